"""CPU tests of the paged cache's entries at the edges of their arguments."""

import os
import struct
import subprocess
import sys

import pytest

import mlxvs_b200 as mv
from mlxvs_b200 import paged
from tests.test_paged_args import AT, cache, lib, queries, refused  # noqa: F401


def test_selected_ends_past_32_bits(lib):  # noqa: F811
    """first + last may pass 2^31."""
    top = 2 ** 31 - 1
    for first, last in ((top, 1), (1, top), (top, top), (top, 0), (0, 5)):
        refused(lib, lib.mlxvs_paged_select_device(cache(), queries(), 4, first, last, AT, None),
                "together at most n")


def test_all_names_without_torch():
    """The package and all its names are imported without torch, which the
    paged functions import when they are called."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import sys; sys.modules['torch'] = None\n"
            "from mlxvs_b200 import *\n"
            "assert brute_force_knn and paged_store and PagedTables\n")
    subprocess.run([sys.executable, "-c", code], cwd=root, check=True)
    code = ("import sys; from mlxvs_b200 import *\n"
            "assert 'torch' not in sys.modules\n"
            "try: paged_store(1, 2, 3, 4, 5)\n"
            "except ValueError as e: assert 'CUDA tensor' in str(e)\n"
            "assert 'torch' in sys.modules\n")
    subprocess.run([sys.executable, "-c", code], cwd=root, check=True)


def test_whole_numbers_past_32_bits():
    """What is left of a larger number in 32 bits is not taken for it."""
    wide = 2 ** 32
    for n, kw in ((wide + 4, {}), (4, dict(page_size=wide + 16)), (4, dict(first=wide + 1)),
                  (4, dict(last=-wide + 1)), (0, {}), (257, {})):
        with pytest.raises(ValueError, match="must be"):
            mv.paged_select(None, None, None, None, None, kw.pop("page_size", 16), n, **kw)
    with pytest.raises(ValueError, match="page_size must be in"):
        mv.paged_tables(None, None, None, None, wide + 16, 4)
    for tokens in (-1, 2 ** 31, wide + 4):
        with pytest.raises(ValueError, match="num_tokens must be in"):
            mv.paged_tables(None, None, None, None, 16, tokens)


CACHE_FIELDS = """keys values key_page_stride key_row_stride key_head_stride value_page_stride
    value_row_stride value_head_stride pages codes scales page_size heads dim type key_scale
    value_scale""".split()
QUERY_FIELDS = """q tokens token_stride head_stride table rows width requests lengths heads
    type""".split()


def test_struct_fields_lie_where_the_header_has_them(tmp_path):
    """Offset and size of every field, by a C compiler from the header."""
    lines = []
    for name, fields in (("mlxvs_paged_cache", CACHE_FIELDS), ("mlxvs_paged_queries", QUERY_FIELDS)):
        for f in fields:
            lines.append(f'printf("%zu %zu ", offsetof({name}, {f}), sizeof((({name}*)0)->{f}));')
        lines.append(f'printf("%zu\\n", sizeof({name}));')
    source = tmp_path / "fields.c"
    source.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"mlxvs_c.h\"\n"
                      "int main(void) {\n" + "\n".join(lines) + "\nreturn 0;\n}\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    program = str(tmp_path / "fields")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), "-o", program, str(source)],
                   check=True)
    got = subprocess.run([program], check=True, capture_output=True, text=True).stdout.split("\n")
    for line, packed, fields in ((got[0], paged._CACHE, CACHE_FIELDS),
                                 (got[1], paged._QUERIES, QUERY_FIELDS)):
        *pairs, size = map(int, line.split())
        kinds = packed.format[1:]
        assert packed.format[0] == "=" and len(kinds) == len(fields) and size == packed.size
        for i, (offset, width) in enumerate(zip(pairs[::2], pairs[1::2])):
            assert offset == struct.calcsize("=" + kinds[:i]), fields[i]
            assert width == struct.calcsize("=" + kinds[i]), fields[i]


@pytest.mark.parametrize("stride", ["kp", "kr", "kh", "vp", "vr", "vh"])
def test_store_into_rows_that_share_memory(lib, stride):  # noqa: F811
    """A cache with a stride of 0 can be read, not written."""
    c = cache(**{stride: 0})
    refused(lib, lib.mlxvs_paged_store_device(c, AT, AT, 1, 3, 256, 128, 256, 128, AT, None),
            "must lie apart")
