"""CPU tests of the paged cache's entries at the edges of their arguments."""

import os
import subprocess
import sys

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
