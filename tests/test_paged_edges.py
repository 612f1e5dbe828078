"""CPU tests of the paged cache's entries at the edges of their arguments."""

from tests.test_paged_args import AT, cache, lib, queries, refused  # noqa: F401


def test_selected_ends_past_32_bits(lib):  # noqa: F811
    """first + last may pass 2^31."""
    top = 2 ** 31 - 1
    for first, last in ((top, 1), (1, top), (top, top), (top, 0), (0, 5)):
        refused(lib, lib.mlxvs_paged_select_device(cache(), queries(), 4, first, last, AT, None),
                "together at most n")
