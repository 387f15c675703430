"""CPU checks of the serving operators' C ABI at the ends of its ranges: refusals before any
launch, and workspace sizes."""

import ctypes

from test_serving_abi import Batch, Blocks, State, _attention, _batch, _blocks, _s, _state, i32, lib, vp  # noqa: F401


def test_a_sequence_ends_before_31_bits(lib):
    """Positions past the last key, by some tiles, are still computed."""
    def both(width, page):
        b = _batch(table_width=width, table_stride=width, page_size=page, num_pages=0)
        s = _s(64, 64, 64)
        return (_attention(lib, batch=b), lib.ltv_paged_cache_append(
            1, vp(16), s, vp(16), s, vp(16), s, vp(16), s, ctypes.byref(b), 2, 64, None))

    for width, page in ((2 ** 31 - 1, 1), (2 ** 31 - 1023, 1), (2 ** 27 - 1, 16), (2 ** 11, 2 ** 20)):
        assert both(width, page) == (2, 2), (width, page)
    # (in range: as far as the workspace, and nothing to append without pages)
    for width, page in ((2 ** 31 - 1024, 1), (2 ** 27 - 64, 16), (2 ** 11 - 1, 2 ** 20)):
        assert both(width, page) == (4, 0), (width, page)


def test_scale_times_log2_e_is_finite(lib):
    assert _attention(lib, scale=3e38) == 1
    assert _attention(lib, scale=2e38) == 4  # (as far as the workspace)
