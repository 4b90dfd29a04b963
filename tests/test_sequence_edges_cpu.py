"""CPU: what the sequence operators' C entries answer, or refuse, before anything is launched."""
import pytest

from simvg_amd import _lib


@pytest.mark.parametrize("T,Hq,causal", [(1571, 3, 0), (8191, 1, 1), (2501, 1, 1), (3000, 1, 1), (2900, 3, 0)])
def test_the_parts_sums_of_a_forward_pass_start_at_multiples_of_16_bytes(T, Hq, causal):
    """the workspace of a sequence that is cut over its keys: statistics, then sums of D values, which are written 16 bytes at a time"""
    size = lambda D: _lib.load().simvg_packed_attn_ws_floats(T, 1, Hq, 1, D, causal, 0)  # noqa: E731
    rows = (size(72) - size(64)) // 8                                       # parts x T x Hq
    assert rows > T * Hq and rows % (T * Hq) == 0 and size(128) - size(64) == 64 * rows
    stats = size(64) - 64 * rows
    assert stats >= 2 * rows and stats % 4 == 0
