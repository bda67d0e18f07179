"""How the balance loss's forward cuts a batch, from the workspace that it asks for (no GPU needed)."""

import pytest

from nanopysche_amd import _lib


def pieces(T, E, S):
    """Places of a piece in the workspace, at least: E fp32 sums and E counts each, two words more, 16 bytes to 16 columns of a sequence."""
    nbytes = _lib.load().fm_balance_workspace_bytes(T, E, S)
    return (nbytes - 16 * S * ((E + 15) // 16) - 6 * 256) // (8 * E + 8)


@pytest.mark.parametrize("E", [257, 259, 301, 511])
@pytest.mark.parametrize("T,S", [(65536, 1), (65536, 64), (20000, 1), (131072, 100)])
def test_rows_of_sixteen_values_a_lane_are_cut_for_four_waves(T, S, E):
    """Sixteen waves of such rows have no kernel: a piece of them would be one wave's, 256 tokens after another."""
    run = max(16, -(-T // 4096 // 16) * 16) * 4
    assert pieces(T, E, S) >= T // run


@pytest.mark.parametrize("E", [256, 260, 508, 512, 255, 64])
def test_others_for_sixteen(E):
    assert pieces(65536, E, 1) < 65536 // 64
