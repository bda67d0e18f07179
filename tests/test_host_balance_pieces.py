"""How the balance loss's forward cuts a batch, from the workspace that it asks for (no GPU needed)."""

import pytest

from nanopysche_amd import _lib


def asked(T, E, S):
    return _lib.load().fm_balance_workspace_bytes(T, E, S)


def room(runs, E, S):
    """Of a batch cut in so many runs: a place for each, for each sequence and for the tokens before and behind them (E fp32 sums and E
    counts, two words more), 16 bytes to 16 columns of a sequence."""
    places = runs + S + 2
    parts = (places * E, places * E, places, places, 4 * S * ((E + 15) // 16))
    return 256 + sum((4 * n + 255) // 256 * 256 for n in parts)


@pytest.mark.parametrize("E", [257, 259, 301, 511])
@pytest.mark.parametrize("T,S", [(65536, 1), (65536, 64), (20000, 1), (131072, 100)])
def test_rows_of_sixteen_values_a_lane_are_cut_for_four_waves(T, S, E):
    """Sixteen waves of such rows have no kernel: a piece of them would be one wave's, 256 tokens after another."""
    run = max(16, -(-T // 4096 // 16) * 16) * 4
    assert asked(T, E, S) == room(-(-T // run), E, S)


@pytest.mark.parametrize("E", [256, 260, 508, 512, 255, 64])
def test_others_for_sixteen(E):
    assert asked(65536, E, 1) == room(256, E, 1)


@pytest.mark.parametrize("T,E,run", [(512, 8, 32), (576, 8, 128), (1024, 8, 128), (2048, 8, 128), (4096, 4, 256), (1024, 16, 64), (1024, 7, 64)])
def test_one_launch_gives_its_waves_a_piece_each(T, E, run):
    """Sixteen waves, a piece of a run or of four each: pieces cut for sixteen waves would be four waves' at 2048 of 8 experts."""
    assert asked(T, E, 1) == room(-(-T // run), E, 1)


@pytest.mark.parametrize("T,E", [(1700, 7), (2340, 7), (2080, 8)])
def test_more_than_the_waves_take_three_launches(T, E):
    """Beyond sixteen pieces of four runs, or 16384 logits: cut for workgroups of sixteen waves."""
    assert asked(T, E, 1) < room(16, E, 1)
