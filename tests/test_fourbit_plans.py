"""How the attention over 4-bit pages cuts its work: every page is somebody's, what merges as a cluster can be one, no limit is passed."""
import pytest

from hos_b200.parts import attention4


@pytest.fixture(autouse=True)
def sms(monkeypatch):
    monkeypatch.setattr(attention4.ops, "sm_count", lambda: 148)


@pytest.mark.parametrize("window", [None, 1, 64, 1000])
@pytest.mark.parametrize("fill", [1.0, 0.5, 0.01])
def test_shares(window, fill):
    for rows in (1, 2, 3, 7, 12, 48, 100, 3000):
        for items in (1, 4, 5, 16):
            for longest in (1, 64, 65, 700, 8192, 131072, 10 ** 7):
                share, splits, cluster = attention4.shares(rows, items, longest, window, fill)
                pages = -(-min(longest, window or longest) // 64) + (1 if window and longest > window else 0)
                assert share >= 1 and (splits - 1) * share < pages <= splits * share and splits <= attention4.MAX_SHARES
                if cluster:
                    assert splits == 2 or splits in (4, 8) and rows * items * splits <= 256


def test_shares_of_tiles():
    for blocks in (1, 3, 40, 1000):
        for kv in (1, 4, 16):
            for longest, new, window in ((1, 1, None), (300, 300, None), (8192, 739, None), (8192, 739, 4096), (10 ** 6, 5, 100)):
                share, splits = attention4.tile_shares(blocks, kv, longest, new, window)
                pages = -(-(min(longest, window + new) if window else longest) // 64) + (1 if window and longest > window else 0)
                assert (splits - 1) * share < pages <= splits * share and (splits == 1 or share >= attention4.TILE_LEAST)
                assert splits <= attention4.MAX_SHARES


def test_long_pieces_take_tiles_and_short_ones_few_rows():
    def faster(new, longest, heads=8, kv=4, dim=256):
        size, per = 128 // (heads // kv), heads // kv
        blocks = -(-new // size)
        return attention4.tiles_are_faster(blocks * kv, attention4.tile_shares(blocks, kv, longest, new, None), new / (blocks * size),
                                           -(-new // max(1, 8 // per)) * kv * -(-per // 8) * attention4._pages(longest, None), 1.0, dim)
    assert faster(739, 8192) and faster(400, 3000) and faster(1000, 16000, 16, 2, 64)
    assert not faster(16, 600) and not faster(64, 600) and not faster(16, 16000) and not faster(128, 1000)
