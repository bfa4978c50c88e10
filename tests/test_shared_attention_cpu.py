"""Which decode steps read shared pages once, and how many pieces a unit falls into (host arithmetic)."""
import pytest
import torch

from torchless_rs_b200.csrc.attention_shared import BLOCK_ROWS, MAX_PARTS, WORTH, shared_plan, worth_sharing

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_bound_is_crossed_where_the_saved_bytes_say(dtype):
    least, share = WORTH[dtype]
    token = 2 * 8 * 128 * dtype.itemsize
    pages = int(least / (3 * 64 * token))                     # common pages of 4 rows that save just less than the bound
    for c, want in ((pages, False), (pages + 1, True)):
        assert worth_sharing([4], [c * 64], [c], 8, 128, None, dtype) is want
    # two groups save together what one would
    assert worth_sharing([4, 4], [pages * 64] * 2, [pages] * 2, 8, 128, None, dtype)
    # rows by themselves save nothing, and count as own keys
    assert not worth_sharing([1] * 64, [100000] * 64, [0] * 64, 8, 128, None, dtype)
    lone = int(least / token) * 20
    assert worth_sharing([4, 1], [(pages + 1) * 64, lone], [pages + 1, 0], 8, 128, None, dtype) is (share == 0)


@pytest.mark.parametrize("groups,nkv,hd", [(16, 4, 64), (16, 2, 128), (4, 8, 128)])
def test_short_prompts_in_32_bit_are_read_per_row(groups, nkv, hd):
    """One common page and 20 tokens in four beams each: the per-row kernel takes 8.7 and 9.6 us there, the other one 14.5 and 20.9."""
    assert not worth_sharing([4] * groups, [84] * groups, [1] * groups, nkv, hd, None, F32)
    assert worth_sharing([4] * groups, [276] * groups, [4] * groups, nkv, hd, None, F32)


def test_keys_before_the_window_are_not_counted():
    assert worth_sharing([8], [65536], [1000], 8, 128, None, BF16)
    assert not worth_sharing([8], [65536], [1000], 8, 128, 1536, BF16)      # the window begins where the common pages end
    assert not worth_sharing([8], [0], [0], 8, 128, None, BF16)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("group", [1, 3, 6, 16])
@pytest.mark.parametrize("blocks", [4, 148, 296])
def test_there_is_room_for_every_piece_of_the_longest_unit(dtype, group, blocks):
    """A line of tiles cut into stretches of ceil(total / blocks): the longest unit lies across at most ceil(longest / share) + 1."""
    for lens, shared, rows, window in (((70,), (1,), 2, 0), ((9000, 65, 1, 0), (140, 1, 0, 0), 9, 0), ((64000,), (1000,), 4, 0),
                                       ((5000, 5000), (78, 10), 40, 700)):
        row_blocks, parts = shared_plan(lens, shared, rows, 4, group, window, dtype, blocks)
        assert row_blocks * (BLOCK_ROWS[dtype] // group) >= rows > (row_blocks - 1) * (BLOCK_ROWS[dtype] // group)
        assert 2 <= parts <= MAX_PARTS
        beams, tile, units = -(-rows // row_blocks), 2 if dtype == BF16 else 1, []
        for n, c in zip(lens, shared):
            first = max(0, n - window) // 64 if window else 0
            end = -(-n // 64)
            border = min(max(c, first), end)
            units += [-(-(border - first + (end - border) * beams) // tile)] * (row_blocks * 4)
        cut = max(1, -(-sum(units) // blocks))
        assert parts >= min(MAX_PARTS, -(-max(units) // cut) + 1)
