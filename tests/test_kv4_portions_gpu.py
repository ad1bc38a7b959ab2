"""Portions behind long contexts over 4-bit pages: contexts that are cut over blocks and joined, contexts that are read back in several
batches, against 64 bits."""
import math

import pytest
import torch

from tests.plain import kv4_plain as plain
from tests.test_kv4_gpu import attend_case, attend_check, attend_run, kv4

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture
def splits(monkeypatch):
    """The numbers of splits that were chosen."""
    from qwen_inference_lab_b200.kernels import attention_tc
    rule, chosen = attention_tc.keys16_splits, []

    def watched(blocks, tiles):
        chosen.append(rule(blocks, tiles))
        return chosen[-1]

    monkeypatch.setattr(attention_tc, "keys16_splits", watched)
    return chosen


SPLIT = [  # hq, hkv, dim, page, starts, lens, window
    (8, 2, 32, 16, [2500, 1000], [100, 60], 0),
    (4, 4, 64, 16, [3000], [130], 1200),                      # the window's first tile lies inside a split's range
    (8, 2, 96, 8, [2000, 0, 700], [150, 40, 30], 0),          # a tile of queries with one tile of keys, fewer than splits
    (32, 8, 128, 16, [6001], [300], 0),                       # splits of more than 32 tiles of keys
    (8, 2, 128, 16, [5000, 3], [64, 50], 1100),
    (5, 1, 128, 64, [1500], [33], 0),                         # five heads share a key: one a tile
    (40, 1, 64, 16, [2100], [5], 0),                          # eight of forty heads a tile, 16 tokens
]


@pytest.mark.parametrize("case", SPLIT, ids=[f"{c[0]}_{c[1]}x{c[2]}_{i}" for i, c in enumerate(SPLIT)])
def test_contexts_cut_over_blocks(case, splits):
    *sizes, window = case
    built = attend_case(*sizes, BF16, seed=21)
    out = attend_run(built, window)
    assert max(splits) > 1
    attend_check(built, out, window)
    assert torch.equal(attend_run(built, window), out)


def test_splits_agree_with_one(monkeypatch):
    """Any number of splits, more than there are tiles of keys among them, gives what one block gives, to a bfloat16 rounding and that of the
    weights, which are counted from another maximum (two roundings of 2^-11 each way)."""
    from qwen_inference_lab_b200.kernels import attention_tc
    built = attend_case(8, 2, 128, 16, [1500, 2], [40, 70], BF16, seed=22)
    outs = {}
    for count in (1, 2, 3, 7, 24, 40):
        monkeypatch.setattr(attention_tc, "keys16_splits", lambda blocks, tiles: count)
        outs[count] = attend_run(built).float().cpu()
        attend_check(built, outs[count])
    size = torch.cat([plain.attention(built["q"][first:first + n].view(n, 8, 128), *held, torch.arange(start, start + n), 128 ** -0.5)[1]
                      for first, start, n, held in zip((0, 40), built["starts"], built["lens"], built["held"])]).view(110, -1)
    for count, out in outs.items():
        assert ((out - outs[1]).abs().double() <= 2 * 2.0 ** -8 * outs[1].abs() + 4 * 2.0 ** -11 * size).all(), count


@pytest.mark.parametrize("window", [0, 1100])
def test_nan_values_in_one_split(window, splits):
    """A NaN group of a value reaches the rows that see it, whichever split read it, and no others."""
    built = attend_case(8, 2, 64, 16, [3000, 2500], [80, 40], BF16, seed=23)
    at = ((0, 0, 1500, 1), (0, 1, 3040, 0), (1, 0, 2, 0))                 # request, kv head, position, group
    for row, head, pos, group in at:
        page = int(built["table"][row, pos // 16])
        codes, pairs = plain.get(built["pages"], page, 1, head, pos % 16)
        pairs[group] = math.nan
        plain.put(built["pages"], page, 1, head, pos % 16, codes, pairs)
    out = attend_run(built, window)
    assert max(splits) > 1
    out = out.float().cpu().view(120, 2, 4, 2, 32)                          # token, kv head, head of it, group
    expected = torch.zeros(120, 2, 4, 2, dtype=torch.bool)
    for row, head, pos, group in at:
        first, start, n = ((0, 3000, 80), (80, 2500, 40))[row]
        for t in range(n):
            if pos <= start + t and (not window or pos > start + t - window):
                expected[first + t, head, :, group] = True
    assert torch.equal(out.isnan().any(-1), expected) and torch.equal(out.isnan().all(-1), expected)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("starts,lens", [
    ([700, 40, 2000, 300, 1100, 90], [1, 3, 70, 40, 30, 64]),     # batches of portions beside single and few tokens
    ([2000, 1900, 100, 10], [4, 6, 80, 40]),                      # the first batches hold short segments only
], ids=["all_kinds", "short_first"])
def test_contexts_read_back_in_batches(starts, lens, dtype, monkeypatch):
    module = kv4()
    monkeypatch.setattr(module, "MOST_READ", 1024)
    built = attend_case(8, 2, 64, 16, starts, lens, dtype, seed=24)
    plan = module.StepPlan.of_segments(range(len(lens)), starts, lens, "cuda")
    assert len(plan.portion_lens) > 2
    for window in (0, 250):
        attend_check(built, attend_run(built, window, plan=plan), window)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_portions_are_cut_by_their_own_contexts(dtype, splits):
    """A fresh prompt beside a few tokens behind a long context: one or two tiles of keys are not cut, whatever lies beside them."""
    built = attend_case(8, 2, 64, 16, [2400, 0, 2000], [4, 70, 1], dtype, seed=25)
    out = attend_run(built)
    assert splits == ([1] if dtype == BF16 else [])
    attend_check(built, out)
