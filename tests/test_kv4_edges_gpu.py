"""Numbers at the edges of their types in the 4-bit cache: what is infinite, nearly infinite or next to nothing, and where it may be seen."""
import math

import pytest
import torch

from tests.plain import kv4_plain as plain
from tests.test_kv4_gpu import BF16, F32, attend_case, attend_check, attend_run, kv4, store_case, store_plain, store_run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("layout", [0, 1], ids=["halves", "neighbours"])
@pytest.mark.parametrize("rot", [0, 30, 32])
def test_infinite_queries_where_nothing_turns(dtype, layout, rot):
    """A dimension that is not turned is what it was, and nothing of its neighbour's."""
    case = store_case(2, 1, 64, 8, "none", "freq" if rot else None, rot, layout, 1.0, [3, 0], [4, 2], dtype)
    rows = case["proj"].view(6, 4, 64)
    rows[:, 0, 40], rows[:, 1, 63], rows[2, :2, 32] = math.inf, -math.inf, math.inf
    pages = torch.zeros((case["n_pages"], *kv4().page_shape(1, 64, 8)), dtype=torch.uint8, device="cuda")
    got, (expected, _, _) = store_run(case, pages).cpu().double().view(6, 2, 64), store_plain(case)
    finite = expected.isfinite()
    assert not expected.isnan().any() and finite.sum() == expected.numel() - 6 - 6 - 2
    assert torch.equal(got[~finite], expected[~finite])
    unit = 2.0 ** -8 if dtype == BF16 else 0.0                       # the bounds of the other store tests
    size = expected.where(finite, torch.zeros_like(expected)).abs().amax()
    assert ((got - expected)[finite].abs() <= unit * expected[finite].abs() + 16 * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("plane", [0, 1], ids=["keys", "values"])
def test_groups_whose_values_pass_the_largest_float(plane):
    """The steps of a group from -3.07e38 to the largest bfloat16 number are rounded up, and its largest value is held as 3.41e38, more than float32
    has.  A portion's rows in front of it are finite whatever it is.  Held as a value it weighs as what it is in the rows behind it; next to it a
    page's other values count as nothing (2^-33 of the page's largest at most)."""
    lens = [50, 70]
    built = attend_case(8, 2, 64, 16, [0, 0], lens, BF16, seed=31)
    rows = [[held[i].float() for i in (0, 1)] for held in built["held"]]
    rows[0][plane][20, 1, 5], rows[0][plane][20, 1, 9] = torch.finfo(BF16).max, -3.0705166702631557e38
    pages, table, held = plain.build([r[0] for r in rows], [r[1] for r in rows], lens, 16, seed=3)
    assert held[0][plane].abs().max() > torch.finfo(F32).max
    built.update(pages=pages, table=table, held=held)
    out = attend_run(built).cpu().double().view(-1, 8, 64)
    assert out[:20].isfinite().all() and out[:, :4].isfinite().all() and out[50:].isfinite().all()
    if plane == 0:
        return
    exact, size = plain.attention(built["q"][:50].view(50, 8, 64), *held[0], torch.arange(50), 64 ** -0.5)
    held_off = (out[20:50] - exact[20:]).abs() <= 8 * 2.0 ** -8 * size[20:] + 2.0 ** -33 * 3.42e38
    assert held_off[exact[20:].abs() < 3.38e38].all()
    assert ((out[:20] - exact[:20]).abs() <= 8 * 2.0 ** -8 * size[:20] + 2.0 ** -33 * 3.42e38).all()


@pytest.mark.parametrize("before", ["zeros", "unseen", "ordinary"])
@pytest.mark.parametrize("size", [1e-30, 1e-34])
def test_tiny_values_behind_others(before, size, monkeypatch):
    """Values of 1e-30 behind 128 positions of zeros (steps of 0), or of ordinary values that weigh 2^-300, or that weigh much: as exact as
    others in what they add.  Single and few tokens; a warp takes every fourth tile of 32 positions, so each has other ones first where a context is
    not cut."""
    monkeypatch.setattr(kv4(), "_spans", lambda *rule: 1)
    lens = [1, 4]
    starts = [500 - n for n in lens]
    built = attend_case(8, 2, 64, 16, starts, lens, BF16, seed=33)
    rows = [[held[i].float() for i in (0, 1)] for held in built["held"]]
    built["q"] = built["q"].float().abs().to(BF16)
    for keys, values in rows:
        values[128:] *= size
        if before == "zeros":
            values[:128] = 0.0
        elif before == "unseen":
            keys[:128] = -keys[:128].abs() - 60.0
    pages, table, held = plain.build([r[0] for r in rows], [r[1] for r in rows], [500, 500], 16, seed=2)
    built.update(pages=pages, table=table, held=held)
    attend_check(built, attend_run(built))
