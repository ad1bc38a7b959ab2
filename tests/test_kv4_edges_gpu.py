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
