"""How near single and few bfloat16 tokens come to 64 bits: beside the rounding of the result nothing counts."""
import pytest
import torch

from tests.plain import kv4_plain as plain
from tests.test_kv4_gpu import BF16, attend_case, attend_run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,dim,starts,lens", [(32, 8, 128, [900, 333], [1, 1]), (8, 2, 64, [700, 60], [5, 2]), (6, 2, 96, [500], [12]),
                                                    (4, 1, 256, [400, 300], [1, 3]), (16, 2, 32, [800], [1])])
@pytest.mark.parametrize("flat", [True, False], ids=["flat", "peaked"])
def test_the_result_is_rounded_and_nothing_else(hq, hkv, dim, starts, lens, flat):
    """A weight is two bfloat16 parts and so is its product with a step: the second part of a product is off by 2^-15 of the whole, that of a
    weight by 2^-16, and so are what a weight adds to the sum of bases and to the sum that divides (with them a score's last bits: the exponent is a
    number of up to 2^7 with 24 bits).  Element by element these add up to 2^-14 of all that is weighed, codes and bases; as rounding errors
    that do not know of each other, to 2^-15 of the root of the sum of squares, three of which are allowed."""
    built = attend_case(hq, hkv, dim, 16, starts, lens, BF16, seed=51, loud=1.0 if flat else 3.0)
    scale = dim ** -0.5 * (0.3 if flat else 1.0)
    got, first = attend_run(built, scale=scale).cpu().double().view(-1, hq, dim), 0
    for start, n, (keys, values) in zip(starts, lens, built["held"]):
        q, at = built["q"][first:first + n].view(n, hq, dim), torch.arange(start, start + n)
        exact, size = plain.attention(q, keys, values, at, scale)
        groups = values.unflatten(-1, (-1, 32))
        base = groups.amin(-1, keepdim=True).expand_as(groups).flatten(-2)
        _, codes = plain.attention(q, keys, values - base, at, scale)
        _, bases = plain.attention(q, keys, base, at, scale)
        share = hq // hkv
        scores = (torch.einsum("nhd,thd->hnt", q.double(), keys.repeat_interleave(share, 1)) * scale).masked_fill(torch.arange(len(keys)) > at[:, None], -torch.inf)
        squares = torch.einsum("hnt,thd->nhd", scores.softmax(-1).square(), ((values - base).square() + base.square()).repeat_interleave(share, 1))
        most = scale * torch.einsum("nhd,thd->nht", q.double().abs(), keys.repeat_interleave(share, 1).abs()).amax(-1, keepdim=True)
        off = (got[first:first + n] - exact).abs()
        assert (off <= 2.0 ** -8 * exact.abs() + 2.0 ** -14 * (codes + bases + size) + 2 * dim * 2.0 ** -24 * most * size).all()
        rounding = (exact.to(BF16).double() - exact).norm()
        assert off.norm() <= rounding + 3 * 2.0 ** -15 * squares.sqrt().norm() + 2.0 ** -15 * exact.norm() + (dim ** 0.5 * 2.0 ** -24 * most * size).norm(), \
            (float(off.norm() / exact.norm()), float(rounding / exact.norm()))
        first += n
