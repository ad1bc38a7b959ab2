"""The endings of a context that is cut over blocks of the 4-bit attention: one block, a cluster, the last block to arrive."""
import pytest
import torch

from tests.plain import kv4_plain as plain
from tests.test_kv4_gpu import BF16, F32, attend_case, attend_check, attend_run, kv4

pytestmark = pytest.mark.gpu

CASES = {"single": ([2100, 700, 31], [1, 1, 1], 0), "few_8_rows": ([2100, 90], [2, 1], 0), "few_16_rows": ([2100, 90], [4, 3], 0),
         "few_48_rows": ([2000, 0], [12, 9], 0), "window": ([2100, 700], [1, 3], 600)}


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("name", CASES)
def test_any_number_of_spans_gives_what_one_gives(name, dtype, monkeypatch):
    """Numbers that are clusters and others, more than there are steps of keys among them, clusters or not.  In float32 the sums' order differs
    (2^-24 of what is summed, a few times over); in bfloat16 weights are counted from another maximum, so that their two roundings and the result's
    fall elsewhere (2^-8 of what is weighed each)."""
    module = kv4()
    starts, lens, window = CASES[name]
    built = attend_case(8, 2, 64, 16, starts, lens, dtype, seed=41)
    outs = {}
    for clusters in (module.CLUSTERS, {1: (), 2: ()}):
        monkeypatch.setattr(module, "CLUSTERS", clusters)
        for count in (1, 2, 3, 4, 8, 16, 40):
            monkeypatch.setattr(module, "_spans", lambda *rule: count)
            out = attend_run(built, window)
            attend_check(built, out, window)
            assert torch.equal(attend_run(built, window), out)
            outs[count, bool(clusters[1])] = out.cpu().double().view(-1, 8, 64)
    assert torch.equal(outs[1, True], outs[1, False])
    firsts = torch.tensor([0, *lens]).cumsum(0).tolist()
    size = torch.cat([plain.attention(built["q"][first:first + n].view(n, 8, 64), *held, torch.arange(start, start + n), 64 ** -0.5, window)[1]
                      for first, start, n, held in zip(firsts, starts, lens, built["held"])])
    bar = (6 * 2.0 ** -8 if dtype == BF16 else 64 * 2.0 ** -24) * size
    for key, out in outs.items():
        assert ((out - outs[1, True]).abs() <= bar).all(), key


@pytest.mark.parametrize("dim,lens", [(256, [2, 3]), (160, [1, 4])])
def test_clusters_of_large_heads(dim, lens, monkeypatch):
    """Heads of which an SM takes one or two blocks: clusters of 2 to 16 of them are placed, and join as one block does."""
    module = kv4()
    built, outs = attend_case(16, 2, dim, 16, [1500, 1900], lens, BF16, seed=42), {}
    for count in (1, 2, 4, 8, 16):
        monkeypatch.setattr(module, "_spans", lambda *rule: count)
        outs[count] = attend_run(built)
        attend_check(built, outs[count])
