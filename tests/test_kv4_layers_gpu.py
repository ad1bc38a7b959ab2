"""Layers over 4-bit pages through the step function that the models of other tests do not have."""
import pytest
import torch

from tests import harness
from tests.plain import kv4_plain
from tests.test_kv4_engine_gpu import NarrowPart, held
from tests.test_parts_gpu import fill
from tests.tiny_configs import TINY_D

pytestmark = pytest.mark.gpu

F32 = torch.float32


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 96), (2, 1, 160), (3, 3, 64)])
def test_float32_portions_of_any_head_size(heads, kv_heads, dim):
    """Portions of heads that the float32 tile kernel takes and of others, which go token by token, beside single tokens."""
    from qwen_inference_lab_b200.cache import CacheManager
    from qwen_inference_lab_b200.engine import StepEntry, StepRunner
    from qwen_inference_lab_b200.parts import GroupedQueryAttention, RotaryFrequencies
    hidden, eps, lengths = 80, 1e-5, (70, 45)
    turn = RotaryFrequencies(32, 1e4)
    part = GroupedQueryAttention(hidden, heads, kv_heads, dim, names={k: k for k in ("q", "k", "v", "o", "q_norm", "k_norm")}, position=turn, qk_norm_eps=eps)
    w = {name: value.double() for name, value in fill(part, 4, F32).items()}
    x = torch.randn(sum(lengths), hidden, generator=torch.Generator().manual_seed(9))
    model = NarrowPart(part, hidden, F32, lambda ctx, rows, view: part.forward(ctx, rows, view))
    cache = CacheManager(model.cache_specs(), num_pages=20, page_size=8, max_requests=2, max_context=128, dtype=F32, device="cuda")
    cache.poison()
    runner = StepRunner(model, cache, use_graphs=False)
    model.inputs = x.cuda()
    done, first, rows = [0, 0], (0, lengths[0]), [[], []]
    for name in (0, 1):
        cache.admit(name)
    for sizes in ((40, 1), (1, 20), (9, 1), (1, 23), (19, 0)):
        taken = [(name, size) for name, size in enumerate(sizes) if size]
        runner.run([StepEntry(name, list(range(first[name] + done[name], first[name] + done[name] + size)), []) for name, size in taken])
        out, at = model.outputs.pop(), 0
        for name, size in taken:
            rows[name].append(out[at:at + size])
            at += size
            done[name] += size
    assert done == list(lengths)
    for name, n in enumerate(lengths):
        y = x[first[name]:first[name] + n].double()
        q, k, v = ((y @ w[f"{letter}.weight"].t()).view(n, -1, dim) for letter in "qkv")
        angles = torch.arange(n).double()[:, None] * torch.tensor(turn.frequencies(), dtype=torch.float64).float().double()
        q, k = (kv4_plain.turned(kv4_plain.normed(t, w[f"{letter}_norm.weight"], eps), angles, 32, turn.layout) for letter, t in (("q", q), ("k", k)))
        out, _ = kv4_plain.attention(q, held(k), held(v), torch.arange(n), dim ** -0.5)
        expected = out.reshape(n, -1) @ w["o.weight"].t()
        got = torch.cat(rows[name]).double()
        # float32 projections: a code tips now and then and moves an output by a step of one key's share at most
        assert (got - expected).norm() <= 2e-3 * expected.norm(), float((got - expected).norm() / expected.norm())


def test_recorded_steps_do_not_remember_who_recorded_them(tmp_path, monkeypatch):
    """A step whose contexts are nearly as long as each other after one with a single long context, the same bits as without any recording.
    The rule is replaced by one that shows the difference at these sizes."""
    from qwen_inference_lab_b200.cache import CacheManager
    from qwen_inference_lab_b200.engine import StepEntry, StepRunner
    from qwen_inference_lab_b200.kernels import kv4
    from qwen_inference_lab_b200.loading import load_model
    asked = []
    monkeypatch.setattr(kv4, "_spans", lambda blocks, step_us, size, reach, *rest: asked.append(reach.fill) or (2 if reach.fill > 0.7 else 4))
    harness.write_folder(TINY_D, 3, tmp_path)
    model, rows = load_model(tmp_path, device="cuda", dtype=F32), {}
    tokens = [harness.random_tokens(TINY_D, 520, 90 + i) for i in range(3)]
    for graphs in (True, False):
        cache = CacheManager(model.cache_specs(kv_bits=4), num_pages=120, page_size=16, max_requests=3, max_context=model.max_positions, dtype=F32,
                             device=model.device)
        runner, done = StepRunner(model, cache, max_step_tokens=1024, use_graphs=graphs), [0, 0, 0]
        for i in range(3):
            cache.admit(i)

        def step(sizes, want):
            entries = []
            for i, size in enumerate(sizes):
                if size:
                    entries.append(StepEntry(i, tokens[i][done[i]:done[i] + size], [size - 1] if want else []))
                    done[i] += size
            return runner.run(entries)

        step((500, 20, 20), False)
        ragged = step((1, 1, 1), True).clone()
        step((0, 460, 470), False)
        even = [step((1, 1, 1), True).clone() for _ in range(2)]
        runner.check()
        rows[graphs] = torch.stack([ragged, *even])
        assert len(runner._graphs) == (2 if graphs else 0)
    assert torch.equal(rows[True], rows[False]) and {1.0, 0.5} <= set(asked)
