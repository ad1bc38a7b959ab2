"""Models whose cache keeps keys and values in 4 bits: the step function under several cuts, generation, the command line, an attention
part with the options that the step function's models do not have."""
import dataclasses
import json
import subprocess
import sys

import pytest
import torch

from tests import harness
from tests.plain import kv4_plain, qwen3_plain
from tests.test_parts_gpu import fill
from tests.tiny_configs import TINY_B, TINY_D

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def held(x):
    return kv4_plain.values(*kv4_plain.coded(x))


def narrow_rows(requests, weights, cfg, monkeypatch):
    """The plain implementation's rows, keys and values as the cache holds them."""
    exact = qwen3_plain.causal_attention
    with monkeypatch.context() as patch:
        patch.setattr(qwen3_plain, "causal_attention", lambda q, k, v, scale, window=0: exact(q, held(k).float(), held(v).float(), scale, window))
        return harness.plain_rows(requests, weights, cfg)


def runner_of(folder, dtype, *, num_pages, page_size, max_requests=4):
    from qwen_inference_lab_b200.cache import CacheManager
    from qwen_inference_lab_b200.engine import StepRunner
    from qwen_inference_lab_b200.loading import load_model
    model = load_model(folder, device="cuda", dtype=dtype)
    cache = CacheManager(model.cache_specs(kv_bits=4), num_pages=num_pages, page_size=page_size, max_requests=max_requests,
                         max_context=model.max_positions, dtype=dtype, device=model.device)
    cache.poison()
    return cache, StepRunner(model, cache, max_step_tokens=1024)


def off(rows, others):
    """Root mean square of the differences of two sets of rows."""
    return torch.stack([(rows[k] - others[k]).square().mean() for k in others]).mean().sqrt().item()


SCHEDULES = {"whole": harness.whole_schedule, "chunks": harness.chunk_schedule, "tail": harness.tail_decode_schedule,
             "mixed": harness.mixed_schedule}


@pytest.mark.parametrize("cut", SCHEDULES)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("name,lengths,pages", [("B", (5, 90, 41, 130), 60), ("D", (3, 300, 150), 40)])
def test_steps(tmp_path, monkeypatch, name, lengths, pages, dtype, cut):
    """In float32 the engine is as far from the plain implementation over held values as a few codes that a rounding of the activations
    tips: each is one step where holding costs every element 0.3 of one on average, so a hundredth of what holding costs leaves room for
    one in ten thousand... of all elements (0.01^2 x 0.083 steps^2).  In bfloat16 activations are off by 2^-8 of a value of up to
    15 steps, which tips at most an eighth of the codes: (1/8) / 0.083 = 1.5 times the variance that holding costs, beside what
    bfloat16 costs the plain implementation."""
    cfg = {"B": TINY_B, "D": TINY_D}[name]
    weights = harness.write_folder(cfg, 3, tmp_path)
    requests = {f"r{i}": harness.random_tokens(cfg, n, 40 + i) for i, n in enumerate(lengths)}
    cache, runner = runner_of(tmp_path, dtype, num_pages=pages, page_size=16)
    rows = harness.run_schedule(runner, cache, SCHEDULES[cut](requests))
    exact = harness.plain_rows(requests, weights, cfg)
    narrow = narrow_rows(requests, weights, cfg, monkeypatch)
    cost = off(narrow, exact)
    assert set(rows) == set(narrow) and all(torch.isfinite(v).all() for v in rows.values())
    if dtype == F32:
        assert off(rows, narrow) <= 0.1 * cost, (off(rows, narrow), cost)
    else:
        rounding = off(harness.plain_rows(requests, weights, cfg, BF16), exact)
        assert off(rows, narrow) <= 1.25 * cost + 1.5 * rounding, (off(rows, narrow), cost, rounding)
    if cut in ("tail", "mixed"):
        assert runner._graphs                      # single tokens were recorded and replayed


def test_generation_and_what_it_holds(tmp_path):
    from qwen_inference_lab_b200 import Engine, Qwen3
    harness.write_folder(TINY_B, 1, tmp_path)
    prompts = [harness.random_tokens(TINY_B, n, 50 + n) for n in (1, 9, 40, 75)]
    for dtype in (F32, BF16):
        model = Qwen3.from_directory(tmp_path, device="cuda", dtype=dtype)
        runs = []
        for _ in range(2):
            engine = Engine(model, num_pages=40, page_size=8, token_budget=48, prefill_chunk=32, max_active=3, kv_bits=4)
            assert engine.cache.kv_groups[0].storage.dtype == torch.uint8
            runs.append([row["token_ids"] for row in engine.generate(prompts, max_new_tokens=20, ignore_eos=True)])
            assert engine.idle and engine.cache.free_pages() == 40 and all(len(t) == 20 for t in runs[-1])
            engine.close()
        assert runs[0] == runs[1]
        # both kinds of cache serve the same model one after the other
        engine = Engine(model, num_pages=40, page_size=8, max_active=3)
        assert engine.cache.kv_groups[0].storage.dtype == dtype
        assert [len(row["token_ids"]) for row in engine.generate(prompts, max_new_tokens=3, ignore_eos=True)] == [3] * 4


def test_command_line_and_replay(tmp_path):
    harness.write_folder(TINY_B, 1, tmp_path)
    run = lambda module, *args, **kw: subprocess.run([sys.executable, "-m", module, "--model", str(tmp_path), "--dtype", "float32", "--kv-bits", "4", *args],
                                                     capture_output=True, text=True, check=True, timeout=300, **kw).stdout
    answer = json.loads(run("qwen_inference_lab_b200", "--token-ids", "[1, 2, 3]", "--max-new-tokens", "4", "--ignore-eos"))
    assert len(answer["token_ids"]) == 4
    step = json.dumps({"step": 0, "entries": [{"id": "a", "tokens": [5, 17, 3], "want": [2]}], "end": ["a"]})
    assert "done 0" in run("qwen_inference_lab_b200.engine.replay", "--out", str(tmp_path / "out"), "--max-tokens", "64", input=step + "\n")
    assert (tmp_path / "out" / "0.f32").stat().st_size == 4 * TINY_B["vocab_size"]


class NarrowPart(harness.OnePartModel):
    def cache_specs(self):
        return [dataclasses.replace(self.part.cache_spec(), bits=4)]


@pytest.mark.parametrize("options", [dict(position="interleaved", unit=True, window=0), dict(position="halves", unit=False, window=21, gate=True),
                                     dict(position="ramp", unit=True, window=0, from_keys=True)], ids=["unit", "window_gate", "ramp_keys"])
def test_attention_part_with_frequencies(options):
    """Rotation by frequencies in both layouts and of part of the head, heads of unit size, a window, an output gate, keys as values."""
    from qwen_inference_lab_b200.cache import CacheManager
    from qwen_inference_lab_b200.engine import StepEntry, StepRunner
    from qwen_inference_lab_b200.parts import GroupedQueryAttention, RotaryFrequencies
    hidden, n_q, n_kv, d, eps, rot = 80, 6, 2, 64, 1e-5, 32
    turn = RotaryFrequencies(rot, 1e4, layout="interleaved" if options["position"] == "interleaved" else "halves",
                             ramp=(8.0, 64, 32, 1) if options["position"] == "ramp" else None)
    gate, from_keys = options.get("gate"), options.get("from_keys", False)
    part = GroupedQueryAttention(hidden, n_q, n_kv, d, names={k: k for k in ("q", "k", "v", "o", "q_norm", "k_norm")}, position=turn,
                                 qk_norm_eps=None if options["unit"] else eps, unit_qk_norm_eps=eps if options["unit"] else None,
                                 window=options["window"], head_gate="g" if gate else None, values_from_keys=from_keys)
    w = {name: value.double() for name, value in fill(part, 4, F32).items()}
    x = torch.randn(70, hidden, generator=torch.Generator().manual_seed(9))

    def body(ctx, rows, view):
        return part.forward(ctx, rows, view)

    model = NarrowPart(part, hidden, F32, body)
    cache = CacheManager(model.cache_specs(), num_pages=16, page_size=8, max_requests=2, max_context=128, dtype=F32, device="cuda")
    cache.poison()
    runner = StepRunner(model, cache, use_graphs=False)
    cache.admit("a")
    model.inputs = x.cuda()
    done = 0
    for size in (40, 1, 1, 5, 20, 3):
        runner.run([StepEntry("a", list(range(done, done + size)), [])])
        done += size
    got = torch.cat(model.outputs).double()
    y = x.double()
    q, k = ((y @ w[f"{name}.weight"].t()).view(70, -1, d) for name in ("q", "k"))
    v = k if from_keys else (y @ w["v.weight"].t()).view(70, n_kv, d)
    angles = torch.arange(70).double()[:, None] * torch.tensor(turn.frequencies(), dtype=torch.float64).float().double()
    def tail(t, weight):
        if not options["unit"]:
            t = kv4_plain.normed(t, w[weight], eps)
        t = kv4_plain.turned(t, angles, rot, turn.layout, turn.gain)
        return kv4_plain.normed(t, None, eps) if options["unit"] else t
    out, _ = kv4_plain.attention(tail(q, "q_norm.weight"), held(tail(k, "k_norm.weight")), held(v), torch.arange(70), d ** -0.5, options["window"])
    if gate:
        out = out * torch.sigmoid(y @ w["g.weight"].t())[..., None]
    expected = out.reshape(70, -1) @ w["o.weight"].t()
    # float32 projections: a code tips now and then and moves an output by a step of one key's share at most
    assert (got - expected).norm() <= 2e-3 * expected.norm(), float((got - expected).norm() / expected.norm())
