"""Other architectures whose cache keeps keys and values in 4 bits: attention beside a state, with its products joined to the other mixer's and
its result in float32, through the step function and the engine."""
import importlib

import pytest
import torch

from tests import bugidra_cases, harness
from tests.bugidra_cases import delta, left, pair, right, rot
from tests.lotazen_cases import CASE_D
from tests.test_kv4_engine_gpu import held, off, runner_of

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
BUGIDRA = bugidra_cases.config(173, 128, 1e-5, 2.0,
                               delta(4, 2, 32, 40, 4, ff=96),
                               pair(left(4, 2, 64, 64, 0.12, rot(100000.0, 48, (2.0, 256, 32.0, 1.0))), right(24, 16, rot(500.0, 8), (0.97, 1.0, 0.5)), 80),
                               pair(left(3, 1, 96, 96, 0.1, rot(10000.0, 96)), right(32, 40, rot(1e5, 32), (0.98, 0.9995))),
                               delta(2, 2, 16, 24, 3))
MODELS = {"lotazen": (CASE_D, "window_attention"), "bugidra": (BUGIDRA, "causal_attention")}
SCHEDULES = {"chunks": harness.chunk_schedule, "tail": harness.tail_decode_schedule, "mixed": harness.mixed_schedule}
_rows: dict = {}


def plain_of(name, folder_cases, requests, weights, cfg):
    """(rows, rows over held keys and values, rows of the bfloat16 yardstick), made once."""
    if name not in _rows:
        plain, attention = folder_cases.plain, MODELS[name][1]
        exact = getattr(plain, attention)
        rows, low = folder_cases.plain_rows(requests, weights, cfg), folder_cases.plain_rows(requests, weights, cfg, BF16)
        with pytest.MonkeyPatch.context() as patch:
            patch.setattr(plain, attention, lambda q, k, v, *rest: exact(q, held(k).to(q.dtype), held(v).to(q.dtype), *rest))
            narrow = folder_cases.plain_rows(requests, weights, cfg)
        _rows[name] = rows, narrow, low
    return _rows[name]


@pytest.mark.parametrize("cut", SCHEDULES)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("name", MODELS)
def test_steps(tmp_path, name, dtype, cut):
    """The bounds of the dense model's steps: in float32 a tenth of what holding costs the plain implementation (a code that tips is one step
    where holding costs every element 0.3 of one); in bfloat16 1.25 of it, and 1.5 of what bfloat16 costs."""
    folder_cases, cfg = importlib.import_module(f"tests.{name}_cases"), MODELS[name][0]
    weights = folder_cases.write_folder(cfg, 8, tmp_path)
    requests = {f"r{i}": folder_cases.random_tokens(cfg, n, 60 + i) for i, n in enumerate((150, 3, 61, 110))}
    exact, narrow, low = plain_of(name, folder_cases, requests, weights, cfg)
    cache, runner = runner_of(tmp_path, dtype, num_pages=60, page_size=16)
    assert all(group.storage.dtype == torch.uint8 for group in cache.kv_groups)
    rows = harness.run_schedule(runner, cache, SCHEDULES[cut](requests))
    cost = off(narrow, exact)
    assert set(rows) == set(narrow) and all(torch.isfinite(v).all() for v in rows.values())
    bar = 0.1 * cost if dtype == F32 else 1.25 * cost + 1.5 * off(low, exact)
    assert off(rows, narrow) <= bar, (off(rows, narrow), cost, off(low, exact))
    if cut in ("tail", "mixed"):
        assert runner._graphs                      # single tokens were recorded and replayed


@pytest.mark.parametrize("name", MODELS)
def test_generation(tmp_path, name):
    """Twice the same tokens, with steps ahead of the host or not, and every page given back."""
    from qwen_inference_lab_b200 import Engine
    from qwen_inference_lab_b200.loading import load_model
    folder_cases, cfg = importlib.import_module(f"tests.{name}_cases"), MODELS[name][0]
    folder_cases.write_folder(cfg, 8, tmp_path)
    prompts = [folder_cases.random_tokens(cfg, n, 70 + n) for n in (1, 9, 40, 75)]
    model, runs = load_model(tmp_path, device="cuda", dtype=BF16), []
    for overlap in (False, True):
        engine = Engine(model, num_pages=40, page_size=8, token_budget=48, prefill_chunk=32, max_active=3, kv_bits=4, overlap=overlap)
        runs.append([row["token_ids"] for row in engine.generate(prompts, max_new_tokens=12, ignore_eos=True)])
        assert engine.idle and engine.cache.free_pages() == 40
        engine.close()
    assert runs[0] == runs[1] and all(len(tokens) == 12 for tokens in runs[0])
