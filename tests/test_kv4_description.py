"""The description of a step over 4-bit pages: how much memory it takes, what it leaves out (no GPU)."""
import random

import numpy as np
import pytest
import torch

from qwen_inference_lab_b200.cache import CacheManager
from qwen_inference_lab_b200.engine import StepEntry, StepRunner
from qwen_inference_lab_b200.kernels import kv4
from qwen_inference_lab_b200.parts import KVCacheSpec, LayerCall
from qwen_inference_lab_b200.parts.attention import PagedAttentionPlanner


class FakeModel:
    device, dtype = torch.device("cpu"), torch.bfloat16
    vocab_size, max_positions = 1000, 40000
    order = [LayerCall(0)]

    def is_graph_safe(self):
        return False

    def step_planners(self):
        return {PagedAttentionPlanner.key: PagedAttentionPlanner()}


def make(budget, rows, pages=6000, page_size=16):
    model = FakeModel()
    cache = CacheManager([KVCacheSpec(1, 32, bits=4)], num_pages=pages, page_size=page_size, max_requests=rows,
                         max_context=model.max_positions, dtype=model.dtype, device="cpu")
    return cache, StepRunner(model, cache, max_step_tokens=budget, use_graphs=False)


def test_recorded_steps_outlive_a_prompt_in_chunks():
    """Two prompts that come in chunks of 64 behind longer and longer contexts: their descriptions fit the memory that recorded steps point to."""
    cache, runner = make(128, 4)
    cache.admit("a")
    cache.admit("b")
    buffer, runner._graphs["recorded"] = runner._meta_dev, object()
    for start in range(0, 32000, 64):
        entries = [StepEntry(name, [1] * 64) for name in "ab"]
        for entry in entries:
            cache.ensure(entry.request_id, start + 64)
        runner._upload(runner._describe(entries).packed)
        for entry in entries:
            cache.advance(entry.request_id, start + 64)
    assert runner._meta_dev is buffer and "recorded" in runner._graphs


def test_memory_that_is_too_small_doubles():
    cache, runner = make(16, 2, pages=40)
    sizes = []
    for ints in range(runner._capacity + 1, 20 * runner._capacity, 7):
        runner._reserve(ints)
        sizes.append(runner._capacity)
    assert len(set(sizes)) <= 6


@pytest.mark.parametrize("seed", range(8))
def test_no_description_is_beyond_its_bound(seed, monkeypatch):
    monkeypatch.setattr(kv4, "MOST_READ", 1 << random.Random(seed).choice([6, 9, 16]))
    rng = random.Random(seed)
    for _ in range(60):
        requests, context = rng.randint(1, 40), int(2 ** rng.uniform(0, 15))
        lens = np.array([min(context, rng.choice([1, 1, 2, 3, 8, 9, 33, 64, 65, 300])) for _ in range(rng.randint(1, requests))])
        starts = np.array([rng.choice([0, context - n, rng.randint(0, context - n)]) for n in lens])
        arrays = kv4.describe_segments(np.cumsum(lens) - lens, starts, lens, np.arange(len(lens)), portion_tokens=False)
        ints = sum(max(4, -(-len(values) // 4) * 4) for values in arrays.values())
        assert ints <= kv4.most_ints(int(lens.sum()), requests, context)


def test_tokens_of_portions_are_described_where_they_are_asked_for():
    whole = kv4.describe_segments([0, 1, 10], [5, 7, 100], [1, 9, 20], [2, 0, 1])
    lean = kv4.describe_segments([0, 1, 10], [5, 7, 100], [1, 9, 20], [2, 0, 1], portion_tokens=False)
    assert set(whole) - set(lean) == {"portion_tokens"} and all((whole[name] == lean[name]).all() for name in lean)
    expected = [[1 + i, 7 + i, 0, 120] for i in range(9)] + [[10 + i, 100 + i, 1, 120] for i in range(20)]
    assert whole["portion_tokens"].reshape(-1, 4).tolist() == expected
    plan = kv4.StepPlan.of_segments([2, 0, 1], [5, 7, 100], [1, 9, 20], "cpu")
    array, tokens = plan.portion_tokens()
    assert tokens == 29 and array.view(-1, 4).tolist() == expected


def test_steps_do_not_upload_the_tokens_of_portions():
    cache, runner = make(128, 4, pages=40)
    cache.admit("a")
    cache.ensure("a", 64)
    assert not any(name.endswith("portion_tokens") for name in runner._describe([StepEntry("a", [1] * 64)]).offsets)


def test_a_recorded_step_goes_by_what_it_is_found_by():
    """Steps that share a recording (the number of requests, the bucket of the longest context and what the planner says) are planned alike,
    whichever of them came first."""
    from types import SimpleNamespace
    from qwen_inference_lab_b200.parts.attention import NarrowCachePlanner
    rng, found, planner = random.Random(3), {}, NarrowCachePlanner()
    for _ in range(400):
        n, longest = rng.choice([1, 2, 48]), rng.randint(513, 1024)
        starts = np.array([longest - 1] + [rng.randint(0, int((longest - 1) * rng.random())) for _ in range(n - 1)])
        lens, rows = np.ones(n, dtype=np.int64), np.arange(n)
        arrays = kv4.describe_segments(rows, starts, lens, rows)
        view = SimpleNamespace(array=arrays, count={name: len(values) for name, values in arrays.items()})
        ctx = SimpleNamespace(plans={kv4.PLAN_KEY: view}, h_seg_start=rows, h_seg_pos0=starts, h_seg_len=lens, h_seg_row=rows, max_context=1024, min_context=513)
        key = n, planner.recording(SimpleNamespace(starts=starts, lens=lens))
        found.setdefault(key, set()).add(kv4.StepPlan.of_step(ctx).singles)
    # one request fills its longest context, 48 drawn so do not
    assert {(1, 1.0), (2, 1.0), (2, 0.5), (48, 0.5)} <= set(found) and all(len(plans) == 1 for plans in found.values())


@pytest.mark.parametrize("rows,starts,lens", [([0], [2**31 - 1], [1]), ([0], [2**32 + 5], [1]), ([2**31], [0], [1]), ([0], [2**31 - 1000], [1]),
                                              ([0, 2**40], [0, 1], [1, 1])])
def test_a_plan_of_numbers_beyond_32_bits_is_refused(rows, starts, lens):
    with pytest.raises(kv4.KernelError, match="32-bit"):
        kv4.StepPlan.of_segments(rows, starts, lens, "cpu")


def test_segments_are_planned_by_their_own_contexts():
    """Spans of single tokens, of a few and of many go by the contexts of their own kind."""
    plan = kv4.StepPlan.of_segments(range(5), [9000, 96, 40, 5000, 60], [1, 4, 40, 1000, 20], "cpu")
    assert plan.singles == (9001, 0, 1.0) and plan.multi.max_context == 6000
    assert plan.few.max_context == plan.few_tokens.max_context == 100 and plan.few_tokens.fill == 1.0 and plan.few.fill == round(16 * 260 / 3 / 100) / 16
    assert plan.long == (6000, 0, round(16 * (80 + 6000 + 80) / 3 / 6000) / 16)
    one = kv4.StepPlan.of_segments([0], [50], [3], "cpu")
    assert one.few == one.few_tokens == one.multi == (53, 0, 1.0) and one.long == kv4.Reach(1, 0, 1.0)


def test_a_plan_of_the_callers_is_one_upload():
    starts, lens = [9000, 96, 40, 5000, 60, 3], [1, 4, 40, 1001, 20, 1]
    plan = kv4.StepPlan.of_segments(range(6), starts, lens, "cpu")
    expected = kv4.describe_segments(np.cumsum(lens) - lens, starts, lens, range(6))
    assert set(plan.array) == set(expected) and len({array.untyped_storage().data_ptr() for array in plan.array.values()}) == 1
    for name, values in expected.items():
        array = plan.array[name]
        assert array.tolist() == values.tolist() and plan.count[name] == len(values) and array.dtype == torch.int32
        assert (array.data_ptr() - plan.array["singles"].data_ptr()) % 16 == 0


def test_three_tiles_of_rows_are_not_cut_into_clusters_of_sixteen():
    """One request of 12 tokens with 4 heads on a key: 24 clusters of 16 blocks do not run at the same time."""
    reach = kv4.Reach(4012, 0, 1.0)
    spans = lambda blocks: kv4._spans(blocks, kv4.STEP_US[2][:3], 1.0, reach, 0, 128, kv4.JOINS_US[2], kv4.CLUSTERS[2])
    assert spans(24) == 8 and kv4._clustered(8, 24, kv4.STEP_US[2][:3], kv4.CLUSTERS[2])
    assert not kv4._clustered(16, 24, kv4.STEP_US[2][:3], kv4.CLUSTERS[2]) and kv4._clustered(16, 16, kv4.STEP_US[2][:3], kv4.CLUSTERS[2])
