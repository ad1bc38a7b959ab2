"""The cache of 4 bits without a GPU: its pages in the cache manager, which models can have it, the plan of a step, the plain
implementation itself."""
import numpy as np
import pytest
import torch

from qwen_inference_lab_b200.cache import CacheError, CacheManager
from qwen_inference_lab_b200.config import registry
from qwen_inference_lab_b200.kernels import kv4
from qwen_inference_lab_b200.kernels.ops import KernelError
from qwen_inference_lab_b200.parts import GroupedQueryAttention, KVCacheSpec, RotaryFrequencies, StateSpec
from tests.plain import kv4_plain as plain
from tests.tiny_configs import TINY_A, TINY_B, TINY_D


def build(cfg):
    return registry.lookup(cfg).build(registry.lookup(cfg).config_class.from_dict(cfg))


def manager(specs, page_size=16):
    return CacheManager(specs, num_pages=6, page_size=page_size, max_requests=2, max_context=64, dtype=torch.float32, device="cpu")


def test_pages_of_the_manager():
    spec = KVCacheSpec(2, 64, bits=4)
    cache = manager([spec, KVCacheSpec(2, 64), spec, (KVCacheSpec(1, 32, window=20, bits=4), StateSpec((3,)))])
    views = cache.views()
    assert views[0].pages.dtype == torch.uint8 and views[0].pages.shape == (6, 2, 2, 2, 320) and views[0].bits == 4
    assert views[1].pages.dtype == torch.float32 and views[1].bits == 0 and views[2].pages.data_ptr() != views[0].pages.data_ptr()
    assert views[3][0].pages.shape == (6, 2, 1, 2, 160) and views[3][0].window == 20
    cache.poison()
    assert (views[0].pages == 255).all() and views[0].pages.view(torch.bfloat16).isnan().all()
    assert list(cache.step_planners()) == [kv4.PLAN_KEY] and manager([KVCacheSpec(2, 64)]).step_planners() == {}
    # 5 bits an element against 32
    assert views[0].pages.numel() * 32 == views[1].pages.numel() * 4 * 5


@pytest.mark.parametrize("spec,page", [(KVCacheSpec(2, 48, bits=4), 16), (KVCacheSpec(2, 288, bits=4), 16), (KVCacheSpec(2, 64, bits=4), 12),
                                       (KVCacheSpec(2, 64, v_head_dim=32, bits=4), 16), (KVCacheSpec(2, 64, shared_rows=True, bits=4), 16),
                                       (KVCacheSpec(2, 64, bits=8), 16)])
def test_the_manager_refuses_what_has_no_such_pages(spec, page):
    with pytest.raises(CacheError):
        manager([spec], page)


def test_which_models_can_have_it():
    model = build(TINY_B)
    specs = model.cache_specs(kv_bits=4)
    assert [s.bits for s in specs] == [4] * 3 and [s.bits for s in model.cache_specs()] == [0] * 3
    assert build(TINY_D).cache_specs(kv_bits=4)[0] == KVCacheSpec(2, 128, bits=4)
    for cfg, bits, why in ((TINY_A, 4, "multiple of 32"), (TINY_B, 8, "4 bits")):
        with pytest.raises(ValueError, match=why):
            build(cfg).cache_specs(kv_bits=bits)


def test_which_attention_can_have_it():
    names = {k: k for k in ("q", "k", "v", "o", "q_norm", "k_norm", "distance_bias", "sink")}
    make = lambda **options: GroupedQueryAttention(64, 4, 2, options.pop("dim", 32), names=names, **options)
    turn = lambda **options: RotaryFrequencies(16, 1e4, **options)
    for options in (dict(), dict(qk_norm_eps=1e-6), dict(window=9), dict(position=turn(layout="interleaved"), unit_qk_norm_eps=1e-6),
                    dict(position=turn(ramp=(4.0, 100, 32, 1)), qk_norm_eps=1e-5, head_gate="g", values_from_keys=True), dict(reads_shared_cache=True)):
        assert make(**options).kv_bits_refusal(4) is None
    for options in (dict(dim=48), dict(dim=288), dict(v_head_dim=64), dict(softcap=30.0), dict(conv_taps=4), dict(chunk=8), dict(sink=True),
                    dict(distance_slopes=[0.5] * 4), dict(q_temperature=(0.1, 64)), dict(distance_bias=(8, 64)), dict(whole_qk_norm_eps=1e-6),
                    dict(position=turn(), value_mix=("s", False))):
        assert make(**options).kv_bits_refusal(4)


@pytest.mark.parametrize("folder", ["virulix", "debisun", "larolorn", "gogotar", "lotazen", "bugidra"])
def test_other_architectures_say_what_stands_in_the_way(folder):
    """Each has a layer whose scores, norms or sizes the kernels do not have; the message names the layer."""
    import importlib
    cases = importlib.import_module(f"tests.{folder}_cases")
    found = [value for value in vars(cases).values() if isinstance(value, dict) and "architectures" in value]
    for cfg in found:
        try:
            model = build(cfg)
        except Exception:                      # a configuration that needs more than its own text
            continue
        with pytest.raises(ValueError, match=r"layer \d+ cannot keep"):
            model.cache_specs(kv_bits=4)


def test_the_plan_of_a_step():
    first, starts, lens, rows = [0, 1, 6, 306, 307], [5, 9, 100, 70, 0], [1, 5, 300, 1, 64], [0, 3, 2, 1, 4]
    arrays = kv4.describe_segments(first, starts, lens, rows)
    assert arrays["singles"].reshape(-1, 8).tolist() == [[0, 5, 1, 0, 0, 71, 0, 0], [306, 70, 1, 1, 1, 71, 0, 0]]
    assert arrays["few"].reshape(-1, 8).tolist() == [[1, 9, 5, 3, 0, 14, 0, 0]]
    assert arrays["multi"].reshape(-1, 8)[:, :5].tolist() == [[1, 9, 5, 3, 0], [6, 100, 300, 2, 5], [307, 0, 64, 4, 305]]
    assert arrays["few_tokens"].reshape(-1, 4).tolist() == [[1 + i, 9 + i, 3, 14] for i in range(5)]
    # every token of a portion lies in one segment and, beyond a few tokens, in one tile of its batch, whose row is that of the segment's pages
    seen = {}
    batch = 0
    while f"b{batch}.read" in arrays:
        read, table = arrays[f"b{batch}.read"].reshape(-1, 4), arrays[f"b{batch}.table"]
        spread, width = arrays[f"b{batch}.spread"].reshape(-1, 4), len(table) // len(read)
        assert (spread[:, (0, 3)] == read[:, (0, 3)]).all() and (read[:, 1] == 0).all()
        assert (read[:, 2] == np.where(spread[:, 2] - spread[:, 1] > kv4.FEW_TOKENS, spread[:, 2], 0)).all()
        for name, most in (("tiles", 64), ("segments", 1 << 20)):
            for token, pos, count, local in arrays[f"b{batch}.{name}"].reshape(-1, 4):
                row, begin, end, page = spread[local]
                assert begin <= pos and count <= most and pos + count <= end <= width * kv4.READ_PAGE and page == local * width
                for i in range(count):
                    assert (name, token + i) not in seen
                    seen[name, token + i] = (row, pos + i)
        batch += 1
    tiled = {**{6 + i: (2, 100 + i) for i in range(300)}, **{307 + i: (4, i) for i in range(64)}}
    assert seen == {**{(name, t): at for name in ("tiles", "segments") for t, at in tiled.items()},
                    **{("segments", 1 + i): (3, 9 + i) for i in range(5)}}
    # consecutive steps of the same single tokens: positions change, nothing else
    old = kv4.describe_segments([0, 1], [5, 9], [1, 1], [4, 2])
    kv4.refresh_single_tokens(old, np.array([6, 31]))
    new = kv4.describe_segments([0, 1], [6, 31], [1, 1], [4, 2])
    assert all((old[name] == new[name]).all() for name in new) and list(old) == list(new)


def test_long_contexts_are_read_in_batches():
    n = kv4.MOST_READ // kv4.READ_PAGE
    starts = [kv4.READ_PAGE * (n // 2), 3 * kv4.MOST_READ, 10, 20]
    arrays = kv4.describe_segments([0, 50, 100, 150], starts, [50] * 4, [0, 1, 2, 3])
    sizes = [len(arrays[f"b{i}.table"]) * kv4.READ_PAGE for i in range(2)]
    reads = [arrays[f"b{i}.read"].reshape(-1, 4)[:, 0].tolist() for i in range(2)]
    assert reads[0] == [1] and sizes[0] >= 3 * kv4.MOST_READ + 50            # longer than a batch may be: alone
    assert all(sum(len(arrays[f"b{i}.read"]) // 4 for i in range(k)) <= 4 for k in (1, 2))


def test_spans_fill_the_gpu():
    """More requests, fewer spans; a context of one step is not cut; never more spans than there is room for."""
    plan = lambda context: kv4.StepPlan.of_segments([0], [context - 1], [1], "cpu").singles
    spans = lambda blocks, context, window=0, most=128: kv4._spans(blocks, kv4.STEP_US[1], 1.0, plan(context), window, most)
    assert spans(8, 100) == 1 and spans(8, 8192) >= 16 and spans(64, 8192) == 8 and spans(2000, 8192) <= 2
    assert spans(8, 8192, most=3) == 3 and spans(8, 100000, window=100) == spans(8, 228)
    counts = [spans(blocks, 16384) for blocks in (8, 32, 128, 600)]
    assert counts == sorted(counts, reverse=True)
    # ragged contexts are cut more finely than as many of the longest; segments of several tokens do not count among single ones
    ragged = kv4.StepPlan.of_segments(range(49), [*range(0, 16320, 340), 30000], [1] * 48 + [20], "cpu")
    assert ragged.singles.max_context == 15981 and ragged.singles.fill == 0.5 and ragged.multi == (30020, 0, 1.0)
    even = kv4.StepPlan.of_segments(range(48), [15980] * 48, [1] * 48, "cpu")
    assert kv4._spans(384, kv4.STEP_US[1], 1.0, ragged.singles, 0, 128) > kv4._spans(384, kv4.STEP_US[1], 1.0, even.singles, 0, 128)


def test_scratch_that_a_recorded_graph_points_to(monkeypatch):
    """Grown scratch replaces the old one; what was handed out while a graph was recorded stays; counters that are zeroed by the graph
    serve no other call; devices have their own."""
    recording = [False]
    monkeypatch.setattr(kv4, "_capturing", lambda: recording[0])
    extras, cpu = {}, torch.device("cpu")
    small = kv4._scratch(extras, cpu, 2, 4, 3, 32)
    assert kv4._scratch(extras, cpu, 2, 4, 2, 32) is small and "kv4_recorded" not in extras and not small[2].any()
    recording[0] = True
    assert kv4._scratch(extras, cpu, 1, 4, 3, 32) is small and extras["kv4_recorded"] == [small]
    own = kv4._scratch(extras, cpu, 20, 4, 3, 32)
    assert own is not small and len(extras["kv4_recorded"]) == 2 and kv4._scratch(extras, cpu, 20, 4, 3, 32) is not own
    rows = kv4._rows(extras, cpu, 100)
    recording[0] = False
    assert kv4._scratch(extras, cpu, 2, 4, 3, 32) is small
    assert kv4._scratch(extras, cpu, 20, 4, 3, 32) is not own and kv4._rows(extras, cpu, 200) is not rows
    kept = [tensor.data_ptr() for tensors in extras["kv4_recorded"] for tensor in tensors]
    assert small[0].data_ptr() in kept and own[2].data_ptr() in kept and rows.data_ptr() in kept
    assert kv4._scratch(extras, torch.device("meta"), 2, 4, 3, 32)[0].device.type == "meta"


def test_a_plan_of_host_segments():
    plan = kv4.StepPlan.of_segments([2, 0], [7, 0], [1, 20], "cpu")
    assert plan.max_context == 20 and plan.tokens == 21 and len(plan.portion_lens) == 1 and plan.count["singles"] == 8
    empty = kv4.StepPlan.of_segments([], [], [], "cpu")
    assert empty.max_context == 0 and not any(empty.count.values())
    for wrong in (([0], [0], [0]), ([0], [-1], [1]), ([-1], [0], [1]), ([0, 1], [0], [1])):
        with pytest.raises(KernelError):
            kv4.StepPlan.of_segments(*wrong, "cpu")


def test_cpu_tensors_are_refused():
    z = torch.zeros
    with pytest.raises(KernelError, match="CUDA"):
        kv4.store(z(1, 96), (0, 32, 64), z(1, 32), z(1, 2, 1, 1, 160, dtype=torch.uint8), z(1, dtype=torch.int32), z(1, dtype=torch.int32),
                  z(1, 1, dtype=torch.int32), 1, 1, 32, 8)
    with pytest.raises(KernelError):
        kv4.page_shape(2, 40, 16)


def test_the_plain_implementation():
    """The bound that the format promises: no element further off than half a step and the roundings of step and base, 15 2^-9 steps and
    2^-9 |base| (a bfloat16 rounding is 2^-9 of a binade's upper end at most, 2^-8 of the value)."""
    torch.manual_seed(0)
    y = torch.randn(50, 3, 64).double() * torch.logspace(-3, 3, 50).double()[:, None, None]
    codes, pairs = plain.coded(y)
    held = plain.values(codes, pairs)
    groups = y.unflatten(-1, (-1, 32))
    step = (groups.amax(-1) - groups.amin(-1)) / 15
    bar = (0.5 + 15 * 2.0 ** -8) * step * (1 + 2.0 ** -8) + 2.0 ** -8 * groups.amin(-1).abs()
    assert ((held - y).abs().unflatten(-1, (-1, 32)) <= bar[..., None]).all()
    pages = torch.zeros(2, 2, 3, 2, 320, dtype=torch.uint8)
    plain.put(pages, 1, 0, 2, 11, codes[7, 1], pairs[7, 1])
    back = plain.get(pages, 1, 0, 2, 11)
    assert torch.equal(back[0], codes[7, 1]) and torch.equal(back[1].view(torch.int16), pairs[7, 1].view(torch.int16))
    built, table, held = plain.build([y[:20, :, :32]], [y[20:40, :, :32]], [20], 8)
    for t in (0, 7, 8, 19):
        codes, pairs = plain.get(built, int(table[0, t // 8]), 1, 2, t % 8)
        assert torch.equal(plain.values(codes, pairs), held[0][1][t, 2])
