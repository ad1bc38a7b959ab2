"""Which of the other architectures can keep their keys and values in 4 bits: every case is built and asked (no GPU)."""
import importlib

import pytest

from qwen_inference_lab_b200.config import registry
from qwen_inference_lab_b200.parts import KVCacheSpec

FOLDERS = ["virulix", "debisun", "larolorn", "gogotar", "lotazen", "bugidra"]
CASES = [(folder, name) for folder in FOLDERS for name in importlib.import_module(f"tests.{folder}_cases").CASES]
ACCEPTED = {("lotazen", "D")}           # unit heads of 128 and 64 behind windows, beside states; the others have a layer that stands in the way


@pytest.mark.parametrize("folder,name", CASES)
def test_every_case_says_yes_or_which_layer_cannot(folder, name):
    cfg = importlib.import_module(f"tests.{folder}_cases").CASES[name]["config"]
    entry = registry.lookup(cfg)
    model = entry.build(entry.config_class.from_dict(cfg))
    if (folder, name) not in ACCEPTED:
        with pytest.raises(ValueError, match=r"layer \d+ cannot keep keys and values in 4 bits: "):
            model.cache_specs(kv_bits=4)
        return
    flat = lambda specs: [one for spec in specs for one in (spec if isinstance(spec, tuple) else (spec,))]
    narrow, wide = flat(model.cache_specs(kv_bits=4)), flat(model.cache_specs())
    assert [type(one) for one in narrow] == [type(one) for one in wide]
    assert [one.bits for one in narrow if isinstance(one, KVCacheSpec)] == [4, 4]
    assert all(one == other for one, other in zip(narrow, wide) if not isinstance(one, KVCacheSpec))


def test_the_cases_are_there():
    assert len(CASES) == 20 and ACCEPTED <= set(CASES)


def test_scales_that_the_kernels_do_not_take():
    from qwen_inference_lab_b200.parts import GroupedQueryAttention
    names = {k: k for k in "qkvo"}
    assert GroupedQueryAttention(64, 4, 2, 32, names=names, scale=0.1).kv_bits_refusal(4) is None
    for scale in (0.0, -0.2, float("nan")):
        assert "positive" in GroupedQueryAttention(64, 4, 2, 32, names=names, scale=scale).kv_bits_refusal(4)
