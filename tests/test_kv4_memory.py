"""What the 4-bit attention keeps from call to call, as it grows with a prompt that comes in chunks (no GPU)."""
import weakref

import pytest
import torch

from qwen_inference_lab_b200.kernels import kv4

CPU = torch.device("cpu")


def test_rows_of_a_growing_context_are_allocated_a_few_times(monkeypatch):
    """Chunks of 64 tokens behind 0, 64, 128, ...: every call asks for a page more."""
    monkeypatch.setattr(kv4, "_capturing", lambda: False)
    extras, made, page = {}, [], 640
    for pages in range(1, 513):
        buffer = kv4._rows(extras, CPU, pages * page)
        assert pages * page <= buffer.numel() <= 2 * pages * page
        if not made or made[-1] != buffer.numel():
            made.append(buffer.numel())
    assert len(made) <= 10 and made == sorted(made)               # 2^9 pages
    assert kv4._rows(extras, CPU, 3) is buffer


def test_rows_grow_by_so_much_at_most(monkeypatch):
    monkeypatch.setattr(kv4, "_capturing", lambda: False)
    monkeypatch.setattr(kv4, "MOST_GROWTH", 1000)
    extras = {}
    sizes = [kv4._rows(extras, CPU, n).numel() for n in (900, 901, 1801, 2801, 9000)]
    assert sizes == [900, 1800, 2800, 3800, 9000]


@pytest.mark.parametrize("recorded", [False, True])
def test_rows_are_given_back_before_larger_ones_are_asked_for(monkeypatch, recorded):
    capturing = [recorded]
    monkeypatch.setattr(kv4, "_capturing", lambda: capturing[0])
    extras = {}
    old = weakref.ref(kv4._rows(extras, CPU, 100))
    capturing[0] = False
    real, seen = torch.empty, []

    def watched(*args, **kwargs):
        seen.append(old() is None)
        return real(*args, **kwargs)

    monkeypatch.setattr(torch, "empty", watched)
    kv4._rows(extras, CPU, 101)
    assert seen == [not recorded]
