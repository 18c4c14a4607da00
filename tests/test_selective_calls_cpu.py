"""What the selective operators and the masked logits refuse, beside test_selective_cpu.py:
without a GPU, every refusal comes before any launch."""

from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def jl():
    from junqi_amd import _lib
    return _lib


@pytest.mark.parametrize("name,number", [("frequency", 1e39), ("presence", -1e39), ("repetition", 1e39), ("repetition", 1e-50),
                                         ("repetition", 3.4028236e38), ("frequency", float("-inf")), ("repetition", 7e-46)])
def test_penalties_that_float32_does_not_hold(name, number):
    """They would reach the kernel as an infinity, or as a repetition of 0."""
    from torch._subclasses import FakeTensorMode

    from junqi_amd import masks
    with FakeTensorMode():      # a call that is not refused ends at the data, with another error
        x = torch.empty(4, 70, device="cuda")
        recent = torch.empty(4, 5, dtype=torch.int32, device="cuda")
        with pytest.raises(ValueError, match=name):
            masks.action_logits(x, recent=recent, **{name: number})
