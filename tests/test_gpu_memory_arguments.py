"""Arguments at the edges of what the memory operators take, on an MI355X."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def memory():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    from junqi_amd import memory as M
    return M


def test_an_output_that_cannot_be_written_is_refused(memory):
    """Elements that share memory, and an output whose gradient belongs to another result."""
    decay, state = torch.zeros(2, device="cuda"), torch.zeros(3, 2, 8, 8, device="cuda")
    ply = [torch.ones(3, 2, 8, device="cuda") for _ in range(3)]
    shared = torch.zeros(1, 2, 8, device="cuda").expand(3, 2, 8), torch.zeros(3, 1, 8, device="cuda").expand(3, 2, 8)
    learned = torch.zeros(3, 2, 8, device="cuda", requires_grad=True)
    for out in (*shared, learned, learned * 2):
        with pytest.raises(ValueError, match="out"):
            memory.linear_attention_step(*ply, decay, state, out=out)
        assert not state.any()
    one = torch.empty(1, 1, 8, device="cuda").expand(1, 1, 8)
    memory.linear_attention_step(*(x[:1, :1] for x in ply), decay[:1], state[:1, :1].clone(), out=one)
    with torch.no_grad():
        memory.linear_attention_step(*ply, decay, state, out=learned)
    assert learned.any()


@pytest.mark.parametrize("shape", [(0, 2, 3, 2, 8), (2, 3, 0, 2, 8), (2, 3, 4, 0, 8), (2, 3, 0, 0, 8), (2, 0, 8), (0, 2, 8), (3, 4, 0, 8)])
def test_rotary_of_nothing(memory, shape):
    x = torch.empty(shape, device="cuda", requires_grad=True)
    positions = torch.zeros(*shape[:-2], 2, dtype=torch.int64, device="cuda")
    out = memory.rotary(x, positions, memory.rotary_frequencies((2, 2), device="cuda"), (2, 2))
    assert out.shape == shape
    assert torch.autograd.grad(out, x, torch.empty_like(out))[0].shape == shape
