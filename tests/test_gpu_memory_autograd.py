"""What autograd is told of the memory operators' calls on an MI355X."""

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


def _rows(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape))).cuda()


def test_a_state_that_moved_on_is_not_learned_from(memory):
    """A segment saves the state before it for its backward pass: after a ply on the
    same memory the gradient would be of another state, which autograd refuses, as
    it does after any other write in place."""
    state, decay = _rows(3, 2, 8, 8), torch.tensor([-0.1, -0.2], device="cuda")
    q = _rows(3, 5, 2, 8).requires_grad_()
    ply = [_rows(3, 2, 8) for _ in range(3)]
    out = memory.linear_attention(q, q, q, decay, initial_state=state)
    memory.linear_attention_step(*ply, decay, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    # a copy of it, or a view of the same memory: as for any tensor
    out = memory.linear_attention(q, q, q, decay, initial_state=state.clone())
    memory.linear_attention_step(*ply, decay, state)
    out.sum().backward()
    pool = _rows(4, 2, 8, 8)
    out = memory.linear_attention(q, q, q, decay, initial_state=pool[1:])
    memory.linear_attention_step(*ply, decay, pool[1:])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_an_output_that_was_written_again_is_not_learned_from(memory):
    state, decay = _rows(3, 2, 8, 8), torch.tensor([-0.1, -0.2], device="cuda")
    ply = [_rows(3, 2, 8) for _ in range(3)]
    out, weight = torch.empty(3, 2, 8, device="cuda"), torch.ones(3, 2, 8, device="cuda", requires_grad=True)
    memory.linear_attention_step(*ply, decay, state, out=out)
    loss = (out * weight).sum()
    memory.linear_attention_step(*ply, decay, state, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_a_ply_in_inference_mode(memory):
    decay = torch.tensor([-0.1, -0.2], device="cuda")
    ply = [_rows(3, 2, 8) for _ in range(3)]
    state = _rows(3, 2, 8, 8)
    want = memory.linear_attention_step(*ply, decay, state.clone())
    with torch.inference_mode():
        held = state.clone()
        out = memory.linear_attention_step(*ply, decay, held, out=torch.empty_like(want))
    assert torch.equal(out, want) and not torch.equal(held, state)
