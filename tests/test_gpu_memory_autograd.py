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


def test_forward_mode_is_refused(memory):
    """No operator has a forward-mode derivative: an input with a tangent is refused, whether
    it requires a gradient or not, and never taken as a constant."""
    import torch.autograd.forward_ad as fw
    q, decay, state = _rows(2, 5, 2, 8), torch.tensor([-0.1, -0.2], device="cuda"), _rows(2, 2, 8, 8)
    positions = torch.zeros(2, 5, 1, dtype=torch.int32, device="cuda")
    frequencies, weight, bias = memory.rotary_frequencies((4,), device="cuda"), _rows(8), _rows(8)
    ply, low = [x.clone() for x in q[:, 0].expand(3, 2, 2, 8)], decay.clone()

    def attention(q1, k1, v1, d1, s1):
        return memory.linear_attention(q1, k1, v1, d1, initial_state=s1)
    calls = [(attention, [q, q, q, decay, state]), (memory.linear_attention_step, [*ply, low, state]),
             (lambda x, f: memory.rotary(x, positions, f, (4,)), [q, frequencies]), (memory.layer_norm, [q, weight, bias])]
    for call, args in calls:
        plain = call(*args) if call is not memory.linear_attention_step else None
        for i in range(len(args)):
            for grad in (False, True):
                with fw.dual_level():
                    given = [a.detach() for a in args]
                    given[i] = fw.make_dual(given[i].clone().requires_grad_(grad), torch.ones_like(args[i]))
                    before = state.clone()
                    with pytest.raises((NotImplementedError, ValueError)):
                        call(*given)
                    with torch.no_grad(), pytest.raises((NotImplementedError, ValueError)):
                        call(*given)
                    assert torch.equal(state, before)
        if plain is not None:     # inside a level, inputs without tangents are as anywhere else
            with fw.dual_level():
                assert torch.equal(call(*args), plain)
    with pytest.raises(RuntimeError):
        torch.func.jvp(memory.layer_norm, (q,), (torch.ones_like(q),))
