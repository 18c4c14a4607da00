"""The selective operators and the masked logits past 2^31 elements: the last rows of a large
call are those of a call on them alone, bit for bit."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def room():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def _rows(*shape, dtype=BF16, seed=1):
    """Numbers of their own for each place, quickly made."""
    x = torch.empty(shape, dtype=dtype, device="cuda")
    flat = x.view(-1)
    g = torch.Generator("cuda").manual_seed(seed)
    some = torch.randn(9_999_991, generator=g, device="cuda").to(dtype)
    for i in range(0, flat.numel(), some.numel()):
        part = flat[i:i + some.numel()]
        part.copy_(some[:part.numel()])
    return x


def test_scan():
    from junqi_amd import memory
    games, plies, d, n = 70000, 32, 1024, 4        # 2.3e9 elements of u
    u, delta = _rows(games, plies, d), _rows(games, plies, d, seed=2)
    b, c = _rows(games, plies, n, seed=3), _rows(games, plies, n, seed=4)
    a, bias = -torch.rand(d, n, device="cuda"), torch.full((d,), -3.0, device="cuda")

    def call(rows):
        leaves = [t[rows].requires_grad_() for t in (u, delta, b, c)]
        out, state = memory.selective_scan(leaves[0], leaves[1], a, leaves[2], leaves[3], delta_bias=bias, softplus=True, return_state=True)
        return [out.detach()[-3:].clone(), state.detach()[-3:].clone(), *(g[-3:].clone() for g in torch.autograd.grad(out, leaves, u[rows]))]
    whole = call(slice(None))
    for x, y in zip(whole, call(slice(games - 3, games))):
        assert torch.equal(x, y) and x.any()


def test_conv():
    from junqi_amd import memory
    games, plies, d = 70000, 32, 1024
    x = _rows(games, plies, d)
    weight, bias = torch.randn(d, 4, device="cuda"), torch.randn(d, device="cuda")

    def call(rows):
        leaf = x[rows].requires_grad_()
        out, state = memory.causal_conv(leaf, weight, bias, silu=True, return_state=True)
        return [out.detach()[-3:].clone(), state.detach()[-3:].clone(), torch.autograd.grad(out, leaf, x[rows])[0][-3:].clone()]
    whole = call(slice(None))
    for p, q in zip(whole, call(slice(games - 3, games))):
        assert torch.equal(p, q) and p.any()


def test_steps():
    from junqi_amd import memory
    rows, d, n = 140000, 1024, 16                  # 2.3e9 states
    state = _rows(rows, d, n, dtype=torch.float32)
    pick = torch.tensor([rows - 1, 5, rows - 70000], device="cuda")
    small = state[pick].clone()
    first = state[:5].clone()
    u, delta, b, c = (torch.randn(3, k, device="cuda").to(BF16) for k in (d, d, n, n))
    a = -torch.rand(d, n, device="cuda")
    out = memory.selective_scan_step(u, delta, a, b, c, state, softplus=True, rows=pick)
    want = memory.selective_scan_step(u, delta, a, b, c, small, softplus=True)
    assert torch.equal(out, want) and torch.equal(state[pick], small) and torch.equal(state[:5], first)
    del state
    rows = 800000
    held = _rows(rows, 3, d)                       # 2.5e9 inputs
    pick = torch.tensor([rows - 1, 7, rows - 300000], device="cuda")
    small = held[pick].clone()
    weight = torch.randn(d, 4, device="cuda")
    out = memory.causal_conv_step(u, weight, held, rows=pick)
    want = memory.causal_conv_step(u, weight, small)
    assert torch.equal(out, want) and torch.equal(held[pick], small)


def test_logits():
    from junqi_amd import masks
    n, acts = 135000, 16641                        # 2.2e9 logits
    x = _rows(n, acts)
    legal = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, 521), device="cuda", dtype=torch.int32)
    recent = torch.randint(0, acts, (n, 8), device="cuda")
    bias = torch.randn(acts, device="cuda")

    def call(rows):
        leaf = x[rows].requires_grad_()
        out = masks.action_logits(leaf, bias=bias, legal=legal[rows], recent=recent[rows], presence=1.0, repetition=1.5)
        return [out.detach()[-3:].clone(), torch.autograd.grad(out, leaf, x[rows])[0][-3:].clone()]
    whole = call(slice(None))
    for p, q in zip(whole, call(slice(n - 3, n))):
        assert torch.equal(p, q) and p.isfinite().any()


def test_far_plies():
    """Time-major rows more than 256 MiB apart: the scan takes a copy of them."""
    from junqi_amd import memory
    wide, d = 70000, 1024
    u = _rows(4, wide, d, dtype=torch.float32).transpose(0, 1)[:, :, :]     # plies 287 MB apart
    assert u.stride(1) * 4 > 1 << 28
    a = -torch.rand(d, 4, device="cuda")
    b = torch.randn(wide, 4, 4, device="cuda")
    out = memory.selective_scan(u, u, a, b, b, softplus=True)
    few = memory.selective_scan(u[-3:].contiguous(), u[-3:].contiguous(), a, b[-3:], b[-3:], softplus=True)
    assert torch.equal(out[-3:], few)


def test_the_widest_row():
    """As many actions as a call may have: the last columns' ends pass 32 bits."""
    from junqi_amd import masks
    acts, tail = 2 ** 31 - 1 - 4096, 70001
    x = _rows(1, acts)
    recent = torch.tensor([[acts - 1, 3, acts]], device="cuda")
    leaf = x.requires_grad_()
    out = masks.action_logits(leaf, recent=recent, presence=1.0, repetition=2.0)
    d, = torch.autograd.grad(out, leaf, x.detach())
    out = out.detach()
    for at in (slice(0, tail), slice(acts - tail, acts)):
        k = 3 if at.start == 0 else tail - 1
        few = x.detach()[:, at].clone()
        want, grad = few.clone(), few.clone()
        y = few[0, k].float()
        want[0, k] = ((y / 2 if y > 0 else y * 2) - 1).to(BF16)
        grad[0, k] = (y * (0.5 if y > 0 else 2.0)).to(BF16)
        assert torch.equal(out[:, at], want) and torch.equal(d[:, at], grad)
