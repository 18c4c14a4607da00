"""What action_logits tells autograd, keeps and refuses, and its penalties at float32's ends, on
an MI355X."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def masks():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    from junqi_amd import masks as M
    return M


def test_forward_mode_is_refused(masks):
    """An input with a tangent is refused, whether it requires a gradient or not, and never taken
    as a constant: the logits and the bias, and each penalty of the rows' own."""
    import torch.autograd.forward_ad as fw
    recent = torch.tensor([[1, 1, 3]] * 4, device="cuda")
    args = {"logits": torch.randn(4, 9, device="cuda"), "bias": torch.randn(9, device="cuda"),
            "repetition": torch.full((4,), 1.5, device="cuda"), "frequency": torch.rand(4, device="cuda"),
            "presence": torch.rand(4, device="cuda")}

    def call(logits, **kw):
        return masks.action_logits(logits, recent=recent, **kw)
    plain = call(**args)
    for name in args:
        for grad in (False, True):
            with fw.dual_level():
                given = {k: v.detach() for k, v in args.items()}
                given[name] = fw.make_dual(given[name].clone().requires_grad_(grad), torch.ones_like(given[name]))
                for mode in (torch.enable_grad(), torch.no_grad()):
                    with mode, pytest.raises((NotImplementedError, ValueError, RuntimeError)):
                        call(**given)
    with fw.dual_level():     # inside a level, inputs without tangents are as anywhere else
        assert torch.equal(call(**args), plain)


def test_a_second_derivative_is_refused(masks):
    x, bias = torch.randn(4, 9, device="cuda", requires_grad=True), torch.randn(9, device="cuda", requires_grad=True)
    out = masks.action_logits(x, bias=bias, recent=torch.tensor([[1, 3]] * 4, device="cuda"), repetition=1.5)
    weight = torch.randn(4, 9, device="cuda", requires_grad=True)
    g = torch.autograd.grad((out * weight).sum(), [x, bias], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g[0].sum() + g[1].sum(), weight)
    for name in ("repetition", "frequency", "presence"):
        with pytest.raises(ValueError, match="no gradient"):
            masks.action_logits(x, recent=torch.tensor([[1]] * 4, device="cuda"), **{name: torch.ones(4, device="cuda", requires_grad=True)})


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_repetition_divides(masks, dtype):
    """x / repetition is one rounding, and so is its gradient: a product with a rounded
    reciprocal is two, and an infinity for a repetition below 2^-128."""
    g = torch.Generator().manual_seed(3)
    n, acts = 64, 257
    x = (2 * torch.randn(n, acts, generator=g)).to(dtype)
    d = torch.randn(n, acts, generator=g).to(dtype)
    rep = 0.5 + torch.rand(n, generator=g)
    rep[:3] = torch.tensor([1e-39, 2.5e-39, 3e38])       # the first two: float32's reciprocal is an infinity
    x[:2], d[:2] = (1e-10 * x[:2].float()).to(dtype), (1e-10 * d[:2].float()).to(dtype)
    x[2], d[2] = (1e30 * x[2].float().abs()).to(dtype), (1e30 * d[2].float()).to(dtype)
    recent = torch.arange(0, acts, 2).repeat(n, 1)
    named = torch.zeros(acts, dtype=torch.bool)
    named[::2] = True
    v, r = x.float(), rep[:, None]
    want = torch.where(named, torch.where(v > 0, v / r, v * r), v).to(dtype)
    want_d = torch.where(named, torch.where(v > 0, d.float() / r, d.float() * r), d.float()).to(dtype)
    leaf = x.cuda().requires_grad_()
    out = masks.action_logits(leaf, recent=recent.cuda(), repetition=rep.cuda())
    got, = torch.autograd.grad(out, leaf, d.cuda())
    assert want.isfinite().all() and want_d.isfinite().all()
    assert torch.equal(out.detach().cpu(), want)
    assert torch.equal(got.cpu(), want_d)


def test_what_the_backward_pass_keeps(masks):
    """The logits only where recent actions are held against them: else they are free to go, or
    to be changed in place, after the call."""
    legal = torch.rand(40, 16641, device="cuda") < 0.01
    d = torch.randn(40, 16641, device="cuda")
    x = torch.randn(40, 16641, device="cuda").requires_grad_()
    bias = torch.randn(16641, device="cuda").requires_grad_()
    for recent in (None, torch.randint(0, 16641, (40, 8), device="cuda")):
        held = []
        y = x * 1.0
        with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t.data_ptr()) or t, lambda t: t):
            masks.action_logits(y, bias=bias, legal=legal, recent=recent, repetition=1.5)
        assert (y.data_ptr() in held) == (recent is not None)
        out = masks.action_logits(y, bias=bias, legal=legal, recent=recent, repetition=1.5)   # autograd's own check: without hooks
        with torch.no_grad():
            y.mul_(2.0)
        if recent is None:
            g = torch.autograd.grad(out, [x, bias], d)
            assert torch.equal(g[0], torch.where(legal, d, 0.0))
            want = torch.where(legal, d, 0.0).double().sum(0)
            assert ((g[1] - want).abs() <= 40 * 2.0 ** -24 * torch.where(legal, d, 0.0).abs().double().sum(0)).all()
        else:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(out, [x, bias], d)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,recent", [((5, 700), 3000), ((3, 40000), 5000), ((2, 70001), 2049), ((4, 2048), 2048), ((60, 33), 2100)])
def test_long_lists_of_recent_actions(masks, shape, recent, dtype):
    """More of them than a wave's table has room for at once: the rows go in narrower parts."""
    from tests import test_gpu_logits as T
    for packed in (False, True):
        T._check(masks, T._inputs(sum(shape), *shape, dtype=dtype, density=0.3, recent=recent), packed=packed, int64=packed)
    T._check(masks, T._inputs(sum(shape) + 1, *shape, dtype=dtype, density=None, recent=recent, each=True), lengths=False)
