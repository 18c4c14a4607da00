"""Penalties, biases and legal masks on the logits of the actions (junqi_amd.masks.action_logits)
on an MI355X against their definition in 64 bits (tests/selective_oracle.py)."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests import selective_oracle as O  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def masks():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    from junqi_amd import masks as M
    return M


def _pack(legal):
    n, a = legal.shape
    w = -(-a // 32)
    bits = torch.zeros(n, w * 32, dtype=torch.int64)
    bits[:, :a] = legal
    words = (bits.view(n, w, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _inputs(seed, n, a, dtype=F32, density=0.02, recent=9, bias=True, each=False):
    g = torch.Generator().manual_seed(seed)
    x = {"logits": (2 * torch.randn(n, a, generator=g)).to(dtype), "bias": torch.randn(a, generator=g) if bias else None,
         "legal": None if density is None else torch.rand(n, a, generator=g) < density, "recent": None, "recent_lengths": None,
         "repetition": 1.3, "frequency": 0.2, "presence": 0.4, "d_out": torch.randn(n, a, generator=g).to(dtype)}
    if density is not None:
        x["legal"][::7] = False      # a finished game has no legal action
    if recent:
        ids = torch.randint(0, a, (n, max(1, recent // 2)), generator=g).gather(1, torch.randint(0, max(1, recent // 2), (n, recent), generator=g))
        ids[:, ::4] = torch.randint(-3, a + 3, (n, len(range(0, recent, 4))), generator=g)
        x["recent"] = ids.to(torch.int32)
        x["recent_lengths"] = torch.randint(-1, recent + 3, (n,), generator=g, dtype=torch.int32)
        if x["legal"] is not None:       # some of the named actions are legal
            x["legal"].scatter_(1, ids.clamp(0, a - 1)[:, :3], True)
            x["legal"][::7] = False
    if each:
        x["repetition"], x["frequency"], x["presence"] = 0.5 + torch.rand(n, generator=g), torch.randn(n, generator=g), torch.randn(n, generator=g)
    return x


def _check(masks, x, packed=False, wide=0, int64=False, lengths=True):
    if not lengths:
        x["recent_lengths"] = None
    dtype = x["logits"].dtype
    c = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in x.items()}
    # a row's penalties are float32 numbers
    for k in ("repetition", "frequency", "presence"):
        if not isinstance(x[k], torch.Tensor):
            c[k] = float(torch.tensor(x[k], dtype=F32))
    want = O.logits(c)

    def at(t):      # a part of wider rows, at an odd element
        if not wide or t.ndim < 2:
            return t.cuda()
        w = torch.zeros(t.shape[0], t.shape[1] + wide, dtype=t.dtype, device="cuda")
        w[:, 1:1 + t.shape[1]] = t.cuda()
        return w[:, 1:1 + t.shape[1]]
    logits = at(x["logits"]).detach().requires_grad_()
    bias = None if x["bias"] is None else x["bias"].cuda().requires_grad_()
    legal = None if x["legal"] is None else at(_pack(x["legal"]) if packed else x["legal"])
    recent = None if x["recent"] is None else at(x["recent"].long() if int64 else x["recent"])
    rest = {k: x[k].cuda() if isinstance(x[k], torch.Tensor) else x[k] for k in ("repetition", "frequency", "presence", "recent_lengths")}
    out = masks.action_logits(logits, bias=bias, legal=legal, recent=recent, **rest)
    assert out.dtype == dtype
    got = out.detach().double().cpu()
    fine = want["out"].isfinite()
    assert torch.equal(got.isfinite(), fine) and bool((got[~fine] == -torch.inf).all())
    O.close("out", torch.where(fine, got, 0.0), torch.where(fine, want["out"], 0.0), want["size"], 8, dtype)
    leaves = [t for t in (logits, bias) if t is not None]
    g = torch.autograd.grad(out, leaves, at(x["d_out"]))
    O.close("d_logits", g[0], want["d_logits"], want["d_logits"].abs(), 4, dtype)
    if bias is not None:
        O.close("d_bias", g[1], want["d_bias"], want["size_bias"], x["logits"].shape[0], F32)


SHAPES = [(1, 1), (3, 7), (9, 31), (8, 32), (5, 100), (15, 129), (4, 4096), (3, 4097), (10, 8200), (30, 16641), (2, 50001)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("mask", ["none", "bool", "words"])
@pytest.mark.parametrize("shape", SHAPES)
def test_logits(masks, shape, mask, dtype):
    x = _inputs(sum(shape), *shape, dtype=dtype, density=None if mask == "none" else 0.03)
    _check(masks, x, packed=mask == "words")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("what", [{"recent": 0}, {"recent": 1}, {"recent": 700}, {"bias": False}, {"each": True}, {"density": 1.0}, {"density": 0.0}])
def test_logits_options(masks, what, dtype):
    x = _inputs(17, 13, 5003, dtype=dtype, **what)
    for packed in (False, True):
        _check(masks, dict(x), packed=packed, int64=packed, lengths=not packed)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wide", [1, 3, 6])
def test_logits_of_wider_rows(masks, wide, dtype):
    for packed in (False, True):
        _check(masks, _inputs(wide, 11, 4133, dtype=dtype), packed=packed, wide=wide)


def test_rows_of_nothing_and_broadcast_rows(masks):
    out = masks.action_logits(torch.zeros(0, 9, device="cuda"), legal=torch.zeros(0, 9, dtype=torch.bool, device="cuda"))
    assert out.shape == (0, 9)
    bias = torch.zeros(9, device="cuda", requires_grad=True)
    x = torch.zeros(0, 9, device="cuda", requires_grad=True)
    g = torch.autograd.grad(masks.action_logits(x, bias=bias), [x, bias], torch.zeros(0, 9, device="cuda"))
    assert g[0].shape == (0, 9) and not g[1].any()
    one = torch.randn(1, 300, device="cuda")
    legal = (torch.rand(1, 300, device="cuda") < 0.5).expand(5, 300)
    out = masks.action_logits(one.expand(5, 300), legal=legal, recent=torch.tensor([[3, 3]], device="cuda").expand(5, 2), presence=1.0)
    assert torch.equal(out, masks.action_logits(one, legal=legal[:1], recent=torch.tensor([[3, 3]], device="cuda"), presence=1.0).expand(5, 300))


def test_masked_values_do_not_matter(masks):
    """NaN and infinities of logits, biases and gradients at illegal actions; the type's lowest value at legal ones."""
    x = _inputs(23, 9, 1000, density=0.1)
    legal = x["legal"].cuda()
    low = torch.finfo(F32).min
    logits, d = x["logits"].cuda(), x["d_out"].cuda()
    logits[legal] = low
    dirty, dirty_d = logits.clone(), d.clone()
    dirty[~legal], dirty_d[~legal] = float("nan"), float("inf")
    both = []
    for v, g in ((logits, d), (dirty, dirty_d)):
        v = v.requires_grad_()
        bias = x["bias"].cuda().requires_grad_()
        out = masks.action_logits(v, bias=bias, legal=legal, recent=x["recent"].cuda(), repetition=0.5, presence=0.4)
        both.append([out.detach(), *torch.autograd.grad(out, [v, bias], g)])
    for a, b in zip(*both):
        assert torch.equal(a, b)
    assert not both[0][0][legal].isnan().any()


def test_the_environment_s_masks(masks):
    """Its packed masks and its bool masks leave the same actions, those of the CSR rows."""
    import junqi_amd
    r = junqi_amd.GpuRollout(40, show_mode=2)
    r.reset(3)
    got = r.batch.legal(mask_words=True, mask_bool=True)
    logits = torch.randn(40, 16641, device="cuda")
    a = masks.action_logits(logits, legal=got["mask_words"].view(40, -1))
    b = masks.action_logits(logits, legal=got["mask_bool"].view(40, -1).bool())
    assert torch.equal(a, b)
    assert torch.equal(a, logits.masked_fill(~got["mask_bool"].view(40, -1).bool(), -torch.inf))
    assert bool((a.isfinite().sum(1) > 0).all())


def test_logits_on_another_stream_and_in_a_graph(masks):
    x = _inputs(29, 20, 16641)
    there = x["logits"].cuda(), x["bias"].cuda()
    legal, recent, d = _pack(x["legal"]).cuda(), x["recent"].cuda(), x["d_out"].cuda()

    def both():
        logits, bias = (t.detach().requires_grad_() for t in there)   # leaves of this call's own graph
        out = masks.action_logits(logits, bias=bias, legal=legal, recent=recent, repetition=1.5, frequency=0.1)
        return [out, *torch.autograd.grad(out, [logits, bias], d)]
    want = [v.detach().clone() for v in both()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        got = both()
    for _ in range(4):
        for v in got:
            v.detach().fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want))
        both()
        torch.cuda.synchronize()
