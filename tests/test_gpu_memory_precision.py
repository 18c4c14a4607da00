"""Mean errors of linear attention's results on an MI355X against the definition in
64 bits: bfloat16 results are rounded once, from sums that are held in float32."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests import memory_oracle as O  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def memory():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    from junqi_amd import memory as M
    return M


def _check(memory, seed, b, t, h, dk, dv, dtype, *, starts=0.02, lengths=None, time_major=False):
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape, to=F32):
        return torch.randn(shape, generator=g, device="cuda").to(to)

    def rows(d):
        x = randn(*((t, b) if time_major else (b, t)), h, d, to=dtype)
        return x.transpose(0, 1) if time_major else x
    q, k, v, d_out = rows(dk), rows(dk), rows(dv), rows(dv)
    state, d_state = randn(b, h, dk, dv), randn(b, h, dk, dv)
    decay = -torch.exp2(-8 * torch.rand(h, generator=g, device="cuda"))      # memories of 1 to 256 plies
    begins = torch.rand(b, t, generator=g, device="cuda") < starts
    if lengths is not None:
        lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    scale = dk ** -0.5
    args = (*(x.double() for x in (q, k, v, decay)), begins, lengths, state.double(), scale, d_out.double(), d_state.double())
    want, terms = O.define(*args), O.spread(*args)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, state)]
    out, last = memory.linear_attention(*leaves[:3], decay, starts=begins, lengths=lengths, initial_state=leaves[3],
                                        return_state=True)
    got = (out, last, *torch.autograd.grad([out, last], leaves, [d_out, d_state]))
    for name, x, w, s in zip(O.NAMES, got, want, terms):
        O.check_rms(name, x.detach(), w, s, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(64, 8, 2, 32, 32), (16, 33, 2, 64, 64), (8, 40, 2, 128, 128), (9, 70, 3, 40, 56), (5, 300, 2, 64, 36),
                                   (3, 200, 2, 24, 128), (4, 129, 1, 128, 96), (2, 500, 2, 16, 16), (40, 1, 2, 64, 64)])
def test_attention_errors_in_the_mean(memory, shape, dtype):
    print(f"[attention] {shape} {dtype}", flush=True)
    _check(memory, sum(shape), *shape, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,lengths,starts", [((2, 900, 3, 64, 40), (730, 900), 0.002), ((2, 1100, 2, 128, 72), (1100, 645), 0.002),
                                                  ((3, 700, 4, 96, 128), (700, 0, 333), 0.0), ((2, 1300, 2, 32, 24), (1, 1299), 0.005),
                                                  ((8, 560, 8, 128, 128), None, 0.001), ((40, 530, 5, 64, 64), None, 0.001)])
def test_attention_in_segments(memory, shape, lengths, starts, dtype):
    """Long axes that are split: heads of every width, keys and values of different dims, games
    that end inside a segment or before it, states that are carried over several."""
    print(f"[segments] {shape} {dtype}", flush=True)
    _check(memory, sum(shape), *shape, dtype, starts=starts, lengths=lengths, time_major=shape[0] == 3)
