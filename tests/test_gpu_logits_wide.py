"""The bias of rows so wide that a block for each 16 of their columns would be more threads
than a launch may have."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,acts", [(1, 2 ** 28 + 17), (3, 2 ** 24 + 5)])
def test_the_bias_of_wide_rows(rows, acts):
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    from junqi_amd import masks
    torch.cuda.empty_cache()
    x = torch.randn(9_999_991, device="cuda", generator=torch.Generator("cuda").manual_seed(acts)).to(torch.bfloat16)

    def numbers(n):
        return x.repeat(-(-n // x.numel()))[:n]
    logits = torch.zeros(rows, acts, dtype=torch.bfloat16, device="cuda")
    bias = numbers(acts).float().requires_grad_()
    d_out = numbers(rows * acts).view(rows, acts)
    out = masks.action_logits(logits, bias=bias)
    d_bias, = torch.autograd.grad(out, bias, d_out)
    assert torch.equal(out.detach()[0], bias.detach().to(torch.bfloat16))
    want = d_out[0].float()
    for r in range(1, rows):
        want += d_out[r]        # three terms: two roundings of at most their sum
    size = sum(d_out[r].float().abs() for r in range(rows))
    assert ((d_bias - want).abs() <= (4 * 2.0 ** -24 if rows > 1 else 0) * size).all()
    del logits, out, d_out, d_bias, bias, want, size
    torch.cuda.empty_cache()
