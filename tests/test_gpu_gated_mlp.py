"""nsw.GatedMLP at every width that its gated product takes: forward and backward."""
import math

import pytest
import torch

import nsw
from nsw import ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def close(got, want, mag, terms, dtype, before=None):
    """Within (terms + 8) u of the sum of magnitudes, and one rounding to the type.  before: what a residual is added to;
    the GEMM's epilogue stages it in the output's type, so it is rounded, too: half a step of it (and of its own error e,
    as the last rounding) more, (e + step (|before| + e)) (1 + step) + step |want| in all."""
    step = torch.finfo(dtype).eps / 2
    assert got.dtype == dtype and got.shape == want.shape
    err = mag * (terms + 8) * U
    if before is not None:
        err = err + step * (1 + 1e-6) * (before.abs() + err)
    over = (got.double() - want).abs() - (err * (1 + step) + want.abs() * step * (1 + 1e-6))
    assert (over <= torch.finfo(dtype).tiny).all(), over.max().item()


@pytest.mark.parametrize("epi", [0, 1, 3])
@pytest.mark.parametrize("M,N,K", [(1, 8, 16), (300, 8, 16), (129600, 512, 16), (1, 8, 48), (5, 104, 80), (300, 520, 112), (4100, 512, 1360), (2000, 1024, 176),
                                   (16203, 2056, 240), (700, 4096, 16 * 63), (8100, 1024, 304)])
def test_bf16_products_of_half_a_step_more(device, epi, M, N, K):
    """K 16 more than whole steps of 32, on all tile sizes."""
    g = torch.Generator().manual_seed(K)
    r = lambda *s: torch.randn(*s, generator=g).to(device=device, dtype=BF16)
    x, w, b, res = r(M, K), r(N, K) * K ** -0.5, r(N), r(M, N)
    y = ops.linear(x, w, b if epi else None, res if epi == 3 else None, epilogue=epi)
    want, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    if epi:
        want, mag = want + b.double(), mag + b.double().abs()
    before = want if epi == 3 else None
    if epi == 3:
        want, mag = want + res.double(), mag + res.double().abs()
    close(y, want, mag, K + 2, BF16, before)


@pytest.mark.parametrize("epi", [2, 4])
@pytest.mark.parametrize("M,N,K", [(5, 104, 80), (2000, 1024, 176), (16203, 2056, 240), (8100, 1024, 304)])
def test_gelu_of_half_a_step_more(device, epi, M, N, K):
    """|GELU'| <= 1.13; the erf form in bf16 is within 0.15 of half a step and 2^-24, the tanh form within 16 u."""
    g = torch.Generator().manual_seed(K)
    r = lambda *s: torch.randn(*s, generator=g).to(device=device, dtype=BF16)
    x, w, b = r(M, K), r(N, K) * K ** -0.5, r(N)
    y = ops.linear(x, w, b, epilogue=epi)
    v = x.double() @ w.double().t() + b.double()
    err = (x.double().abs() @ w.double().abs().t() + b.double().abs()) * (K + 8) * U * 1.13
    step = torch.finfo(BF16).eps / 2
    if epi == 2:
        want = 0.5 * v * torch.erfc(-v / math.sqrt(2))
        err = err + 0.15 * step * v.abs() + U
    else:
        want = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
        err = err + 16 * U * v.abs() + 1e-37
    over = (y.double() - want).abs() - (err * (1 + step) + want.abs() * step * (1 + 1e-6))
    assert (over <= torch.finfo(BF16).tiny).all(), over.max().item()


def test_half_a_step_more_and_what_is_not_finite(device):
    """A NaN or infinity in the last 16 values, or in the row that follows, stays in its row."""
    g = torch.Generator().manual_seed(3)
    x, w = (torch.randn(s, 80, generator=g).to(device=device, dtype=BF16) for s in (300, 136))
    clean = ops.linear(x, w)
    x[17, 79], x[40, 0], w[5, 64] = float("nan"), float("inf"), float("nan")
    y = ops.linear(x, w)
    rows = [i for i in range(300) if i not in (17, 40)]
    cols = [i for i in range(136) if i != 5]
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])
    assert y[17].isnan().all() and y[:, 5].isnan().all() and not y[40, cols].isfinite().any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,C,H,out", [(77, 64, 48, 64), (500, 512, 1360, 512), (130, 96, 176, 104), (1, 32, 16 * 3, 8), (70, 64, 16, 40)])
def test_training_step(device, dtype, M, C, H, out):
    """The down projection and its gradients from the h that the gated product gives; the rest from its dh."""
    torch.manual_seed(H)
    m = nsw.GatedMLP(C, H, out)
    with torch.no_grad():
        for t in m.parameters():
            t.copy_(torch.randn_like(t) * (t.shape[-1] ** -0.5 if t.dim() == 2 else 0.3))
    m = m.to(device=device, dtype=dtype)
    x = torch.randn(M, C, device=device).to(dtype).requires_grad_()
    r = torch.randn(M, out, device=device).to(dtype).requires_grad_()
    dy = torch.randn(M, out, device=device).to(dtype)
    y = m(x, r)
    y.backward(dy)
    w1, b1, w2, b2 = (t.detach() for t in (m.fc1.weight, m.bias1.bias, m.fc2.weight, m.bias2.bias))
    h = ops.gated_linear(x.detach(), w1, b1)
    h64, d64, w64 = h.double(), dy.double(), w2.double()
    before = h64 @ w64.t() + b2.double()
    close(y, before + r.double(), h64.abs() @ w64.abs().t() + b2.double().abs() + r.double().abs(), H + 2, dtype, before)
    close(m.fc2.weight.grad, d64.t() @ h64, d64.abs().t() @ h64.abs(), M, dtype)
    close(m.bias2.bias.grad, d64.sum(0), d64.abs().sum(0), 512, dtype)
    assert torch.equal(r.grad, dy)
    dh = ops.linear_backward(dy, h, w2, needs=(True, False, False))[0]
    close(dh, d64 @ w64, d64.abs() @ w64.abs(), out, dtype)
    want = ops.gated_linear_backward(dh, x.detach(), w1, b1)
    for got, v in zip((x.grad, m.fc1.weight.grad, m.bias1.bias.grad), want):
        assert torch.equal(got, v)
