"""nsw.GatedMLP at every width that its gated product takes: forward and backward."""
import contextlib
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


@pytest.mark.parametrize("dtype,M,K", [(F32, 150_003, 4096), (BF16, 270_011, 4096), (BF16, 800_009, 1360)])
@pytest.mark.parametrize("epi", [0, 3])
def test_rows_of_more_than_2_gib(device, dtype, M, K, epi):
    """x goes in pieces of rows: those on both sides of a border and the last ones, from float64 sums; with a residual."""
    N = 40
    g = torch.Generator(device=device).manual_seed(K)
    x = torch.empty(M, K, dtype=dtype, device=device).normal_(0, 1, generator=g)
    w = torch.empty(N, K, device=device).normal_(0, K ** -0.5, generator=g).to(dtype)
    b, r = torch.randn(N, device=device).to(dtype), torch.randn(M, N, device=device).to(dtype)
    y = ops.linear(x, w, b if epi else None, r if epi else None)
    piece = (2 ** 31 - 1) // (K * x.element_size()) // 256 * 256
    assert 0 < piece < M
    for rows in (slice(0, 300), slice(piece - 300, piece + 300), slice(M - 300, M)):
        a = x[rows].double()
        want, mag = a @ w.double().t(), a.abs() @ w.double().abs().t()
        before = None
        if epi:
            before = want + b.double()
            want, mag = before + r[rows].double(), mag + b.double().abs() + r[rows].double().abs()
        close(y[rows], want, mag, K + 2, dtype, before)


def test_gated_mlp_with_more_than_2_gib_of_hidden_rows(device):
    """Forward and backward; the last rows are those of a pass over them alone, within the sums' and the roundings' bounds."""
    M, C, H = 150_003, 32, 4096
    torch.manual_seed(0)
    m = nsw.GatedMLP(C, H).to(device=device, dtype=F32)
    with torch.no_grad():
        for t in m.parameters():
            t.copy_(torch.randn_like(t) * (t.shape[-1] ** -0.5 if t.dim() == 2 else 0.3))
    x = torch.randn(M, C, device=device).requires_grad_()
    dy = torch.randn(M, C, device=device)
    y = m(x)
    gx, gw = torch.autograd.grad(y, (x, m.fc2.weight), dy)
    n = 500
    xt = x.detach()[-n:].clone().requires_grad_()
    yt = m(xt)
    gt, = torch.autograd.grad(yt, xt, dy[-n:])
    # relative 2-norm: sums of at most 4096 terms, two one after the other, 4096 2^-24 = 2.5e-4 each at worst
    for a, c in ((y[-n:], yt), (gx[-n:], gt)):
        assert (a - c).norm() <= 1e-3 * c.norm()
    ref = torch.zeros(C, H, dtype=torch.float64, device=device)
    w1, b1 = m.fc1.weight.detach().double(), m.bias1.bias.detach().double()
    for i in range(0, M, 30_000):
        g, u = (x.detach()[i:i + 30_000].double() @ w1.t() + b1).chunk(2, -1)
        ref += dy[i:i + 30_000].double().t() @ (g * torch.sigmoid(g) * u)
    assert (gw.double() - ref).norm() <= 1e-3 * ref.norm()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_rows(device, dtype):
    """Empty outputs, gradients of zero rows and zeros for the parameters, as from the gated product and the norms."""
    m = nsw.GatedMLP(64, 48, 40).to(device=device, dtype=dtype)
    x, r = (torch.empty(2, 0, n, device=device, dtype=dtype).requires_grad_() for n in (64, 40))
    y = m(x, r)
    assert y.shape == (2, 0, 40) and y.dtype == dtype
    y.sum().backward()
    assert x.grad.shape == x.shape and r.grad.shape == r.shape
    assert all(p.grad.shape == p.shape and not p.grad.any() for p in m.parameters())
    with pytest.raises(ValueError, match="residual"):
        ops.linear(x.detach(), torch.empty(8, 64, device=device, dtype=dtype), torch.empty(8, device=device, dtype=dtype),
                   torch.empty(1, 8, device=device, dtype=dtype))


def test_another_current_device(device, monkeypatch):
    """Every call of the block, forward and backward, makes its tensors' device the current one where another is."""
    m = nsw.GatedMLP(64, 48).to(device=device, dtype=BF16)
    x = torch.randn(5, 64, device=device).to(BF16).requires_grad_()
    want, = torch.autograd.grad(m(x), x, torch.ones(5, 64, device=device, dtype=BF16))
    entered = []

    @contextlib.contextmanager
    def enter(index):
        entered.append(index)
        yield

    monkeypatch.setattr(ops, "_current_index", lambda: 7)
    monkeypatch.setattr(torch.cuda, "device", enter)
    y = m(x)
    assert entered == [0, 0]                                      # the gated product, the down projection
    got, = torch.autograd.grad(y, x, torch.ones(5, 64, device=device, dtype=BF16))
    assert entered == [0] * 4 and torch.equal(got, want)
