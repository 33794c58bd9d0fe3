"""Gradients of torch.ops.nsw.linear: where some operands are frozen, the bits of those
with everything trained; for every width that the forward pass takes."""
import pytest
import torch

import nsw
from nsw import ops, torch_ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", [(3, 96, 64), (300, 1024, 256), (1000, 64, 512)])
def test_frozen_operands(device, dtype, M, N, K):
    g = torch.Generator().manual_seed(M)
    r = lambda *s: torch.randn(*s, generator=g).to(device=device, dtype=dtype)
    t = {"x": r(M, K), "w": r(N, K) * K ** -0.5, "b": r(N), "r": r(M, N)}
    dy = r(M, N)

    def grads(names):
        a = {n: v.clone().requires_grad_(n in names) for n, v in t.items()}
        y = torch_ops.linear_epi(a["x"], a["w"], a["b"], a["r"])
        return dict(zip(names, torch.autograd.grad(y, [a[n] for n in names], dy)))

    full = grads("xwbr")
    assert torch.equal(full["r"], dy)
    for names in ("x", "w", "b", "r", "xb", "wr"):
        for n, v in grads(names).items():
            assert torch.equal(v, full[n]), (names, n)
    dx, dw, db = ops.linear_backward(dy, None, t["w"], needs=(True, False, True))
    assert dw is None and torch.equal(dx, full["x"]) and torch.equal(db, full["b"])
    with pytest.raises(ValueError, match="dweight"):
        ops.linear_backward(dy, None, t["w"])


def test_gelu_mlp_behind_frozen_parameters(device):
    """With fc1 frozen the second product's gradients are whole; h is what fc1 gives."""
    torch.manual_seed(0)
    m = nsw.MLP(64, 128).to(device=device, dtype=F32)
    x, dy = torch.randn(50, 64, device=device), torch.randn(50, 64, device=device)
    with pytest.raises(NotImplementedError):
        m(x).backward(dy)
    for p in (m.fc1.weight, m.bias1.bias):
        p.requires_grad_(False)
    m(x).backward(dy)
    h = torch_ops.linear_epi(x, m.fc1.weight, m.bias1.bias, epilogue=m.gelu_epilogue)
    _, dw, db = ops.linear_backward(dy, h, m.fc2.weight.detach(), needs=(False, True, True))
    assert torch.equal(m.fc2.weight.grad, dw) and torch.equal(m.bias2.bias.grad, db)


@pytest.mark.parametrize("dtype,M,N,K", [(BF16, 1, 8, 32), (BF16, 70, 40, 64), (BF16, 300, 1000, 256), (BF16, 4100, 1112, 160),
                                         (F32, 1, 8, 16), (F32, 70, 24, 48), (F32, 300, 1000, 256), (F32, 4100, 1112, 176)])
def test_every_width_of_the_forward_pass(device, dtype, M, N, K):
    """N a multiple of 8.  Bounds: (terms + 8) 2^-24 of the sums of magnitudes, and one rounding; db in at most 512 steps.
    A row of dy that is not finite stays a row of dx."""
    g = torch.Generator().manual_seed(N + K)
    dy, x, w = (torch.randn(*s, generator=g).to(device=device, dtype=dtype) for s in ((M, N), (M, K), (N, K)))
    a = [t.clone().requires_grad_() for t in (x, w, dy[0])]
    y = torch_ops.linear_epi(*a)
    got = torch.autograd.grad(y, a, dy)
    d, xx, ww = dy.double(), x.double(), w.double()
    want = ((d @ ww, d.abs() @ ww.abs() * (N + 8)), (d.t() @ xx, d.abs().t() @ xx.abs() * (M + 8)),
            (d.sum(0), d.abs().sum(0) * 512))
    step = torch.finfo(dtype).eps / 2
    for t, (v, mag) in zip(got, want):
        assert t.dtype == dtype and t.shape == v.shape and t.is_contiguous()
        over = (t.double() - v).abs() - (mag * 2.0 ** -24 * (1 + step) + v.abs() * step * (1 + 1e-6))
        assert (over <= torch.finfo(dtype).tiny).all(), over.max().item()
    if M > 1:
        clean = ops.linear_backward(dy, x, w, needs=(True, False, False))[0]
        dy[M // 2, N - 1] = float("nan")
        dx = ops.linear_backward(dy, x, w, needs=(True, False, False))[0]
        keep = torch.arange(M, device=device) != M // 2
        assert torch.equal(dx[keep], clean[keep]) and dx[M // 2].isnan().all()


def test_widths_without_rows(device):
    dx, dw, db = ops.linear_backward(torch.empty(0, 40, device=device), torch.empty(0, 16, device=device),
                                     torch.ones(40, 16, device=device))
    assert dx.shape == (0, 16) and dw.shape == (40, 16) and not dw.any() and db.shape == (40,) and not db.any()


def test_fp32_gradients_of_more_than_2_gib(device):
    """dy of more than 2^31 bytes: dx goes in pieces of rows (262143 and the rest here) and dw by itself.  dx on both sides of
    the border and at the end from float64 sums, dw and db from sums over all rows; the same bits each on its own."""
    M, N, K = 270_011, 2048, 32
    g = torch.Generator(device=device).manual_seed(4)
    dy = torch.empty(M, N, device=device).normal_(0, 1, generator=g)
    x = torch.empty(M, K, device=device).normal_(0, 1, generator=g)
    w = torch.empty(N, K, device=device).normal_(0, 0.02, generator=g)
    piece = (2 ** 31 - 1) // (N * 4)
    assert 0 < piece < M
    dx, dw, db = ops.linear_backward(dy, x, w)
    for rows in (slice(0, 300), slice(piece - 300, piece + 300), slice(M - 300, M)):
        d, ww = dy[rows].double(), w.double()
        over = (dx[rows].double() - d @ ww).abs() - (d.abs() @ ww.abs()) * (N + 8) * 2.0 ** -24
        assert (over <= 0).all(), over.max().item()
    dw64, mag, db64, dmag = 0, 0, 0, 0
    for m in range(0, M, 50_000):
        d, xx = dy[m:m + 50_000].double(), x[m:m + 50_000].double()
        dw64, mag = dw64 + d.t() @ xx, mag + d.abs().t() @ xx.abs()
        db64, dmag = db64 + d.sum(0), dmag + d.abs().sum(0)
    assert ((dw.double() - dw64).abs() <= mag * (M + 8) * 2.0 ** -24).all()
    assert (dw.double() - dw64).norm() <= 2e-5 * dw64.norm()        # by chance the square root of the terms, sqrt(M) 2^-24 = 3e-5 / 2
    # a column sum is of at most M / 64 + 64 steps one after the other (rows of a part, parts)
    assert ((db.double() - db64).abs() <= dmag * (M // 64 + 64) * 2.0 ** -24).all()
    assert torch.equal(ops.linear_backward(dy, x, w, needs=(True, False, False))[0], dx)
    assert torch.equal(ops.linear_backward(dy, x, w, needs=(False, True, False))[1], dw)


def test_a_bias_of_another_size_is_refused(device):
    x, w = torch.zeros(3, 64, device=device), torch.zeros(32, 64, device=device)
    for n in (8, 31, 64):
        with pytest.raises(ValueError, match="bias"):
            ops.linear(x, w, torch.zeros(n, device=device))
        with pytest.raises(ValueError, match="bias"):
            torch_ops.linear_epi(x, w, torch.zeros(n, device=device))


@pytest.mark.parametrize("M,N,K", [(1, 32, 16), (77, 64, 48), (1000, 160, 1008), (40, 1600, 336), (2000, 4096, 1008), (8000, 2080, 176),
                                   (16200, 4096, 1040), (64800, 1024, 16)])
def test_bf16_rows_of_half_a_step_more(device, M, N, K):
    """K 16 more than whole steps of 32, on all kernels of the gradients: the bounds as above."""
    g = torch.Generator().manual_seed(K)
    dy, x, w = (torch.randn(*s, generator=g).to(device=device, dtype=BF16) for s in ((M, N), (M, K), (N, K)))
    got = ops.linear_backward(dy, x, w)
    d, xx, ww = dy.double(), x.double(), w.double()
    want = ((d @ ww, d.abs() @ ww.abs() * (N + 8)), (d.t() @ xx, d.abs().t() @ xx.abs() * (M + 8)),
            (d.sum(0), d.abs().sum(0) * (512 + M // 64)))
    step = torch.finfo(BF16).eps / 2
    for t, (v, mag) in zip(got, want):
        over = (t.double() - v).abs() - (mag * 2.0 ** -24 * (1 + step) + v.abs() * step * (1 + 1e-6))
        assert (over <= torch.finfo(BF16).tiny).all(), over.max().item()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", [(70, 40, 64), (700, 1000, 112)])
def test_replays_of_padded_gradients(device, dtype, M, N, K):
    """Widths that go through copies, captured: every replay the eager result, with eager work between."""
    g = torch.Generator().manual_seed(N)
    dy, x, w = (torch.randn(*s, generator=g).to(device=device, dtype=dtype) for s in ((M, N), (M, K), (N, K)))
    want = ops.linear_backward(dy, x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.linear_backward(dy, x, w)
    for i in range(4):
        dy.copy_(torch.randn(M, N, generator=g))
        want = ops.linear_backward(dy, x, w)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
