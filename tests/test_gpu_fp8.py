"""nsw.ops.quantize_fp8 and linear_fp8.

The quantiser is exact: its values and scales are those of the definition, formed
in float64 on the CPU.  A product is off by its fp32 sums alone, (K + 8) u of the sum
of magnitudes (u = 2^-24), for bf16 results 7 * 2^-13 more (the 8-bit instructions
add groups of 8 products; one that is not the largest loses what lies below 2^-13 of
the largest's power of two, so a group loses less than 7 * 2^-13 of its largest
product, which is at most its sum of magnitudes), plus the activation's error (erf form 1.5e-7 |v| in fp32,
0.15 of half a step in bf16, tanh form 16 u) and one rounding to the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


def quantized(x, rows):
    """(values [R, Kp], scale exponents [blocks, Kb]) of the definition, float64 on the CPU.  NaN where x is not finite."""
    x = x.double().cpu()
    R, K = x.shape
    Kp, Rp = -(-K // 128) * 128, -(-R // rows) * rows
    p = torch.zeros(Rp, Kp, dtype=torch.float64)
    p[:R, :K] = x
    b = p.view(Rp // rows, rows, Kp // 128, 128)
    fin = torch.where(b.isfinite(), b, torch.zeros_like(b))
    top = fin.abs().amax((1, 3))
    m, e = torch.frexp(top)                                       # top = m 2^e, 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(top > 0, e, torch.full_like(e, -127)).clamp(min=-127)
    v = torch.ldexp(fin, -e[:, None, :, None])
    _, ev = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (ev - 1).clamp(min=-6) - 3)
    q = torch.where(b.isfinite(), torch.round(v / step) * step, torch.full_like(v, float("nan")))
    return q.view(Rp, Kp)[:R], e


def widen(q, scale, rows):
    e = scale.view(torch.uint8).double() - 127
    return q.double() * torch.exp2(e).repeat_interleave(rows, 0)[:q.shape[0]].repeat_interleave(128, 1)


def data(R, K, dtype, seed=0, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g)
    if spread:
        x = x * torch.exp2(torch.randint(-12, 12, (R, 1), generator=g).float())
        x[:, ::17] *= 30
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("R,K", [(1, 8), (1, 128), (5, 136), (127, 200), (128, 256), (129, 1000), (700, 384), (3, 4096)])
def test_quantize_is_the_definition(device, dtype, rows, R, K):
    from nsw import ops
    x = data(R, K, dtype, seed=R + K)
    q, s = ops.quantize_fp8(x.to(device), rows=rows)
    want, e = quantized(x, rows)
    assert q.shape == want.shape and s.shape == e.shape
    assert torch.equal(s.view(torch.uint8).cpu().int() - 127, e.int())
    assert torch.equal(q.cpu().double(), want)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_borders(device, rows):
    """Ties, e4m3's subnormals, blocks of zeros, tiny and huge magnitudes, 448 and its neighbours."""
    from nsw import ops
    x = torch.zeros(12, 128, dtype=F32)
    x[0] = torch.arange(128) * 3.5                                 # to 444.5: ties at every step
    x[1, :4] = torch.tensor([448.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10])
    x[2, :2] = torch.tensor([448.0 * (1 + 2 ** -23), 1.0])         # just past: the next scale
    x[3, :2] = torch.tensor([-448.0, 16.5])
    x[4, 0] = 2.0 ** -149                                          # the smallest fp32
    x[5, 0] = 2.0 ** -119
    x[6, 0], x[6, 1] = 3.4e38, -1e38
    x[7, :3] = torch.tensor([1.75, 1.0625, 1.1875])
    x[8, :3] = torch.tensor([float("nan"), 2.0, -3.0])
    x[9, :3] = torch.tensor([float("inf"), 2.0, -3.0])
    x[10, :3] = torch.tensor([-0.0, 1e-30, 1e30])
    if rows == 128:
        x = torch.cat([x[i:i + 1].expand(128, -1) for i in range(12)])
    q, s = ops.quantize_fp8(x.to(device), rows=rows)
    want, e = quantized(x, rows)
    assert torch.equal(s.view(torch.uint8).cpu().int() - 127, e.int())
    assert torch.equal(q.cpu().double().nan_to_num(777.0), want.nan_to_num(777.0))


def operands(device, M, N, K, dtype, seed=0):
    from nsw import ops
    x = data(M, K, dtype, seed)
    w = data(N, K, dtype, seed + 1, spread=False) * K ** -0.5
    g = torch.Generator().manual_seed(seed + 2)
    b, r = torch.randn(N, generator=g).to(dtype), torch.randn(M, N, generator=g).to(dtype)
    x, w, b, r = (t.to(device) for t in (x, w, b, r))
    return ops.quantize_fp8(x), ops.quantize_fp8(w, rows=128), b, r


def reference(xq, wq, b, r, epi, dtype):
    x, w = widen(*xq, 1), widen(*wq, 128)
    v, mag = x @ w.t(), x.abs() @ w.abs().t()
    step = torch.finfo(dtype).eps / 2
    if epi:
        v, mag = v + b.double(), mag + b.double().abs()
    tol = mag * ((x.shape[1] + 8) * U + (7 * 2.0 ** -13 if dtype == BF16 else 0.0))
    if epi == 2:
        v, tol = 0.5 * v * torch.erfc(-v / math.sqrt(2)), tol * 1.13
        tol = tol + (1.5e-7 * mag if dtype == F32 else 0.15 * step * v.abs() + U)
    elif epi == 4:
        v, tol = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)), tol * 1.13
        tol = tol + 16 * U * v.abs() + 1e-37
    elif epi == 3:
        v, tol = v + r.double(), tol + U * (mag + r.double().abs())
    return v, tol


def check(y, want, tol, dtype):
    step = torch.finfo(dtype).eps / 2
    over = (y.double() - want).abs() - (tol * (1 + step) + want.abs() * step * (1 + 1e-6))
    assert y.dtype == dtype and (over <= torch.finfo(dtype).tiny).all(), over.max().item()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("epi", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("M,N,K", [(1, 8, 128), (1, 4096, 1024), (17, 72, 256), (33, 136, 384), (130, 264, 200), (300, 1336, 1000)])
def test_linear(device, dtype, epi, M, N, K):
    from nsw import ops
    xq, wq, b, r = operands(device, M, N, K, dtype, seed=M + epi)
    y = ops.linear_fp8(*xq, *wq, None if epi == 0 else b, r if epi == 3 else None, epilogue=epi, dtype=dtype)
    want, tol = reference(xq, wq, b, r, epi, dtype)
    check(y, want, tol, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_far_scales(device, dtype):
    """Rows of very small and very large values: scales near both ends, their products within fp32."""
    from nsw import ops
    x = data(6, 256, F32, spread=False) * torch.tensor([1e-38, 1e-30, 1.0, 1e30, 3e37, 1e-44])[:, None]
    w = data(16, 256, F32, 1, False) * 1e-3
    w[3] *= 1e-4
    xq, wq = ops.quantize_fp8(x.to(device)), ops.quantize_fp8(w.to(device), rows=128)
    v, tol = reference(xq, wq, None, None, 0, dtype)
    check(ops.linear_fp8(*xq, *wq, dtype=dtype), v, tol + 2.0 ** -126, dtype)   # subnormal sums may be flushed


@pytest.mark.parametrize("M", [2, 8, 15, 16, 31, 32, 48, 63, 64, 65, 96, 127, 128, 129, 255, 257, 640, 2049])
def test_rows(device, M):
    from nsw import ops
    xq, wq, b, r = operands(device, M, 520, 640, BF16, seed=M)
    y = ops.linear_fp8(*xq, *wq, b, r, dtype=BF16)
    want, tol = reference(xq, wq, b, r, 3, BF16)
    check(y, want, tol, BF16)


@pytest.mark.parametrize("M,N,K", [(16203, 2056, 128), (8200, 4096, 512), (700, 1024, 4096), (40, 264, 16128)])
def test_large(device, M, N, K):
    from nsw import ops
    xq, wq, b, r = operands(device, M, N, K, BF16, seed=K)
    y = ops.linear_fp8(*xq, *wq, b, epilogue=2, dtype=BF16)
    want, tol = reference(xq, wq, b, r, 2, BF16)
    check(y, want, tol, BF16)


def test_default_epilogues_and_shapes(device):
    from nsw import ops
    xq, wq, b, r = operands(device, 24, 64, 128, BF16)
    x3 = (xq[0].view(2, 12, 128), xq[1].view(2, 12, 1))
    assert torch.equal(ops.linear_fp8(*x3, *wq).view(24, 64), ops.linear_fp8(*xq, *wq, epilogue=0))
    assert torch.equal(ops.linear_fp8(*xq, *wq, b), ops.linear_fp8(*xq, *wq, b, epilogue=1))
    assert torch.equal(ops.linear_fp8(*x3, *wq, b, r.view(2, 12, 64)).view(24, 64), ops.linear_fp8(*xq, *wq, b, r, epilogue=3))


def test_nan_stays_in_its_row(device):
    from nsw import ops
    x = data(40, 256, BF16).to(device)
    wq = ops.quantize_fp8(data(64, 256, BF16, 1, False).to(device), rows=128)
    clean = ops.linear_fp8(*ops.quantize_fp8(x), *wq)
    x[7, 3], x[9, 200] = float("nan"), float("inf")
    y = ops.linear_fp8(*ops.quantize_fp8(x), *wq)
    keep = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(y[keep], clean[keep]) and y[7].isnan().all() and y[9].isnan().all()


def test_no_rows(device):
    from nsw import ops
    q, s = ops.quantize_fp8(torch.empty(0, 200, device=device, dtype=BF16))
    assert q.shape == (0, 256) and s.shape == (0, 2)
    wq = ops.quantize_fp8(torch.ones(64, 200, device=device, dtype=BF16), rows=128)
    assert ops.linear_fp8(q, s, *wq).shape == (0, 64)


@pytest.mark.parametrize("M", [5, 1300])
def test_graph_replays_and_another_stream(device, M):
    from nsw import ops
    x = data(M, 384, BF16).to(device)
    wq = ops.quantize_fp8(data(264, 384, BF16, 1, False).to(device), rows=128)
    step = lambda: ops.linear_fp8(*ops.quantize_fp8(x), *wq)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for i in range(3):
        x.copy_(data(M, 384, BF16, seed=20 + i))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_rows_past_32_bit_offsets(device):
    """x of more than 2^32 quantised bytes: the last rows are those of a call on them alone, bit for bit."""
    from nsw import ops
    M, K, N = 4_300_003, 1024, 264
    x = torch.empty(M, K, dtype=BF16, device=device)
    x.random_(-6, 7)
    wq = ops.quantize_fp8(data(N, K, BF16, 1, False).to(device), rows=128)
    y = ops.linear_fp8(*ops.quantize_fp8(x), *wq)
    tail = ops.linear_fp8(*ops.quantize_fp8(x[-2000:].contiguous()), *wq)
    v, tol = reference(ops.quantize_fp8(x[-2000:].contiguous()), wq, None, None, 0, BF16)
    check(y[-2000:], v, tol, BF16)
    check(tail, v, tol, BF16)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [5, 700])
def test_a_scale_that_is_not_a_number(device, dtype, M):
    from nsw import ops
    xq, wq, _, _ = operands(device, M, 136, 256, dtype)
    xq[1].view(torch.uint8)[3, 1] = 255
    y = ops.linear_fp8(*xq, *wq, dtype=dtype)
    assert y[3].isnan().all() and not y[:3].isnan().any() and not y[4:].isnan().any()
