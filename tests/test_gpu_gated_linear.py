"""nsw.ops.gated_linear, gated_linear_backward and linear_backward against the
formulas in float64 (evaluated on the GPU from the same rounded inputs).

Tolerances, per element, u = 2^-24 and r = finfo(type).eps / 2 (one rounding).
A product over n terms is off by at most (n + 8) u of its sum of magnitudes
(fp32 accumulation; the split fp32 products keep within (n / 8 + 4) u).  The
activations: SiLU and the tanh form 16 u of themselves; the erf form 1.5e-7 |g|
in fp32 (the formula's own error) and 0.15 r of itself in bf16; derivatives 16 u
(1 + |g|)^3, the erf form 1.5e-7 more.  |act'| <= 1.13.  dg and du are rounded
to the type before the products of the backward pass: r of each, twice in all
with the result's."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACTS = ["silu", "gelu", "gelu_tanh"]
BF16, F32 = torch.bfloat16, torch.float32


def case(device, dtype, M, K, H, bias, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    t = dict(x=r(M, K), w=r(2 * H, K) * K ** -0.5, b=0.3 * r(2 * H) if bias else None, dh=r(M, H))
    return {k: None if v is None else v.to(device=device, dtype=dtype) for k, v in t.items()}


def act64(g, act):
    if act == "gelu":
        s = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        return g * s, s + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    c = 1.0 if act == "silu" else 2 * math.sqrt(2 / math.pi)
    z, dz = (g, 1.0) if act == "silu" else (c * (g + 0.044715 * g ** 3), c * (1 + 0.134145 * g * g))
    s = torch.sigmoid(z)
    return g * s, s + g * s * torch.sigmoid(-z) * dz


def reference(t, act):
    """{name: (value, bound of the error before the final rounding)} in float64."""
    dtype, (M, K) = t["x"].dtype, t["x"].shape
    r = torch.finfo(dtype).eps / 2
    x, w, dh = t["x"].double(), t["w"].double(), t["dh"].double()
    H = w.shape[0] // 2
    b = torch.zeros(2 * H, dtype=torch.float64, device=x.device) if t["b"] is None else t["b"].double()
    p, ep = x @ w.t() + b, (x.abs() @ w.abs().t() + b.abs()) * (K + 8) * U
    g, u, eg, eu = p[:, :H], p[:, H:], ep[:, :H], ep[:, H:]
    a, d = act64(g, act)
    ea = a.abs() * 16 * U + 1.13 * eg
    ed = 16 * U * (1 + g.abs()) ** 3 + 2 * eg          # |act''| < 2
    if act == "gelu":
        ea = ea + (0.15 * r * a.abs() + 2.0 ** -24 if dtype == BF16 else 1.5e-7 * g.abs())
        ed = ed + 1.5e-7
    out = {"h": (a * u, ea * u.abs() + (a.abs() + ea) * eu)}
    if act == "gelu":                                  # the backward pass has the fp32 form for both types
        ea = a.abs() * 16 * U + 1.13 * eg + 1.5e-7 * g.abs()
    dp = torch.cat([dh * u * d, dh * a], 1)
    ed = torch.cat([dh.abs() * (u.abs() * ed + d.abs() * eu + ed * eu), dh.abs() * ea], 1) + 4 * U * dp.abs()
    out["db"] = (dp.sum(0), ed.sum(0) + dp.abs().sum(0) * 512 * U)
    ed = ed + r * (dp.abs() + ed)                      # rounded before the products
    mp = dp.abs() + ed
    out["dx"] = (dp @ w, ed @ w.abs() + (mp @ w.abs()) * (2 * H + 8) * U)
    out["dw"] = (dp.t() @ x, ed.t() @ x.abs() + (mp.t() @ x.abs()) * (M + 8) * U)
    return out


def check(got, want, dtype):
    r = torch.finfo(dtype).eps / 2
    for name, g in got.items():
        v, tol = want[name]
        assert g.dtype == dtype and g.shape == v.shape, name
        over = (g.double() - v).abs() - (tol * (1 + r) + v.abs() * r * (1 + 1e-6))
        assert (over <= torch.finfo(dtype).tiny).all(), (name, over.max().item(), v.abs().max().item())


def run(t, act, needs=(True, True, True)):
    from nsw import ops
    h = ops.gated_linear(t["x"], t["w"], t["b"], act=act)
    got = ops.gated_linear_backward(t["dh"], t["x"], t["w"], t["b"], act=act, needs=needs)
    out = {"h": h}
    out.update({n: v for n, v in zip(("dx", "dw", "db"), got) if v is not None})
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [1, 2, 31, 64, 65, 129, 257])
@pytest.mark.parametrize("K,H", [(32, 16), (64, 48), (96, 144), (160, 272)])
def test_sizes(device, dtype, M, K, H):
    act = ACTS[(M + K) % 3]
    t = case(device, dtype, M, K, H, M % 2 == 1, seed=M + K)
    check(run(t, act), reference(t, act), dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [True, False])
def test_activations(device, dtype, act, bias):
    t = case(device, dtype, 200, 128, 80, bias, seed=3)
    t["x"] *= 4                                       # gates well into both tails
    got = run(t, act)
    assert ("db" in got) == bias
    check(got, reference(t, act), dtype)


@pytest.mark.parametrize("dtype,M,K,H", [(BF16, 4100, 512, 1360), (BF16, 16203, 96, 2064), (F32, 4100, 176, 1040),
                                         (F32, 777, 16, 32), (BF16, 33, 1024, 4096)])
def test_large_tiles(device, dtype, M, K, H):
    t = case(device, dtype, M, K, H, True, seed=5)
    check(run(t, "silu"), reference(t, "silu"), dtype)


@pytest.mark.parametrize("dtype,M,K,H", [(BF16, 4100, 256, 2048), (BF16, 2600, 512, 4096), (BF16, 12961, 512, 1360),
                                         (F32, 4100, 256, 4096), (F32, 6000, 512, 2048)])
def test_rows_in_two_launches(device, dtype, M, K, H):
    """Whole rounds of large tiles, then the rest: few rows (4 of 4100) and many."""
    t = case(device, dtype, M, K, H, True, seed=9)
    check(run(t, "gelu_tanh"), reference(t, "gelu_tanh"), dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True)])
def test_gradients_on_their_own(device, dtype, needs):
    t = case(device, dtype, 130, 64, 48, True, seed=6)
    got, every = run(t, "gelu", needs), run(t, "gelu")
    assert set(got) == {"h"} | {n for n, k in zip(("dx", "dw", "db"), needs) if k}
    for n in got:
        assert torch.equal(got[n], every[n]), n


def test_extreme_gates(device):
    """Gates far out: act(g) is 0 or g, its derivative 0 or 1, nothing overflows to NaN."""
    from nsw import ops
    g = torch.tensor([-1e30, -3e4, -200.0, -90.0, 0.0, 90.0, 200.0, 3e4, 1e15], dtype=F32, device=device)
    x = torch.zeros(9, 16, device=device)
    x[:, 0] = g
    x[:, 1] = 1
    w = torch.zeros(32, 16, device=device)
    w[:16, 0] = 1                                     # the gate is g, the up projection 1
    w[16:, 1] = 1
    dh = torch.ones(9, 16, device=device)
    for act in ACTS:
        h = ops.gated_linear(x, w, act=act)
        dx, _, _ = ops.gated_linear_backward(dh, x, w, act=act)
        assert torch.equal(h[:, 0], g.clamp(min=0)), act
        want = (g > 0).float() + 0.5 * (g == 0).float()
        assert torch.allclose(dx[:, 0] / 16, want, atol=1e-6), act


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_are_not_finite_stay_alone(device, dtype):
    t = case(device, dtype, 300, 64, 48, False, seed=7)
    clean = run(t, "silu", (True, False, False))
    t["x"][17, 3] = float("nan")
    t["x"][200, 0] = float("inf")
    got = run(t, "silu", (True, False, False))
    keep = [i for i in range(300) if i not in (17, 200)]
    for n in ("h", "dx"):
        assert torch.equal(got[n][keep], clean[n][keep]), n
    assert got["h"][17].isnan().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", [(1, 32, 32), (63, 64, 96), (300, 160, 64), (4100, 512, 1376), (2500, 1024, 128)])
def test_linear_backward(device, dtype, M, N, K):
    from nsw import ops
    g = torch.Generator().manual_seed(M)
    dy, x = (torch.randn(M, n, generator=g).to(device, dtype) for n in (N, K))
    w = (torch.randn(N, K, generator=g) * K ** -0.5).to(device, dtype)
    dx, dw, db = ops.linear_backward(dy, x, w)
    d, xx, ww = dy.double(), x.double(), w.double()
    want = {"dx": (d @ ww, (d.abs() @ ww.abs()) * (N + 8) * U), "dw": (d.t() @ xx, (d.abs().t() @ xx.abs()) * (M + 8) * U),
            "db": (d.sum(0), d.abs().sum(0) * 512 * U)}
    check({"dx": dx, "dw": dw, "db": db}, want, dtype)
    one = ops.linear_backward(dy, x, w, needs=(False, True, False))
    assert one[0] is None and one[2] is None and torch.equal(one[1], dw)


@pytest.mark.parametrize("M,N,K", [(77, 96, 64), (1031, 176, 208), (3, 16, 16)])
def test_infinite_gradients_in_fp32(device, M, N, K):
    """An infinity stays in its row of dx and its row of dw, with the signs of what it meets; all else as without it."""
    from nsw import ops
    g = torch.Generator().manual_seed(K)
    dy, x, w = (torch.randn(*s, generator=g).to(device) for s in ((M, N), (M, K), (N, K)))
    clean = ops.linear_backward(dy, x, w)
    m, n = M - 1, N - 3
    dy[m, n] = math.inf
    dx, dw, db = ops.linear_backward(dy, x, w)
    assert torch.equal(dx[m], math.inf * w[n]) and torch.equal(dw[n], math.inf * x[m]) and db[n] == math.inf
    for got, want, i in ((dx, clean[0], m), (dw, clean[1], n), (db, clean[2], n)):
        keep = torch.arange(got.shape[0], device=device) != i
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("M,N,K", [(1, 1024, 32), (1, 4096, 64), (1000, 160, 32), (2000, 4096, 1024), (3000, 4096, 512),
                                   (8000, 2080, 160), (16200, 4096, 1024)])
def test_gradients_side_by_side(device, M, N, K):
    """bf16: dx, dw and db in one launch or after one another, whole or in parts, the longer parts first; and the same bits
    whichever of them are asked for."""
    from nsw import ops
    g = torch.Generator().manual_seed(N)
    dy, x = (torch.randn(M, n, generator=g).to(device, BF16) for n in (N, K))
    w = (torch.randn(N, K, generator=g) * K ** -0.5).to(device, BF16)
    got = dict(zip(("dx", "dw", "db"), ops.linear_backward(dy, x, w)))
    d, xx, ww = dy.double(), x.double(), w.double()
    want = {"dx": (d @ ww, (d.abs() @ ww.abs()) * (N + 8) * U), "dw": (d.t() @ xx, (d.abs().t() @ xx.abs()) * (M + 8) * U),
            "db": (d.sum(0), d.abs().sum(0) * 512 * U)}
    check(got, want, BF16)
    for needs in ((True, False, False), (False, True, True), (True, False, True), (False, False, True)):
        for n, t in zip(got, ops.linear_backward(dy, x, w, needs=needs)):
            assert t is None or torch.equal(t, got[n]), (needs, n)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_rows(device, dtype):
    from nsw import ops
    t = case(device, dtype, 0, 64, 48, True)
    got = run(t, "silu")
    assert got["h"].shape == (0, 48) and got["dx"].shape == (0, 64)
    assert torch.count_nonzero(got["dw"]) == 0 and torch.count_nonzero(got["db"]) == 0
    dx, dw, db = ops.linear_backward(torch.empty(0, 96, device=device, dtype=dtype), t["x"],
                                     torch.ones(96, 64, device=device, dtype=dtype))
    assert dx.shape == (0, 64) and torch.count_nonzero(dw) == 0 and torch.count_nonzero(db) == 0


def test_same_bits_every_time_and_on_another_stream(device):
    t = case(device, BF16, 3001, 256, 336, True, seed=8)
    want = run(t, "gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(t, "gelu")
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_graph_replays(device, dtype):
    t = case(device, dtype, 333, 96, 112, True, seed=9)
    run(t, "silu")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(t, "silu")
    for i in range(3):
        t["x"].copy_(torch.randn(t["x"].shape, generator=torch.Generator().manual_seed(i)))
        want = run(t, "silu")
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for n in want:
            assert torch.equal(out[n], want[n]), n


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(device, act):
    """fp32 directional derivatives of sum(h * dh): h^2 / 6 times the third derivative (1e-4 / 6 of values of order
    100) and the rounding of sums of 50 x 32 products of order 1 over 2h (1e-7 * 1600 / 2e-2 = 8e-3)."""
    from nsw import ops
    t = case(device, F32, 50, 48, 32, True, seed=10)
    grads = dict(zip(("x", "w", "b"), ops.gated_linear_backward(t["dh"], t["x"], t["w"], t["b"], act=act)))
    h = 1e-2
    for n in grads:
        e = torch.randn(t[n].shape, generator=torch.Generator().manual_seed(4)).to(device)
        e = e / e.norm()

        def f(s):
            v = {**t, n: t[n] + s * e}
            return (ops.gated_linear(v["x"], v["w"], v["b"], act=act).double() * t["dh"]).sum().item()

        want = (grads[n].double() * e).sum().item()
        assert abs((f(h) - f(-h)) / (2 * h) - want) < 2e-2 * max(1.0, abs(want)), n


@pytest.mark.parametrize("dtype,M,K", [(BF16, 2_200_003, 512), (F32, 1_100_003, 512)])
def test_rows_past_32_bit_offsets(device, dtype, M, K):
    """x of more than 2^31 bytes: the last rows within the bounds, dW and db against float64 sums over all rows."""
    from nsw import ops
    H = 16
    g = torch.Generator(device=device).manual_seed(1)
    x = torch.empty(M, K, dtype=dtype, device=device).normal_(0, 1, generator=g)
    t = {k: v for k, v in case(device, dtype, 1, K, H, True, seed=2).items()}
    dh = torch.empty(M, H, dtype=dtype, device=device).normal_(0, 1, generator=g)
    h = ops.gated_linear(x, t["w"], t["b"], act="silu")
    dx, dw, db = ops.gated_linear_backward(dh, x, t["w"], t["b"], act="silu")
    n = 300
    tail = {"x": x[-n:].contiguous(), "w": t["w"], "b": t["b"], "dh": dh[-n:].contiguous()}
    want = reference(tail, "silu")
    check({"h": h[-n:], "dx": dx[-n:]}, {k: want[k] for k in ("h", "dx")}, dtype)
    r, dw64, db64 = torch.finfo(dtype).eps / 2, 0, 0
    for m in range(0, M, 100_000):                   # dg and du are rounded once, sums of random signs: r by chance
        p = x[m:m + 100_000].double() @ t["w"].double().t() + t["b"].double()
        a, d = act64(p[:, :H], "silu")
        d64 = dh[m:m + 100_000].double()
        dp = torch.cat([d64 * p[:, H:] * d, d64 * a], 1)
        dw64, db64 = dw64 + dp.t() @ x[m:m + 100_000].double(), db64 + dp.sum(0)
    for got, ref in ((dw, dw64), (db, db64)):
        assert (got.double() - ref).norm() <= (3 * r + 2e-5) * ref.norm()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", [(40, 1600, 320), (9, 640, 928), (700, 1600, 320), (1000, 96, 4096), (130, 4096, 64)])
def test_split_contractions(device, dtype, M, N, K):
    """Few results and long sums, either way: pieces that are added afterwards."""
    from nsw import ops
    g = torch.Generator().manual_seed(M)
    dy, x = (torch.randn(M, n, generator=g).to(device, dtype) for n in (N, K))
    w = (torch.randn(N, K, generator=g) * K ** -0.5).to(device, dtype)
    dx, dw, _ = ops.linear_backward(dy, x, w, needs=(True, True, False))
    d, xx, ww = dy.double(), x.double(), w.double()
    check({"dx": dx, "dw": dw}, {"dx": (d @ ww, (d.abs() @ ww.abs()) * (N + 8) * U),
                                 "dw": (d.t() @ xx, (d.abs().t() @ xx.abs()) * (M + 8) * U)}, dtype)
