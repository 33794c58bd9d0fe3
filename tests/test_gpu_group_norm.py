"""nsw.ops.group_norm and its gradients against the formulas in float64.

Tolerances, per element.  u = 2^-24.  A lane joins at most 128 batches of rows here (the
large samples are split over workgroups), then lanes, groups and workgroups are joined in
chains of at most 256: with three roundings a step the mean is off by at most
1200 u of the group's mean magnitude A, so (x - mean) by that and one rounding; the centred
squares, sums of squares of values that are off so, by 2400 u of A / std relative to the
variance at most, where A / std is at least 1; half of that in rs.  With h the bound of
xh's error these give xh within (1200 A rs + 1200 A rs |xh| + 4 |xh|) u =: h.  n = xh w + b
adds two roundings; the activations used have slopes of at most 1.13 and are themselves
within 4 u of |n| and 1.5e-7 |n| (GELU, fp32); y is rounded once, half a step
(finfo.eps / 2), and a bf16 GELU is within 0.15 of half a step more.  The slope of an
activation changes by at most 1.2 for a change of n by 1 and is within 4e-7.  Sums over rows
are chains of at most 1200 terms: 1200 u of the sum of magnitudes, beside the errors of
the terms.  In practice errors are a hundredth of this: the chains' roundings do not add up."""
import pytest
import torch
from torch import nn

import nsw
from nsw import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
K = 1200


def case(dtype, B, R, C, affine=True, seed=0, offset=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    t = dict(x=r(B, R, C) * (0.5 * r(C)).exp() + offset * r(C), dy=r(B, R, C), weight=1 + 0.2 * r(C) if affine else None,
             bias=0.3 * r(C) if affine else None)
    return {k: None if v is None else v.to(dtype) for k, v in t.items()}


def activation(n, act):
    """(value, slope) in float64."""
    n = n.detach().requires_grad_()
    f = {"none": lambda v: v * 1, "silu": nn.functional.silu, "gelu": nn.functional.gelu,
         "gelu_tanh": lambda v: nn.functional.gelu(v, approximate="tanh")}[act]
    a = f(n)
    return a.detach(), torch.autograd.grad(a.sum(), n)[0]


def reference(t, groups, act, eps):
    """{name: (value, bound of the error before the last rounding)} in float64."""
    d = {k: None if v is None else v.double() for k, v in t.items()}
    B, R, C = d["x"].shape
    x = d["x"].view(B, R, groups, -1)
    var, mean = torch.var_mean(x, (1, 3), correction=0, keepdim=True)
    rs = (var + eps).rsqrt()
    A = x.abs().mean((1, 3), keepdim=True)
    xh = ((x - mean) * rs)
    h = (K * A * rs * (1 + xh.abs()) + 4 * xh.abs()) * U
    w = torch.ones(C, dtype=torch.float64) if d["weight"] is None else d["weight"]
    b = torch.zeros(C, dtype=torch.float64) if d["bias"] is None else d["bias"]
    xh, h = xh.reshape(B, R, C), h.reshape(B, R, C)
    n = xh * w + b
    hn = h * w.abs() + 2 * U * (n.abs() + (xh * w).abs())
    a, s = activation(n, act)
    out = {"y": (a, 1.13 * hn + (4 * U + 1.5e-7) * n.abs())}
    if t["dy"] is None:
        return out
    dn, hs = d["dy"] * s, d["dy"].abs() * (1.2 * hn + 4e-7)
    s1, s2 = dn, dn * xh
    e1, e2 = hs, hs * (xh.abs() + h) + dn.abs() * h
    rows = lambda v: v.sum((0, 1))
    out["dbias"] = (rows(s1), rows(e1) + K * U * rows(s1.abs() + e1))
    out["dweight"] = (rows(s2), rows(e2) + K * U * rows(s2.abs() + e2))
    over = lambda v: v.view(B, R, groups, -1).mean((1, 3), keepdim=True).expand(B, R, groups, C // groups).reshape(B, R, C)
    m1, m2 = over(s1 * w), over(s2 * w)
    h1, h2 = over((e1 + K * U * (s1.abs() + e1)) * w.abs()), over((e2 + K * U * (s2.abs() + e2)) * w.abs())
    r = rs.expand(B, R, groups, C // groups).reshape(B, R, C)
    in_ = dn * w - m1 - xh * m2
    big = (dn * w).abs() + m1.abs() + (xh * m2).abs()
    rel = (K * A * rs).expand(B, R, groups, C // groups).reshape(B, R, C) * U
    out["dx"] = (r * in_, r * (hs * w.abs() + h1 + (xh.abs() + h) * h2 + h * m2.abs() + 4 * U * big + rel * in_.abs()))
    return out


def run(t, groups, act, eps, device):
    d = {k: None if v is None else v.to(device) for k, v in t.items()}
    y, stats = ops.group_norm(d["x"], groups, d["weight"], d["bias"], act=act, eps=eps)
    got = {"y": y, "stats": stats}
    if t["dy"] is not None:
        got.update(zip(("dx", "dweight", "dbias"),
                       ops.group_norm_backward(d["dy"], d["x"], stats, groups, d["weight"], d["bias"], act=act)))
    return got


def check(got, want, dtype):
    step = torch.finfo(dtype).eps / 2 * (1.15 if dtype == torch.bfloat16 else 1.0)
    for name, (v, tol) in want.items():
        g = got[name]
        if g is None:
            continue
        assert g.dtype == dtype and g.shape == v.shape, name
        err = (g.double().cpu() - v).abs() - (v.abs() * step + tol * (1 + step))
        assert (err <= torch.finfo(dtype).tiny).all(), (name, err.max().item())


DTYPES = [torch.float32, torch.bfloat16]
WIDTHS = {torch.bfloat16: [(8, 1), (8, 8), (24, 8), (64, 4), (200, 8), (192, 6), (1024, 32), (2048, 64), (2056, 8), (4096, 4096)],
          torch.float32: [(4, 2), (20, 5), (200, 8), (256, 1), (512, 32), (1024, 1024), (1028, 4), (2048, 16)]}


@pytest.mark.parametrize("dtype,C,groups", [(d, c, g) for d, cs in WIDTHS.items() for c, g in cs])
@pytest.mark.parametrize("B,R", [(2, 19), (1, 1300)])
def test_widths(device, dtype, C, groups, B, R):
    t = case(dtype, B, R, C, seed=C)
    check(run(t, groups, "silu", 1e-5, device), reference(t, groups, "silu", 1e-5), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,R", [(1, 1), (3, 1), (1, 2), (5, 7), (300, 3), (1, 4099), (3, 2501), (700, 129)])
def test_rows(device, dtype, B, R):
    t = case(dtype, B, R, 64, seed=R)
    check(run(t, 8, "gelu", 1e-5, device), reference(t, 8, "gelu", 1e-5), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("affine", [True, False])
@pytest.mark.parametrize("R", [31, 3000])
def test_options(device, dtype, act, affine, R):
    t = case(dtype, 2, R, 120, affine, seed=9)
    got = run(t, 5, act, 1e-3, device)
    check(got, reference(t, 5, act, 1e-3), dtype)
    assert (got["dweight"] is None) == (not affine) and (got["dbias"] is None) == (not affine)


@pytest.mark.parametrize("R", [50, 3000])
def test_a_mean_far_from_zero(device, R):
    """A mean of 300 times the spread: squares less the mean's square would lose the variance."""
    t = case(torch.float32, 2, R, 64, seed=3, offset=0.0)
    t["x"] += 300.0
    got = run(t, 8, "none", 1e-6, device)
    check(got, reference(t, 8, "none", 1e-6), torch.float32)
    var, mean = torch.var_mean(t["x"].double().view(2, R, 8, 8), (1, 3), correction=0)
    rs = (var + 1e-6).rsqrt()
    assert ((got["stats"][..., 0].double().cpu() - mean).abs() <= K * U * mean.abs()).all()
    # centred values: the relative error of rs does not see the mean
    assert ((got["stats"][..., 1].double().cpu() / rs - 1).abs() <= 1e-4).all()


@pytest.mark.parametrize("R", [40, 3000])
def test_constant_groups(device, R):
    """No spread at all: rs = 1 / sqrt(eps), results the bias."""
    x = torch.full((1, R, 64), 2.5)
    t = dict(x=x, weight=torch.ones(64), bias=torch.linspace(-1, 1, 64), dy=None)
    got = run(t, 4, "none", 1e-4, device)
    assert torch.equal(got["y"].cpu(), t["bias"].expand(1, R, 64))
    assert torch.allclose(got["stats"][..., 1].cpu(), torch.full((1, 4), 100.0))


@pytest.mark.parametrize("R", [40, 3000])
def test_not_a_number_stays_in_its_group(device, R):
    t = case(torch.float32, 2, R, 64, seed=5)
    want = run(t, 8, "silu", 1e-5, device)
    t["x"][0, R // 2, 17] = float("nan")
    got = run(t, 8, "silu", 1e-5, device)
    for name in ("y", "dx"):
        assert got[name][0, :, 16:24].isnan().all(), name
        for part in ((0, slice(None), slice(0, 16)), (0, slice(None), slice(24, None)), (1,)):
            assert torch.equal(got[name][part], want[name][part]), name


@pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True), (False, True, True),
                                   (False, False, False)])
@pytest.mark.parametrize("R", [40, 3000])
def test_some_gradients(device, needs, R):
    t = {k: v.to(device) for k, v in case(torch.bfloat16, 2, R, 64, seed=6).items()}
    y, stats = ops.group_norm(t["x"], 8, t["weight"], t["bias"], act="silu")
    args = (t["dy"], t["x"], stats, 8, t["weight"], t["bias"])
    whole = ops.group_norm_backward(*args, act="silu")
    for n, a, b in zip(needs, ops.group_norm_backward(*args, act="silu", needs=needs), whole):
        assert (a is None) == (not n) and (a is None or torch.equal(a, b))


def test_no_rows(device):
    for shape in ((0, 5, 64), (2, 0, 64)):
        x = torch.empty(shape, device=device)
        w = torch.ones(64, device=device)
        y, stats = ops.group_norm(x, 8, w, w)
        dx, dw, db = ops.group_norm_backward(x, x, stats, 8, w, w)
        assert y.shape == dx.shape == shape and stats.shape == (shape[0], 8, 2)
        assert not dw.any() and not db.any()


def test_zeros_at_the_c_entry(device):
    from nsw import _lib
    dw = torch.ones(64, device=device)
    ws = torch.empty(4096, dtype=torch.uint8, device=device)
    for B, R in ((0, 3), (3, 0)):
        dw.fill_(1)
        _lib.check(_lib.lib().nsw_group_norm_backward(None, None, None, None, None, None, dw.data_ptr(), None, B, R, 64, 8, 0,
                                                      _lib.NSW_DTYPE_F32, ws.data_ptr(), ws.numel(),
                                                      torch.cuda.current_stream().cuda_stream))
        assert not dw.any()


def test_in_place_at_the_c_entry(device):
    """y over x and dx over dy, whole samples and split ones."""
    from nsw import _lib
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for B, R in ((3, 20), (2, 3000)):
        t = {k: v.to(device) for k, v in case(torch.bfloat16, B, R, 64, seed=8).items()}
        y, stats = ops.group_norm(t["x"], 8, t["weight"], t["bias"], act="silu")
        dx, dw, db = ops.group_norm_backward(t["dy"], t["x"], stats, 8, t["weight"], t["bias"], act="silu")
        ws = torch.empty(1 << 22, dtype=torch.uint8, device=device)
        dy, x, st2 = t["dy"].clone(), t["x"].clone(), torch.empty_like(stats)
        _lib.check(L.nsw_group_norm_backward(dy.data_ptr(), x.data_ptr(), stats.data_ptr(), t["weight"].data_ptr(),
                                             t["bias"].data_ptr(), dy.data_ptr(), None, None, B, R, 64, 8, _lib.NSW_ACT_SILU,
                                             _lib.NSW_DTYPE_BF16, ws.data_ptr(), ws.numel(), st))
        _lib.check(L.nsw_group_norm(x.data_ptr(), t["weight"].data_ptr(), t["bias"].data_ptr(), x.data_ptr(), st2.data_ptr(), B,
                                    R, 64, 8, 1e-5, _lib.NSW_ACT_SILU, _lib.NSW_DTYPE_BF16, ws.data_ptr(), ws.numel(), st))
        assert torch.equal(dy, dx) and torch.equal(x, y) and torch.equal(st2, stats)


def test_refusals(device):
    x = torch.zeros(2, 5, 64, device=device)
    w = torch.ones(64, device=device)
    y, stats = ops.group_norm(x, 8)
    for bad in (lambda: ops.group_norm(x, 7), lambda: ops.group_norm(x, 0), lambda: ops.group_norm(x, 8, w[:32].contiguous()),
                lambda: ops.group_norm(x, 8, act="tanh"), lambda: ops.group_norm(x[0, 0], 8),
                lambda: ops.group_norm_backward(x[:1].contiguous(), x, stats, 8),
                lambda: ops.group_norm_backward(x, x, stats[:1].contiguous(), 8),
                lambda: ops.group_norm_backward(x, x, stats.double(), 8)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.group_norm(x, 8, w.bfloat16())
    with pytest.raises(TypeError):
        ops.group_norm(x.half(), 8)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.group_norm(x.transpose(1, 2).contiguous().transpose(1, 2), 8)


def test_more_than_32_bits_of_bytes(device):
    """A sample whose last rows lie past 2^32 bytes, against its own first rows' formula."""
    R, C = 2_200_000, 1024
    x = torch.empty(1, R, C, dtype=torch.bfloat16, device=device)
    g = torch.Generator(device=device).manual_seed(1)
    x.normal_(generator=g)
    y, stats = ops.group_norm(x, 32)
    sums = torch.zeros(2, 32, dtype=torch.float64, device=device)
    for r in range(0, R, 100_000):
        v = x[0, r:r + 100_000].view(-1, 32, 32).double()
        sums += torch.stack([v.sum((0, 2)), (v * v).sum((0, 2))])
    n = R * 32.0
    mean = sums[0] / n
    rs = (sums[1] / n - mean * mean + 1e-5).rsqrt()
    tail = x[0, -1000:].view(-1, 32, 32).double()
    want = ((tail - mean[:, None]) * rs[:, None]).view(-1, C)
    err = (y[0, -1000:].double() - want).abs()
    # split over 512 workgroups: chains of 540 batches
    assert (err <= want.abs() * 2 ** -8 + 4 * K * U * (1 + want.abs())).all(), err.max()


def test_many_large_samples(device):
    """More groups and columns in all than one launch joins: the first, a middle and the last sample, and the
    parameters' gradients, sums of all of them."""
    B, R, C, groups, eps = 16400, 25, 4096, 2048, 1e-5
    g = torch.Generator(device=device).manual_seed(5)
    x = torch.empty(B, R, C, dtype=torch.bfloat16, device=device).normal_(generator=g)
    dy = torch.empty_like(x).normal_(generator=g)
    w = torch.empty(C, dtype=torch.bfloat16, device=device).normal_(1.0, 0.2, generator=g)
    b = torch.empty_like(w).normal_(generator=g)
    y, stats = ops.group_norm(x, groups, w, b, eps=eps)
    dx, dw, db = ops.group_norm_backward(dy, x, stats, groups, w, b)
    for i in (0, 8201, B - 1):
        t = {"x": x[i:i + 1].cpu(), "dy": dy[i:i + 1].cpu(), "weight": w.cpu(), "bias": b.cpu()}
        want = reference(t, groups, "none", eps)
        check({"y": y[i:i + 1], "dx": dx[i:i + 1]}, {k: want[k] for k in ("y", "dx")}, torch.bfloat16)
    sums = torch.zeros(4, C, dtype=torch.float64, device=device)
    for i in range(0, B, 1000):
        v = x[i:i + 1000].double().view(-1, R, groups, C // groups)
        var, mean = torch.var_mean(v, (1, 3), correction=0, keepdim=True)
        xh = ((v - mean) * (var + eps).rsqrt()).view(-1, R, C)
        d = dy[i:i + 1000].double()
        sums += torch.stack([x_.sum((0, 1)) for x_ in (d, d.abs(), d * xh, (d * xh).abs())])
    for got, v, mag in ((db, sums[0], sums[1]), (dw, sums[2], sums[3] + sums[1])):
        # xh is off by h of reference(), at most 4 K u a term here, the sums by K u
        err = (got.double() - v).abs() - (v.abs() * 2 ** -8 + 5 * K * U * mag * (1 + 2 ** -8))
        assert (err <= 0).all(), err.max()


# ------------------------------------------------- autograd, modules, graphs ---

def module(dtype, device, seed=1):
    torch.manual_seed(seed)
    m = nsw.GroupNorm(8, 64, act_layer=nn.SiLU)
    with torch.no_grad():
        m.weight.normal_(1, 0.2)
        m.bias.normal_(0, 0.3)
    return m.to(device=device, dtype=dtype)


@pytest.mark.parametrize("R", [(3, 7), (40, 70)])
def test_module_gradients(device, R):
    m = module(torch.float32, device)
    t = case(torch.float32, 2, R[0] * R[1], 64, seed=11)
    t["weight"], t["bias"] = m.weight.detach().cpu(), m.bias.detach().cpu()
    x = t["x"].view(2, *R, 64).to(device).requires_grad_()
    y = m(x)
    y.backward(t["dy"].view(2, *R, 64).to(device))
    got = {"y": y.detach().view(2, -1, 64), "dx": x.grad.view(2, -1, 64), "dweight": m.weight.grad, "dbias": m.bias.grad}
    check(got, reference(t, 8, "silu", 1e-5), torch.float32)


def test_gradients_against_differences(device):
    """The directional derivative against central differences of the forward kernel."""
    m = module(torch.float32, device)
    g = torch.Generator(device=device).manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, device=device)
    x, dy, v = rnd(2, 30, 64), rnd(2, 30, 64), rnd(2, 30, 64)
    xr = x.clone().requires_grad_()
    (m(xr) * dy).sum().backward()
    with torch.no_grad():
        e = 2.0 ** -6
        f = lambda t: (m(t).double() * dy.double()).sum()
        diff = (f(x + e * v) - f(x - e * v)) / (2 * e)
    got = (xr.grad.double() * v.double()).sum()
    # rounding: 3840 results within 1e-6 of 4, of random signs, over 2 e: 2e-2 at 5 sigma is far above; the third
    # derivative, of at most 3 a value: 3840 * 3 * e^2 / 6 at worst, a hundredth of it with random signs
    assert abs(got - diff) <= 0.05 * (1 + 0.02 * abs(diff)), (got, diff)


def test_strided_inputs_and_gradients(device):
    m = module(torch.bfloat16, device)
    base = torch.randn(2, 64, 50, device=device).bfloat16()
    x = base.transpose(1, 2).detach().requires_grad_()           # channels first in memory
    dy = torch.randn(2, 100, 64, device=device).bfloat16()[:, ::2]
    y = m(x)
    y.backward(dy)
    xc = x.detach().contiguous().requires_grad_()
    yc = m(xc)
    yc.backward(dy.contiguous())
    assert torch.equal(y, yc) and torch.equal(x.grad, xc.grad)


def test_statistics_have_no_gradient(device):
    x = torch.randn(2, 5, 64, device=device, requires_grad=True)
    _, stats = torch.ops.nsw.group_norm(x, 8, None, None, "none", 1e-5)
    with pytest.raises(NotImplementedError, match="statistics"):
        stats.sum().backward()


def test_compiled(device):
    m = module(torch.float32, device)
    x = torch.randn(2, 50, 64, device=device)
    xs = [x.clone().requires_grad_() for _ in range(2)]
    ys = [m(xs[0]), torch.compile(m, fullgraph=True, backend="aot_eager")(xs[1])]
    for y in ys:
        y.square().sum().backward()
    assert torch.equal(ys[0], ys[1]) and torch.equal(xs[0].grad, xs[1].grad)


@pytest.mark.parametrize("R", [40, 3000])
def test_captured_and_replayed(device, R):
    """Forward and backward in one graph, replayed with other inputs and eager work between."""
    t = {k: v.to(device) for k, v in case(torch.bfloat16, 2, R, 64, seed=12).items()}
    def step():
        y, stats = ops.group_norm(t["x"], 8, t["weight"], t["bias"], act="silu")
        return (y,) + ops.group_norm_backward(t["dy"], t["x"], stats, 8, t["weight"], t["bias"], act="silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        t["x"].normal_()
        t["dy"].normal_()
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), k


def test_two_streams_at_once(device):
    ts = [{k: v.to(device) for k, v in case(torch.bfloat16, 1, 5000, 64, seed=s).items()} for s in (1, 2)]
    def step(t):
        y, stats = ops.group_norm(t["x"], 8, t["weight"], t["bias"], act="gelu")
        return (y,) + ops.group_norm_backward(t["dy"], t["x"], stats, 8, t["weight"], t["bias"], act="gelu")
    want = [step(t) for t in ts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ts]
    for _ in range(5):
        got = []
        for t, s in zip(ts, streams):
            with torch.cuda.stream(s):
                got.append(step(t))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))
