"""nsw.ops.residual_norm and its gradients against the formulas in float64.

Tolerances, per element.  u = 2^-24.  A row sum of C terms is taken on lanes that
add at most 32 terms each and then a tree of at most 8: its relative error is below
40 u, that of the reciprocal root half of it plus three roundings: below 24 u.  A
value that passes one norm is off by at most 32 u of the magnitudes it is made of,
one that passes two by 80 u, a gradient (three sums) by 160 u; then one rounding to
the result's type, half a step (finfo.eps / 2).  Sums over the rows are chains of
fewer than 64 terms (at most 4099 rows over at least 64 slots) and a tree of 32 + 8:
160 u more of the sum of magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def case(dtype, G, R, C, post, gate, pre, seed=0):
    g = torch.Generator().manual_seed(seed)
    M = G * R
    r = lambda *s: torch.randn(*s, generator=g)
    t = dict(branch=r(M, C) * 0.5, skip=r(M, C) * 2, dy=r(M, C), dz=r(M, C) if pre else None,
             post_weight=1 + 0.2 * r(C) if post else None, norm_weight=1 + 0.2 * r(C) if pre else None,
             gate={"none": None, "channel": 0.5 * r(C), "sample": 0.5 * r(G, C)}[gate])
    return {k: None if v is None else v.to(dtype) for k, v in t.items()}


def reference(t, alpha, eps):
    """{name: (value, magnitude that its error is a share of)} in float64."""
    d = {k: None if v is None else v.double() for k, v in t.items()}
    M, C = d["branch"].shape
    o, x = d["branch"], d["skip"]
    gate = torch.ones(1, C, dtype=torch.float64) if d["gate"] is None else d["gate"].reshape(-1, C)
    gate = gate.repeat_interleave(M // gate.shape[0], 0)
    w = torch.ones(C, dtype=torch.float64) if d["post_weight"] is None else d["post_weight"]
    ro = torch.ones(M, 1, dtype=torch.float64) if d["post_weight"] is None else (o.pow(2).mean(1, True) + eps).rsqrt()
    oh = o * ro
    y = alpha * x + gate * w * oh
    my = (alpha * x).abs() + (gate * w * oh).abs()
    out = {"y": (y, my * 32 * U)}
    dy = torch.zeros_like(o) if d["dy"] is None else d["dy"]
    dd, md = dy, dy.abs()
    if d["norm_weight"] is not None:
        ry = (y.pow(2).mean(1, True) + eps).rsqrt()
        yh, myh = y * ry, my * ry
        out["z"] = (yh * d["norm_weight"], myh * d["norm_weight"].abs() * 80 * U)
        if d["dz"] is not None:
            tt = d["dz"] * d["norm_weight"]
            dd = dd + ry * (tt - yh * (tt * yh).mean(1, True))
            md = md + ry * (tt.abs() + myh * (tt.abs() * myh).mean(1, True))
            out["dnorm"] = ((d["dz"] * yh).sum(0), (d["dz"].abs() * myh).sum(0) * 240 * U)
    out["dskip"] = (alpha * dd, abs(alpha) * md * 160 * U)
    G = 1 if d["gate"] is None else d["gate"].reshape(-1, C).shape[0]
    S, mS = (dd * oh).view(G, -1, C).sum(1), (md * oh.abs()).view(G, -1, C).sum(1)
    if d["gate"] is not None:
        out["dgate"] = ((w * S).reshape(t["gate"].shape), ((w.abs() * mS) * 320 * U).reshape(t["gate"].shape))
    if d["post_weight"] is not None:
        gg = gate.view(G, -1, C)[:, 0] if M else gate
        out["dpost"] = ((gg * S).sum(0), (gg.abs() * mS).sum(0) * 320 * U)
    s, ms = dd * gate * w, md * (gate * w).abs()
    if d["post_weight"] is not None:
        s = ro * (s - oh * (s * oh).mean(1, True))
        ms = ro * (ms + oh.abs() * (ms * oh.abs()).mean(1, True))
    out["dbranch"] = (s, ms * 200 * U)
    return out


def run(t, alpha, eps, device):
    from nsw import ops
    d = {k: None if v is None else v.to(device) for k, v in t.items()}
    kw = dict(post_weight=d["post_weight"], gate=d["gate"], alpha=alpha, norm_weight=d["norm_weight"], eps=eps)
    y, z = ops.residual_norm(d["branch"], d["skip"], **kw)
    got = ops.residual_norm_backward(d["dy"], d["dz"], d["branch"], d["skip"], **kw)
    return dict(zip(("y", "z", "dbranch", "dskip", "dpost", "dgate", "dnorm"), (y, z) + got))


def check(got, want, dtype):
    step = torch.finfo(dtype).eps / 2
    for name, (v, tol) in want.items():
        g = got[name]
        assert g.dtype == dtype and g.shape == v.shape, name
        err = (g.double().cpu() - v).abs() - (v.abs() * step * (1 + 1e-3) + tol * (1 + step))
        assert (err <= 1e-300 + torch.finfo(dtype).tiny).all(), (name, err.max().item())


WIDTHS = {torch.bfloat16: [8, 64, 128, 136, 256, 264, 512, 520, 1024, 1032, 2048, 4096, 4104, 8192],
          torch.float32: [4, 64, 68, 128, 132, 200, 256, 260, 512, 516, 2048, 2052, 4096]}


@pytest.mark.parametrize("dtype,C", [(d, c) for d, cs in WIDTHS.items() for c in cs])
def test_widths(device, dtype, C):
    t = case(dtype, 2, 19, C, True, "sample", True, seed=C)
    check(run(t, 0.8, 1e-5, device), reference(t, 0.8, 1e-5), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G,R", [(1, 1), (1, 2), (3, 1), (1, 17), (5, 333), (1, 4099)])
def test_rows(device, dtype, G, R):
    t = case(dtype, G, R, 200, True, "sample", True, seed=R)
    check(run(t, 1.0, 1e-5, device), reference(t, 1.0, 1e-5), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", ["none", "channel", "sample"])
@pytest.mark.parametrize("pre", [True, False])
def test_options(device, dtype, post, gate, pre):
    t = case(dtype, 3, 41, 136, post, gate, pre, seed=9)
    got = run(t, -1.5, 1e-6, device)
    check(got, reference(t, -1.5, 1e-6), dtype)
    assert (got["z"] is None) == (not pre) and (got["dnorm"] is None) == (not pre)
    assert (got["dpost"] is None) == (not post) and (got["dgate"] is None) == (gate == "none")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("missing", ["dy", "dz"])
def test_one_gradient_only(device, dtype, missing):
    t = case(dtype, 1, 50, 64, True, "channel", True, seed=5)
    t[missing] = None
    got = run(t, 1.0, 1e-5, device)
    want = reference(t, 1.0, 1e-5)
    if missing == "dz":
        assert torch.count_nonzero(got["dnorm"]) == 0
    check(got, want, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_zero_rows_of_data(device, dtype):
    """Rows of zeros (padding) meet eps alone."""
    t = case(dtype, 1, 33, 128, True, "channel", True, seed=6)
    for k in ("branch", "skip"):
        t[k][5:9] = 0
    check(run(t, 1.0, 1e-3, device), reference(t, 1.0, 1e-3), dtype)


@pytest.mark.parametrize("C", [64, 1024, 4096])
def test_rows_that_are_not_finite_stay_alone(device, C):
    t = case(torch.bfloat16, 1, 40, C, True, "channel", True, seed=7)
    clean = run(t, 1.0, 1e-5, device)
    t["branch"][3, 1] = float("nan")
    t["skip"][9, 0] = float("inf")
    got = run(t, 1.0, 1e-5, device)
    keep = [i for i in range(40) if i not in (3, 9)]
    for n in ("y", "z", "dbranch", "dskip"):
        assert torch.equal(got[n][keep], clean[n][keep]), n
    assert got["y"][3, 1].isnan() and got["z"][3].isnan().all() and got["y"][9, 0].isinf()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows(device, dtype):
    t = case(dtype, 1, 0, 64, True, "channel", True)
    got = run(t, 1.0, 1e-5, device)
    assert got["y"].shape == (0, 64) and got["z"].shape == (0, 64) and got["dbranch"].shape == (0, 64)
    for n in ("dpost", "dgate", "dnorm"):
        assert torch.count_nonzero(got[n]) == 0


def test_same_bits_every_time_and_on_another_stream(device):
    t = case(torch.bfloat16, 2, 3001, 512, True, "sample", True, seed=8)
    want = run(t, 1.0, 1e-5, device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(t, 1.0, 1e-5, device)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_graph_replays(device):
    from nsw import ops
    t = {k: None if v is None else v.to(device) for k, v in case(torch.bfloat16, 2, 77, 256, True, "sample", True).items()}
    kw = dict(post_weight=t["post_weight"], gate=t["gate"], norm_weight=t["norm_weight"], eps=1e-5)

    def step():
        y, z = ops.residual_norm(t["branch"], t["skip"], **kw)
        return (y, z) + ops.residual_norm_backward(t["dy"], t["dz"], t["branch"], t["skip"], **kw)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        t["branch"].copy_(torch.randn(t["branch"].shape, generator=torch.Generator().manual_seed(i)))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_gradients_against_differences(device):
    """fp32 directional derivatives: (f(v + h e) - f(v - h e)) / 2h.  The difference of two sums of 3 x 40 x 64
    products is off by their rounding over 2h (2e-7 * 200 / 2e-2 = 2e-3) and by h^2 times the third derivative
    (1e-4 times values of order 100)."""
    from nsw import ops
    t = {k: v.to(device) for k, v in case(torch.float32, 2, 20, 64, True, "sample", True, seed=10).items()}
    names = ["branch", "skip", "post_weight", "gate", "norm_weight"]

    def f(**v):
        y, z = ops.residual_norm(v["branch"], v["skip"], post_weight=v["post_weight"], gate=v["gate"], alpha=0.9,
                                 norm_weight=v["norm_weight"], eps=1e-5)
        return ((y.double() * t["dy"]).sum() + (z.double() * t["dz"]).sum()).item()

    grads = ops.residual_norm_backward(t["dy"], t["dz"], t["branch"], t["skip"], post_weight=t["post_weight"],
                                       gate=t["gate"], alpha=0.9, norm_weight=t["norm_weight"], eps=1e-5)
    grads = dict(zip(["branch", "skip", "post_weight", "gate", "norm_weight"], grads))
    h = 1e-2
    for n in names:
        e = torch.randn(t[n].shape, generator=torch.Generator().manual_seed(3)).to(device)
        e = e / e.norm()
        v = {k: t[k] for k in names}
        up, down = f(**{**v, n: t[n] + h * e}), f(**{**v, n: t[n] - h * e})
        want = (grads[n].double() * e).sum().item()
        assert abs((up - down) / (2 * h) - want) < 2e-2 * max(1.0, abs(want)), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G", [8, 9, 300])
def test_many_samples(device, dtype, G):
    """Gates of many samples, whose sums are split over workgroups, down to a row each."""
    for R in (1, 7):
        t = case(dtype, G, R, 136, True, "sample", True, seed=G)
        check(run(t, 1.0, 1e-5, device), reference(t, 1.0, 1e-5), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G,R", [(3, 30), (3, 100), (2, 300), (4, 300), (40, 300), (70, 100), (300, 33)])
def test_sums_of_samples_of_unlike_length(device, dtype, G, R):
    """Few and many samples whose partial sums are few, some and many."""
    t = case(dtype, G, R, 136, True, "sample", True, seed=G + R)
    check(run(t, 1.0, 1e-5, device), reference(t, 1.0, 1e-5), dtype)


def test_rows_past_32_bit_offsets(device):
    """More than 2^32 bytes a tensor: the last rows are those of a call on them alone, bit for bit."""
    from nsw import ops
    rows, C = 1_100_001, 2048
    branch = torch.empty(rows, C, dtype=torch.bfloat16, device=device)
    branch.random_(-3, 4)
    skip, dy = branch.flip(0), branch.roll(1, 0)
    w = torch.linspace(0.5, 1.5, C, device=device).to(torch.bfloat16)
    kw = dict(post_weight=w, norm_weight=w, eps=1e-5)
    y, z = ops.residual_norm(branch, skip, **kw)
    db, ds, dp, _, dn = ops.residual_norm_backward(dy, branch, branch, skip, **kw)
    n = 4099
    tail = [t[-n:].clone() for t in (branch, skip, dy)]
    y2, z2 = ops.residual_norm(tail[0], tail[1], **kw)
    db2, ds2, _, _, _ = ops.residual_norm_backward(tail[2], tail[0], tail[0], tail[1], **kw)
    for a, b in ((y, y2), (z, z2), (db, db2), (ds, ds2)):
        assert torch.equal(a[-n:], b)
    assert dp.isfinite().all() and dn.isfinite().all()
