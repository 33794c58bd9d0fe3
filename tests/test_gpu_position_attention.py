"""nsw.ops.position_attention and its gradients against the formulas in float64.

Tolerances, per element.  u = 2^-24, h = 2^-8 for bf16 (a rounding is off by at most half a
step), 0 for fp32.  A logit is a dot product of hd terms, a product, one or two sums: off by at most
e = (hd + 6) u (scale |q||k| + |bias| + min(|mask|, 1e4)) (the reference forms mask sums in fp32 too,
so that a large mask rounds alike).  Its difference to the row's maximum, product with log2 e and
exp2 add 4 u (1 + |z - m|).  So p is off by the factor 1 + f, f = 2 (e + e_max) + 8 u (1 + |z - m|)
+ (L + 8) u, the last for the sum of L terms.  o: f and the rounding of p, h, on the sum of
p |v|, L u for the product, then one rounding to the type.  With the error t_o of o
and of the bits that its rounding lost, an eighth of a step at most (a half is 2^-8), D = do o is off by
|do| t_o + hd u |do||o|, dp by hd u |do||v|, and dz = p (dp - D) by p (those) + f |dz|.
dz and p are rounded once more (h) for dq, dk and dv, which sum L terms; dtable sums windows L^2
terms at most, in chains: (64 + Bw L) u of the sum of magnitudes."""
import math

import pytest
import torch

import nsw
from nsw import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LOWEST = torch.finfo(torch.float32).min


def pairs(T, A, W):
    t, a, w = (v.reshape(-1) for v in torch.meshgrid(torch.arange(T), torch.arange(A), torch.arange(W), indexing="ij"))
    d = lambda v, n: v[:, None] - v[None, :] + n - 1
    return (d(t, T) * (2 * A - 1) + d(a, A)) * (2 * W - 1) + d(w, W)


def case(dtype, Bw, extent, heads, hd, seed=0, buckets=None, nb=None, std=0.5):
    g = torch.Generator().manual_seed(seed)
    L, C, R = math.prod(extent), heads * hd, ops.window_displacements(extent)
    if buckets is None:
        buckets, nb = torch.arange(R, dtype=torch.int32), R
    r = lambda *s: torch.randn(*s, generator=g)
    return dict(qkv=r(Bw, L, 3 * C).to(dtype), table=(std * r(nb, heads)).to(dtype), do=r(Bw, L, C).to(dtype), buckets=buckets,
                extent=extent, heads=heads, scale=hd ** -0.5)


def reference(t, mask=None):
    """{name: (value, tolerance before the last rounding)} in float64.  mask: fp32 [nW, L, L] or None."""
    dtype, heads = t["qkv"].dtype, t["heads"]
    h = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    Bw, L, C3 = t["qkv"].shape
    hd = C3 // 3 // heads
    q, k, v = t["qkv"].double().view(Bw, L, 3, heads, hd).permute(2, 0, 3, 1, 4)
    b = t["buckets"].long()
    there = (b >= 0) & (b < t["table"].shape[0])
    rel = torch.where(there[:, None], t["table"].double()[b.clamp(0, t["table"].shape[0] - 1)], 0.0)
    idx = pairs(*t["extent"])
    bias = rel[idx].permute(2, 0, 1)
    z = t["scale"] * q @ k.mT + bias
    e = (hd + 6) * U * (abs(t["scale"]) * q.abs() @ k.abs().mT + bias.abs())
    if mask is not None:
        m = mask.repeat(Bw // mask.shape[0], 1, 1)[:, None]
        z = (z.float() + m).double()
        e = e + (hd + 6) * U * torch.where(m.isfinite(), m.abs(), torch.zeros_like(m)).clamp(max=1e4)
    top = z.amax(-1, keepdim=True)
    empty = top == -math.inf
    d = torch.where(empty, torch.full_like(z, -math.inf), z - top.masked_fill(empty, 0.0))
    p = d.exp()
    s = p.sum(-1, keepdim=True)
    p = p / s.masked_fill(empty, 1.0)
    far = torch.where(p > 0, d.abs(), torch.zeros_like(d))
    f = 2 * (e + e.amax(-1, keepdim=True)) + 8 * U * (1 + far) + (L + 8) * U
    o, do = p @ v, t["do"].double().view(Bw, L, heads, hd).transpose(1, 2)
    to = (p * (f + h + L * U)) @ v.abs()
    stored = to + (o.abs() + to) * (h / 4 if h else U)
    dp = do @ v.mT
    D = (do * o).sum(-1, keepdim=True)
    err = hd * U * (do.abs() @ v.abs().mT) + (do.abs() * (stored + hd * U * o.abs())).sum(-1, keepdim=True)
    dz = p * (dp - D)
    if L == 1:
        dz, err = dz * 0, err * 0
    tz = p * err + f * dz.abs()
    wide = tz + (h + L * U) * (dz.abs() + tz)
    sc = abs(t["scale"])
    flat = lambda x: x.transpose(1, 2).reshape(Bw, L, -1)
    out = {"o": (flat(o), flat(to))}
    dq = (t["scale"] * dz @ k, sc * wide @ k.abs())
    dk = (t["scale"] * dz.mT @ q, sc * wide.mT @ q.abs())
    dv = (p.mT @ do, (p * (f + h + L * U)).mT @ do.abs())
    out["dqkv"] = tuple(torch.cat([flat(x[i]) for x in (dq, dk, dv)], -1) for i in (0, 1))
    rows = lambda x: x.sum(0).reshape(heads, L * L).T
    at = b[idx].reshape(-1)
    keep = there[idx].reshape(-1)
    add = lambda x: torch.zeros(t["table"].shape, dtype=torch.float64).index_add_(0, at[keep], rows(x)[keep])
    out["dtable"] = (add(dz), add(tz + (64 + Bw * L) * U * (dz.abs() + tz)))
    return out


def run(t, device, mask=None, geometry=None):
    d = {k: v.to(device) if torch.is_tensor(v) else v for k, v in t.items()}
    mask = None if mask is None else mask.to(device)
    args = (d["heads"], d["scale"], d["table"], d["buckets"], d["extent"])
    o, stats = ops.position_attention(d["qkv"], *args, mask=mask, geometry=geometry)
    dqkv, dtable = ops.position_attention_backward(d["do"], d["qkv"], o, stats, *args, mask=mask, geometry=geometry)
    return {"o": o, "dqkv": dqkv, "dtable": dtable, "stats": stats}


def check(got, want, dtype):
    step = torch.finfo(dtype).eps / 2
    for name, (v, tol) in want.items():
        g = got[name]
        assert g.dtype == dtype and g.shape == v.shape, name
        err = (g.double().cpu() - v).abs() - (v.abs() * step + tol * (1 + step))
        assert (err <= 1e-30).all(), (name, err.max().item(), v.flatten()[err.argmax()].item())


DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [4, 8, 16, 32, 64, 128])
@pytest.mark.parametrize("extent", [(1, 3, 5), (1, 7, 7), (1, 9, 18), (2, 9, 18)])
def test_head_dims(device, dtype, hd, extent):
    t = case(dtype, 3, extent, 2, hd, seed=hd)
    check(run(t, device), reference(t), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent", [(1, 1, 1), (1, 1, 2), (1, 1, 15), (1, 1, 16), (1, 1, 17), (1, 1, 33), (1, 1, 63), (1, 1, 64),
                                    (1, 1, 65), (1, 1, 127), (1, 8, 16), (1, 1, 129), (1, 1, 191), (1, 12, 16), (1, 1, 193),
                                    (3, 6, 9), (1, 1, 257), (5, 1, 7), (4, 4, 1), (1, 40, 2)])
def test_extents(device, dtype, extent):
    t = case(dtype, 2, extent, 2, 32, seed=math.prod(extent))
    check(run(t, device), reference(t), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent", [(1, 5, 6), (1, 9, 18), (1, 1, 200)])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-8, 1e-6, 1e6, 1e8])
def test_scales(device, dtype, extent, scale):
    t = case(dtype, 3, extent, 2, 64, seed=12)
    if abs(scale) >= 1e6:
        t["qkv"][..., :128] /= 4 * scale
    t["scale"] = scale
    check(run(t, device), reference(t), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,n", [(16, 700), (64, 1023), (128, 900)])
def test_sequences(device, dtype, hd, n):
    """Lengths whose accumulators the groups of a wave share, buckets that widen with the distance."""
    buckets, nb = nsw.position_buckets((1, 1, n), 32, 128)
    t = case(dtype, 1, (1, 1, n), 2, hd, seed=n, buckets=buckets, nb=nb)
    check(run(t, device), reference(t), dtype)


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 4), (torch.bfloat16, 128), (torch.float32, 128)])
def test_the_most_displacements(device, dtype, hd):
    """8191 of them: the waves of a workgroup share one accumulator."""
    t = case(dtype, 1, (1, 1, 4096), 2, hd, seed=2) if hd == 4 else case(dtype, 1, (1, 1, 3100), 1, hd, seed=2)
    check(run(t, device), reference(t), dtype)


def masks(kind, nW, L, seed=3):
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(nW, L, L, generator=g)
    if kind == "float":
        return torch.randn(nW, L, L, generator=g)
    m = torch.where(u < 0.4, torch.tensor(-math.inf if kind in ("infinite", "empty") else LOWEST), torch.tensor(0.0))
    if kind == "empty":
        m[:, L // 3] = -math.inf                # a query without keys
        m[:, :, L // 2] = -math.inf             # a key without queries
        m[0] = -math.inf                        # a window without any pair
    elif kind == "one":
        m = torch.full((nW, L, L), -math.inf)
        m[:, torch.arange(L), (torch.arange(L) * 7 + 3) % L] = 0.0
    elif kind == "lowest":
        m[:, L // 3] = LOWEST                   # uniform over all keys, as in fp32 on the formula
    elif kind == "large":
        m = torch.where(u < 0.4, torch.tensor(-1e9), torch.tensor(0.0))
        m[:, L // 3] = -1e9
    return m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent,hd", [((1, 3, 5), 16), ((1, 9, 18), 32), ((1, 9, 18), 64), ((2, 9, 18), 64), ((1, 1, 70), 128)])
@pytest.mark.parametrize("kind", ["float", "infinite", "empty", "one", "lowest", "large"])
def test_masks(device, dtype, extent, hd, kind):
    t = case(dtype, 4, extent, 2, hd, seed=5)
    m = masks(kind, 2, math.prod(extent))
    got = run(t, device, mask=m)
    check(got, reference(t, m), dtype)
    if kind == "empty":
        L = math.prod(extent)
        assert not got["o"][:, L // 3].any() and not got["o"][0].any()
        assert not got["dqkv"][0].any() and not got["dqkv"][:, L // 3, :2 * hd].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent", [(1, 9, 18), (2, 5, 6)])
def test_boolean_mask(device, dtype, extent):
    """True marks the pairs that take part."""
    t = case(dtype, 2, extent, 2, 32, seed=6)
    keep = masks("infinite", 1, math.prod(extent)) == 0
    got = run(t, device, mask=keep)
    check(got, reference(t, torch.zeros(keep.shape).masked_fill_(~keep, -math.inf)), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent,shift,hd", [((1, 9, 18), (4, 9), 64), ((1, 3, 5), (1, 2), 16), ((2, 6, 6), (3, 0), 32),
                                             ((2, 9, 18), (0, 9), 32)])
def test_shift_mask_from_the_geometry(device, dtype, extent, shift, hd):
    """Both forms of the mask within their tolerance of the formula, so of each other within twice that."""
    T, A, W = extent
    H, Wi = 3 * A, 2 * W
    t = case(dtype, 12, extent, 2, hd, seed=7)
    m = nsw.swin_helpers.attention_mask_closed_form(H, Wi, (A, W), shift, T)
    got = run(t, device, geometry=(H, Wi, (A, W), shift, T))
    want = reference(t, m)
    check(got, want, dtype)
    check(run(t, device, mask=m), want, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_buckets_outside_the_table(device, dtype):
    """They count as no bias and have no gradient; several displacements to a bucket, buckets that none has."""
    extent = (1, 5, 6)
    g = torch.Generator().manual_seed(1)
    b = torch.randint(-3, 15, (ops.window_displacements(extent),), generator=g).int()
    b[0], b[1] = -2 ** 31, 2 ** 31 - 1
    t = case(dtype, 3, extent, 2, 16, seed=8, buckets=b, nb=300)
    t["table"] = torch.cat([t["table"][:10], t["table"][10:]])
    got = run(t, device)
    check(got, reference(t), dtype)
    assert not got["dtable"][15:].any()


def test_one_token_has_no_gradient_through_its_weight(device):
    for dtype in DTYPES:
        t = case(dtype, 70, (1, 1, 1), 4, 16, seed=9)
        got = run(t, device)
        assert torch.equal(got["o"].cpu(), t["qkv"][..., 128:]) and torch.equal(got["dqkv"][..., 128:].cpu(), t["do"])
        assert not got["dqkv"][..., :128].any() and not got["dtable"].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_statistics(device, dtype):
    t = case(dtype, 2, (1, 5, 7), 2, 32, seed=10)
    t["qkv"] *= 4
    got = run(t, device)["stats"].double().cpu()
    q, k, _ = t["qkv"].double().view(2, 35, 3, 2, 32).permute(2, 0, 3, 1, 4)
    z = t["scale"] * q @ k.mT + t["table"].double()[pairs(1, 5, 7)].permute(2, 0, 1)
    top = z.amax(-1) * math.log2(math.e)
    assert ((got[..., 0] - top).abs() <= 1e-4 * (1 + top.abs())).all()
    total = (z * math.log2(math.e) - top[..., None]).exp2().sum(-1).log2()
    assert ((got[..., 1] - total).abs() <= 1e-4).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent", [(1, 9, 18), (2, 9, 18), (1, 1, 700)])
def test_the_same_bits_every_time(device, dtype, extent):
    t = case(dtype, 5, extent, 2, 32, seed=11)
    a, b = run(t, device), run(t, device)
    assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("needs", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("extent", [(1, 9, 18), (2, 9, 18)])
def test_some_gradients(device, needs, extent):
    t = case(torch.bfloat16, 3, extent, 2, 32, seed=12)
    d = {k: v.to(device) if torch.is_tensor(v) else v for k, v in t.items()}
    args = (d["heads"], d["scale"], d["table"], d["buckets"], d["extent"])
    o, stats = ops.position_attention(d["qkv"], *args)
    whole = ops.position_attention_backward(d["do"], d["qkv"], o, stats, *args)
    for n, a, b in zip(needs, ops.position_attention_backward(d["do"], d["qkv"], o, stats, *args, needs=needs), whole):
        assert (a is None) == (not n) and (a is None or torch.equal(a, b))


def test_not_a_number_stays_in_its_window(device):
    for extent in ((1, 9, 18), (2, 9, 18)):
        t = case(torch.float32, 3, extent, 2, 32, seed=13)
        want = run(t, device)
        t["qkv"][1, 7, 40] = math.nan               # a query value of head 1
        got = run(t, device)
        for name in ("o", "dqkv"):
            assert torch.equal(got[name][::2], want[name][::2])
        assert got["o"][1, 7, 32:].isnan().all() and torch.equal(got["o"][1, :, :32], want["o"][1, :, :32])
        assert torch.equal(got["o"][1, :7], want["o"][1, :7])
        assert got["dtable"][:, 1].isnan().any() and torch.equal(got["dtable"][:, 0], want["dtable"][:, 0])


def test_no_windows(device):
    t = case(torch.bfloat16, 0, (1, 3, 5), 2, 32)
    got = run(t, device)
    assert got["o"].shape == (0, 15, 64) and got["dqkv"].shape == (0, 15, 192) and not got["dtable"].any()


def test_more_than_32_bits_of_bytes(device):
    """The windows past 2^32 bytes against the same windows alone."""
    extent, heads, hd, Bw = (1, 9, 18), 8, 64, 9300
    t = case(torch.bfloat16, 4, extent, heads, hd, seed=14)
    qkv = torch.empty(Bw, 162, 3 * heads * hd, dtype=torch.bfloat16, device=device)
    do = torch.empty(Bw, 162, heads * hd, dtype=torch.bfloat16, device=device)
    qkv.normal_()
    do.normal_()
    table, buckets = t["table"].to(device), t["buckets"].to(device)
    args = (heads, t["scale"], table, buckets, extent)
    o, stats = ops.position_attention(qkv, *args)
    dqkv, dtable = ops.position_attention_backward(do, qkv, o, stats, *args)
    o2, stats2 = ops.position_attention(qkv[-4:].clone(), *args)
    dqkv2, _ = ops.position_attention_backward(do[-4:].clone(), qkv[-4:].clone(), o2, stats2, *args)
    assert torch.equal(o[-4:], o2) and torch.equal(stats[-4:], stats2) and torch.equal(dqkv[-4:], dqkv2)
    assert dtable.isfinite().all()


def test_refusals(device):
    z = lambda *s, **k: torch.zeros(*s, device=device, **k)
    qkv, table, b = z(4, 15, 192), z(45, 2), z(45, dtype=torch.int32)
    o, stats = ops.position_attention(qkv, 2, 0.2, table, b, (1, 3, 5))
    f = lambda qkv=qkv, table=table, b=b, extent=(1, 3, 5), **k: ops.position_attention(qkv, 2, 0.2, table, b, extent, **k)
    g = lambda do=o, o=o, stats=stats: ops.position_attention_backward(do, qkv, o, stats, 2, 0.2, table, b, (1, 3, 5))
    geo = (6, 10, (3, 5), (1, 2), 1)
    for bad in (lambda: f(extent=(1, 3, 4)), lambda: f(extent=(1, 1, 15)), lambda: f(table=z(45, 3)), lambda: f(table=z(0, 2)),
                lambda: f(b=z(44, dtype=torch.int32)), lambda: f(b=z(45, dtype=torch.int64)), lambda: f(mask=z(3, 15, 15)),
                lambda: f(mask=z(15, 15)), lambda: f(mask=z(4, 15, 14)), lambda: f(mask=z(1, 15, 15), geometry=geo),
                lambda: f(geometry=(6, 10, (5, 3), (1, 2), 1)), lambda: f(geometry=(6, 15, (3, 5), (1, 2), 1)),
                lambda: f(qkv=z(4, 15, 190)), lambda: f(qkv=z(60, 192)), lambda: g(do=z(4, 15, 32)), lambda: g(stats=stats[:2]),
                lambda: g(stats=stats.double())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        f(table=table.bfloat16())
    with pytest.raises(TypeError):
        f(qkv=qkv.half(), table=table.half())
    with pytest.raises(RuntimeError, match="contiguous"):
        f(qkv=z(4, 192, 15).transpose(1, 2))


# ------------------------------------------------- autograd, modules, graphs ---

def test_gradients_against_differences(device):
    """Directional derivatives to qkv and to the table against central differences of the forward kernel."""
    t = case(torch.float32, 2, (1, 5, 7), 2, 32, seed=15)
    got = run(t, device)
    g = torch.Generator().manual_seed(4)
    for name, grad in (("qkv", "dqkv"), ("table", "dtable")):
        v = torch.randn(t[name].shape, generator=g)
        e = 2.0 ** -7
        f = lambda s: (run({**t, name: t[name] + s * e * v}, device)["o"].double().cpu() * t["do"].double()).sum()
        diff = (f(1) - f(-1)) / (2 * e)
        exact = (got[grad].double().cpu() * v.double()).sum()
        # rounding: 4480 results within 2e-6, of random signs, over 2 e: 0.03 at 3 sigma; the third derivative's part
        # is e^2 / 6 of it, with a factor of at most 30 here
        assert abs(exact - diff) <= 0.1 + 2e-3 * abs(diff), (name, exact, diff)


def branch(device, dtype=torch.float32, **kw):
    torch.manual_seed(3)
    m = nsw.PositionAttentionBranch(64, 2, (6, 10), (3, 5), 2, (1, 2), num_groups=8, act_layer=torch.nn.SiLU, **kw)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(torch.randn_like(p) * (0.1 if p.dim() > 1 else 0.2))
    return m.to(device=device, dtype=dtype)


def branch_reference(x, prm, buckets):
    """PositionAttentionBranch's formula on float64 tensors."""
    B, T, H, W, C = x.shape
    g = x.view(B, -1, 8, 8)
    var, mean = torch.var_mean(g, (1, 3), correction=0, keepdim=True)
    n = ((g - mean) / (var + 1e-5).sqrt()).reshape(B, T, H, W, C) * prm["norm.weight"] + prm["norm.bias"]
    n = n * n.sigmoid()
    w = n.roll((-1, -2), (2, 3)).view(B, T, 2, 3, 2, 5, C).permute(0, 2, 4, 1, 3, 5, 6).reshape(-1, 30, C)
    q, k, v = (w @ prm["attn.qkv.weight"].T + prm["attn.biasqkv.bias"]).view(-1, 30, 3, 2, 32).permute(2, 0, 3, 1, 4)
    m = nsw.swin_helpers.attention_mask_closed_form(6, 10, (3, 5), (1, 2), 2).double()
    z = 32 ** -0.5 * q @ k.mT + prm["attn.position.table"][buckets.long()[pairs(2, 3, 5)]].permute(2, 0, 1)
    o = (z + m.repeat(B, 1, 1)[:, None]).softmax(-1) @ v
    o = o.transpose(1, 2).reshape(-1, 30, C) @ prm["attn.proj.weight"].T + prm["attn.biasproj.bias"]
    o = o.view(B, 2, 2, T, 3, 5, C).permute(0, 3, 1, 4, 2, 5, 6).reshape(B, T, H, W, C)
    return x + o.roll((1, 2), (2, 3))


@pytest.mark.parametrize("kw", [{}, dict(num_buckets=8, max_distance=8)])
def test_branch(device, kw):
    """Group norm, roll and partition, projections, attention and the way back together, with every gradient,
    to 2e-5 of each result's norm (fp32 throughout; sums of at most a few hundred terms in a chain of seven operators)."""
    m = branch(device, **kw)
    g = torch.Generator().manual_seed(5)
    x, dy = torch.randn(3, 2, 6, 10, 64, generator=g), torch.randn(3, 2, 6, 10, 64, generator=g)
    xd = x.to(device).requires_grad_()
    y = m(xd)
    y.backward(dy.to(device))
    prm = {k: v.detach().double().cpu().requires_grad_() for k, v in m.named_parameters()}
    x64 = x.double().requires_grad_()
    y64 = branch_reference(x64, prm, m.attn.position.buckets.cpu())
    y64.backward(dy.double())
    near = lambda a, b: (a.double().cpu() - b).norm() <= 2e-5 * b.norm()
    assert near(y.detach(), y64.detach()) and near(xd.grad, x64.grad)
    for k, v in m.named_parameters():
        assert near(v.grad, prm[k].grad), k


def test_branch_in_bf16_runs_with_gradients(device):
    m = branch(device, torch.bfloat16)
    x = torch.randn(2, 2, 6, 10, 64, device=device).bfloat16().requires_grad_()
    m(x).float().square().mean().backward()
    assert x.grad.isfinite().all() and all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters())


def test_compiled(device):
    m = branch(device)
    x = torch.randn(2, 2, 6, 10, 64, device=device)
    xs = [x.clone().requires_grad_() for _ in range(2)]
    ys = [m(xs[0]), torch.compile(m, fullgraph=True, backend="aot_eager")(xs[1])]
    for y in ys:
        y.square().sum().backward()
    assert torch.equal(ys[0], ys[1]) and torch.equal(xs[0].grad, xs[1].grad)


def test_gradient_of_a_mask_is_refused(device):
    t = case(torch.float32, 2, (1, 3, 5), 2, 32)
    qkv = t["qkv"].to(device).requires_grad_()
    mask = torch.zeros(1, 15, 15, device=device, requires_grad=True)
    o = nsw.torch_ops.position_attention(qkv, 2, 0.2, t["table"].to(device), t["buckets"].to(device), (1, 3, 5), mask=mask)
    with pytest.raises(NotImplementedError, match="mask"):
        o.sum().backward()
    o, stats = torch.ops.nsw.position_attention(qkv, 2, 0.2, t["table"].to(device), t["buckets"].to(device), [1, 3, 5], None, [])
    with pytest.raises(NotImplementedError, match="statistics"):
        stats.sum().backward()


def test_strided_inputs_and_gradients(device):
    t = case(torch.bfloat16, 4, (1, 3, 5), 2, 32, seed=16)
    wide = torch.randn(4, 15, 200, device=device).bfloat16()
    args = (2, t["scale"], t["table"].to(device), t["buckets"].to(device), (1, 3, 5))
    a = wide[..., 3:195].detach().requires_grad_()                    # rows of 200, 6 bytes off
    b = wide[..., 3:195].contiguous().detach().requires_grad_()
    do = torch.randn(4, 64, 15, device=device).bfloat16().transpose(1, 2)
    for x in (a, b):
        nsw.torch_ops.position_attention(x, *args).backward(do if x is a else do.contiguous())
    assert torch.equal(a.grad, b.grad)


@pytest.mark.parametrize("R", [(1, 1, 1), (2, 2, 4)])
def test_window_maps_have_gradients(device, R):
    """A permutation: the gradient is the other map."""
    x = torch.randn(2, 2, 6, 10, 8, device=device, requires_grad=True)
    w = torch.ops.nsw.roll_window_partition(x, [3, 5], [1, 2])
    dw = torch.randn_like(w)
    w.backward(dw)
    assert torch.equal(x.grad, torch.ops.nsw.window_reverse_roll(dw, [3, 5], [6, 10], [1, 2]))
    v = torch.randn(8, 2, 3, 5, 8, device=device, requires_grad=True)
    y = torch.ops.nsw.window_reverse(v, [3, 5], [6, 10])
    dy = torch.randn_like(y)
    y.backward(dy)
    assert torch.equal(v.grad, torch.ops.nsw.window_partition(dy, [3, 5]))


@pytest.mark.parametrize("extent", [(1, 9, 18), (2, 9, 18)])
def test_captured_and_replayed(device, extent):
    """Forward and backward in one graph, replayed with other inputs and eager work between."""
    t = {k: v.to(device) if torch.is_tensor(v) else v for k, v in case(torch.bfloat16, 4, extent, 2, 32, seed=17).items()}
    args = (t["heads"], t["scale"], t["table"], t["buckets"], t["extent"])
    def step():
        o, stats = ops.position_attention(t["qkv"], *args)
        return (o,) + ops.position_attention_backward(t["do"], t["qkv"], o, stats, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        for n in ("qkv", "do", "table"):
            t[n].normal_()
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), k


def test_two_streams_at_once(device):
    ts = [{k: v.to(device) if torch.is_tensor(v) else v for k, v in case(torch.bfloat16, 40, (1, 9, 18), 2, 64, seed=s).items()}
          for s in (1, 2)]
    def step(t):
        args = (t["heads"], t["scale"], t["table"], t["buckets"], t["extent"])
        o, stats = ops.position_attention(t["qkv"], *args)
        return (o,) + ops.position_attention_backward(t["do"], t["qkv"], o, stats, *args)
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
