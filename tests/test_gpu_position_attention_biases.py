"""nsw.ops.position_attention with table entries far from zero, as a table holds them for
displacements that take no part, against the formula in float64 on logits rounded to fp32 as
fp32 forms them (half an fp32 step at 1e8 and beyond is larger than the products here, a sixteenth
of a case's, so that a row of such entries alone is uniform).

Tolerances: those of test_gpu_position_attention, a logit's error e without the far
entry's share.  Entries of one far value cancel exactly in the difference to the row's maximum
where the row has no other, and have p = 0 exactly where it has (the next logit is more than
200 away)."""
import math

import pytest
import torch

from test_gpu_position_attention import DTYPES, U, case, check, pairs, run
from test_gpu_position_attention import reference as masked_reference

pytestmark = pytest.mark.gpu


def far_case(dtype, Bw, extent, heads, hd, far, which, seed=20):
    """A case whose table is `far` at every displacement ("all"), or where the query is not behind the key
    ("causal": the first token's row has nothing else)."""
    t = case(dtype, Bw, extent, heads, hd, seed=seed)
    middle = t["table"].shape[0] // 2
    t["qkv"][..., :2 * heads * hd] *= 0.25
    if abs(far) < 1e8:                          # half a step is less than a product: none at all
        t["qkv"][..., :heads * hd] = 0
    t["table"][:None if which == "all" else middle + 1] = far
    return t


def reference(t, far):
    """{name: (value, tolerance before the last rounding)} in float64, and the row's maximum and log2 of its sum."""
    dtype, heads = t["qkv"].dtype, t["heads"]
    h = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    far = t["table"].new_tensor(far).double()
    Bw, L, C3 = t["qkv"].shape
    hd = C3 // 3 // heads
    q, k, v = t["qkv"].double().view(Bw, L, 3, heads, hd).permute(2, 0, 3, 1, 4)
    rel = t["table"].double()[t["buckets"].long()]
    idx = pairs(*t["extent"])
    bias = rel[idx].permute(2, 0, 1)
    z = (t["scale"] * q @ k.mT + bias).float().double()
    e = (hd + 6) * U * (abs(t["scale"]) * q.abs() @ k.abs().mT + torch.where(bias == far, 0.0, bias.abs()))
    top = z.amax(-1, keepdim=True)
    p = (z - top).exp()
    total = p.sum(-1, keepdim=True)
    p = p / total
    far_off = torch.where(p > 0, z - top, 0.0).abs()
    f = 2 * (e + e.amax(-1, keepdim=True)) + 8 * U * (1 + far_off) + (L + 8) * U
    flat = lambda x: x.transpose(1, 2).reshape(Bw, L, -1)
    o, do = p @ v, t["do"].double().view(Bw, L, heads, hd).transpose(1, 2)
    to = (p * (f + h + L * U)) @ v.abs()
    out = {"o": (flat(o), flat(to))}
    stored = to + (o.abs() + to) * (h / 4 if h else U)
    dp, D = do @ v.mT, (do * o).sum(-1, keepdim=True)
    err = hd * U * (do.abs() @ v.abs().mT) + (do.abs() * (stored + hd * U * o.abs())).sum(-1, keepdim=True)
    dz = p * (dp - D)
    if L == 1:
        dz, err = dz * 0, err * 0
    tz = p * err + f * dz.abs()
    wide = tz + (h + L * U) * (dz.abs() + tz)
    sc = abs(t["scale"])
    dq = (t["scale"] * dz @ k, sc * wide @ k.abs())
    dk = (t["scale"] * dz.mT @ q, sc * wide.mT @ q.abs())
    dv = (p.mT @ do, (p * (f + h + L * U)).mT @ do.abs())
    out["dqkv"] = tuple(torch.cat([flat(x[i]) for x in (dq, dk, dv)], -1) for i in (0, 1))
    add = lambda x: torch.zeros(rel.shape, dtype=torch.float64).index_add_(0, t["buckets"].long()[idx].reshape(-1),
                                                                          x.sum(0).reshape(heads, L * L).T)
    out["dtable"] = (add(dz), add(tz + (64 + Bw * L) * U * (dz.abs() + tz)))
    return out, top[..., 0] * math.log2(math.e), total[..., 0].log2(), f.amax(-1)


FAR = [-1e4, -1e6, 1e6, -1e8, -1e10, -1e30, -1e38, 1e10, 1e30]
EXTENTS = [(1, 1, 1), (1, 3, 5), (1, 1, 70), (1, 9, 18), (1, 12, 16), (2, 9, 18)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent", EXTENTS)
@pytest.mark.parametrize("which", ["all", "causal"])
@pytest.mark.parametrize("far", FAR)
def test_forward(device, dtype, extent, which, far):
    """A row of far entries alone is a mean of v, neither zeros nor NaN."""
    for hd in (32, 64):
        t = far_case(dtype, 3, extent, 2, hd, far, which)
        got = run(t, device)
        want, top, total, f = reference(t, far)
        check(got, {"o": want["o"]}, dtype)
        stats = got["stats"].double().cpu()
        assert ((stats[..., 0] - top).abs() <= 8 * U * top.abs() + f).all()
        assert ((stats[..., 1] - total).abs() <= 2 * f + 4 * U * total).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent", EXTENTS)
@pytest.mark.parametrize("which", ["all", "causal"])
@pytest.mark.parametrize("far", FAR)
def test_gradients(device, dtype, extent, which, far):
    """Probabilities formed again from statistics whose maximum is far from zero."""
    for hd in (32, 64):
        t = far_case(dtype, 3, extent, 2, hd, far, which)
        check(run(t, device), reference(t, far)[0], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent", EXTENTS)
@pytest.mark.parametrize("which", ["all", "causal"])
@pytest.mark.parametrize("far", ["lowest", "highest", -2.4e38, 2.4e38])
def test_the_largest_table_values(device, dtype, extent, which, far):
    """Finite values whose product with log2 e is not: they stay what they are among others, and uniform by themselves."""
    far = {"lowest": torch.finfo(dtype).min, "highest": torch.finfo(dtype).max}.get(far, far)
    t = far_case(dtype, 3, extent, 2, 32, far, which)
    check(run(t, device), reference(t, far)[0], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent", [e for e in EXTENTS if math.prod(e) > 1])
@pytest.mark.parametrize("high", [torch.finfo(torch.float32).max, 2.4e38])
def test_the_largest_mask_values(device, dtype, extent, high):
    """The keys that a mask lifts above all others share a row's weight."""
    t = case(dtype, 4, extent, 2, 32, seed=21)
    L = math.prod(extent)
    m = torch.zeros(2, L, L)
    m[0, L // 2, :L // 2 + 1] = high
    m[1, :, L // 3] = high
    m[1, L - 1] = -math.inf
    check(run(t, device, mask=m), masked_reference(t, m), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent,kind", [(e, k) for e in [(1, 3, 5), (1, 9, 18), (2, 9, 18), (1, 1, 700)]
                                         for k in ["none", "shift", "mask"] if k != "shift" or e[1] > 1])
@pytest.mark.parametrize("hd", [16, 64, 128])
def test_probabilities_add_up_whatever_the_logits(device, dtype, extent, kind, hd):
    """With ones for the gradient of o, dv summed over the keys is the sum of all probabilities: L, if the backward pass
    forms each logit as the forward pass did.  Logits of 1e7 and more, whose fp32 steps change a probability by any factor.

    A probability's exponent z - m - l: z - m is exact at the maximum and off by u |z - m| elsewhere, where p < 1 makes p
    |z - m| at most 1/e a term; l, log2 of a sum of L terms, by (L + 8) u and a step of up to 2^-20; the sum over keys by
    L u: (3 L + 64) u of L in all, and 16 u for l's step.  bf16: p and dv are rounded by 2^-8 each."""
    T, A, W = extent
    L, C = math.prod(extent), 2 * hd
    tol = (3 * L + 80) * U + (2 * 2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
    g = torch.Generator().manual_seed(25)
    how = {"none": {}, "shift": dict(geometry=(3 * A, 2 * W, (A, W), (A // 2, W // 2), T)),
           "mask": dict(mask=torch.randn(2, L, L, generator=g))}[kind]
    for factor in (1.0, 30.0, 300.0, 3000.0):
        for std in (0.5, 1e6):
            t = case(dtype, 6, extent, 2, hd, seed=26, std=std)
            t["qkv"][..., :2 * C] *= factor
            t["do"] = torch.ones_like(t["do"])
            total = run(t, device, **how)["dqkv"][..., 2 * C:].double().sum(1) / L
            assert ((total - 1).abs() <= tol).all(), (factor, std, (total - 1).abs().max().item(), tol)
