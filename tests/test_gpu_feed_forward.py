"""The feed-forward half of a block as it is used: the norms around it, the gated
block, the gradients of all of it against float64 autograd of the formulas; the
same half served in 8-bit floating point, stage by stage."""
import math

import pytest
import torch
from torch import nn

import nsw
from nsw import _lib, ops, torch_ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


class Half(nn.Module):
    """y, z = norms(branch, skip); the gated block on z; the norms after it."""

    def __init__(self, C, H, act):
        super().__init__()
        self.first = nsw.ResidualNorm(C, alpha=0.9)
        self.mlp = nsw.GatedMLP(C, H, act_layer=act)
        self.last = nsw.ResidualNorm(C, layer_scale=0.7)

    def forward(self, branch, skip, gate):
        y, z = self.first(branch, skip, gate)
        return self.last(self.mlp(z), y)


def plain(p, branch, skip, gate, act, eps):
    rms = lambda t, w: t * (t.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w
    y = 0.9 * skip + gate.repeat_interleave(branch.shape[0] // gate.shape[0], 0) * rms(branch, p["first.post_norm.norm.weight"])
    z = rms(y, p["first.next_norm.norm.weight"])
    g, u = (z @ p["mlp.fc1.weight"].t() + p["mlp.bias1.bias"]).chunk(2, -1)
    o = (act(g) * u) @ p["mlp.fc2.weight"].t() + p["mlp.bias2.bias"]
    y = y + p["last.gamma"] * rms(o, p["last.post_norm.norm.weight"])
    return y, rms(y, p["last.next_norm.norm.weight"])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", [nn.SiLU, nn.GELU])
def test_training_step(device, dtype, act):
    """Relative 2-norm.  fp32: six sums of at most 333 terms one after the other, each within 333 * 2^-24 = 2e-5 of
    its magnitudes at worst, by chance the square root of that (1e-6): 2e-5 in all.  bf16: at most 12 values rounded
    one after the other on the way to a gradient (z, h, the down projection, y, z; dz, dy, the two branches', dg and
    du, dx, the parameter's), half a step (2^-8) each at most."""
    C, H, G, R = 96, 160, 3, 111
    torch.manual_seed(1)
    m = Half(C, H, act)
    with torch.no_grad():
        for n, t in m.named_parameters():
            t.copy_(torch.randn_like(t) * (t.shape[-1] ** -0.5 if t.dim() == 2 else 0.3) + (1.0 if "norm" in n else 0.0))
    m = m.to(device=device, dtype=dtype)
    ins = [torch.randn(s).to(device=device, dtype=dtype).requires_grad_() for s in ((G * R, C), (G * R, C), (G, C))]
    up = [torch.randn(G * R, C).to(device=device, dtype=dtype) for _ in range(2)]
    out = m(*ins)
    leaves = ins + list(m.parameters())
    got = torch.autograd.grad(out, leaves, up)
    p64 = {n: t.detach().double().requires_grad_() for n, t in m.named_parameters()}
    i64 = [t.detach().double().requires_grad_() for t in ins]
    ref = plain(p64, *i64, nn.functional.silu if act is nn.SiLU else nn.functional.gelu, torch.finfo(dtype).eps)
    want = torch.autograd.grad(ref, i64 + list(p64.values()), [t.double() for t in up])
    tol = 2e-5 if dtype == F32 else 12 * 2.0 ** -8
    for a, b in list(zip(out, ref)) + list(zip(got, want)):
        assert a.dtype == dtype and a.shape == b.shape
        assert (a.double() - b).norm() <= tol * b.norm(), ((a.double() - b).norm() / b.norm()).item()


def test_training_step_in_a_graph(device):
    torch.manual_seed(2)
    m = Half(64, 96, nn.SiLU).to(device=device, dtype=BF16)
    ins = [torch.randn(s, device=device).to(BF16) for s in ((150, 64), (150, 64), (2, 64))]
    up = [torch.randn(150, 64, device=device).to(BF16) for _ in range(2)]
    params = list(m.parameters())

    def step():
        return torch.autograd.grad(m(*ins), params, up)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i in range(3):
        ins[0].copy_(torch.randn(150, 64, generator=torch.Generator().manual_seed(i)))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_linear_gradients_of_views(device, dtype):
    """Gradients that arrive transposed, expanded and sliced off alignment give those of their copies."""
    x = torch.randn(64, 96, device=device).to(dtype).requires_grad_()
    w = torch.randn(64, 96, device=device).to(dtype).requires_grad_()
    b = torch.randn(64, device=device).to(dtype).requires_grad_()
    for up in (torch.randn(64, 64, device=device).to(dtype).t(), torch.ones(1, 1, device=device, dtype=dtype).expand(64, 64),
               torch.randn(64 * 64 + 1, device=device).to(dtype)[1:].view(64, 64)):
        y = torch_ops.linear_epi(x, w, b)
        a = torch.autograd.grad(y, (x, w, b), up)
        c = torch.autograd.grad(torch_ops.linear_epi(x, w, b), (x, w, b), up.clone(memory_format=torch.contiguous_format))
        for s, t in zip(a, c):
            assert torch.equal(s, t)


def test_gradients_that_nobody_asks_for(device):
    x, s = (torch.randn(8, 64, device=device) for _ in range(2))
    w = torch.ones(64, device=device, requires_grad=True)
    y, z = torch_ops.residual_norm(x, s, w, None, 1.0, w.detach())
    g, = torch.autograd.grad(y.sum(), w)                       # z unused
    full = torch.ops.nsw.residual_norm_backward(torch.ones_like(y), None, x, s, w.detach(), None, 1.0, w.detach(),
                                                torch.finfo(F32).eps)
    assert torch.equal(g, full[2])


def test_mlp_keeps_its_results_without_gradients(device):
    m = nsw.MLP(64, 128).to(device)
    x = torch.randn(10, 64, device=device)
    with torch.no_grad():
        want = m(x)
    assert torch.equal(m(x), want)


def held(q, scale, rows):
    e = scale.view(torch.uint8).double() - 127
    return q.double() * torch.exp2(e).repeat_interleave(rows, 0)[:q.shape[0]].repeat_interleave(128, 1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tanh", [False, True])
def test_served_mlp(device, dtype, tanh):
    """Each product from the values that its operands hold (the quantiser is exact, tests/test_gpu_fp8.py): fp32 within
    (K + 8) 2^-24 of its sums of magnitudes, bf16 7 * 2^-13 more, and one rounding."""
    C, H, M = 200, 328, 77
    torch.manual_seed(3)
    mlp = nsw.MLP(C, H, act_layer=lambda: nn.GELU(approximate="tanh" if tanh else "none"))
    with torch.no_grad():
        for t in mlp.parameters():
            t.copy_(torch.randn_like(t) * (t.shape[-1] ** -0.5 if t.dim() == 2 else 0.3))
    mlp = mlp.to(device=device, dtype=dtype)
    fp8 = mlp.to_fp8()
    assert set(fp8.state_dict()) == {f"fc{i}.{n}" for i in (1, 2) for n in ("weight", "weight_scale", "bias")}
    with torch.no_grad():
        x, r = torch.randn(M, C, device=device).to(dtype), torch.randn(M, C, device=device).to(dtype)
        y = fp8(x, r)
        h = fp8.fc1(x)
        assert torch.equal(fp8.fc2(h, r), y)
        assert torch.allclose(fp8(x), (y.double() - r.double()).to(dtype), atol=0.1)
    step = torch.finfo(dtype).eps / 2
    for layer, inp, out, add in ((fp8.fc1, x, h, None), (fp8.fc2, h, y, r)):
        a, w = held(*ops.quantize_fp8(inp), 1), held(layer.weight, layer.weight_scale, 128)
        v = a @ w.t() + layer.bias.double()
        tol = (a.abs() @ w.abs().t() + layer.bias.double().abs()) * ((a.shape[1] + 8) * 2.0 ** -24
                                                                     + (7 * 2.0 ** -13 if dtype == BF16 else 0.0))
        if add is None:
            act = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)) if tanh \
                else 0.5 * v * torch.erfc(-v / math.sqrt(2))
            tol = 1.13 * tol + 1.5e-7 * v.abs() + 0.15 * step * act.abs() + 2.0 ** -24
            v = act
        else:
            v = v + add.double()
            tol = tol + 2.0 ** -24 * v.abs()
        over = (out.double() - v).abs() - (tol * (1 + step) + v.abs() * step * (1 + 1e-6))
        assert (over <= 0).all(), over.max().item()


def test_served_half_block(device):
    """Norms, 8-bit block and residual in one run, captured and replayed."""
    torch.manual_seed(4)
    C = 128
    norm, fp8 = nsw.ResidualNorm(C).to(device=device, dtype=BF16), nsw.MLP(C, 4 * C).to(device=device, dtype=BF16).to_fp8()
    branch, skip = (torch.randn(2, 81, C, device=device).to(BF16) for _ in range(2))

    def run():
        with torch.no_grad():
            y, z = norm(branch, skip)
            return fp8(z, y)

    want = run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(3):
        branch.copy_(torch.randn(branch.shape, generator=torch.Generator().manual_seed(i)))
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_fp8_linear_refusals(device):
    lin = nsw.LinearLayer(64, 32).to(device)
    q = nsw.Fp8Linear.from_layers(lin)
    x = torch.randn(3, 64, device=device)
    with pytest.raises(NotImplementedError, match="residual"):
        q(x, residual=torch.zeros(3, 32, device=device))
    with pytest.raises(TypeError):
        ops.linear_fp8(*ops.quantize_fp8(x), q.weight, q.weight_scale, torch.zeros(32, device=device), dtype=BF16)
    with pytest.raises(ValueError, match="scales"):
        xq, xs = ops.quantize_fp8(x)
        ops.linear_fp8(xq, xs[:2].contiguous(), q.weight, q.weight_scale, dtype=F32)
    assert q(x).dtype == F32 and q.epilogue is None and _lib.NSW_EPI_NONE == 0


def test_fp8_parts_that_an_epilogue_lacks(device):
    """A bias or residual that the epilogue would leave out is refused, not dropped."""
    mlp = nsw.MLP(64, 128).to(device=device, dtype=BF16).to_fp8()
    x = torch.randn(3, 64, device=device).to(BF16)
    with torch.no_grad():
        with pytest.raises(NotImplementedError, match="GELU"):
            mlp.fc1(x, residual=torch.zeros(3, 128, device=device, dtype=BF16))
        xq, w = ops.quantize_fp8(x), (mlp.fc1.weight, mlp.fc1.weight_scale)
        r = torch.zeros(3, 128, device=device, dtype=BF16)
        with pytest.raises(ValueError, match="residual"):
            ops.linear_fp8(*xq, *w, None, r)
        with pytest.raises(ValueError, match="residual"):
            ops.linear_fp8(*xq, *w, mlp.fc1.bias, r, epilogue=_lib.NSW_EPI_BIAS_GELU)
        with pytest.raises(ValueError, match="bias"):
            ops.linear_fp8(*xq, *w, mlp.fc1.bias, epilogue=_lib.NSW_EPI_NONE)


def test_fp8_module_keeps_its_bytes_under_a_change_of_dtype(device):
    torch.manual_seed(5)
    mlp = nsw.MLP(128, 256).to(device=device, dtype=F32).to_fp8()
    held_ = [t.clone() for t in (mlp.fc1.weight, mlp.fc1.weight_scale)]
    mlp = mlp.to(BF16)
    x = torch.randn(5, 128, device=device).to(BF16)
    assert mlp.fc1.bias.dtype == BF16 and mlp(x).dtype == BF16
    for t, want in zip((mlp.fc1.weight, mlp.fc1.weight_scale), held_):
        assert t.dtype == want.dtype and torch.equal(t.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_two_streams_and_two_graphs_at_once(device, dtype):
    """Calls that overlap share nothing: the same bits as one after the other."""
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g).to(device=device, dtype=dtype)
    w, b, nw = r(2 * 160, 96) * 96 ** -0.5, r(2 * 160), r(96)
    ins = [(r(700, 96), r(700, 160), r(700, 96), r(4, 96)) for _ in range(2)]

    def step(x, dh, s, gate):
        h = ops.gated_linear(x, w, b)
        y, z = ops.residual_norm(x, s, nw, gate, 1.0, nw)
        return (h, y, z, *ops.gated_linear_backward(dh, x, w, b), *ops.residual_norm_backward(y, z, x, s, nw, gate, 1.0, nw),
                *ops.quantize_fp8(z))

    same = lambda a, b: all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))
    want = [step(*i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(step(*ins[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(same(o, want[k]) for o in got[k])
    graphs, outs = [], []
    for i in ins:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*i))
    for _ in range(3):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert all(same(o, w_) for o, w_ in zip(outs, want))
        step(*ins[0])
