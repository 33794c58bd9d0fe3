"""The feed-forward modules and their custom operators without a GPU: shape
functions, state-dict keys, initialisation, refusals, tracing as single nodes."""
import pytest
import torch
from torch import nn

import nsw
from nsw import torch_ops


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, device="meta", dtype=dtype)


def test_shape_functions():
    n = torch.ops.nsw
    x, w, b = meta(2, 5, 64), meta(96, 64), meta(96)
    assert n.gated_linear(x, w, b, "silu").shape == (2, 5, 48)
    dx, dw, db = n.gated_linear_backward(meta(2, 5, 48), x, w, b, "silu", [True, False, True])
    assert dx.shape == x.shape and dw.shape == (0,) and db.shape == (96,)
    dx, dw, db = n.linear_backward(meta(2, 5, 96), x, w, [False, True, True])
    assert dx.shape == (0,) and dw.shape == w.shape and db.shape == (96,)
    q, s = n.quantize_fp8(meta(2, 5, 200), 1)
    assert q.shape == (2, 5, 256) and q.dtype == torch.float8_e4m3fn
    assert s.shape == (2, 5, 2) and s.dtype == torch.float8_e8m0fnu
    wq, ws = n.quantize_fp8(meta(300, 200), 128)
    assert wq.shape == (300, 256) and ws.shape == (3, 2)
    y = n.linear_fp8(q, s, wq, ws, None, None, 0, torch.float32)
    assert y.shape == (2, 5, 300) and y.dtype == torch.float32
    y, z = torch_ops.residual_norm(x, x, meta(64), meta(2, 64), 1.0, meta(64))
    assert y.shape == x.shape and z.shape == x.shape
    assert torch_ops.residual_norm(x, x)[1] is None


def test_gradients_have_shapes_on_meta():
    x, w, b = (t.requires_grad_() for t in (meta(2, 5, 64), meta(96, 64), meta(96)))
    g = torch.autograd.grad(torch.ops.nsw.gated_linear(x, w, b, "gelu"), (x, w, b), meta(2, 5, 48))
    assert [t.shape for t in g] == [x.shape, w.shape, b.shape]
    r = meta(2, 5, 96).requires_grad_()
    g = torch.autograd.grad(torch_ops.linear_epi(x, w, b, r), (x, w, b, r), meta(2, 5, 96))
    assert [t.shape for t in g] == [x.shape, w.shape, b.shape, r.shape]
    gate, wn = meta(2, 64).requires_grad_(), meta(64).requires_grad_()
    y, z = torch_ops.residual_norm(x, x.detach(), wn, gate, 1.0, wn)
    assert [t.shape for t in torch.autograd.grad(z, (x, gate, wn), meta(2, 5, 64))] == [x.shape, gate.shape, wn.shape]


def test_gelu_epilogue_has_no_gradient():
    x, w = meta(5, 64).requires_grad_(), meta(96, 64)
    y = torch.ops.nsw.linear(x, w, meta(96), None, 2)
    with pytest.raises(NotImplementedError, match="GatedMLP"):
        torch.autograd.grad(y, x, meta(5, 96))


def test_gated_mlp_parameters():
    m = nsw.GatedMLP(64, 48, 32)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "fc1.weight": (96, 64), "bias1.bias": (96,), "fc2.weight": (32, 48), "bias2.bias": (32,)}
    assert m.act_name == "silu" and nsw.GatedMLP(64, act_layer=nn.GELU).act_name == "gelu"
    assert nsw.GatedMLP(64, act_layer=lambda: nn.GELU(approximate="tanh")).act_name == "gelu_tanh"
    assert float(m.bias1.bias.abs().max()) == 0 and 0.015 < float(m.fc1.weight.std()) < 0.025
    with pytest.raises(NotImplementedError, match="gates"):
        nsw.GatedMLP(64, act_layer=nn.ReLU).act_name
    with pytest.raises(NotImplementedError, match="dropout"):
        nsw.GatedMLP(64, 48, drop=0.1).train()(torch.zeros(1, 64))


def test_residual_norm_parameters():
    m = nsw.ResidualNorm(64, layer_scale=0.1)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "post_norm.norm.weight": (64,), "next_norm.norm.weight": (64,), "gamma": (64,)}
    assert torch.allclose(m.gamma, torch.full((64,), 0.1))
    assert not nsw.ResidualNorm(64, post_norm=False, next_norm=False).state_dict()
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="gate"):
        m(x, x, gate=torch.zeros(64))
    m.next_norm.norm.eps = 1e-3
    with pytest.raises(NotImplementedError, match="eps"):
        m(x, x)


def test_half_block_traces_into_one_graph():
    class Half(nn.Module):
        def __init__(self):
            super().__init__()
            self.norm, self.mlp = nsw.ResidualNorm(64, layer_scale=1.0), nsw.GatedMLP(64, 48)

        def forward(self, branch, skip):
            y, z = self.norm(branch, skip)
            return self.mlp(z, y)

    torch._dynamo.reset()
    graphs = []

    def capture(gm, _):
        graphs.append([n.target for n in gm.graph.nodes if n.op == "call_function" and "nsw" in str(n.target)])
        return lambda *a: (torch.zeros(3, 64),)

    with torch.no_grad():
        torch.compile(Half(), backend=capture, fullgraph=True)(torch.zeros(3, 64), torch.zeros(3, 64))
    torch._dynamo.reset()
    assert len(graphs) == 1
    assert [str(t).split(".")[-1] for t in graphs[0]] != []
    assert sum("gated_linear" in str(t) for t in graphs[0]) == 1 and sum("residual_norm" in str(t) for t in graphs[0]) == 1
