"""Which gradients torch.ops.nsw.linear and the modules on it give, without a GPU
(meta tensors): all of those that are asked for, or an error, never some of them."""
import pytest
import torch

import nsw
from nsw import torch_ops


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, device="meta", dtype=dtype)


def test_attention_gives_no_partial_gradients():
    m = nsw.WindowMultiHeadAttention(64, 2, (3, 4)).to(device="meta", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="linear_forward"):
        m(meta(2, 12, 64)).sum().backward()
    assert all(p.grad is None for p in m.parameters())
    for p in m.parameters():
        p.requires_grad_(False)
    m.k_norm.norm.weight.requires_grad_()
    m.proj.weight.requires_grad_()
    with pytest.raises(RuntimeError, match="linear_forward"):
        m(meta(2, 12, 64)).sum().backward()
    with torch.no_grad():
        assert m(meta(2, 12, 64)).shape == (2, 12, 64)


def test_attention_trains_what_it_can_train_whole():
    m = nsw.WindowMultiHeadAttention(64, 2, (3, 4)).to(device="meta", dtype=torch.bfloat16)
    for n, p in m.named_parameters():
        p.requires_grad_(n.startswith(("proj", "biasproj")))
    m(meta(2, 12, 64)).sum().backward()
    assert {n for n, p in m.named_parameters() if p.grad is not None} == {"proj.weight", "biasproj.bias"}
    x = meta(2, 12, 64).requires_grad_()          # the gradient of x passes through attention, which has none
    with pytest.raises((RuntimeError, NotImplementedError)):
        m(x).sum().backward()


def test_patch_embedding_gives_no_partial_gradients():
    c = nsw.PatchEmbedLayer(4, 3, 32, [8], [16]).to(device="meta", dtype=torch.bfloat16)
    x, r = meta(1, 1, 3, 8, 16, dtype=torch.float32), meta(8, 32).requires_grad_()
    with pytest.raises(RuntimeError, match="linear_forward"):
        c.tokens(x, residual=r).sum().backward()
    assert r.grad is None
    for p in c.parameters():
        p.requires_grad_(False)
    c.tokens(x, residual=r).sum().backward()
    assert r.grad.shape == r.shape


@pytest.mark.parametrize("epilogue,wants", [(0, "bias"), (0, "residual"), (1, "residual"), (None, "residual")])
def test_no_gradient_of_what_the_epilogue_left_out(epilogue, wants):
    x, w = meta(5, 64).requires_grad_(), meta(96, 64)
    b, r = meta(96), meta(5, 96)
    (b if wants == "bias" else r).requires_grad_()
    y = torch_ops.linear_epi(x, w, None if epilogue is None else b, r, epilogue)
    with pytest.raises(ValueError, match=wants):
        y.sum().backward()
    b, r = b.detach(), r.detach()                  # present, but asked for nothing: x has its gradient
    g, = torch.autograd.grad(torch_ops.linear_epi(x, w, None if epilogue is None else b, r, epilogue), x, meta(5, 96))
    assert g.shape == x.shape


def kept(f):
    """Shapes of what autograd keeps for a backward pass through f."""
    shapes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: shapes.append(tuple(t.shape)) or t, lambda t: t):
        y = f()
    assert y.requires_grad
    return shapes


def test_linear_keeps_only_what_a_gradient_reads():
    x, w, b = meta(7, 64), meta(96, 64), meta(96)
    assert (7, 64) in kept(lambda: torch_ops.linear_epi(x, w.requires_grad_(), b))
    w = w.detach()
    assert (7, 64) not in kept(lambda: torch_ops.linear_epi(x.requires_grad_(), w, b))
    g, = torch.autograd.grad(torch_ops.linear_epi(x, w, b), x, meta(7, 96))
    assert g.shape == (7, 64)
    x, b = x.detach(), b.requires_grad_()
    assert (7, 64) not in kept(lambda: torch_ops.linear_epi(x, w, b))
    g, = torch.autograd.grad(torch_ops.linear_epi(x, w, b), b, meta(7, 96))
    assert g.shape == (96,)


def test_gelu_mlp_keeps_no_hidden_rows():
    m = nsw.MLP(64, 256).to(device="meta", dtype=torch.bfloat16)
    for r in (None, meta(7, 64)):
        assert (7, 256) not in kept(lambda: m(meta(7, 64), r))
        with pytest.raises(NotImplementedError):
            m(meta(7, 64), r).sum().backward()
    assert all(p.grad is None for p in m.parameters())
    for p in (m.fc1.weight, m.bias1.bias):
        p.requires_grad_(False)
    m(meta(7, 64)).sum().backward()               # what follows the frozen half
    assert m.fc2.weight.grad.shape == (64, 256) and m.bias2.bias.grad.shape == (64,)


def test_linear_backward_without_x():
    dy, x, w = meta(2, 3, 96), meta(2, 3, 64), meta(96, 64)
    dx, dw, db = torch.ops.nsw.linear_backward(dy, None, w, [True, False, True])
    assert dx.shape == x.shape and dw.shape == (0,) and db.shape == (96,)
