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
