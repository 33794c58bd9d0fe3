"""Gradients of torch.ops.nsw.linear where some operands are frozen: the bits of
those with everything trained."""
import pytest
import torch

import nsw
from nsw import ops, torch_ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", [(3, 96, 64), (300, 1024, 256), (1000, 64, 512)])
def test_frozen_operands(device, dtype, M, N, K):
    g = torch.Generator().manual_seed(M)
    r = lambda *s: torch.randn(*s, generator=g).to(device=device, dtype=dtype)
    t = {"x": r(M, K), "w": r(N, K) * K ** -0.5, "b": r(N), "r": r(M, N)}
    dy = r(M, N)

    def grads(names):
        a = {n: v.clone().requires_grad_(n in names) for n, v in t.items()}
        y = torch_ops.linear_epi(a["x"], a["w"], a["b"], a["r"])
        return dict(zip(names, torch.autograd.grad(y, [a[n] for n in names], dy)))

    full = grads("xwbr")
    assert torch.equal(full["r"], dy)
    for names in ("x", "w", "b", "r", "xb", "wr"):
        for n, v in grads(names).items():
            assert torch.equal(v, full[n]), (names, n)
    dx, dw, db = ops.linear_backward(dy, None, t["w"], needs=(True, False, True))
    assert dw is None and torch.equal(dx, full["x"]) and torch.equal(db, full["b"])
    with pytest.raises(ValueError, match="dweight"):
        ops.linear_backward(dy, None, t["w"])


def test_gelu_mlp_behind_frozen_parameters(device):
    """With fc1 frozen the second product's gradients are whole; h is what fc1 gives."""
    torch.manual_seed(0)
    m = nsw.MLP(64, 128).to(device=device, dtype=F32)
    x, dy = torch.randn(50, 64, device=device), torch.randn(50, 64, device=device)
    with pytest.raises(NotImplementedError):
        m(x).backward(dy)
    for p in (m.fc1.weight, m.bias1.bias):
        p.requires_grad_(False)
    m(x).backward(dy)
    h = torch_ops.linear_epi(x, m.fc1.weight, m.bias1.bias, epilogue=m.gelu_epilogue)
    _, dw, db = ops.linear_backward(dy, h, m.fc2.weight.detach(), needs=(False, True, True))
    assert torch.equal(m.fc2.weight.grad, dw) and torch.equal(m.bias2.bias.grad, db)
