"""Gradients of the four window maps: permutations, so every value equals torch's own roll, view and permute."""
import pytest
import torch

import nsw  # noqa: F401

pytestmark = pytest.mark.gpu

MAPS = ["window_partition", "roll_window_partition", "window_reverse", "window_reverse_roll"]
# B, T, bands, across, window, shift, C
SIZES = [(2, 1, 2, 2, (3, 5), (1, 2), 8), (1, 2, 3, 2, (3, 5), (2, 0), 24), (3, 3, 1, 1, (4, 6), (0, 5), 8), (1, 1, 4, 1, (1, 7), (0, 3), 16),
         (2, 2, 2, 3, (9, 18), (4, 9), 192)]


def plain(name, x, B, T, H, W, ws, shift):
    """The map by torch operators: [B, T, H, W, C] -> [windows, T, ws0, ws1, C], or back."""
    n0, n1 = H // ws[0], W // ws[1]
    if "partition" in name:
        if "roll" in name:
            x = x.roll((-shift[0], -shift[1]), (2, 3))
        x = x.view(B, T, n0, ws[0], n1, ws[1], -1).permute(0, 2, 4, 1, 3, 5, 6)
        return x.reshape(B * n0 * n1, T, ws[0], ws[1], -1)
    x = x.view(B, n0, n1, T, ws[0], ws[1], -1).permute(0, 3, 1, 4, 2, 5, 6).reshape(B, T, H, W, -1)
    return x.roll(shift, (2, 3)) if "roll" in name else x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", MAPS)
@pytest.mark.parametrize("size", SIZES)
def test_gradient(device, dtype, name, size):
    B, T, bands, across, ws, shift, C = size
    H, W = bands * ws[0], across * ws[1]
    args = [list(ws)] if "partition" in name else [list(ws), [H, W]]
    if "roll" in name:
        args.append(list(shift))
    g = torch.Generator().manual_seed(50)
    shape = (B, T, H, W, C) if "partition" in name else (B * bands * across, T, *ws, C)
    x = torch.randn(shape, generator=g).to(dtype)
    xc = x.clone().requires_grad_()
    want = plain(name, xc, B, T, H, W, ws, shift)
    xd = x.to(device).requires_grad_()
    y = getattr(torch.ops.nsw, name)(xd, *args)
    assert torch.equal(y.detach().cpu(), want.detach())
    dy = torch.randn(want.shape, generator=g).to(dtype)
    for of in (lambda d: d, lambda d: d[..., :1].expand(d.shape), lambda d: d.transpose(2, 3).contiguous().transpose(2, 3)):
        xd.grad = xc.grad = None
        want.backward(of(dy), retain_graph=True)
        y.backward(of(dy.to(device)), retain_graph=True)
        assert torch.equal(xd.grad.cpu(), xc.grad)
