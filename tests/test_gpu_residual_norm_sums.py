"""Gradients of nsw.ops.residual_norm's parameters over more than 2^32 bytes a tensor,
from float64 sums over all rows."""
import pytest
import torch

from nsw import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def test_parameter_sums_past_32_bit_offsets(device):
    """dy, dz and the branch alike, so that the sums' terms have one sign: a workgroup's rows (1075 of 1,100,001) left out or
    counted twice are 1e-3 of a sum.  Bounds: a term's error as in test_gpu_residual_norm (160 u through the gradient, 80 u
    through z), a chain of 1075 rows, one of 4 workgroups and a tree of 40: less than 1200 u of the magnitudes, 8e-5 in all."""
    rows, C = 1_100_001, 1024
    g = torch.Generator(device=device).manual_seed(6)
    branch = torch.empty(rows, C, device=device).normal_(0, 1, generator=g)
    skip = branch.flip(0)
    dy = branch.abs().mul_(branch.sign())
    w = torch.linspace(0.5, 1.5, C, device=device)
    _, _, dp, _, dn = ops.residual_norm_backward(dy, branch, branch, skip, post_weight=w, norm_weight=w, eps=1e-5)
    w64 = w.double()
    sums = [torch.zeros(C, dtype=torch.float64, device=device) for _ in range(4)]
    for i in range(0, rows, 50_000):
        o, x, d = (t[i:i + 50_000].double() for t in (branch, skip, dy))
        oh = o * (o.pow(2).mean(1, True) + 1e-5).rsqrt()
        y, my = x + w64 * oh, x.abs() + (w64 * oh).abs()
        ry = (y.pow(2).mean(1, True) + 1e-5).rsqrt()
        yh, myh, tt = y * ry, my * ry, o * w64
        dd = d + ry * (tt - yh * (tt * yh).mean(1, True))
        md = d.abs() + ry * (tt.abs() + myh * (tt.abs() * myh).mean(1, True))
        for s, v in zip(sums, (dd * oh, md * oh.abs(), o * yh, o.abs() * myh)):
            s += v.sum(0)
    for got, want, mag, own in ((dp, sums[0], sums[1], 160), (dn, sums[2], sums[3], 80)):
        assert (want > 0.2 * mag).all()                       # one sign: what is left out shows
        over = (got.double() - want).abs() - mag * (1200 + own) * U - want.abs() * U
        assert (over <= 0).all(), over.max().item()
