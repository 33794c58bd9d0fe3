"""nsw.ops.position_attention with more windows than workgroups share a head: what a workgroup keeps from one window
to the next (the sums of dz for the table, biases, buffers) and what it must not, against the formula in float64.
Tolerances: test_gpu_position_attention's."""
import math

import pytest
import torch

import nsw
from nsw import _lib, ops

from test_gpu_position_attention import case, check, reference, run

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def turns(t):
    """Whether a workgroup of the backward pass takes several windows: its sums of dz are [heads, parts, L, L]."""
    Bw, L, C3 = t["qkv"].shape
    n = _lib.lib().nsw_position_attention_backward_workspace_size(Bw, L, C3 // 3, t["heads"], *t["extent"], ops.dtype_code(t["qkv"]))
    return 0 < n < 4 * t["heads"] * Bw * L * L


def check_two_heads(t, got, dtype, mask=None):
    """The first head and the last against float64: heads have nothing in common."""
    heads = t["heads"]
    picked = [0, heads - 1]
    rows = lambda x, parts: x.unflatten(-1, (parts, heads, -1))[:, :, :, picked].flatten(-3)
    few = dict(t, heads=2, qkv=rows(t["qkv"], 3), do=rows(t["do"], 1), table=t["table"][:, picked])
    check({"o": rows(got["o"], 1), "dqkv": rows(got["dqkv"], 3), "dtable": got["dtable"][:, picked]}, reference(few, mask), dtype)


# windows in a workgroup of 4, 8 and 12 waves, k and v in one buffer and in two; longer ones (from 65 tokens on with
# 512-byte rows, 129 with 256-byte rows, 193 otherwise)
CASES = [
    (BF16, 40, (1, 5, 6), 64, 16), (F32, 40, (1, 5, 6), 64, 16), (F32, 70, (1, 7, 7), 32, 128), (BF16, 70, (1, 3, 5), 32, 128),
    (BF16, 35, (1, 8, 16), 32, 64), (F32, 35, (1, 8, 16), 32, 64), (BF16, 35, (1, 8, 16), 32, 128), (F32, 35, (1, 8, 15), 32, 32),
    (BF16, 20, (1, 9, 18), 32, 64), (F32, 20, (1, 9, 18), 32, 32), (BF16, 20, (1, 12, 16), 32, 16), (F32, 20, (1, 12, 16), 32, 32),
    (BF16, 20, (2, 9, 18), 16, 64), (F32, 12, (2, 9, 18), 16, 64), (F32, 14, (2, 9, 18), 16, 32), (BF16, 16, (1, 1, 259), 16, 128),
    (F32, 12, (1, 9, 18), 32, 128), (BF16, 16, (1, 9, 18), 32, 128),
]


@pytest.mark.parametrize("dtype,Bw,extent,heads,hd", CASES)
def test_windows_in_turn(device, dtype, Bw, extent, heads, hd):
    t = case(dtype, Bw, extent, heads, hd, seed=30)
    assert turns(t)
    check_two_heads(t, run(t, device), dtype)


@pytest.mark.parametrize("dtype,Bw,extent,heads,hd", CASES)
def test_masks_in_turn(device, dtype, Bw, extent, heads, hd):
    """A mask of its own for each window, some rows of them empty."""
    t = case(dtype, Bw, extent, heads, hd, seed=31)
    assert turns(t)
    L = math.prod(extent)
    g = torch.Generator().manual_seed(32)
    m = torch.randn(Bw, L, L, generator=g)
    m[torch.rand(Bw, L, L, generator=g) < 0.3] = -math.inf
    m[::3, L // 2] = -math.inf
    m[1] = -math.inf
    check_two_heads(t, run(t, device, mask=m), dtype, m)


@pytest.mark.parametrize("dtype,Bw,extent,heads,hd", [c for c in CASES if c[2][1] > 1])
def test_shifts_in_turn(device, dtype, Bw, extent, heads, hd):
    """Windows inside an image and of its last band in one workgroup."""
    T, A, W = extent
    bands, across = 3, 2
    Bw = (Bw + 5) // 6 * 6
    t = case(dtype, Bw, extent, heads, hd, seed=33)
    assert turns(t)
    H, Wi, shift = bands * A, across * W, (A // 2, W // 2)
    m = nsw.swin_helpers.attention_mask_closed_form(H, Wi, (A, W), shift, T)
    check_two_heads(t, run(t, device, geometry=(H, Wi, (A, W), shift, T)), dtype, m)
