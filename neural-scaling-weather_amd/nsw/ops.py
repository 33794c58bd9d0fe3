"""Tensor-level wrappers of the libnsw C ABI.

Every op takes / returns torch tensors on the GPU, enqueues HIP kernels on
torch's current stream and allocates its outputs with torch (plumbing only:
all arithmetic runs in libnsw's kernels).  Inputs must be contiguous,
16-byte aligned, fp32 or bf16, on a HIP device; anything else raises.
"""
from __future__ import annotations

import functools
import threading
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from ._lib import check, lib

_DTYPES = {torch.float32: _lib.NSW_DTYPE_F32, torch.bfloat16: _lib.NSW_DTYPE_BF16}


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"libnsw supports float32 and bfloat16 tensors, got {t.dtype}") from None


def _dev(*ts: Optional[torch.Tensor]) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("libnsw ops run on the GPU only; got a tensor on " + str(t.device))
        if not t.is_contiguous():
            raise RuntimeError("libnsw ops need contiguous tensors")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError("libnsw op arguments are on different devices")
    return dev


def _same_dtype(ref: torch.Tensor, *ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and t.dtype != ref.dtype:
            raise TypeError(f"dtype mismatch: {t.dtype} vs {ref.dtype}")


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


# the current stream's handle without a Stream object around it (0.1 us, not 1.9), and
# the current device's index without the check that the GPU is initialised
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_index = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _stream(dev: torch.device):
    if dev.index is not None:
        return _raw_stream(dev.index)
    return torch.cuda.current_stream(dev).cuda_stream


def default_eps(dtype: torch.dtype) -> float:
    """nn.RMSNorm(eps=None) uses finfo(input dtype).eps."""
    return float(torch.finfo(dtype).eps)


# ------------------------------------------------------------------ index ---

def roll_hw(x: torch.Tensor, shifts: Tuple[int, int]) -> torch.Tensor:
    """torch.roll(x, shifts, dims=(-3, -2)) of a [B,T,H,W,C] tensor."""
    B, T, H, W, C = x.shape
    dev = _dev(x)
    y = torch.empty_like(x)
    check(lib().nsw_roll_hw(x.data_ptr(), y.data_ptr(), B, T, H, W, C, int(shifts[0]), int(shifts[1]),
                            dtype_code(x), _stream(dev)), "roll_hw")
    return y


def window_partition(x: torch.Tensor, window_size: Tuple[int, int]) -> torch.Tensor:
    B, T, H, W, C = x.shape
    ws0, ws1 = window_size
    if H % ws0 or W % ws1:
        raise ValueError(f"image {H}x{W} is not divisible by window {window_size}")
    dev = _dev(x)
    out = torch.empty((B * (H // ws0) * (W // ws1), T, ws0, ws1, C), dtype=x.dtype, device=dev)
    check(lib().nsw_window_partition(x.data_ptr(), out.data_ptr(), B, T, H, W, C, ws0, ws1,
                                     dtype_code(x), _stream(dev)), "window_partition")
    return out


def window_reverse(windows: torch.Tensor, window_size: Tuple[int, int],
                   img_size: Tuple[int, int]) -> torch.Tensor:
    H, W = img_size
    ws0, ws1 = window_size
    T, C = windows.shape[1], windows.shape[-1]
    nw = (H // ws0) * (W // ws1)
    if windows.shape[0] % nw:
        raise ValueError("number of windows is not a multiple of the image's windows")
    B = windows.shape[0] // nw
    dev = _dev(windows)
    out = torch.empty((B, T, H, W, C), dtype=windows.dtype, device=dev)
    check(lib().nsw_window_reverse(windows.data_ptr(), out.data_ptr(), B, T, H, W, C, ws0, ws1,
                                   dtype_code(windows), _stream(dev)), "window_reverse")
    return out


def roll_window_partition(x: torch.Tensor, window_size, shift_size) -> torch.Tensor:
    """window_partition(torch.roll(x, -shift, (H, W)), window_size) in one pass."""
    B, T, H, W, C = x.shape
    ws0, ws1 = window_size
    dev = _dev(x)
    out = torch.empty((B * (H // ws0) * (W // ws1), T, ws0, ws1, C), dtype=x.dtype, device=dev)
    check(lib().nsw_roll_window_partition(x.data_ptr(), out.data_ptr(), B, T, H, W, C, ws0, ws1,
                                          int(shift_size[0]), int(shift_size[1]), dtype_code(x),
                                          _stream(dev)), "roll_window_partition")
    return out


def window_reverse_roll(windows: torch.Tensor, window_size, img_size, shift_size) -> torch.Tensor:
    """torch.roll(window_reverse(windows), +shift, (H, W)) in one pass."""
    H, W = img_size
    ws0, ws1 = window_size
    T, C = windows.shape[1], windows.shape[-1]
    B = windows.shape[0] // ((H // ws0) * (W // ws1))
    dev = _dev(windows)
    out = torch.empty((B, T, H, W, C), dtype=windows.dtype, device=dev)
    check(lib().nsw_window_reverse_roll(windows.data_ptr(), out.data_ptr(), B, T, H, W, C, ws0, ws1,
                                        int(shift_size[0]), int(shift_size[1]), dtype_code(windows),
                                        _stream(dev)), "window_reverse_roll")
    return out


def make_attention_mask(H: int, W: int, window_size: Tuple[int, int], shift_size: Tuple[int, int],
                        T: int, device) -> torch.Tensor:
    ws0, ws1 = window_size
    nW = (H // ws0) * (W // ws1)
    L = T * ws0 * ws1
    m = torch.empty((nW, L, L), dtype=torch.float32, device=device)
    check(lib().nsw_make_attention_mask(m.data_ptr(), H, W, ws0, ws1, int(shift_size[0]),
                                        int(shift_size[1]), T, _stream(m.device)), "make_attention_mask")
    return m


# ------------------------------------------------------------------- norms ---

def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: Optional[float] = None) -> torch.Tensor:
    dev = _dev(x, weight)
    _same_dtype(x, weight)
    C = x.shape[-1]
    if weight.numel() != C:
        raise ValueError(f"norm weight has {weight.numel()} elements, input has {C} features")
    eps = default_eps(x.dtype) if eps is None else float(eps)
    y = torch.empty_like(x)
    check(lib().nsw_rmsnorm(x.data_ptr(), weight.data_ptr(), eps, y.data_ptr(), x.numel() // C, C,
                            dtype_code(x), _stream(dev)), "rms_norm")
    return y


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
               eps: float = 1e-5) -> torch.Tensor:
    """nn.LayerNorm over the last dim (biased variance); weight / bias may be
    None (elementwise_affine=False)."""
    dev = _dev(x, weight, bias)
    _same_dtype(x, weight, bias)
    C = x.shape[-1]
    for t in (weight, bias):
        if t is not None and t.numel() != C:
            raise ValueError(f"layer-norm parameter has {t.numel()} elements, input has {C} features")
    y = torch.empty_like(x)
    check(lib().nsw_layernorm(x.data_ptr(), _p(weight), _p(bias), float(eps), y.data_ptr(), x.numel() // C, C,
                              dtype_code(x), _stream(dev)), "layer_norm")
    return y


def rmsnorm_roll_partition(x: torch.Tensor, weight: torch.Tensor, window_size, shift_size,
                           eps: Optional[float] = None) -> torch.Tensor:
    """norm1 + roll by -shift + window_partition, as [B*nW, T*wa, C]."""
    B, T, H, W, C = x.shape
    dev = _dev(x, weight)
    _same_dtype(x, weight)
    eps = default_eps(x.dtype) if eps is None else float(eps)
    ws0, ws1 = window_size
    out = torch.empty((B * (H // ws0) * (W // ws1), T * ws0 * ws1, C), dtype=x.dtype, device=dev)
    check(lib().nsw_rmsnorm_roll_partition(x.data_ptr(), weight.data_ptr(), eps, out.data_ptr(), B, T, H, W,
                                           C, ws0, ws1, int(shift_size[0]), int(shift_size[1]),
                                           dtype_code(x), _stream(dev)), "rmsnorm_roll_partition")
    return out


def _at(*ts: Optional[torch.Tensor]) -> int:
    """Index of the device of ts (the first is given) after the checks of _dev, which raises what is found."""
    at = ts[0].get_device()
    for t in ts:
        if t is not None and (t.get_device() != at or not t.is_contiguous()):
            break
    else:
        if at >= 0:
            return at
    _dev(*ts)
    return at


def _uniform(*ts: Optional[torch.Tensor]) -> int:
    """_at of ts after _same_dtype, too."""
    at, dt = ts[0].get_device(), ts[0].dtype
    for t in ts:
        if t is not None and (t.dtype is not dt or t.get_device() != at or not t.is_contiguous()):
            break
    else:
        if at >= 0:
            return at
    _dev(*ts)
    _same_dtype(ts[0], *ts)
    return at


def _run(what: str, at: int, fn, *args) -> None:
    """fn(*args, stream) with device ``at`` as the current one, its error raised."""
    if _current_index() == at:
        rc = fn(*args, _raw_stream(at))
    else:
        with torch.cuda.device(at):
            rc = fn(*args, _raw_stream(at))
    if rc:
        check(rc, what)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(handle, name, *sizes) -> int:
    """The library's answer for these sizes (0.2 us, not up to 3)."""
    return int(getattr(handle, name)(*sizes))


def _residual_norm_args(what, branch, skip, post_weight, gate, norm_weight, eps):
    """(device index, rows, C, G, eps) of a residual_norm, its arguments checked."""
    at = _uniform(branch, skip, post_weight, gate, norm_weight)
    shape = branch.shape
    if not shape or shape != skip.shape:
        raise ValueError(f"{what}: branch {tuple(branch.shape)} and skip {tuple(skip.shape)} must have one shape")
    C = shape[-1]
    if C == 0:
        raise ValueError(f"{what}: no features")
    rows = branch.numel() // C
    if post_weight is not None and post_weight.shape != (C,):
        raise ValueError(f"{what}: post_weight has shape {tuple(post_weight.shape)}, expected ({C},)")
    if norm_weight is not None and norm_weight.shape != (C,):
        raise ValueError(f"{what}: norm_weight has shape {tuple(norm_weight.shape)}, expected ({C},)")
    G = 1
    if gate is not None:
        if gate.dim() not in (1, 2) or gate.shape[-1] != C or gate.numel() == 0:
            raise ValueError(f"{what}: gate has shape {tuple(gate.shape)}, expected ({C},) or (G, {C})")
        G = gate.numel() // C
        if rows % G:
            raise ValueError(f"{what}: {rows} rows are not a multiple of the gate's {G}")
    return at, rows, C, G, default_eps(branch.dtype) if eps is None else float(eps)


def residual_norm(branch: torch.Tensor, skip: torch.Tensor, post_weight: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, alpha: float = 1.0,
                  norm_weight: Optional[torch.Tensor] = None, eps: Optional[float] = None
                  ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(y, z): y = alpha * skip + gate * RMSNorm(branch; post_weight) and
    z = RMSNorm(y; norm_weight), the end of one residual branch and the norm
    before the next, in one pass.  branch and skip [..., C]; post_weight None:
    the branch is not normalised; gate [C] (a layer scale) or [G, C], the rows
    of G equal parts of the batch each under their own gate, None: 1;
    norm_weight None: z is None.  Statistics, and z's y, in fp32."""
    at, rows, C, G, eps = _residual_norm_args("residual_norm", branch, skip, post_weight, gate, norm_weight, eps)
    y = torch.empty_like(branch)
    z = None if norm_weight is None else torch.empty_like(branch)
    _run("residual_norm", at, lib().nsw_residual_norm, branch.data_ptr(), skip.data_ptr(), _p(post_weight), _p(gate),
         _p(norm_weight), y.data_ptr(), _p(z), rows, C, G, float(alpha), eps, dtype_code(branch))
    return y, z


def residual_norm_backward(dy: Optional[torch.Tensor], dz: Optional[torch.Tensor], branch: torch.Tensor,
                           skip: torch.Tensor, post_weight: Optional[torch.Tensor] = None,
                           gate: Optional[torch.Tensor] = None, alpha: float = 1.0,
                           norm_weight: Optional[torch.Tensor] = None, eps: Optional[float] = None):
    """(dbranch, dskip, dpost_weight, dgate, dnorm_weight) of residual_norm from
    the gradients of y and z, None for what was None.  dy or dz may be None
    (zero)."""
    what = "residual_norm_backward"
    at, rows, C, G, eps = _residual_norm_args(what, branch, skip, post_weight, gate, norm_weight, eps)
    if dy is None and dz is None:
        raise ValueError(f"{what}: dy or dz is required")
    if dz is not None and norm_weight is None:
        raise ValueError(f"{what}: dz without norm_weight")
    _uniform(branch, dy, dz)
    for t in (dy, dz):
        if t is not None and t.shape != branch.shape:
            raise ValueError(f"{what}: gradient of shape {tuple(t.shape)}, expected {tuple(branch.shape)}")
    db, ds = torch.empty_like(branch), torch.empty_like(branch)
    dp = None if post_weight is None else torch.empty_like(post_weight)
    dg = None if gate is None else torch.empty_like(gate)
    # without dz the norm before the next branch has no part in the gradients
    dn = None if norm_weight is None else torch.zeros_like(norm_weight) if dz is None else torch.empty_like(norm_weight)
    nw = None if dz is None else norm_weight
    code = dtype_code(branch)
    nbytes = _workspace_bytes(lib(), "nsw_residual_norm_backward_workspace_size", rows, C, G, code)
    ws = branch.new_empty(max(nbytes, 16), dtype=torch.uint8)
    _run(what, at, lib().nsw_residual_norm_backward, _p(dy), _p(dz), branch.data_ptr(), skip.data_ptr(),
         _p(post_weight), _p(gate), _p(nw), db.data_ptr(), ds.data_ptr(), _p(dp), _p(dg), None if dz is None else _p(dn),
         rows, C, G, float(alpha), eps, code, ws.data_ptr(), nbytes)
    return db, ds, dp, dg, dn


_NORM_ACTS = {"none": _lib.NSW_ACT_NONE, "silu": _lib.NSW_ACT_SILU, "gelu": _lib.NSW_ACT_GELU,
              "gelu_tanh": _lib.NSW_ACT_GELU_TANH}


def _group_norm_args(what, x, groups, weight, bias, act):
    """(device index, B, R, C, act code) of a group norm, its arguments checked."""
    at = _uniform(x, weight, bias)
    if act not in _NORM_ACTS:
        raise ValueError(f"{what}: act must be one of {sorted(_NORM_ACTS)}, got {act!r}")
    shape = x.shape
    if len(shape) < 2:
        raise ValueError(f"{what}: x has shape {tuple(shape)}, expected [B, ..., C]")
    B, C = shape[0], shape[-1]
    if C == 0 or groups < 1 or C % groups:
        raise ValueError(f"{what}: {C} channels are not a multiple of {groups} groups")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != (C,):
            raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected ({C},)")
    return at, B, x.numel() // (B * C) if B else 0, C, _NORM_ACTS[act]


def group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               act: str = "none", eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, stats): y = act(GroupNorm(x) * weight + bias) of x [B, ..., C], channels
    last, the mean and variance over a sample's rows and a group's channels; act "none",
    "silu", "gelu" (exact erf) or "gelu_tanh".  stats [B, groups, 2] fp32: mean and
    1 / sqrt(var + eps), for group_norm_backward (zeros where a sample has no rows)."""
    at, B, R, C, code = _group_norm_args("group_norm", x, groups, weight, bias, act)
    y = torch.empty_like(x)
    if B == 0 or R == 0:
        return y, x.new_zeros((B, groups, 2), dtype=torch.float32)
    dt = dtype_code(x)
    stats = x.new_empty((B, groups, 2), dtype=torch.float32)
    nbytes = _workspace_bytes(lib(), "nsw_group_norm_workspace_size", B, R, C, groups, dt)
    ws = x.new_empty(max(nbytes, 16), dtype=torch.uint8)
    _run("group_norm", at, lib().nsw_group_norm, x.data_ptr(), _p(weight), _p(bias), y.data_ptr(), stats.data_ptr(), B, R, C,
         groups, float(eps), code, dt, ws.data_ptr(), nbytes)
    return y, stats


def group_norm_backward(dy: torch.Tensor, x: torch.Tensor, stats: torch.Tensor, groups: int,
                        weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, act: str = "none",
                        needs: Sequence[bool] = (True, True, True)):
    """(dx, dweight, dbias) of group_norm from the gradient of y and the forward
    pass's stats, None where ``needs`` says so or there is no such parameter."""
    what = "group_norm_backward"
    at, B, R, C, code = _group_norm_args(what, x, groups, weight, bias, act)
    _uniform(x, dy)
    if dy.shape != x.shape:
        raise ValueError(f"{what}: dy has shape {tuple(dy.shape)}, expected {tuple(x.shape)}")
    _dev(x, stats)
    if stats.dtype != torch.float32 or stats.shape != (B, groups, 2):
        raise ValueError(f"{what}: stats is {stats.dtype} {tuple(stats.shape)}, expected float32 {(B, groups, 2)}")
    dx, dw, db = _grads(needs, x, weight, bias)
    if B == 0 or R == 0:
        return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_()
    dt = dtype_code(x)
    nbytes = _workspace_bytes(lib(), "nsw_group_norm_backward_workspace_size", B, R, C, groups, dt)
    ws = x.new_empty(max(nbytes, 16), dtype=torch.uint8)
    _run(what, at, lib().nsw_group_norm_backward, dy.data_ptr(), x.data_ptr(), stats.data_ptr(), _p(weight), _p(bias),
         _p(dx), _p(dw), _p(db), B, R, C, groups, code, dt, ws.data_ptr(), nbytes)
    return dx, dw, db


# -------------------------------------------------------------------- GEMM ---

def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           residual: Optional[torch.Tensor] = None, epilogue: Optional[int] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = epi(x . weight^T): F.linear with an optional fused bias / GELU / residual.
    An epilogue leaves out what it has no part for (a residual without a bias: NSW_EPI_NONE).
    ``out`` (contiguous, x.shape[:-1] + (N,), x's dtype) receives y if given."""
    at = _uniform(x, weight, bias, residual, out)
    K = x.shape[-1]
    N, Kw = weight.shape
    if Kw != K:
        raise ValueError(f"linear: x has {K} features, weight expects {Kw}")
    if bias is not None and bias.numel() != N:
        raise ValueError(f"linear: bias has {bias.numel()} elements, expected {N}")
    M = x.numel() // K
    if epilogue is None:
        epilogue = _lib.NSW_EPI_NONE if bias is None else (
            _lib.NSW_EPI_BIAS if residual is None else _lib.NSW_EPI_BIAS_RESIDUAL)
    if out is not None:
        if out.numel() != M * N:
            raise ValueError(f"linear: out has {out.numel()} elements, expected {M * N}")
        y = out.view(x.shape[:-1] + (N,))
    else:
        y = x.new_empty(x.shape[:-1] + (N,))
    if residual is not None and residual.shape != y.shape:
        raise ValueError(f"residual shape {tuple(residual.shape)} != output {tuple(y.shape)}")
    if M == 0:
        return y
    _run("linear", at, lib().nsw_linear, x.data_ptr(), weight.data_ptr(), _p(bias), _p(residual), y.data_ptr(), M, N, K,
         int(epilogue), dtype_code(x))
    return y


_ACTS = {"silu": _lib.NSW_ACT_SILU, "gelu": _lib.NSW_ACT_GELU, "gelu_tanh": _lib.NSW_ACT_GELU_TANH}


def _gated_args(what, x, weight, bias, act):
    """(device index, M, H, K, act code) of a gated linear, its arguments checked."""
    at = _uniform(x, weight, bias)
    if act not in _ACTS:
        raise ValueError(f"{what}: act must be one of {sorted(_ACTS)}, got {act!r}")
    shape, wshape = x.shape, weight.shape
    if not shape or len(wshape) != 2 or wshape[1] != shape[-1] or wshape[0] % 2:
        raise ValueError(f"{what}: x {tuple(x.shape)} and weight {tuple(weight.shape)}, expected [..., K] and [2H, K]")
    K, H = wshape[1], wshape[0] // 2
    if K == 0 or H == 0:
        raise ValueError(f"{what}: no features")
    if bias is not None and bias.shape != (2 * H,):
        raise ValueError(f"{what}: bias has shape {tuple(bias.shape)}, expected ({2 * H},)")
    return at, x.numel() // K, H, K, _ACTS[act]


def gated_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 act: str = "silu") -> torch.Tensor:
    """h [..., H] = act(x Wg^T + bg) * (x Wu^T + bu), both projections, the
    activation and the product of a gated feed-forward block in one kernel.
    weight [2H, K] stacks Wg over Wu, bias [2H] bg over bu; act "silu",
    "gelu" (exact erf) or "gelu_tanh"."""
    at, M, H, K, code = _gated_args("gated_linear", x, weight, bias, act)
    h = x.new_empty(x.shape[:-1] + (H,))
    if M == 0:
        return h
    _run("gated_linear", at, lib().nsw_gated_linear, x.data_ptr(), weight.data_ptr(), _p(bias), h.data_ptr(), M, H, K,
         code, dtype_code(x))
    return h


def _grads(needs, *ts):
    """Empty gradients of the tensors that are given and asked for."""
    return [torch.empty_like(t) if n and t is not None else None for n, t in zip(needs, ts)]


def gated_linear_backward(dh: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                          bias: Optional[torch.Tensor] = None, act: str = "silu",
                          needs: Sequence[bool] = (True, True, True)):
    """(dx, dweight, dbias) of gated_linear from the gradient of h, None where
    ``needs`` says so or there is no bias.  The projections are formed again
    from x and weight; their gradients are rounded to x's dtype before the
    products that give dx and dweight."""
    what = "gated_linear_backward"
    at, M, H, K, code = _gated_args(what, x, weight, bias, act)
    _uniform(x, dh)
    if dh.shape != x.shape[:-1] + (H,):
        raise ValueError(f"{what}: dh has shape {tuple(dh.shape)}, expected {tuple(x.shape[:-1]) + (H,)}")
    dx, dw, db = _grads(needs, x, weight, bias)
    if M == 0:
        return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_()
    nbytes = _workspace_bytes(lib(), "nsw_gated_linear_backward_workspace_size", M, H, K, dtype_code(x))
    ws = x.new_empty(max(nbytes, 16), dtype=torch.uint8)
    _run(what, at, lib().nsw_gated_linear_backward, dh.data_ptr(), x.data_ptr(), weight.data_ptr(), _p(bias), _p(dx),
         _p(dw), _p(db), M, H, K, code, dtype_code(x), ws.data_ptr(), nbytes)
    return dx, dw, db


def linear_backward(dy: torch.Tensor, x: Optional[torch.Tensor], weight: torch.Tensor,
                    needs: Sequence[bool] = (True, True, True)):
    """(dx, dweight, dbias) = (dy W, dy^T x, column sums of dy) of linear without
    an activation, None where ``needs`` says so.  x may be None where dweight is
    not needed.  N a multiple of 8 as linear's: the kernel's contraction of dx goes
    in steps of 32 (bf16) / 16 (fp32), other N through copies with columns of zeros."""
    what = "linear_backward"
    at = _uniform(dy, x, weight)
    if x is None and needs[1]:
        raise ValueError(f"{what}: dweight needs x")
    shape = dy.shape[:-1] + weight.shape[1:]                # of x
    if dy.dim() < 1 or weight.dim() != 2 or dy.shape[-1] != weight.shape[0] or (x is not None and x.shape != shape):
        raise ValueError(f"{what}: dy {tuple(dy.shape)}, x {None if x is None else tuple(x.shape)} and weight "
                         f"{tuple(weight.shape)} do not match")
    N, K = weight.shape
    if K == 0 or N == 0:
        raise ValueError(f"{what}: no features")
    M = dy.numel() // N
    Np = N
    if N % 8 == 0 and N % (16 if dy.dtype == torch.float32 else 32):
        Np = (N + 31) // 32 * 32
        dy = torch.nn.functional.pad(dy, (0, Np - N))
        if needs[0]:                                        # dw and db do not read it
            weight = torch.nn.functional.pad(weight, (0, 0, 0, Np - N))
    dx = dy.new_empty(shape) if needs[0] else None
    dw = dy.new_empty(Np, K) if needs[1] else None
    db = dy.new_empty(Np) if needs[2] else None
    if M == 0:
        dw, db = (None if t is None else t.zero_() for t in (dw, db))
    else:
        nbytes = _workspace_bytes(lib(), "nsw_linear_backward_workspace_size", M, Np, K, dtype_code(dy))
        ws = dy.new_empty(max(nbytes, 16), dtype=torch.uint8)
        _run(what, at, lib().nsw_linear_backward, dy.data_ptr(), _p(x), weight.data_ptr(), _p(dx), _p(dw), _p(db), M,
             Np, K, dtype_code(dy), ws.data_ptr(), nbytes)
    if Np != N:
        dw, db = (None if t is None else t[:N] for t in (dw, db))
    return dx, dw, db


FP8_BLOCK = 128     # values along k under one scale


def quantize_fp8(x: torch.Tensor, rows: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of x [..., K]: q float8_e4m3fn [..., Kp], the last dim padded
    with zeros to a multiple of 128, and a power-of-two scale (float8_e8m0fnu)
    for each block of ``rows`` x 128 values: rows=1 for activations (scale
    [..., Kp / 128]), rows=128 for a weight matrix [N, K] (scale
    [ceil(N / 128), Kp / 128])."""
    at = _at(x)
    if rows not in (1, FP8_BLOCK):
        raise ValueError(f"quantize_fp8: rows must be 1 or {FP8_BLOCK}, got {rows}")
    if x.dim() < 1 or x.shape[-1] == 0 or (rows != 1 and x.dim() != 2):
        raise ValueError(f"quantize_fp8: x has shape {tuple(x.shape)}, expected [..., K], with rows={FP8_BLOCK} [N, K]")
    K = x.shape[-1]
    Kb = (K + FP8_BLOCK - 1) // FP8_BLOCK
    R = x.numel() // K
    code = dtype_code(x)
    lead = x.shape[:-1]
    q = x.new_empty(lead + (Kb * FP8_BLOCK,), dtype=torch.float8_e4m3fn)
    scale = x.new_empty((lead if rows == 1 else ((R + rows - 1) // rows,)) + (Kb,), dtype=torch.float8_e8m0fnu)
    if R:
        _run("quantize_fp8", at, lib().nsw_quantize_fp8, x.data_ptr(), q.data_ptr(), scale.data_ptr(), R, K, rows, code)
    return q, scale


def linear_fp8(xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
               bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
               epilogue: Optional[int] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """linear of operands from quantize_fp8 (x with rows=1, the weight with
    rows=128): y [..., N] in ``dtype`` (bfloat16 or float32; bias and residual
    in it too), the epilogues of linear.  Sums of float32 results in fp32; those
    of bfloat16 results keep 13 bits within a group of 8 products (at most
    7 2^-13 of the sum of magnitudes), the groups are added in fp32."""
    what = "linear_fp8"
    at = _at(xq, x_scale, wq, w_scale, bias, residual)
    if dtype not in _DTYPES:
        raise TypeError(f"{what}: the result is float32 or bfloat16, got {dtype}")
    if (xq.dtype != torch.float8_e4m3fn or wq.dtype != torch.float8_e4m3fn or x_scale.dtype != torch.float8_e8m0fnu
            or w_scale.dtype != torch.float8_e8m0fnu):
        raise TypeError(f"{what}: expected float8_e4m3fn values and float8_e8m0fnu scales, got "
                        f"{xq.dtype}, {x_scale.dtype}, {wq.dtype}, {w_scale.dtype}")
    shape, wshape = xq.shape, wq.shape
    if not shape or len(wshape) != 2 or wshape[1] != shape[-1] or wshape[1] % FP8_BLOCK or wshape[1] == 0:
        raise ValueError(f"{what}: xq {tuple(xq.shape)} and wq {tuple(wq.shape)}, expected [..., K] and [N, K] with K a "
                         f"multiple of {FP8_BLOCK}")
    N, K = wshape
    Kb = K // FP8_BLOCK
    if x_scale.shape != shape[:-1] + (Kb,) or w_scale.shape != ((N + FP8_BLOCK - 1) // FP8_BLOCK, Kb):
        raise ValueError(f"{what}: scales {tuple(x_scale.shape)} and {tuple(w_scale.shape)} do not match "
                         f"{tuple(xq.shape)} and {tuple(wq.shape)}")
    for t in (bias, residual):
        if t is not None and t.dtype != dtype:
            raise TypeError(f"dtype mismatch: {t.dtype} vs {dtype}")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"{what}: bias has shape {tuple(bias.shape)}, expected ({N},)")
    if epilogue is None:
        epilogue = _lib.NSW_EPI_NONE if bias is None else (
            _lib.NSW_EPI_BIAS if residual is None else _lib.NSW_EPI_BIAS_RESIDUAL)
    if (bias is not None and epilogue == _lib.NSW_EPI_NONE) or (residual is not None and epilogue != _lib.NSW_EPI_BIAS_RESIDUAL):
        raise ValueError(f"{what}: epilogue {int(epilogue)} has no part for the {'bias' if residual is None else 'residual'}")
    y = xq.new_empty(shape[:-1] + (N,), dtype=dtype)
    if residual is not None and residual.shape != y.shape:
        raise ValueError(f"residual shape {tuple(residual.shape)} != output {tuple(y.shape)}")
    if y.numel():
        _run(what, at, lib().nsw_linear_fp8, xq.data_ptr(), x_scale.data_ptr(), wq.data_ptr(), w_scale.data_ptr(),
             _p(bias), _p(residual), y.data_ptr(), xq.numel() // K, N, K, int(epilogue), _DTYPES[dtype])
    return y


def qkv_projection(x: torch.Tensor, wqkv: torch.Tensor, bqkv: torch.Tensor, qn_w: torch.Tensor,
                   kn_w: torch.Tensor, num_heads: int, eps: Optional[float] = None) -> torch.Tensor:
    """[.., C] -> [.., 3C]: q|k|v = x W^T + b with per-head RMSNorm on q and k."""
    dev = _dev(x, wqkv, bqkv, qn_w, kn_w)
    _same_dtype(x, wqkv, bqkv, qn_w, kn_w)
    C = x.shape[-1]
    M = x.numel() // C
    eps = default_eps(x.dtype) if eps is None else float(eps)
    y = torch.empty(x.shape[:-1] + (3 * C,), dtype=x.dtype, device=dev)
    check(lib().nsw_qkv_projection(x.data_ptr(), wqkv.data_ptr(), bqkv.data_ptr(), qn_w.data_ptr(),
                                   kn_w.data_ptr(), eps, y.data_ptr(), M, C, num_heads, dtype_code(x),
                                   _stream(dev)), "qkv_projection")
    return y


# --------------------------------------------------------------- attention ---

def window_attention(qkv: torch.Tensor, num_heads: int, scale: float, mask: Optional[torch.Tensor] = None,
                     geometry: Optional[Tuple[int, int, Tuple[int, int], Tuple[int, int], int]] = None
                     ) -> torch.Tensor:
    """qkv [Bw, L, 3C] -> o [Bw, L, C].  ``mask`` [nW, L, L] or None, with
    F.scaled_dot_product_attention's meaning (models/swin_helpers.py:247): a
    float mask is added to the scaled logits, a boolean mask marks the keys
    that take part (True) and is applied as 0 / -inf.  ``geometry`` = (H, W,
    window_size, shift_size, T) computes the reference's shift mask from
    indices instead (ignored when mask is given)."""
    Bw, L, C3 = qkv.shape
    C = C3 // 3
    dev = _dev(qkv, mask)
    if mask is not None:
        if mask.dtype == torch.bool:
            mask = torch.zeros(mask.shape, dtype=torch.float32, device=mask.device).masked_fill_(
                ~mask, float("-inf"))
        elif mask.dtype != torch.float32:
            mask = mask.float().contiguous()
        if mask.shape[-2:] != (L, L):
            raise ValueError(f"mask shape {tuple(mask.shape)} does not match L={L}")
        nWm = mask.shape[0]
    else:
        nWm = 0
    H = W = ws0 = ws1 = 1
    s0 = s1 = 0
    T = 1
    if geometry is not None and mask is None:
        H, W, (ws0, ws1), (s0, s1), T = geometry
    o = torch.empty((Bw, L, C), dtype=qkv.dtype, device=dev)
    check(lib().nsw_window_attention(qkv.data_ptr(), o.data_ptr(), _p(mask), nWm, Bw, L, C, num_heads,
                                     float(scale), H, W, ws0, ws1, s0, s1, T, dtype_code(qkv),
                                     _stream(dev)), "window_attention")
    return o


def window_displacements(extent: Sequence[int]) -> int:
    """Displacements between tokens of a window of T x A x W: (2T-1)(2A-1)(2W-1)."""
    n = 1
    for e in extent:
        n *= 2 * int(e) - 1
    return n


def _position_args(what, qkv, num_heads, table, buckets, extent, mask, geometry):
    """(device index, Bw, L, C, mask, the sizes of the C entries after the scale) of a position attention."""
    at = _uniform(qkv, table)
    _dev(qkv, buckets, mask)
    if qkv.dim() != 3 or qkv.shape[-1] % 3:
        raise ValueError(f"{what}: qkv has shape {tuple(qkv.shape)}, expected [Bw, L, 3C]")
    Bw, L, C = qkv.shape[0], qkv.shape[1], qkv.shape[2] // 3
    T, A, W = (int(e) for e in extent)
    if min(T, A, W) < 1 or T * A * W != L:
        raise ValueError(f"{what}: extent {(T, A, W)} does not hold {L} tokens")
    if table.dim() != 2 or table.shape[1] != num_heads or table.shape[0] == 0:
        raise ValueError(f"{what}: table has shape {tuple(table.shape)}, expected [buckets, {num_heads}]")
    R = window_displacements((T, A, W))
    if buckets.dtype != torch.int32 or buckets.shape != (R,):
        raise ValueError(f"{what}: buckets is {buckets.dtype} {tuple(buckets.shape)}, expected int32 ({R},)")
    if mask is not None and geometry is not None:
        raise ValueError(f"{what}: a mask or a geometry")
    nW = 0
    H = Wi = s0 = s1 = 0
    if mask is not None:
        if mask.dtype == torch.bool:
            mask = torch.zeros(mask.shape, dtype=torch.float32, device=mask.device).masked_fill_(~mask, float("-inf"))
        elif mask.dtype != torch.float32:
            mask = mask.float()
        if mask.dim() != 3 or mask.shape[1:] != (L, L) or mask.shape[0] == 0 or Bw % mask.shape[0]:
            raise ValueError(f"{what}: mask has shape {tuple(mask.shape)}, expected [nW, {L}, {L}] with nW a divisor of {Bw}")
        nW = mask.shape[0]
    elif geometry is not None:
        H, Wi, ws, (s0, s1), Tg = geometry
        if (Tg, *ws) != (T, A, W):
            raise ValueError(f"{what}: geometry of windows {(Tg, *ws)}, extent {(T, A, W)}")
    return at, Bw, L, C, mask, nW, (table.shape[0], T, A, W, H, Wi, int(s0), int(s1), dtype_code(qkv))


def position_stats_width(qkv: torch.Tensor, num_heads: int) -> int:
    """Floats of a row of position_attention's stats."""
    return 2 + (qkv.shape[-1] // 3 // max(num_heads, 1) + 7) // 8 if qkv.dtype == torch.bfloat16 else 2


def position_attention(qkv: torch.Tensor, num_heads: int, scale: float, table: torch.Tensor, buckets: torch.Tensor,
                       extent: Sequence[int], mask: Optional[torch.Tensor] = None,
                       geometry: Optional[Tuple[int, int, Tuple[int, int], Tuple[int, int], int]] = None
                       ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(o, stats): window_attention with a learned position bias, o [Bw, L, C] of qkv [Bw,
    L, 3C] with the logits scale q k^T + table[buckets[r], head] + mask.  ``extent``
    (T, A, W) lays out the L tokens of a window (a sequence: (1, 1, L)); r numbers the
    displacements of a query from a key, ((dt + T-1) (2A-1) + da + A-1) (2W-1) + dw + W-1;
    buckets [(2T-1)(2A-1)(2W-1)] int32 (at most 8192), table [buckets, num_heads] in
    qkv's dtype.  ``mask`` [nW, L, L] or ``geometry`` as window_attention; a row whose
    mask leaves nothing gives zeros (k and v have to be finite also where they are masked, as
    for the formula).  Finite table and mask values may be as large as they go: a row of the lowest
    alone is uniform, as in fp32.  stats [Bw, num_heads, L, position_stats_width] fp32 for
    position_attention_backward: each row's maximum m of z log2(e), log2 of its sum of
    2^(z log2(e) - m); bf16: then the bits that o's rounding lost."""
    what = "position_attention"
    at, Bw, L, C, mask, nW, sizes = _position_args(what, qkv, num_heads, table, buckets, extent, mask, geometry)
    o = qkv.new_empty((Bw, L, C))
    stats = qkv.new_empty((Bw, num_heads, L, position_stats_width(qkv, num_heads)), dtype=torch.float32)
    _run(what, at, lib().nsw_position_attention, qkv.data_ptr(), table.data_ptr(), buckets.data_ptr(), _p(mask), nW,
         o.data_ptr(), stats.data_ptr(), Bw, L, C, num_heads, float(scale), *sizes)
    return o, stats


def position_attention_backward(do: torch.Tensor, qkv: torch.Tensor, o: torch.Tensor, stats: torch.Tensor, num_heads: int,
                                scale: float, table: torch.Tensor, buckets: torch.Tensor, extent: Sequence[int],
                                mask: Optional[torch.Tensor] = None, geometry=None,
                                needs: Sequence[bool] = (True, True)):
    """(dqkv, dtable) of position_attention from the gradient of o, o itself and stats,
    None where ``needs`` says so.  The mask has no gradient."""
    what = "position_attention_backward"
    at, Bw, L, C, mask, nW, sizes = _position_args(what, qkv, num_heads, table, buckets, extent, mask, geometry)
    _uniform(qkv, do, o)
    _dev(qkv, stats)
    if do.shape != (Bw, L, C) or o.shape != (Bw, L, C):
        raise ValueError(f"{what}: do {tuple(do.shape)} and o {tuple(o.shape)}, expected {(Bw, L, C)}")
    rows = (Bw, num_heads, L, position_stats_width(qkv, num_heads))
    if stats.dtype != torch.float32 or stats.shape != rows:
        raise ValueError(f"{what}: stats is {stats.dtype} {tuple(stats.shape)}, expected float32 {rows}")
    if not any(needs):
        return None, None
    dqkv = torch.empty_like(qkv)
    dtable = torch.empty_like(table) if needs[1] else None
    nbytes, ws = 0, None
    if needs[1]:
        nbytes = _workspace_bytes(lib(), "nsw_position_attention_backward_workspace_size", Bw, L, C, num_heads, *sizes[1:4],
                                  sizes[-1])
        ws = qkv.new_empty(max(nbytes, 16), dtype=torch.uint8)
    _run(what, at, lib().nsw_position_attention_backward, do.data_ptr(), qkv.data_ptr(), o.data_ptr(), stats.data_ptr(),
         table.data_ptr(), buckets.data_ptr(), _p(mask), nW, dqkv.data_ptr(), _p(dtable), Bw, L, C, num_heads, float(scale),
         *sizes, _p(ws), nbytes)
    return dqkv if needs[0] else None, dtable


def proj_reverse_residual(o: torch.Tensor, wproj: torch.Tensor, bproj: torch.Tensor, skip: torch.Tensor,
                          window_size, shift_size) -> torch.Tensor:
    """skip + roll(window_reverse(o W^T + b), +shift) with skip [B,T,H,W,C]."""
    B, T, H, W, C = skip.shape
    dev = _dev(o, wproj, bproj, skip)
    _same_dtype(o, wproj, bproj, skip)
    y = torch.empty_like(skip)
    check(lib().nsw_proj_reverse_residual(o.data_ptr(), wproj.data_ptr(), bproj.data_ptr(), skip.data_ptr(),
                                          y.data_ptr(), B, T, H, W, C, window_size[0], window_size[1],
                                          int(shift_size[0]), int(shift_size[1]), dtype_code(o),
                                          _stream(dev)), "proj_reverse_residual")
    return y


def proj_reverse_residual_sumsq(o: torch.Tensor, wproj: torch.Tensor, bproj: torch.Tensor, skip: torch.Tensor,
                                window_size, shift_size):
    """proj_reverse_residual that also returns the partial sums of squares of
    each output row [B*T*H*W, P] (fp32, one per 512 bytes of row), the
    statistics of the RMSNorm that follows."""
    B, T, H, W, C = skip.shape
    dev = _dev(o, wproj, bproj, skip)
    _same_dtype(o, wproj, bproj, skip)
    y = torch.empty_like(skip)
    P = int(lib().nsw_row_sumsq_parts(C, dtype_code(skip)))
    ss = torch.empty(B * T * H * W, P, dtype=torch.float32, device=dev)
    check(lib().nsw_proj_reverse_residual_sumsq(o.data_ptr(), wproj.data_ptr(), bproj.data_ptr(),
                                                skip.data_ptr(), y.data_ptr(), ss.data_ptr(), B, T, H, W, C,
                                                window_size[0], window_size[1], int(shift_size[0]),
                                                int(shift_size[1]), dtype_code(o), _stream(dev)),
          "proj_reverse_residual_sumsq")
    return y, ss


def linear_rowscale(x: torch.Tensor, w_n: torch.Tensor, row_sumsq: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    residual: Optional[torch.Tensor] = None, epilogue: Optional[int] = None,
                    eps: Optional[float] = None) -> torch.Tensor:
    """y = epi(RMSNorm(x) . W^T) with w_n = W * norm_w and the rows' sums of
    squares given as partials row_sumsq [M, P] (from proj_reverse_residual_sumsq)."""
    dev = _dev(x, w_n, bias, residual, row_sumsq)
    _same_dtype(x, w_n, bias, residual)
    K = x.shape[-1]
    N, Kw = w_n.shape
    if Kw != K:
        raise ValueError(f"linear_rowscale: x has {K} features, weight expects {Kw}")
    M = x.numel() // K
    if row_sumsq.dtype != torch.float32 or row_sumsq.dim() != 2 or row_sumsq.shape[0] != M \
            or not row_sumsq.is_contiguous():
        raise ValueError("linear_rowscale: row_sumsq must be a contiguous fp32 [M, P] tensor")
    if epilogue is None:
        epilogue = _lib.NSW_EPI_NONE if bias is None else (
            _lib.NSW_EPI_BIAS if residual is None else _lib.NSW_EPI_BIAS_RESIDUAL)
    eps = default_eps(x.dtype) if eps is None else float(eps)
    y = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=dev)
    check(lib().nsw_linear_rowscale(x.data_ptr(), w_n.data_ptr(), _p(bias), _p(residual), y.data_ptr(),
                                    row_sumsq.data_ptr(), row_sumsq.shape[1], M, N, K, int(epilogue), eps,
                                    dtype_code(x), _stream(dev)), "linear_rowscale")
    return y


def qkv_projection_rowscale(x: torch.Tensor, wqkv_n: torch.Tensor, bqkv: torch.Tensor, qn_w: torch.Tensor,
                            kn_w: torch.Tensor, row_sumsq: torch.Tensor, num_heads: int,
                            eps: Optional[float] = None) -> torch.Tensor:
    """[M, C] -> [M, 3C]: q|k|v of RMSNorm(x) (norm1's weight folded into
    wqkv_n) with the row statistics given as partial sums of squares
    row_sumsq [M, P] (from window_partition_sumsq or linear_remap_residual)."""
    dev = _dev(x, wqkv_n, bqkv, qn_w, kn_w, row_sumsq)
    _same_dtype(x, wqkv_n, bqkv, qn_w, kn_w)
    C = x.shape[-1]
    M = x.numel() // C
    if row_sumsq.dtype != torch.float32 or row_sumsq.dim() != 2 or row_sumsq.shape[0] != M:
        raise ValueError("qkv_projection_rowscale: row_sumsq must be a contiguous fp32 [M, P] tensor")
    eps = default_eps(x.dtype) if eps is None else float(eps)
    y = torch.empty(x.shape[:-1] + (3 * C,), dtype=x.dtype, device=dev)
    check(lib().nsw_qkv_projection_rowscale(x.data_ptr(), wqkv_n.data_ptr(), bqkv.data_ptr(), qn_w.data_ptr(),
                                            kn_w.data_ptr(), eps, y.data_ptr(), row_sumsq.data_ptr(),
                                            row_sumsq.shape[1], M, C, num_heads, dtype_code(x), _stream(dev)),
          "qkv_projection_rowscale")
    return y


def linear_remap_residual(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor, residual: torch.Tensor,
                          map_mode: int, image=None, window_size=(1, 1), shift_size=(0, 0), next_shift=(0, 0)):
    """(y, row_sumsq): y[map(m)] = x[m] . w^T + bias + residual[m] for window
    rows of ``image`` = (B, T, H, W) with ``window_size`` / ``shift_size``:
    map_mode 0 identity, 1 to token order, 2 to the window order of the
    same image rolled by ``next_shift``, 3 from token-ordered rows into the
    window order with ``shift_size``; row_sumsq [M, P] fp32 (the stored
    rows' partial sums of squares, at the stored rows) for modes 0, 2 and 3,
    None for mode 1."""
    dev = _dev(x, w, bias, residual)
    _same_dtype(x, w, bias, residual)
    K = x.shape[-1]
    N = w.shape[0]
    M = x.numel() // K
    B, T, H, W = image if image is not None else (1, 1, 1, M)
    y = torch.empty(M, N, dtype=x.dtype, device=dev)
    ss = None
    if map_mode != 1:
        ss = torch.empty(M, lib().nsw_row_sumsq_parts(N, dtype_code(x)), dtype=torch.float32, device=dev)
    check(lib().nsw_linear_remap_residual(x.data_ptr(), w.data_ptr(), bias.data_ptr(), residual.data_ptr(),
                                          y.data_ptr(), _p(ss), M, N, K, int(map_mode), B, T, H, W,
                                          window_size[0], window_size[1], int(shift_size[0]), int(shift_size[1]),
                                          int(next_shift[0]), int(next_shift[1]), dtype_code(x), _stream(dev)),
          "linear_remap_residual")
    return y, ss


# ------------------------------------------------------------------- block ---

_ws_lock = threading.Lock()
_workspaces = {}      # (device index, stream) -> [buffer, handed out under graph capture]
_ws_retired = []      # replaced buffers that a captured graph may still address


def workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """Grow-only scratch buffer per (device, stream), reused by every block
    launched on that stream (kernels on one stream run in order).  A buffer
    handed out while the stream was being captured into a CUDA graph is
    never freed: when a later, larger call replaces it, it moves to a list
    kept for the life of the process, so that replays of the graph keep
    writing memory they own."""
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    capturing = torch.cuda.is_current_stream_capturing()
    with _ws_lock:
        ent = _workspaces.get(key)
        if ent is None or ent[0].numel() < nbytes:
            if ent is not None and ent[1]:
                _ws_retired.append(ent[0])
            ent = [torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device), False]
            _workspaces[key] = ent
        if capturing:
            ent[1] = True
        return ent[0]


def block_shape(x: torch.Tensor, num_heads: int, window_size, shift_size, hidden: int,
                eps: Optional[float], gelu_tanh: bool = False) -> _lib.BlockShape:
    B, T, H, W, C = x.shape
    eps = default_eps(x.dtype) if eps is None else float(eps)
    return _lib.BlockShape(B, T, H, W, C, num_heads, window_size[0], window_size[1],
                           int(shift_size[0]), int(shift_size[1]), hidden, eps, dtype_code(x),
                           1 if gelu_tanh else 0)


def swin_block_forward(x: torch.Tensor, packed: dict, num_heads: int, window_size, shift_size,
                       eps: Optional[float] = None, out: Optional[torch.Tensor] = None,
                       gelu_tanh: bool = False) -> torch.Tensor:
    """Whole Block.forward through one C-ABI call.  ``packed`` holds the
    tensors named like the fields of nsw_block_params; ``gelu_tanh`` selects
    the tanh-form GELU (the reference's TE block) instead of the erf form."""
    dev = _dev(x, *packed.values())
    _same_dtype(x, *packed.values())
    hidden = packed["w1"].shape[0]
    shp = block_shape(x, num_heads, window_size, shift_size, hidden, eps, gelu_tanh)
    params = _lib.BlockParams(*[_p(packed.get(n)) for n, _ in _lib.BlockParams._fields_])
    nbytes = lib().nsw_block_workspace_size(shp)
    ws = workspace(nbytes, dev)
    y = torch.empty_like(x) if out is None else out
    check(lib().nsw_swin_block_forward(x.data_ptr(), y.data_ptr(), params, shp, ws.data_ptr(), ws.numel(),
                                       _stream(dev)), "swin_block_forward")
    return y


def swin_blocks_forward(x: torch.Tensor, packs, num_heads: int, window_size, shifts, eps: Optional[float] = None,
                        out: Optional[torch.Tensor] = None, gelu_tanh: bool = False,
                        row_sumsq: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The blocks loop ``for blk in blocks: x = blk(x)`` through one C-ABI
    call that keeps the residual stream in window order between blocks.
    ``packs[i]`` is block i's dict of nsw_block_params tensors and must hold
    the norm-folded ``wqkv_n1`` and ``w1_n2``; ``shifts[i]`` its shift.  With
    ``row_sumsq`` ([rows, P] fp32, as window_partition_sumsq returns), x holds
    block 0's input already in block 0's window order (same [B, T, H, W, C]
    shape, rows in window order) and those are its norm1 sums of squares;
    the result is in token order either way."""
    packs = list(packs)
    if not packs or len(packs) != len(shifts):
        raise ValueError("swin_blocks_forward: one pack and one shift per block")
    tensors = [t for pk in packs for t in pk.values()]
    dev = _dev(x, *tensors)
    _same_dtype(x, *tensors)
    if x.dim() != 5 or not x.is_contiguous():
        raise ValueError("swin_blocks_forward: x must be a contiguous [B, T, H, W, C] tensor")
    depth = len(packs)
    hidden = packs[0]["w1"].shape[0]
    shapes = (_lib.BlockShape * depth)(*[block_shape(x, num_heads, window_size, shifts[i], hidden, eps, gelu_tanh)
                                         for i in range(depth)])
    params = (_lib.BlockParams * depth)(*[_lib.BlockParams(*[_p(pk.get(n)) for n, _ in _lib.BlockParams._fields_])
                                          for pk in packs])
    nbytes = lib().nsw_blocks_workspace_size(shapes, depth)
    if nbytes == 0:
        raise ValueError("swin_blocks_forward: malformed block shape")
    ws = workspace(nbytes, dev)
    y = torch.empty_like(x) if out is None else out
    if row_sumsq is None:
        check(lib().nsw_swin_blocks_forward(x.data_ptr(), y.data_ptr(), params, shapes, depth, ws.data_ptr(),
                                            ws.numel(), _stream(dev)), "swin_blocks_forward")
    else:
        if row_sumsq.dtype != torch.float32 or not row_sumsq.is_contiguous() or row_sumsq.device != dev:
            raise ValueError("swin_blocks_forward: row_sumsq must be a contiguous float32 tensor on x's device")
        if row_sumsq.numel() != (x.numel() // x.shape[-1]) * lib().nsw_row_sumsq_parts(x.shape[-1], dtype_code(x)):
            raise ValueError("swin_blocks_forward: row_sumsq must be [rows, nsw_row_sumsq_parts(C)]")
        check(lib().nsw_swin_blocks_forward_windowed(x.data_ptr(), row_sumsq.data_ptr(), y.data_ptr(), params,
                                                     shapes, depth, ws.data_ptr(), ws.numel(), _stream(dev)),
              "swin_blocks_forward")
    return y


def window_partition_sumsq(x: torch.Tensor, window_size, shift_size):
    """(windows, row_sumsq): x [B,T,H,W,C] rolled by -shift and split into
    windows [B*nW, T, ws0, ws1, C], and fp32 [rows, nparts] partial sums of
    squares of each stored row (512-byte parts)."""
    dev = _dev(x)
    if x.dim() != 5 or not x.is_contiguous():
        raise ValueError("window_partition_sumsq: x must be a contiguous [B, T, H, W, C] tensor")
    B, T, H, W, C = x.shape
    ws0, ws1 = window_size
    nW = (H // ws0) * (W // ws1)
    xw = torch.empty((B * nW, T, ws0, ws1, C), dtype=x.dtype, device=dev)
    nparts = lib().nsw_row_sumsq_parts(C, dtype_code(x))
    ss = torch.empty((x.numel() // C, nparts), dtype=torch.float32, device=dev)
    check(lib().nsw_window_partition_sumsq(x.data_ptr(), xw.data_ptr(), ss.data_ptr(), B, T, H, W, C, ws0, ws1,
                                           int(shift_size[0]), int(shift_size[1]), dtype_code(x), _stream(dev)),
          "window_partition_sumsq")
    return xw, ss


# ----------------------------------------------------------------- metrics ---

def weighted_metrics(pred: torch.Tensor, target: torch.Tensor, weights: torch.Tensor,
                     clim: Optional[torch.Tensor] = None):
    """Per-(b,t,c) weighted RMSE and (if clim is given) ACC, float64 [B,T,C].
    ``weights``: [H], [H, 1] (cos-lat) or [H, W] (a full map)."""
    if pred.shape != target.shape or pred.dim() != 5:
        raise ValueError("pred and target must be [B, T, C, H, W] of the same shape")
    if pred.dtype != torch.float32 or target.dtype != torch.float32:
        raise TypeError("weighted metrics take float32 fields")
    B, T, C, H, W = pred.shape
    dev = _dev(pred, target, clim)
    w = weights.to(device=dev, dtype=torch.float64).contiguous()
    if w.numel() == H:
        w_cols = 1
    elif w.numel() == H * W and (w.dim() < 2 or tuple(w.shape[-2:]) == (H, W)):
        w_cols = W
    else:
        raise ValueError(f"weights of shape {tuple(weights.shape)} do not match a {H}x{W} field")
    if clim is not None:
        clim = clim.reshape(-1).to(torch.float32).contiguous()
        if clim.numel() != C:
            raise ValueError("climatology must have one value per channel")
    P = B * T * C
    rmse = torch.empty(P, dtype=torch.float64, device=dev)
    acc = torch.empty(P, dtype=torch.float64, device=dev) if clim is not None else None
    nbytes = lib().nsw_weighted_metrics_workspace_size(P, H, W)
    ws = torch.empty(max(nbytes, 8), dtype=torch.uint8, device=dev)
    check(lib().nsw_weighted_metrics(pred.data_ptr(), target.data_ptr(), w.data_ptr(), w_cols, _p(clim), P,
                                     H, W, C,
                                     rmse.data_ptr(), _p(acc), ws.data_ptr(), ws.numel(), _stream(dev)),
          "weighted_metrics")
    rmse = rmse.view(B, T, C)
    return rmse, (acc.view(B, T, C) if acc is not None else None)


# ------------------------------------------------------------ model layout ---

def k_granule(dtype: torch.dtype) -> int:
    """K padding of the patch matrix: one 128-byte operand stage of the GEMM,
    64 (bf16) / 32 (f32) elements, so that its rows start on whole cache
    lines (the GEMM itself takes K a multiple of 32 / 16)."""
    return 64 if dtype == torch.bfloat16 else 32


def patch_im2col(x: torch.Tensor, p: int, Kp: int, dtype: torch.dtype,
                 invariants: Optional[torch.Tensor] = None, frame0: int = 0) -> torch.Tensor:
    """Patch matrix of the stride-p patch convolution: x [B, T, C_x, H, W]
    (+ invariants [C_inv, H, W] as extra channels; frame t read from slot
    (t + frame0) mod T) -> [B*T*(H/p)*(W/p), Kp] in ``dtype``."""
    if x.dim() != 5:
        raise ValueError("patch_im2col: x must be [B, T, C, H, W]")
    B, T, Cx, H, W = x.shape
    if invariants is not None:
        if invariants.dtype != x.dtype:
            raise TypeError("patch_im2col: invariants must have x's dtype")
        if invariants.dim() != 3 or tuple(invariants.shape[1:]) != (H, W):
            raise ValueError("patch_im2col: invariants must be [C_inv, H, W]")
    dev = _dev(x, invariants)
    Cinv = 0 if invariants is None else invariants.shape[0]
    M = B * T * (H // p) * (W // p)
    out = torch.empty(M, Kp, dtype=dtype, device=dev)
    check(lib().nsw_patch_im2col(x.data_ptr(), _p(invariants), B, T, Cx, Cinv, H, W, p, int(frame0), Kp,
                                 out.data_ptr(), dtype_code(x), _DTYPES[dtype], _stream(dev)), "patch_im2col")
    return out


def unpatchify(y: torch.Tensor, B: int, C_out: int, H: int, W: int, p: int,
               dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Head layout: y [B*(H/p)*(W/p), p*p*C_out] -> [B, 1, C_out, H, W].  With
    ``out`` (a [B, 1, C_out, H, W] tensor whose frames are contiguous, e.g.
    one slot of a [B, T, C, H, W] ring buffer) the result is written there in
    out's dtype."""
    if out is not None:
        if tuple(out.shape) != (B, 1, C_out, H, W):
            raise ValueError(f"unpatchify: out must be [{B}, 1, {C_out}, {H}, {W}]")
        if out.stride()[2:] != (H * W, W, 1) or out.stride(0) < C_out * H * W:
            raise ValueError("unpatchify: every frame of out must be contiguous")
        if not out.is_cuda:
            raise RuntimeError("libnsw ops run on the GPU only")
        bstride = out.stride(0)
        dst = out
    else:
        dst = torch.empty(B, 1, C_out, H, W, dtype=dtype or y.dtype, device=y.device)
        bstride = C_out * H * W
    dev = _dev(y)
    if dst.device != dev:
        raise RuntimeError("libnsw op arguments are on different devices")
    check(lib().nsw_unpatchify(y.data_ptr(), dst.data_ptr(), B, C_out, H, W, p, bstride, dtype_code(y),
                               dtype_code(dst), _stream(dev)), "unpatchify")
    return dst


def head_weight_perm(weight: torch.Tensor, C_out: int, p: int) -> torch.Tensor:
    """The head weight [p*p*C_out, E] (reference row (u*p + v)*C_out + c,
    models/swin.py:201-209,293-299) with its rows reordered to c*p*p + u*p + v,
    the order nsw_head_unpatchify takes."""
    E = weight.shape[-1]
    if weight.shape[0] != p * p * C_out:
        raise ValueError(f"head weight has {weight.shape[0]} rows, expected p*p*C_out = {p * p * C_out}")
    return weight.view(p * p, C_out, E).transpose(0, 1).reshape(C_out * p * p, E).contiguous()


def head_unpatchify(x: torch.Tensor, w_perm: torch.Tensor, B: int, C_out: int, H: int, W: int, p: int,
                    dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """unpatchify(x . W^T) in one launch: x [B*(H/p)*(W/p), E] tokens, w_perm
    from head_weight_perm -> [B, 1, C_out, H, W] in ``dtype`` (x's dtype or
    float32), or into ``out`` (frames contiguous, e.g. one slot of a ring
    buffer) in out's dtype."""
    if x.dim() != 2 or x.shape[0] != B * (H // p) * (W // p):
        raise ValueError("head_unpatchify: x must be [B*(H/p)*(W/p), E]")
    if w_perm.shape != (C_out * p * p, x.shape[1]):
        raise ValueError(f"head_unpatchify: w_perm must be [{C_out * p * p}, {x.shape[1]}]")
    if out is not None:
        if tuple(out.shape) != (B, 1, C_out, H, W):
            raise ValueError(f"head_unpatchify: out must be [{B}, 1, {C_out}, {H}, {W}]")
        if out.stride()[2:] != (H * W, W, 1) or out.stride(0) < C_out * H * W:
            raise ValueError("head_unpatchify: every frame of out must be contiguous")
        bstride = out.stride(0)
        dst = out
    else:
        dst = torch.empty(B, 1, C_out, H, W, dtype=dtype or x.dtype, device=x.device)
        bstride = C_out * H * W
    dev = _dev(x, w_perm)
    if dst.device != dev:
        raise RuntimeError("libnsw op arguments are on different devices")
    _same_dtype(x, w_perm)
    check(lib().nsw_head_unpatchify(x.data_ptr(), w_perm.data_ptr(), dst.data_ptr(), B, C_out, H, W, p,
                                    x.shape[1], bstride, dtype_code(x), dtype_code(dst), _stream(dev)),
          "head_unpatchify")
    return dst


def skip_conv_accumulate(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor,
                         invariants: Optional[torch.Tensor] = None, frame0: int = 0,
                         model_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The big skip of SwinTransformer.forward (models/swin.py:310-319) in
    place: out [B, 1, C_out, H, W] += Conv2d 1x1 (``weight`` [C_out, C_in]
    or [C_out, C_in, 1, 1], no bias) of x's last frame (ring slot (T - 1 +
    frame0) mod T of x [B, T, C_x, H, W]) with the invariant planes
    [C_inv, H, W] appended; values rounded to ``model_dtype`` (weight's
    dtype by default) as the reference's model-dtype conv and add."""
    if x.dim() != 5 or out.dim() != 5:
        raise ValueError("skip_conv_accumulate: x and out must be [B, T, C, H, W] / [B, 1, C_out, H, W]")
    B, T, C_x, H, W = x.shape
    C_inv = 0 if invariants is None else invariants.shape[0]
    w2 = weight.reshape(weight.shape[0], -1)
    C_out = w2.shape[0]
    if w2.shape[1] != C_x + C_inv:
        raise ValueError(f"skip_conv_accumulate: weight has {w2.shape[1]} input channels, x + invariants "
                         f"{C_x + C_inv}")
    if tuple(out.shape) != (B, 1, C_out, H, W) or out.stride()[2:] != (H * W, W, 1):
        raise ValueError(f"skip_conv_accumulate: out must be [{B}, 1, {C_out}, {H}, {W}] with contiguous frames")
    if invariants is not None and (tuple(invariants.shape) != (C_inv, H, W) or invariants.dtype != x.dtype):
        raise ValueError("skip_conv_accumulate: invariants must be [C_inv, H, W] in x's dtype")
    xc = x.contiguous()
    inv = None if invariants is None else invariants.contiguous()
    wf = w2.detach().to(torch.float32).contiguous()
    dev = _dev(xc, wf, inv)
    if out.device != dev:                      # out may be a strided ring slot (frames contiguous)
        raise RuntimeError("libnsw op arguments are on different devices")
    md = model_dtype or weight.dtype
    check(lib().nsw_skip_conv_accumulate(xc.data_ptr(), _p(inv), wf.data_ptr(), out.data_ptr(), B, T, C_x, C_inv,
                                         C_out, H, W, int(frame0), out.stride(0), dtype_code(xc),
                                         _lib.NSW_DTYPE_BF16 if md == torch.bfloat16 else _lib.NSW_DTYPE_F32,
                                         dtype_code(out), _stream(dev)), "skip_conv_accumulate")
    return out


def weighted_metrics_unnorm(pred: torch.Tensor, target: torch.Tensor, std: torch.Tensor, mean: torch.Tensor,
                            weights: torch.Tensor, clim: Optional[torch.Tensor] = None):
    """Weighted RMSE (and ACC with ``clim``) of pred * std + mean against
    target * std + mean, per (b, t, c), float64 [B, T, C].  pred fp32 or
    bf16, target fp32, std / mean per channel; float64 std or mean (stats
    read from a float64 file) make the unnormalised fields float64, as the
    reference's type promotion does, otherwise they are fp32."""
    if pred.shape != target.shape or pred.dim() != 5:
        raise ValueError("pred and target must be [B, T, C, H, W] of the same shape")
    if target.dtype != torch.float32:
        raise TypeError("target must be float32")
    B, T, C, H, W = pred.shape
    dev = _dev(pred, target)
    w = weights.to(device=dev, dtype=torch.float64).contiguous()
    if w.numel() == H:
        w_cols = 1
    elif w.numel() == H * W and (w.dim() < 2 or tuple(w.shape[-2:]) == (H, W)):
        w_cols = W
    else:
        raise ValueError(f"weights of shape {tuple(weights.shape)} do not match a {H}x{W} field")
    f64 = torch.float64 in (torch.as_tensor(std).dtype, torch.as_tensor(mean).dtype)
    sdt = torch.float64 if f64 else torch.float32
    sc = torch.as_tensor(std).reshape(-1).to(device=dev, dtype=sdt).contiguous()
    of = torch.as_tensor(mean).reshape(-1).to(device=dev, dtype=sdt).contiguous()
    if sc.numel() != C or of.numel() != C:
        raise ValueError("std and mean must have one value per channel")
    if clim is not None:
        clim = clim.reshape(-1).to(device=dev, dtype=torch.float32).contiguous()
        if clim.numel() != C:
            raise ValueError("climatology must have one value per channel")
    P = B * T * C
    rmse = torch.empty(P, dtype=torch.float64, device=dev)
    acc = torch.empty(P, dtype=torch.float64, device=dev) if clim is not None else None
    nbytes = lib().nsw_weighted_metrics_workspace_size(P, H, W)
    ws = workspace(max(nbytes, 8), dev)
    fn = lib().nsw_weighted_metrics_unnorm_f64stats if f64 else lib().nsw_weighted_metrics_unnorm
    check(fn(pred.data_ptr(), dtype_code(pred), target.data_ptr(), sc.data_ptr(), of.data_ptr(), w.data_ptr(),
             w_cols, _p(clim), P, H, W, C, rmse.data_ptr(), _p(acc), ws.data_ptr(), ws.numel(), _stream(dev)),
          "weighted_metrics_unnorm")
    rmse = rmse.view(B, T, C)
    return rmse, (acc.view(B, T, C) if acc is not None else None)
