"""The library's functional ops as PyTorch custom operators, ``torch.ops.nsw.*``.

Each op is registered with ``torch.library.custom_op`` and a shape function
(``register_fake``), so the modules built on them (``nsw.Block``,
``WindowMultiHeadAttention``, ``MLP``, ``NormLayer``, ``LinearLayer``,
``SwinTransformer``, ``WeightedRMSE`` ...) trace under ``torch.compile``
without graph breaks: the op bodies call the ctypes layer (``nsw/ops.py``),
which stays opaque to the tracer.  The ops allocate their outputs with torch
and enqueue HIP kernels on the current stream, so they also run under CUDA
graph capture.  Ops that write into a caller's tensor (``out=``) are not
registered; their callers keep the ``nsw.ops`` functions.

``linear`` (without GELU), ``gated_linear``, ``residual_norm``, ``group_norm`` and
``position_attention`` have gradients (``linear_backward``, ``gated_linear_backward``,
``residual_norm_backward``, ``group_norm_backward``, ``position_attention_backward``),
and so have the window maps (each the other); the others are forward only, and so are
the modules that pack their parameters (``WindowMultiHeadAttention``, the blocks, the
patch embedding): a backward pass to those parameters raises.

The block parameters travel as one list in the field order of
``nsw_block_params`` (``BLOCK_PARAMS``), None for absent fields; shapes,
windows and shifts as int lists.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib, ops

BLOCK_PARAMS = [n for n, _ in _lib.BlockParams._fields_]


def block_param_list(packed: dict) -> List[Optional[torch.Tensor]]:
    return [packed.get(n) for n in BLOCK_PARAMS]


def _unpack_block(params: List[Optional[torch.Tensor]]) -> dict:
    if len(params) != len(BLOCK_PARAMS):
        raise ValueError(f"a block takes {len(BLOCK_PARAMS)} parameter slots, got {len(params)}")
    return {n: t for n, t in zip(BLOCK_PARAMS, params) if t is not None}


# ----------------------------------------------------------------- blocks ---

@torch.library.custom_op("nsw::swin_block", mutates_args=())
def swin_block(x: torch.Tensor, params: List[Optional[torch.Tensor]], num_heads: int, window_size: List[int],
               shift_size: List[int], eps: float, gelu_tanh: bool) -> torch.Tensor:
    """Block.forward (models/swin_helpers.py:435-459) through nsw_swin_block_forward."""
    return ops.swin_block_forward(x.contiguous(), _unpack_block(params), num_heads, tuple(window_size),
                                  tuple(shift_size), eps=eps, gelu_tanh=gelu_tanh)


@swin_block.register_fake
def _(x, params, num_heads, window_size, shift_size, eps, gelu_tanh):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


@torch.library.custom_op("nsw::swin_blocks", mutates_args=())
def swin_blocks(x: torch.Tensor, params: List[Optional[torch.Tensor]], num_heads: int, window_size: List[int],
                shifts: List[int], eps: float, gelu_tanh: bool) -> torch.Tensor:
    """``for blk in blocks: x = blk(x)`` (models/swin.py:307-308) as one window-order chain;
    params = the blocks' parameter lists concatenated, shifts = [s0, s1] per block."""
    nb = len(BLOCK_PARAMS)
    depth = len(shifts) // 2
    if depth == 0 or len(shifts) != 2 * depth or len(params) != nb * depth:
        raise ValueError("swin_blocks: one parameter list and one shift pair per block")
    packs = [_unpack_block(params[i * nb:(i + 1) * nb]) for i in range(depth)]
    sh = [(shifts[2 * i], shifts[2 * i + 1]) for i in range(depth)]
    return ops.swin_blocks_forward(x.contiguous(), packs, num_heads, tuple(window_size), sh, eps=eps,
                                   gelu_tanh=gelu_tanh)


@swin_blocks.register_fake
def _(x, params, num_heads, window_size, shifts, eps, gelu_tanh):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


@torch.library.custom_op("nsw::swin_blocks_windowed", mutates_args=())
def swin_blocks_windowed(xw: torch.Tensor, row_sumsq: torch.Tensor, params: List[Optional[torch.Tensor]],
                         num_heads: int, window_size: List[int], shifts: List[int], eps: float,
                         gelu_tanh: bool) -> torch.Tensor:
    """swin_blocks from block 0's window order: xw [B, T, H, W, C] holding the
    rows in block 0's window order, row_sumsq their norm1 partial sums."""
    nb = len(BLOCK_PARAMS)
    depth = len(shifts) // 2
    if depth == 0 or len(shifts) != 2 * depth or len(params) != nb * depth:
        raise ValueError("swin_blocks_windowed: one parameter list and one shift pair per block")
    packs = [_unpack_block(params[i * nb:(i + 1) * nb]) for i in range(depth)]
    sh = [(shifts[2 * i], shifts[2 * i + 1]) for i in range(depth)]
    return ops.swin_blocks_forward(xw.contiguous(), packs, num_heads, tuple(window_size), sh, eps=eps,
                                   gelu_tanh=gelu_tanh, row_sumsq=row_sumsq.contiguous())


@swin_blocks_windowed.register_fake
def _(xw, row_sumsq, params, num_heads, window_size, shifts, eps, gelu_tanh):
    return torch.empty_like(xw, memory_format=torch.contiguous_format)


# ------------------------------------------------------------ linear / norm ---

@torch.library.custom_op("nsw::linear", mutates_args=())
def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], residual: Optional[torch.Tensor],
           epilogue: int) -> torch.Tensor:
    """y = epi(x . weight^T) (F.linear with a fused bias / GELU / residual epilogue)."""
    return ops.linear(x.contiguous(), weight.contiguous(), bias, None if residual is None else residual.contiguous(),
                      epilogue=epilogue)


@linear.register_fake
def _(x, weight, bias, residual, epilogue):
    return x.new_empty(tuple(x.shape[:-1]) + (weight.shape[0],))


@torch.library.custom_op("nsw::linear_forward", mutates_args=())
def linear_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                   residual: Optional[torch.Tensor], epilogue: int) -> torch.Tensor:
    """linear without a gradient: a backward pass that reaches it raises."""
    return ops.linear(x.contiguous(), weight.contiguous(), bias, None if residual is None else residual.contiguous(),
                      epilogue=epilogue)


@linear_forward.register_fake
def _(x, weight, bias, residual, epilogue):
    return x.new_empty(tuple(x.shape[:-1]) + (weight.shape[0],))


def _no_gradient(ctx, dy):
    raise NotImplementedError("nsw.linear_forward: the module's pass is forward only (GELU MLP, attention, patch embedding; "
                              "nsw.GatedMLP has gradients)")


linear_forward.register_autograd(_no_gradient)


def _dense(t: torch.Tensor) -> torch.Tensor:
    """t contiguous and 16-byte aligned (a gradient may be any view)."""
    t = t.contiguous()
    return t.clone() if t.is_cuda and t.data_ptr() % 16 else t


def _or_empty(like: torch.Tensor, *ts: Optional[torch.Tensor]) -> Tuple[torch.Tensor, ...]:
    """ts with an empty tensor in the place of None (custom ops return tensors)."""
    return tuple(like.new_empty((0,)) if t is None else t for t in ts)


@torch.library.custom_op("nsw::linear_backward", mutates_args=())
def linear_backward(dy: torch.Tensor, x: Optional[torch.Tensor], weight: torch.Tensor,
                    needs: List[bool]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias) of a linear without an activation; empty ([0]) where ``needs`` is False.
    x may be None where dweight is not needed."""
    return _or_empty(dy, *ops.linear_backward(_dense(dy), None if x is None else _dense(x), _dense(weight),
                                              needs=tuple(needs)))


@linear_backward.register_fake
def _(dy, x, weight, needs):
    return (dy.new_empty(tuple(dy.shape[:-1]) + (weight.shape[1],) if needs[0] else (0,)),
            dy.new_empty(weight.shape if needs[1] else (0,)), dy.new_empty((weight.shape[0],) if needs[2] else (0,)))


def _linear_setup(ctx, inputs, output):
    x, weight, bias, residual, epilogue = inputs
    ctx.epilogue = epilogue
    if epilogue in (_lib.NSW_EPI_NONE, _lib.NSW_EPI_BIAS, _lib.NSW_EPI_BIAS_RESIDUAL):
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, weight)   # only dweight reads x


def _linear_backward(ctx, dy):
    if ctx.epilogue not in (_lib.NSW_EPI_NONE, _lib.NSW_EPI_BIAS, _lib.NSW_EPI_BIAS_RESIDUAL):
        raise NotImplementedError("nsw.linear with a GELU epilogue has no gradient (nsw.GatedMLP has)")
    need = list(ctx.needs_input_grad)
    if (need[2] and ctx.epilogue == _lib.NSW_EPI_NONE) or (need[3] and ctx.epilogue != _lib.NSW_EPI_BIAS_RESIDUAL):
        raise ValueError(f"nsw.linear: epilogue {ctx.epilogue} left the {'residual' if need[3] else 'bias'} out, which "
                         "needs a gradient (a residual takes part with a bias)")
    x, weight = ctx.saved_tensors
    needs = [need[0], need[1], need[2]]
    dx, dw, db = torch.ops.nsw.linear_backward(dy, x, weight, needs) if any(needs) else (None, None, None)
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, dy if need[3] else None, None)


linear.register_autograd(_linear_backward, setup_context=_linear_setup)


@torch.library.custom_op("nsw::gated_linear", mutates_args=())
def gated_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], act: str) -> torch.Tensor:
    """act(x Wg^T + bg) * (x Wu^T + bu), weight [2H, K] = Wg over Wu."""
    return ops.gated_linear(_dense(x), _dense(weight), bias, act=act)


@gated_linear.register_fake
def _(x, weight, bias, act):
    return x.new_empty(tuple(x.shape[:-1]) + (weight.shape[0] // 2,))


@torch.library.custom_op("nsw::gated_linear_backward", mutates_args=())
def gated_linear_backward(dh: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                          act: str, needs: List[bool]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias) of gated_linear; empty ([0]) where ``needs`` is False or there is no bias."""
    return _or_empty(x, *ops.gated_linear_backward(_dense(dh), _dense(x), _dense(weight), bias, act=act,
                                                   needs=tuple(needs)))


@gated_linear_backward.register_fake
def _(dh, x, weight, bias, act, needs):
    return (x.new_empty(x.shape if needs[0] else (0,)), x.new_empty(weight.shape if needs[1] else (0,)),
            x.new_empty(bias.shape if needs[2] and bias is not None else (0,)))


def _gated_setup(ctx, inputs, output):
    x, weight, bias, act = inputs
    ctx.act, ctx.has_bias = act, bias is not None
    ctx.save_for_backward(x, weight, *([bias] if bias is not None else []))


def _gated_backward(ctx, dh):
    x, weight, *rest = ctx.saved_tensors
    need = list(ctx.needs_input_grad)
    dx, dw, db = torch.ops.nsw.gated_linear_backward(dh, x, weight, rest[0] if ctx.has_bias else None, ctx.act,
                                                     [need[0], need[1], need[2]])
    return dx if need[0] else None, dw if need[1] else None, db if need[2] and ctx.has_bias else None, None


gated_linear.register_autograd(_gated_backward, setup_context=_gated_setup)


@torch.library.custom_op("nsw::quantize_fp8", mutates_args=())
def quantize_fp8(x: torch.Tensor, rows: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """(e4m3 values, E8M0 scales) of x, a scale for each block of rows (1 or 128) x 128."""
    return ops.quantize_fp8(_dense(x), rows=rows)


@quantize_fp8.register_fake
def _(x, rows):
    Kb = (x.shape[-1] + ops.FP8_BLOCK - 1) // ops.FP8_BLOCK
    lead = tuple(x.shape[:-1]) if rows == 1 else ((x.shape[0] + rows - 1) // rows,)
    return (x.new_empty(tuple(x.shape[:-1]) + (Kb * ops.FP8_BLOCK,), dtype=torch.float8_e4m3fn),
            x.new_empty(lead + (Kb,), dtype=torch.float8_e8m0fnu))


@torch.library.custom_op("nsw::linear_fp8", mutates_args=())
def linear_fp8(xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
               bias: Optional[torch.Tensor], residual: Optional[torch.Tensor], epilogue: int,
               dtype: torch.dtype) -> torch.Tensor:
    """nsw.linear on operands from quantize_fp8, the result in dtype."""
    return ops.linear_fp8(xq.contiguous(), x_scale.contiguous(), wq, w_scale, bias,
                          None if residual is None else _dense(residual), epilogue=epilogue, dtype=dtype)


@linear_fp8.register_fake
def _(xq, x_scale, wq, w_scale, bias, residual, epilogue, dtype):
    return xq.new_empty(tuple(xq.shape[:-1]) + (wq.shape[0],), dtype=dtype)


@torch.library.custom_op("nsw::residual_norm", mutates_args=())
def _residual_norm(branch: torch.Tensor, skip: torch.Tensor, post_weight: Optional[torch.Tensor],
                   gate: Optional[torch.Tensor], alpha: float, norm_weight: Optional[torch.Tensor],
                   eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    return _or_empty(branch, *ops.residual_norm(_dense(branch), _dense(skip), post_weight,
                                                None if gate is None else _dense(gate), alpha, norm_weight, eps))


@_residual_norm.register_fake
def _(branch, skip, post_weight, gate, alpha, norm_weight, eps):
    y = torch.empty_like(branch, memory_format=torch.contiguous_format)
    return y, branch.new_empty((0,)) if norm_weight is None else torch.empty_like(y)


@torch.library.custom_op("nsw::residual_norm_backward", mutates_args=())
def _residual_norm_backward(dy: Optional[torch.Tensor], dz: Optional[torch.Tensor], branch: torch.Tensor,
                            skip: torch.Tensor, post_weight: Optional[torch.Tensor], gate: Optional[torch.Tensor],
                            alpha: float, norm_weight: Optional[torch.Tensor], eps: float
                            ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return _or_empty(branch, *ops.residual_norm_backward(
        None if dy is None else _dense(dy), None if dz is None else _dense(dz), _dense(branch), _dense(skip), post_weight,
        None if gate is None else _dense(gate), alpha, norm_weight, eps))


@_residual_norm_backward.register_fake
def _(dy, dz, branch, skip, post_weight, gate, alpha, norm_weight, eps):
    full = lambda t: branch.new_empty((0,) if t is None else t.shape)
    return full(branch), full(skip), full(post_weight), full(gate), full(norm_weight)


def _residual_setup(ctx, inputs, output):
    branch, skip, post_weight, gate, alpha, norm_weight, eps = inputs
    ctx.alpha, ctx.eps = alpha, eps
    ctx.given = [t is not None for t in (post_weight, gate, norm_weight)]
    ctx.save_for_backward(branch, skip, *[t for t in (post_weight, gate, norm_weight) if t is not None])
    ctx.set_materialize_grads(False)


def _residual_backward(ctx, dy, dz):
    branch, skip, *rest = ctx.saved_tensors
    rest = iter(rest)
    post_weight, gate, norm_weight = (next(rest) if g else None for g in ctx.given)
    if norm_weight is None:
        dz = None
    if dy is None and dz is None:
        return (None,) * 7
    db, ds, dp, dg, dn = torch.ops.nsw.residual_norm_backward(dy, dz, branch, skip, post_weight, gate, ctx.alpha,
                                                              norm_weight, ctx.eps)
    return (db, ds, dp if ctx.given[0] else None, dg if ctx.given[1] else None, None, dn if ctx.given[2] else None, None)


_residual_norm.register_autograd(_residual_backward, setup_context=_residual_setup)


def residual_norm(branch: torch.Tensor, skip: torch.Tensor, post_weight: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, alpha: float = 1.0,
                  norm_weight: Optional[torch.Tensor] = None, eps: Optional[float] = None):
    """torch.ops.nsw.residual_norm with ops.residual_norm's defaults: (y, z or None)."""
    y, z = torch.ops.nsw.residual_norm(branch, skip, post_weight, gate, float(alpha), norm_weight,
                                       ops.default_eps(branch.dtype) if eps is None else float(eps))
    return y, None if norm_weight is None else z


@torch.library.custom_op("nsw::group_norm", mutates_args=())
def _group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], act: str,
                eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """(act(GroupNorm(x) * weight + bias), stats) of x [B, ..., C], channels last."""
    return ops.group_norm(_dense(x), groups, None if weight is None else _dense(weight),
                          None if bias is None else _dense(bias), act=act, eps=eps)


@_group_norm.register_fake
def _(x, groups, weight, bias, act, eps):
    return (torch.empty_like(x, memory_format=torch.contiguous_format),
            x.new_empty((x.shape[0], groups, 2), dtype=torch.float32))


@torch.library.custom_op("nsw::group_norm_backward", mutates_args=())
def _group_norm_backward(dy: torch.Tensor, x: torch.Tensor, stats: torch.Tensor, groups: int,
                         weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], act: str,
                         needs: List[bool]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias); empty ([0]) where ``needs`` is False or there is no such parameter."""
    return _or_empty(x, *ops.group_norm_backward(
        _dense(dy), _dense(x), _dense(stats), groups, None if weight is None else _dense(weight),
        None if bias is None else _dense(bias), act=act, needs=tuple(needs)))


@_group_norm_backward.register_fake
def _(dy, x, stats, groups, weight, bias, act, needs):
    return tuple(x.new_empty(t.shape if n and t is not None else (0,)) for n, t in zip(needs, (x, weight, bias)))


def _group_norm_setup(ctx, inputs, output):
    x, groups, weight, bias, act, eps = inputs
    ctx.groups, ctx.act = groups, act
    ctx.given = [t is not None for t in (weight, bias)]
    ctx.save_for_backward(x, output[1], *[t for t in (weight, bias) if t is not None])
    ctx.set_materialize_grads(False)


def _group_norm_grad(ctx, dy, dstats):
    if dstats is not None:
        raise NotImplementedError("nsw.group_norm: the statistics have no gradient of their own")
    if dy is None:
        return (None,) * 6
    x, stats, *rest = ctx.saved_tensors
    rest = iter(rest)
    weight, bias = (next(rest) if g else None for g in ctx.given)
    need = [ctx.needs_input_grad[0], ctx.needs_input_grad[2], ctx.needs_input_grad[3]]
    got = torch.ops.nsw.group_norm_backward(dy, x, stats, ctx.groups, weight, bias, ctx.act, need)
    dx, dw, db = (g if n else None for n, g in zip(need, got))
    return dx, None, dw, db, None, None


_group_norm.register_autograd(_group_norm_grad, setup_context=_group_norm_setup)


def group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               act: str = "none", eps: float = 1e-5) -> torch.Tensor:
    """torch.ops.nsw.group_norm with ops.group_norm's defaults: y alone."""
    return torch.ops.nsw.group_norm(x, int(groups), weight, bias, act, float(eps))[0]


@torch.library.custom_op("nsw::linear_to_window", mutates_args=())
def linear_to_window(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, residual: torch.Tensor,
                     image: List[int], window_size: List[int], shift_size: List[int]) -> Tuple[torch.Tensor,
                                                                                               torch.Tensor]:
    """(y, row_sumsq): token-ordered rows x . weight^T + bias + residual stored
    in the window order of image (B, T, H, W) rolled by -shift, with the
    stored rows' partial sums of squares (nsw_linear_remap_residual mode 3)."""
    return ops.linear_remap_residual(x.contiguous(), weight.contiguous(), bias.contiguous(), residual.contiguous(),
                                     3, image=tuple(image), window_size=tuple(window_size),
                                     shift_size=tuple(shift_size))


@linear_to_window.register_fake
def _(x, weight, bias, residual, image, window_size, shift_size):
    M, N = x.numel() // x.shape[-1], weight.shape[0]
    P = (N * x.element_size() + 511) // 512
    return x.new_empty((M, N)), x.new_empty((M, P), dtype=torch.float32)


def linear_epi(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, epilogue: Optional[int] = None,
               left_out: Sequence[Optional[torch.Tensor]] = ()) -> torch.Tensor:
    """torch.ops.nsw.linear with ops.linear's default epilogue (none / bias / bias + residual).
    ``left_out``: parameters that the arguments were formed from outside the graph (packed,
    detached).  Where one of them needs a gradient the product has none, so that a backward
    pass raises instead of leaving theirs out."""
    if epilogue is None:
        epilogue = _lib.NSW_EPI_NONE if bias is None else (
            _lib.NSW_EPI_BIAS if residual is None else _lib.NSW_EPI_BIAS_RESIDUAL)
    whole = not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in left_out))
    return (torch.ops.nsw.linear if whole else torch.ops.nsw.linear_forward)(x, weight, bias, residual, int(epilogue))


@torch.library.custom_op("nsw::rms_norm", mutates_args=())
def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    return ops.rms_norm(x.contiguous(), weight.contiguous(), eps)


@rms_norm.register_fake
def _(x, weight, eps):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


@torch.library.custom_op("nsw::layer_norm", mutates_args=())
def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
               eps: float) -> torch.Tensor:
    return ops.layer_norm(x.contiguous(), weight, bias, eps)


@layer_norm.register_fake
def _(x, weight, bias, eps):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


# -------------------------------------------------------------- attention ---

@torch.library.custom_op("nsw::qkv_projection", mutates_args=())
def qkv_projection(x: torch.Tensor, wqkv: torch.Tensor, bqkv: torch.Tensor, qn_w: torch.Tensor,
                   kn_w: torch.Tensor, num_heads: int, eps: float) -> torch.Tensor:
    return ops.qkv_projection(x.contiguous(), wqkv, bqkv, qn_w, kn_w, num_heads, eps)


@qkv_projection.register_fake
def _(x, wqkv, bqkv, qn_w, kn_w, num_heads, eps):
    return x.new_empty(tuple(x.shape[:-1]) + (3 * x.shape[-1],))


@torch.library.custom_op("nsw::window_attention", mutates_args=())
def window_attention(qkv: torch.Tensor, num_heads: int, scale: float, mask: Optional[torch.Tensor],
                     geometry: List[int]) -> torch.Tensor:
    """geometry = [H, W, ws0, ws1, s0, s1, T] (shift mask from indices) or []."""
    geo = None
    if len(geometry) == 7:
        H, W, ws0, ws1, s0, s1, T = geometry
        geo = (H, W, (ws0, ws1), (s0, s1), T)
    elif len(geometry) != 0:
        raise ValueError("window_attention: geometry is [H, W, ws0, ws1, s0, s1, T] or empty")
    return ops.window_attention(qkv.contiguous(), num_heads, scale,
                                mask=None if mask is None else mask.contiguous(), geometry=geo)


@window_attention.register_fake
def _(qkv, num_heads, scale, mask, geometry):
    Bw, L, C3 = qkv.shape
    return qkv.new_empty((Bw, L, C3 // 3))


def _position_geometry(geometry: List[int]):
    if len(geometry) == 7:
        H, W, ws0, ws1, s0, s1, T = geometry
        return (H, W, (ws0, ws1), (s0, s1), T)
    if len(geometry) != 0:
        raise ValueError("position_attention: geometry is [H, W, ws0, ws1, s0, s1, T] or empty")
    return None


@torch.library.custom_op("nsw::position_attention", mutates_args=())
def _position_attention(qkv: torch.Tensor, num_heads: int, scale: float, table: torch.Tensor, buckets: torch.Tensor,
                        extent: List[int], mask: Optional[torch.Tensor], geometry: List[int]
                        ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(o, stats): window_attention with a learned position bias; geometry = [H, W, ws0, ws1, s0, s1, T] or []."""
    return ops.position_attention(_dense(qkv), num_heads, scale, table.contiguous(), buckets.contiguous(), tuple(extent),
                                  mask=None if mask is None else mask.contiguous(), geometry=_position_geometry(geometry))


@_position_attention.register_fake
def _(qkv, num_heads, scale, table, buckets, extent, mask, geometry):
    Bw, L, C3 = qkv.shape
    return (qkv.new_empty((Bw, L, C3 // 3)),
            qkv.new_empty((Bw, num_heads, L, ops.position_stats_width(qkv, num_heads)), dtype=torch.float32))


@torch.library.custom_op("nsw::position_attention_backward", mutates_args=())
def _position_attention_backward(do: torch.Tensor, qkv: torch.Tensor, o: torch.Tensor, stats: torch.Tensor, num_heads: int,
                                 scale: float, table: torch.Tensor, buckets: torch.Tensor, extent: List[int],
                                 mask: Optional[torch.Tensor], geometry: List[int], needs: List[bool]
                                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dqkv, dtable); empty ([0]) where ``needs`` is False."""
    return _or_empty(qkv, *ops.position_attention_backward(
        _dense(do), _dense(qkv), _dense(o), stats.contiguous(), num_heads, scale, table.contiguous(), buckets.contiguous(),
        tuple(extent), mask=None if mask is None else mask.contiguous(), geometry=_position_geometry(geometry),
        needs=tuple(needs)))


@_position_attention_backward.register_fake
def _(do, qkv, o, stats, num_heads, scale, table, buckets, extent, mask, geometry, needs):
    return qkv.new_empty(qkv.shape if needs[0] else (0,)), qkv.new_empty(table.shape if needs[1] else (0,))


def _position_setup(ctx, inputs, output):
    qkv, num_heads, scale, table, buckets, extent, mask, geometry = inputs
    ctx.rest = (num_heads, scale, list(extent), list(geometry))
    ctx.masked = mask is not None
    ctx.save_for_backward(qkv, table, buckets, *output, *([mask] if mask is not None else []))
    ctx.set_materialize_grads(False)


def _position_backward(ctx, do, dstats):
    if dstats is not None:
        raise NotImplementedError("nsw.position_attention: the row statistics have no gradient of their own")
    if ctx.needs_input_grad[6]:
        raise NotImplementedError("nsw.position_attention: the mask has no gradient (a learned bias is a table's)")
    if do is None:
        return (None,) * 8
    qkv, table, buckets, o, stats, *rest = ctx.saved_tensors
    num_heads, scale, extent, geometry = ctx.rest
    need = [ctx.needs_input_grad[0], ctx.needs_input_grad[3]]
    got = torch.ops.nsw.position_attention_backward(do, qkv, o, stats, num_heads, scale, table, buckets, extent,
                                                    rest[0] if ctx.masked else None, geometry, need)
    dqkv, dtable = (g if n else None for n, g in zip(need, got))
    return dqkv, None, None, dtable, None, None, None, None


_position_attention.register_autograd(_position_backward, setup_context=_position_setup)


def position_attention(qkv: torch.Tensor, num_heads: int, scale: float, table: torch.Tensor, buckets: torch.Tensor,
                       extent: Sequence[int], mask: Optional[torch.Tensor] = None, geometry=None) -> torch.Tensor:
    """torch.ops.nsw.position_attention with ops.position_attention's arguments: o alone."""
    geo = []
    if geometry is not None:
        H, W, ws, sh, T = geometry
        geo = [int(H), int(W), int(ws[0]), int(ws[1]), int(sh[0]), int(sh[1]), int(T)]
    return torch.ops.nsw.position_attention(qkv, int(num_heads), float(scale), table, buckets, [int(e) for e in extent], mask,
                                            geo)[0]


# ------------------------------------------------------------ window maps ---

@torch.library.custom_op("nsw::window_partition", mutates_args=())
def window_partition(x: torch.Tensor, window_size: List[int]) -> torch.Tensor:
    return ops.window_partition(x.contiguous(), tuple(window_size))


@window_partition.register_fake
def _(x, window_size):
    B, T, H, W, C = x.shape
    return x.new_empty((B * (H // window_size[0]) * (W // window_size[1]), T, window_size[0], window_size[1], C))


@torch.library.custom_op("nsw::window_reverse", mutates_args=())
def window_reverse(windows: torch.Tensor, window_size: List[int], img_size: List[int]) -> torch.Tensor:
    return ops.window_reverse(windows.contiguous(), tuple(window_size), tuple(img_size))


@window_reverse.register_fake
def _(windows, window_size, img_size):
    T, C = windows.shape[1], windows.shape[-1]
    H, W = img_size
    B = windows.shape[0] // ((H // window_size[0]) * (W // window_size[1]))
    return windows.new_empty((B, T, H, W, C))


def _partition_setup(ctx, inputs, output):
    x, window_size, *rest = inputs
    ctx.image = [int(x.shape[2]), int(x.shape[3])]
    ctx.window, ctx.shift = list(window_size), list(rest[0]) if rest else [0, 0]


def _partition_backward(ctx, dw):
    # a permutation of rows: the other map
    dx = torch.ops.nsw.window_reverse_roll(dw, ctx.window, ctx.image, ctx.shift)
    return (dx,) + (None,) * (len(ctx.needs_input_grad) - 1)


def _reverse_setup(ctx, inputs, output):
    _, window_size, _, *rest = inputs
    ctx.window, ctx.shift = list(window_size), list(rest[0]) if rest else [0, 0]


def _reverse_backward(ctx, dx):
    dw = torch.ops.nsw.roll_window_partition(dx, ctx.window, ctx.shift)
    return (dw,) + (None,) * (len(ctx.needs_input_grad) - 1)


@torch.library.custom_op("nsw::roll_hw", mutates_args=())
def roll_hw(x: torch.Tensor, shifts: List[int]) -> torch.Tensor:
    return ops.roll_hw(x.contiguous(), tuple(shifts))


@roll_hw.register_fake
def _(x, shifts):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


@torch.library.custom_op("nsw::roll_window_partition", mutates_args=())
def roll_window_partition(x: torch.Tensor, window_size: List[int], shift_size: List[int]) -> torch.Tensor:
    return ops.roll_window_partition(x.contiguous(), tuple(window_size), tuple(shift_size))


@roll_window_partition.register_fake
def _(x, window_size, shift_size):
    B, T, H, W, C = x.shape
    return x.new_empty((B * (H // window_size[0]) * (W // window_size[1]), T, window_size[0], window_size[1], C))


@torch.library.custom_op("nsw::window_reverse_roll", mutates_args=())
def window_reverse_roll(windows: torch.Tensor, window_size: List[int], img_size: List[int],
                        shift_size: List[int]) -> torch.Tensor:
    return ops.window_reverse_roll(windows.contiguous(), tuple(window_size), tuple(img_size), tuple(shift_size))


@window_reverse_roll.register_fake
def _(windows, window_size, img_size, shift_size):
    T, C = windows.shape[1], windows.shape[-1]
    H, W = img_size
    B = windows.shape[0] // ((H // window_size[0]) * (W // window_size[1]))
    return windows.new_empty((B, T, H, W, C))


for _op in (window_partition, roll_window_partition):
    _op.register_autograd(_partition_backward, setup_context=_partition_setup)
for _op in (window_reverse, window_reverse_roll):
    _op.register_autograd(_reverse_backward, setup_context=_reverse_setup)


# ----------------------------------------------------------- model layout ---

@torch.library.custom_op("nsw::patch_im2col", mutates_args=())
def patch_im2col(x: torch.Tensor, p: int, Kp: int, dtype: torch.dtype, invariants: Optional[torch.Tensor],
                 frame0: int) -> torch.Tensor:
    return ops.patch_im2col(x.contiguous(), p, Kp, dtype,
                            invariants=None if invariants is None else invariants.contiguous(), frame0=frame0)


@patch_im2col.register_fake
def _(x, p, Kp, dtype, invariants, frame0):
    B, T, _, H, W = x.shape
    return x.new_empty((B * T * (H // p) * (W // p), Kp), dtype=dtype)


@torch.library.custom_op("nsw::unpatchify", mutates_args=())
def unpatchify(y: torch.Tensor, B: int, C_out: int, H: int, W: int, p: int,
               dtype: Optional[torch.dtype]) -> torch.Tensor:
    return ops.unpatchify(y.contiguous(), B, C_out, H, W, p, dtype=dtype)


@unpatchify.register_fake
def _(y, B, C_out, H, W, p, dtype):
    return y.new_empty((B, 1, C_out, H, W), dtype=dtype if dtype is not None else y.dtype)


@torch.library.custom_op("nsw::head_unpatchify", mutates_args=())
def head_unpatchify(x: torch.Tensor, w_perm: torch.Tensor, B: int, C_out: int, H: int, W: int, p: int,
                    dtype: Optional[torch.dtype]) -> torch.Tensor:
    """The head GEMM with the head layout in its write-out (w_perm from ops.head_weight_perm)."""
    return ops.head_unpatchify(x.contiguous(), w_perm.contiguous(), B, C_out, H, W, p, dtype=dtype)


@head_unpatchify.register_fake
def _(x, w_perm, B, C_out, H, W, p, dtype):
    return x.new_empty((B, 1, C_out, H, W), dtype=dtype if dtype is not None else x.dtype)


@torch.library.custom_op("nsw::skip_conv_accumulate", mutates_args=("out",))
def skip_conv_accumulate(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor, invariants: Optional[torch.Tensor],
                         frame0: int) -> None:
    """The model's big skip added in place to its predicted frame."""
    ops.skip_conv_accumulate(x, weight, out, invariants=invariants, frame0=frame0)


@skip_conv_accumulate.register_fake
def _(x, weight, out, invariants, frame0):
    return None


# ---------------------------------------------------------------- metrics ---

@torch.library.custom_op("nsw::weighted_metrics", mutates_args=())
def weighted_metrics(pred: torch.Tensor, target: torch.Tensor, weights: torch.Tensor,
                     clim: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """(rmse, acc) float64 [B, T, C]; acc is empty ([0]) without a climatology."""
    rmse, acc = ops.weighted_metrics(pred.contiguous(), target.contiguous(), weights, clim)
    if acc is None:
        acc = rmse.new_empty((0,))
    return rmse, acc


@weighted_metrics.register_fake
def _(pred, target, weights, clim):
    B, T, C = pred.shape[:3]
    rmse = pred.new_empty((B, T, C), dtype=torch.float64)
    acc = pred.new_empty((B, T, C) if clim is not None else (0,), dtype=torch.float64)
    return rmse, acc
