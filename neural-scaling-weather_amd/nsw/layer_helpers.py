"""Parameter wrappers with the reference's names (models/layer_helpers.py:8-119).

Same attributes and state-dict keys as the reference (``weight`` of
``LinearLayer``, ``bias`` of ``BiasLayer``, ``norm.weight`` of ``NormLayer``)
and the same init (trunc-normal std 0.02, zero bias, unit norm weight); the
forward passes run libnsw kernels.  ``comm_metadata`` is kept as an attribute
for API compatibility (every communicator has size 1 here).
"""
from __future__ import annotations

import math

import torch
from torch import nn

from . import _lib, ops, torch_ops

def submodule(module, name: str):
    """``module.name`` for a registered submodule, without the failed instance
    lookup and the Python-level nn.Module.__getattr__ that the attribute takes
    each time.  Whatever is not in the module's own table (a parametrised,
    wrapped or replaced member) is looked up as the attribute.  Block.packed
    looks at 16 parameters on every call: 16 us this way, 39 by attributes on
    one host; a 648-token block, bound by the host, 73 -> 61 us."""
    try:
        m = module._modules.get(name)
    except AttributeError:
        m = None
    return getattr(module, name) if m is None else m


def parameter(module, name: str):
    """``module.name`` for a registered parameter, as ``submodule``."""
    try:
        p = module._parameters.get(name)
    except AttributeError:
        p = None
    return getattr(module, name) if p is None else p


_DEFAULT_META = {"sharded": [None, None], "shared": [], "reduce": []}


def trunc_normal_(tensor: torch.Tensor, mean: float = 0.0, std: float = 1.0, a: float = -2.0,
                  b: float = 2.0) -> torch.Tensor:
    """Truncated normal by the inverse-CDF method with absolute bounds [a, b]
    (models/timm_helpers.py:46-98)."""
    def cdf(v):
        return (1.0 + math.erf(v / math.sqrt(2.0))) / 2.0
    lo, hi = cdf((a - mean) / std), cdf((b - mean) / std)
    with torch.no_grad():
        tensor.uniform_(2 * lo - 1, 2 * hi - 1)
        tensor.erfinv_()
        tensor.mul_(std * math.sqrt(2.0)).add_(mean)
        tensor.clamp_(min=a, max=b)
    return tensor


class LinearLayer(nn.Module):
    """Bias-free ``F.linear`` (models/layer_helpers.py:8-42)."""

    def __init__(self, in_features, out_features, comm_metadata=None):
        super().__init__()
        self.weight = nn.Parameter(torch.empty((out_features, in_features)))
        self.weight.comm_metadata = comm_metadata or dict(_DEFAULT_META)
        trunc_normal_(self.weight, std=0.02)

    def forward(self, x):
        return torch_ops.linear_epi(x, self.weight)


class BiasLayer(nn.Module):
    """Separate bias add (models/layer_helpers.py:45-72)."""

    def __init__(self, dim, comm_metadata=None):
        super().__init__()
        self.bias = nn.Parameter(torch.zeros(dim))
        self.bias.comm_metadata = comm_metadata or {"sharded": [None], "shared": [], "reduce": []}

    def forward(self, x):
        # y = x . I^T + b would waste a GEMM; the blocks fuse the bias into the
        # producing GEMM's epilogue instead.  Stand-alone use is a broadcast add.
        return x + self.bias


class NormLayer(nn.Module):
    """``NormLayer`` (models/layer_helpers.py:75-119): ``rms_norm`` runs the
    libnsw RMSNorm kernel, ``layer_norm`` the libnsw LayerNorm kernel (same
    parameters and eps as the wrapped nn.RMSNorm / nn.LayerNorm)."""

    def __init__(self, normalized_shape, elementwise_affine=True, norm_type="layer_norm",
                 comm_metadata=None):
        super().__init__()
        self.norm_type = norm_type
        if norm_type == "layer_norm":
            self.norm = nn.LayerNorm(normalized_shape, elementwise_affine=elementwise_affine, bias=True)
        elif norm_type == "rms_norm":
            self.norm = nn.RMSNorm(normalized_shape, elementwise_affine=elementwise_affine)
        else:
            raise ValueError(f"Invalid norm type: {norm_type}")
        if elementwise_affine:
            meta = comm_metadata or {"sharded": [None], "shared": [], "reduce": []}
            self.norm.weight.comm_metadata = meta
            if norm_type == "layer_norm":
                self.norm.bias.comm_metadata = meta

    def forward(self, x):
        if self.norm_type == "layer_norm":
            n = self.norm
            if len(n.normalized_shape) != 1:
                raise NotImplementedError("libnsw normalises over the last dim only")
            return torch.ops.nsw.layer_norm(x, n.weight, n.bias, float(n.eps))
        w = self.norm.weight
        if w is None:
            w = torch.ones(x.shape[-1], dtype=x.dtype, device=x.device)
        eps = self.norm.eps
        return torch.ops.nsw.rms_norm(x, w, ops.default_eps(x.dtype) if eps is None else float(eps))


class ResidualNorm(nn.Module):
    """The end of one residual branch and the norm before the next, in one pass
    with gradients (no counterpart in the reference, whose blocks are pre-norm
    without gates): y = alpha * skip + gate * RMSNorm(branch) and z =
    RMSNorm(y).

    post_norm    a norm after the branch (``post_norm.norm.weight``)
    layer_scale  initial value of a learned gate for every channel (``gamma``),
                 None: no learned gate; a gate given to ``forward`` (of a
                 condition: [C], or [B, C] for B equal parts of the rows)
                 multiplies the branch instead
    alpha        scale of the residual
    next_norm    the norm before the next branch (``next_norm.norm.weight``);
                 without it z is None
    """

    def __init__(self, dim, post_norm=True, layer_scale=None, alpha=1.0, next_norm=True, comm_metadata=None):
        super().__init__()
        self.post_norm = NormLayer(dim, norm_type="rms_norm", comm_metadata=comm_metadata) if post_norm else None
        self.next_norm = NormLayer(dim, norm_type="rms_norm", comm_metadata=comm_metadata) if next_norm else None
        self.gamma = None if layer_scale is None else nn.Parameter(torch.full((dim,), float(layer_scale)))
        if self.gamma is not None:
            self.gamma.comm_metadata = comm_metadata or {"sharded": [None], "shared": [], "reduce": []}
        self.alpha = float(alpha)

    def forward(self, branch, skip, gate=None):
        norms = [n.norm for n in (self.post_norm, self.next_norm) if n is not None]
        eps = {n.eps for n in norms}
        if len(eps) > 1:
            raise NotImplementedError("the two norms of a ResidualNorm share eps")
        if gate is not None and self.gamma is not None:
            raise ValueError("ResidualNorm: a gate is given and a layer scale is learned")
        return torch_ops.residual_norm(branch, skip, None if self.post_norm is None else self.post_norm.norm.weight,
                                       self.gamma if gate is None else gate, self.alpha,
                                       None if self.next_norm is None else self.next_norm.norm.weight,
                                       eps.pop() if eps else None)


class Fp8Linear(nn.Module):
    """A linear layer served in 8-bit floating point: the weight is quantised
    once (e4m3, a power-of-two scale for each 128 x 128 block), the rows in
    every call (a scale for each 1 x 128 block); forward only.  ``epilogue`` as
    ``nsw.ops.linear``; the result has the input's dtype."""

    def __init__(self, weight: torch.Tensor, bias=None, epilogue=None):
        super().__init__()
        q, scale = torch.ops.nsw.quantize_fp8(weight.detach(), ops.FP8_BLOCK)
        self.register_buffer("weight", q)
        self.register_buffer("weight_scale", scale)
        self.in_features = weight.shape[1]      # the quantised rows are padded
        self.register_buffer("bias", None if bias is None else bias.detach().clone())
        self.epilogue = epilogue

    @classmethod
    def from_layers(cls, linear: LinearLayer, bias=None, epilogue=None):
        """Of a LinearLayer and the BiasLayer after it, if any."""
        return cls(linear.weight, None if bias is None else bias.bias, epilogue)

    def _apply(self, fn, recurse=True):
        # as bytes: a change of dtype (module.bfloat16()) is for the bias
        self.weight, self.weight_scale = (t.view(torch.uint8) for t in (self.weight, self.weight_scale))
        try:
            return super()._apply(fn, recurse)
        finally:
            self.weight, self.weight_scale = self.weight.view(torch.float8_e4m3fn), self.weight_scale.view(torch.float8_e8m0fnu)

    def forward(self, x, residual=None):
        if x.shape[-1] != self.in_features:
            raise ValueError(f"Fp8Linear: x has {x.shape[-1]} features, weight expects {self.in_features}")
        epi = self.epilogue
        if residual is not None and epi in (_lib.NSW_EPI_BIAS_GELU, _lib.NSW_EPI_BIAS_GELU_TANH):
            raise NotImplementedError("a residual after a GELU is not fused")
        if epi is None or residual is not None:
            epi = _lib.NSW_EPI_NONE if self.bias is None else (
                _lib.NSW_EPI_BIAS if residual is None else _lib.NSW_EPI_BIAS_RESIDUAL)
        if residual is not None and epi != _lib.NSW_EPI_BIAS_RESIDUAL:
            raise NotImplementedError("a residual without a bias is not fused")
        xq, xs = torch.ops.nsw.quantize_fp8(x, 1)
        return torch.ops.nsw.linear_fp8(xq, xs, self.weight, self.weight_scale, self.bias, residual, int(epi), x.dtype)
