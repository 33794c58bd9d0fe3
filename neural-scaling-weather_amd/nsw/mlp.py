"""``MLP`` (models/mlp.py:14-95): fc1 -> +bias1 -> GELU -> fc2 -> +bias2.

Two libnsw GEMM launches: fc1 with the bias + GELU epilogue, fc2 with the
bias epilogue.  The GELU is ``act_layer``'s: nn.GELU() (exact erf, the
reference's default) or nn.GELU(approximate="tanh") (the form of the
reference's Transformer-Engine block, models/swin_helpers_te.py:318-323).
Dropout is the identity in eval (p = 0 in every config); a training-mode
dropout with p > 0 is not implemented and raises.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib, torch_ops
from .layer_helpers import BiasLayer, Fp8Linear, LinearLayer
from .profiler_utils import profile


class MLP(nn.Module):
    def __init__(self, in_features, hidden_features=None, out_features=None, act_layer=nn.GELU, drop=0.0):
        super().__init__()
        out_features = out_features or in_features
        hidden_features = hidden_features or in_features
        self.fc1 = LinearLayer(in_features, hidden_features,
                               comm_metadata={"sharded": ["tp", None], "shared": ["sp1-sp2"], "reduce": ["sp1-sp2"]})
        self.bias1 = BiasLayer(hidden_features,
                               comm_metadata={"sharded": ["tp"], "shared": ["sp1-sp2"], "reduce": ["sp1-sp2"]})
        self.act = act_layer()
        self.fc2 = LinearLayer(hidden_features, out_features,
                               comm_metadata={"sharded": [None, "tp"], "shared": ["sp1-sp2"], "reduce": ["sp1-sp2"]})
        self.bias2 = BiasLayer(out_features,
                               comm_metadata={"sharded": [], "shared": ["tp-sp1-sp2"], "reduce": ["sp1-sp2"]})
        self.drop = nn.Dropout(drop)

    def _check_fusable(self):
        if not (isinstance(self.act, nn.GELU) and self.act.approximate in ("none", "tanh")):
            raise NotImplementedError("libnsw fuses nn.GELU (approximate 'none' or 'tanh') only")
        if self.training and self.drop.p > 0:
            raise NotImplementedError("dropout with p > 0 in training mode is not implemented")

    @property
    def gelu_tanh(self) -> bool:
        return self.act.approximate == "tanh"

    @property
    def gelu_epilogue(self) -> int:
        return _lib.NSW_EPI_BIAS_GELU_TANH if self.gelu_tanh else _lib.NSW_EPI_BIAS_GELU

    def to_fp8(self) -> "Fp8MLP":
        """This MLP for serving in 8-bit floating point (the weights quantised now)."""
        return Fp8MLP(self)

    @profile("mlp")
    def forward(self, x, residual=None):
        """``residual`` (same shape as the output) is added in fc2's epilogue;
        the reference adds the block's skip right after the MLP
        (models/swin_helpers.py:456)."""
        self._check_fusable()
        x = x.contiguous()
        h = torch_ops.linear_epi(x, self.fc1.weight, self.bias1.bias, epilogue=self.gelu_epilogue)
        if residual is None:
            return torch_ops.linear_epi(h, self.fc2.weight, self.bias2.bias, epilogue=_lib.NSW_EPI_BIAS, left_out=(h,))
        return torch_ops.linear_epi(h, self.fc2.weight, self.bias2.bias, residual=residual,
                                    epilogue=_lib.NSW_EPI_BIAS_RESIDUAL, left_out=(h,))


class Fp8MLP(nn.Module):
    """``MLP`` with both products in 8-bit floating point (``Fp8Linear``): fc1
    with the bias + GELU epilogue, fc2 with the bias (and residual); forward
    only."""

    def __init__(self, mlp: MLP):
        super().__init__()
        mlp._check_fusable()
        self.fc1 = Fp8Linear.from_layers(mlp.fc1, mlp.bias1, mlp.gelu_epilogue)
        self.fc2 = Fp8Linear.from_layers(mlp.fc2, mlp.bias2)

    @profile("mlp")
    def forward(self, x, residual=None):
        return self.fc2(self.fc1(x), residual)


class GatedMLP(nn.Module):
    """A gated feed-forward block: fc2(act(g) * u) + bias2 with [g, u] = fc1(x) +
    bias1, the interface and initialisation of ``MLP`` (no counterpart in the
    reference).  fc1 holds the gate's rows over the up projection's
    ([2 hidden, in]); one kernel runs both projections, the activation and
    the product, one the down projection with bias and residual.  Has
    gradients.  act_layer: nn.SiLU or nn.GELU (approximate "none" or "tanh")."""

    def __init__(self, in_features, hidden_features=None, out_features=None, act_layer=nn.SiLU, drop=0.0):
        super().__init__()
        out_features = out_features or in_features
        hidden_features = hidden_features or in_features
        col = {"sharded": ["tp", None], "shared": ["sp1-sp2"], "reduce": ["sp1-sp2"]}
        self.fc1 = LinearLayer(in_features, 2 * hidden_features, comm_metadata=col)
        self.bias1 = BiasLayer(2 * hidden_features,
                               comm_metadata={"sharded": ["tp"], "shared": ["sp1-sp2"], "reduce": ["sp1-sp2"]})
        self.act = act_layer()
        self.fc2 = LinearLayer(hidden_features, out_features,
                               comm_metadata={"sharded": [None, "tp"], "shared": ["sp1-sp2"], "reduce": ["sp1-sp2"]})
        self.bias2 = BiasLayer(out_features,
                               comm_metadata={"sharded": [], "shared": ["tp-sp1-sp2"], "reduce": ["sp1-sp2"]})
        self.drop = nn.Dropout(drop)

    @property
    def act_name(self) -> str:
        if isinstance(self.act, nn.SiLU):
            return "silu"
        if isinstance(self.act, nn.GELU) and self.act.approximate in ("none", "tanh"):
            return "gelu" if self.act.approximate == "none" else "gelu_tanh"
        raise NotImplementedError("libnsw gates with nn.SiLU or nn.GELU (approximate 'none' or 'tanh')")

    @profile("mlp")
    def forward(self, x, residual=None):
        """``residual`` (same shape as the output) is added in fc2's epilogue."""
        if self.training and self.drop.p > 0:
            raise NotImplementedError("dropout with p > 0 in training mode is not implemented")
        h = torch.ops.nsw.gated_linear(x, self.fc1.weight, self.bias1.bias, self.act_name)
        return torch_ops.linear_epi(h, self.fc2.weight, self.bias2.bias, residual=residual)
