"""nsw — MI355X-native shifted-window Swin block of neural-scaling-weather.

Drop-in replacements for the reference's hot-path modules, running HIP
kernels for gfx950 from ``libnsw.so`` through its C ABI (include/nsw.h):

    from nsw import Block, WindowMultiHeadAttention, window_partition, window_reverse
    from nsw import WeightedRMSE, WeightedACC, build_spherical_area_weights
    from nsw import SwinTransformer, TimeStepper, Rollout
    from nsw import GatedMLP, ResidualNorm, GroupNorm, PositionAttentionBranch   # trained: with gradients
    from nsw import Fp8Linear, Fp8MLP                  # served in 8-bit floating point

Build the library first: ``python neural-scaling-weather_amd/build.py``.
"""
from .layer_helpers import BiasLayer, Fp8Linear, GroupNorm, LinearLayer, NormLayer, ResidualNorm, trunc_normal_
from .losses import WeightedACC, WeightedRMSE, weighted_rmse_acc
from .misc_utils import build_spherical_area_weights, create_dummy_metadata, get_spatial_coords
from .mlp import MLP, Fp8MLP, GatedMLP
from .swin_helpers import (Block, PositionAttentionBranch, PositionWindowAttention, RelativePositionBias,
                           SwinTransformerBlock, WindowAttention, WindowMultiHeadAttention, position_buckets,
                           roll_forward_reverseroll_backward, window_partition, window_reverse)
from .swin import Conv2DLayer, PatchEmbedLayer, SwinTransformer, TimeStepper, get_model
from .inference import Rollout
from . import checkpoint, ops, profiler_utils, torch_ops   # torch_ops registers torch.ops.nsw.*

__all__ = [
    "Block", "SwinTransformerBlock", "WindowMultiHeadAttention", "WindowAttention", "MLP",
    "LinearLayer", "BiasLayer", "NormLayer", "trunc_normal_", "window_partition", "window_reverse",
    "roll_forward_reverseroll_backward", "WeightedRMSE", "WeightedACC", "weighted_rmse_acc",
    "build_spherical_area_weights", "get_spatial_coords", "create_dummy_metadata", "checkpoint", "ops",
    "SwinTransformer", "PatchEmbedLayer", "Conv2DLayer", "TimeStepper", "get_model", "Rollout", "torch_ops",
    "profiler_utils", "GatedMLP", "ResidualNorm", "GroupNorm", "PositionAttentionBranch",
    "PositionWindowAttention", "RelativePositionBias", "position_buckets", "Fp8Linear", "Fp8MLP",
]
