"""nsw.Fp8Linear's own checks, without a GPU (meta tensors)."""
import copy

import pytest
import torch

import nsw


def meta(*shape):
    return torch.empty(*shape, device="meta", dtype=torch.bfloat16)


@pytest.mark.parametrize("K", [136, 208, 256, 72])
def test_rows_of_another_width_are_refused(K):
    """Widths that the quantiser pads to the same 256 bytes (or others) as the weight's 200."""
    lin = nsw.Fp8Linear(meta(64, 200), meta(64))
    for layer in (lin, copy.deepcopy(lin)):
        with pytest.raises(ValueError, match="200"):
            layer(meta(3, K))
        assert layer(meta(2, 3, 200)).shape == (2, 3, 64)
    assert set(lin.state_dict()) == {"weight", "weight_scale", "bias"}


def test_mlp_refuses_rows_of_another_width():
    mlp = nsw.MLP(200, 328).to(device="meta", dtype=torch.bfloat16).to_fp8()
    assert mlp(meta(3, 200)).shape == (3, 200)
    with pytest.raises(ValueError, match="200"):
        mlp(meta(3, 256))
