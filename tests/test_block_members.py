"""Feed-forward modules that the fused block does not run are refused by name."""
import pytest
import torch

import nsw


@pytest.mark.parametrize("make", [lambda: nsw.GatedMLP(32, 128), lambda: torch.nn.Linear(32, 32)])
def test_block_refuses_other_feed_forward_modules(make):
    blk = nsw.Block(32, 2, (18, 36), (9, 18), 1).eval()
    blk.mlp = make()
    x = torch.zeros(1, 1, 18, 36, 32)
    with pytest.raises(NotImplementedError, match="GELU MLP.*" + type(blk.mlp).__name__):
        blk(x)


def test_block_keeps_its_own_checks():
    blk = nsw.Block(32, 2, (18, 36), (9, 18), 1, drop=0.1).train()
    with pytest.raises(NotImplementedError, match="dropout"):
        blk(torch.zeros(1, 1, 18, 36, 32))
