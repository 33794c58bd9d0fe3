"""Large tables of nsw.ops.position_attention."""
import pytest
import torch

from nsw import ops

from test_gpu_position_attention import case, check, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,nb,heads", [(torch.bfloat16, 1 << 22, 64), (torch.float32, (1 << 22) + 77, 64), (torch.bfloat16, (1 << 24) - 1, 2)])
def test_a_table_of_very_many_buckets(device, dtype, nb, heads):
    """As many values as 2^28 and more: the buckets that displacements have, and zeros in all the others."""
    extent, hd = (1, 3, 5), 4
    R = ops.window_displacements(extent)
    g = torch.Generator().manual_seed(40)
    used = torch.unique(torch.cat([torch.tensor([0, nb - 1]), torch.randint(0, nb, (R - 5,), generator=g)]))
    at = torch.randint(0, len(used), (R,), generator=g)
    at[:2] = torch.tensor([0, len(used) - 1])
    t = case(dtype, 2, extent, heads, hd, seed=41, buckets=at.int(), nb=len(used))
    d = {k: t[k].to(device) for k in ("qkv", "do")}
    table = torch.zeros(nb, heads, dtype=dtype, device=device)
    table[used.to(device)] = t["table"].to(device)
    args = (heads, t["scale"], table, used[at].int().to(device), extent)
    o, stats = ops.position_attention(d["qkv"], *args)
    dqkv, dtable = ops.position_attention_backward(d["do"], d["qkv"], o, stats, *args)
    del table
    rows = dtable[used.to(device)]
    check({"o": o, "dqkv": dqkv, "dtable": rows}, reference(t), dtype)
    dtable[used.to(device)] = 0
    assert not any(part.any() for part in dtable.split(1 << 20))
