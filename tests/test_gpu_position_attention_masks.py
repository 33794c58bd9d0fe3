"""Mask tensors of nsw.ops.position_attention where rows of L floats do not end on 16 bytes: what a mask holds for
one query is nothing to the others."""
import math

import pytest
import torch

from test_gpu_position_attention import DTYPES, case, check, reference, run

pytestmark = pytest.mark.gpu

EXTENTS = [(1, 1, 2), (1, 3, 5), (1, 7, 7), (1, 1, 70), (1, 9, 18), (1, 1, 179), (1, 1, 191), (1, 1, 193), (2, 9, 18)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent", EXTENTS)
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_query_that_is_not_a_number(device, dtype, extent, value):
    """NaN or infinity at the first key of one query: the other queries and windows keep their bits."""
    L = math.prod(extent)
    t = case(dtype, 4, extent, 2, 32, seed=22)
    g = torch.Generator().manual_seed(23)
    m = torch.randn(2, L, L, generator=g)
    want = run(t, device, mask=m)
    bad = [i for i in range(L) if i % 2]
    m[0, bad, 0] = value
    got = run(t, device, mask=m)
    others = [i for i in range(L) if not i % 2]
    for name, parts in (("o", 64), ("dqkv", 64)):
        a, b = got[name][..., :parts], want[name][..., :parts]               # o, and of dqkv the queries' part
        assert torch.equal(a[::2, others], b[::2, others]), name
        assert a[::2, bad].isnan().all(), name
        assert torch.equal(got[name][1::2], want[name][1::2]), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extent", EXTENTS)
def test_the_last_values_of_a_mask(device, dtype, extent):
    """The last query may see its last key alone; the last key is hidden from all the others."""
    L = math.prod(extent)
    t = case(dtype, 4, extent, 2, 32, seed=24)
    m = torch.zeros(2, L, L)
    m[:, :, L - 1] = -math.inf
    m[:, L - 1] = -math.inf
    m[:, L - 1, L - 1] = 0.0
    check(run(t, device, mask=m), reference(t, m), dtype)
