"""nsw.ops.group_norm on samples of one workgroup, at every width (two 16-byte pieces of a row to a lane beyond 2048 bf16
or 1024 fp32 channels), and on either side of the sizes where a sample is shared.  Tolerances: test_gpu_group_norm's."""
import pytest
import torch

from test_gpu_group_norm import DTYPES, WIDTHS, case, check, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,C,groups", [(d, c, g) for d, cs in WIDTHS.items() for c, g in cs])
@pytest.mark.parametrize("B,R", [(1, 1), (3, 7), (2, 8), (1, 4)])
def test_a_workgroup_a_sample(device, dtype, C, groups, B, R):
    t = case(dtype, B, R, C, seed=C + R)
    check(run(t, groups, "silu", 1e-5, device), reference(t, groups, "silu", 1e-5), dtype)


# samples of 64 KB, of 96 KB from 128 of them on, of 192 KB from 256 of them on, and of a row more
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,kib", [(2, 64), (127, 64), (128, 96), (256, 192)])
@pytest.mark.parametrize("more", [0, 1])
def test_limits_of_a_workgroup(device, dtype, B, kib, more):
    C, groups = (4096, 32) if dtype == torch.bfloat16 else (2048, 2048)
    t = case(dtype, B, kib // 8 + more, C, seed=kib)
    check(run(t, groups, "gelu_tanh", 1e-5, device), reference(t, groups, "gelu_tanh", 1e-5), dtype)
