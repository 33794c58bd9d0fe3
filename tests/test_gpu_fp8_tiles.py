"""Every kernel of nsw.ops.linear_fp8 at sizes that the choice by estimated time sends
there, asserted through nsw_linear_fp8_tile_rows: the 256 x 256 one (bf16 results), the
128 x 128 one in both types, with edges in both directions, odd counts of 128-blocks,
all epilogues, NaN scales and values.  Bounds as in test_gpu_fp8."""
import pytest
import torch

from nsw import _lib, ops
from test_gpu_fp8 import check, data, operands, reference

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def rows(M, N, K, dtype):
    return _lib.lib().nsw_linear_fp8_tile_rows(M, N, -(-K // 128) * 128, _lib.NSW_DTYPE_BF16 if dtype == BF16 else _lib.NSW_DTYPE_F32)


@pytest.mark.parametrize("epi", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("dtype,M,N,K,tile", [
    (BF16, 8100, 2040, 1600, 256), (BF16, 8065, 1928, 2000, 256), (BF16, 7937, 2048, 1664, 256),
    (BF16, 2500, 1336, 1000, 128), (BF16, 3001, 520, 256, 128), (BF16, 4001, 1544, 120, 128),
    (F32, 4051, 1336, 1000, 128), (F32, 2500, 1400, 1160, 128), (F32, 2049, 2056, 120, 128)])
def test_tiled_kernels(device, dtype, epi, M, N, K, tile):
    assert rows(M, N, K, dtype) == tile
    xq, wq, b, r = operands(device, M, N, K, dtype, seed=M + epi)
    y = ops.linear_fp8(*xq, *wq, None if epi == 0 else b, r if epi == 3 else None, epilogue=epi, dtype=dtype)
    want, tol = reference(xq, wq, b, r, epi, dtype)
    check(y, want, tol, dtype)


@pytest.mark.parametrize("dtype,M,N,K,tile", [(BF16, 8100, 2040, 1600, 256), (BF16, 2500, 1336, 1000, 128),
                                              (F32, 4051, 1336, 1000, 128)])
def test_what_is_not_a_number_stays_in_its_row(device, dtype, M, N, K, tile):
    """A scale of 255, a NaN value of x, and those of w in their column and its 128-row block of columns."""
    assert rows(M, N, K, dtype) == tile
    xq, wq, _, _ = operands(device, M, N, K, dtype)
    clean = ops.linear_fp8(*xq, *wq, dtype=dtype)
    xq[1].view(torch.uint8)[3, 1] = 255
    xq[0].view(torch.uint8)[M - 1, 5] = 0x7f
    wq[0].view(torch.uint8)[9, K - 1] = 0x7f
    wq[1].view(torch.uint8)[-1, 0] = 255
    y = ops.linear_fp8(*xq, *wq, dtype=dtype)
    last = (N - 1) // 128 * 128
    keep = torch.ones(M, N, dtype=torch.bool, device=device)
    keep[[3, M - 1]] = False
    keep[:, 9] = False
    keep[:, last:] = False
    assert torch.equal(y[keep], clean[keep]) and y[~keep].isnan().all()


@pytest.mark.parametrize("dtype,M,N,K,tile", [(BF16, 8100, 2040, 1600, 256), (F32, 4051, 1336, 1000, 128)])
def test_replays(device, dtype, M, N, K, tile):
    assert rows(M, N, K, dtype) == tile
    x = data(M, K, dtype).to(device)
    wq = ops.quantize_fp8(data(N, K, dtype, 1, False).to(device), rows=128)
    step = lambda: ops.linear_fp8(*ops.quantize_fp8(x), *wq, dtype=dtype)
    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for i in range(3):
        x.copy_(data(M, K, dtype, seed=20 + i))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_rows_past_32_bit_offsets_bit_for_bit(device):
    """x of more than 2^32 quantised bytes: the last rows are those of a call on them alone that takes the same kernel (a
    result depends on its row of x and column of w alone)."""
    M, K, N, n = 4_300_003, 1024, 264, 20_000
    assert rows(M, N, K, BF16) == rows(n, N, K, BF16) == 128
    x = torch.empty(M, K, dtype=BF16, device=device)
    x.random_(-6, 7)
    wq = ops.quantize_fp8(data(N, K, BF16, 1, False).to(device), rows=128)
    y = ops.linear_fp8(*ops.quantize_fp8(x), *wq)
    assert torch.equal(y[-n:], ops.linear_fp8(*ops.quantize_fp8(x[-n:].contiguous()), *wq))


def test_every_kernel_of_few_rows(device):
    for dtype in (BF16, F32):
        assert [rows(M, 1024, 512, dtype) for M in (1, 16, 17, 32, 33, 64)] == [16, 16, 32, 32, 64, 64]
