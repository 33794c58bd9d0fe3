"""The 8-bit linear's choice of kernel as the host query states it (no GPU)."""
from nsw import _lib

BF16, F32 = _lib.NSW_DTYPE_BF16, _lib.NSW_DTYPE_F32


def rows(M, N, K, dtype=BF16):
    return _lib.lib().nsw_linear_fp8_tile_rows(M, N, K, dtype)


def test_every_kernel_is_chosen():
    sizes = [(M, N, K) for M in (1, 17, 64, 648, 8100, 64800) for N in (8, 1024, 4096) for K in (128, 1024, 4096)]
    assert {rows(*s) for s in sizes} == {16, 32, 64, 128, 256}
    assert {rows(*s, F32) for s in sizes} == {16, 32, 64, 128}


def test_large_products_take_the_large_tile():
    assert rows(64800, 4096, 1024) == 256 and rows(64800, 1024, 4096) == 256 and rows(1, 4096, 1024) == 16


def test_refused():
    assert rows(0, 8, 128) == 0 and rows(4, 12, 128) == 0 and rows(4, 8, 192) == 0 and rows(4, 8, 16256) == 0
    assert rows(4, 8, 128, 9) == 0 and rows(1 << 38, 8, 128) == 0
