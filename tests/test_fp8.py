"""Refusals of the 8-bit quantiser and product that need no GPU."""
import pytest
import torch

from nsw import _lib, ops

BF16, F32 = _lib.NSW_DTYPE_BF16, _lib.NSW_DTYPE_F32
P = 16     # an aligned address that nothing reads


def quantize(R=4, K=64, rows=1, dtype=BF16, x=P, s=P):
    return _lib.lib().nsw_quantize_fp8(x, P, s, R, K, rows, dtype, None)


def linear(M=4, N=64, K=128, epi=0, dtype=BF16, xq=P, b=P, r=P, xs=P):
    return _lib.lib().nsw_linear_fp8(xq, xs, P, P, b, r, P, M, N, K, epi, dtype, None)


@pytest.mark.parametrize("call,kw,says", [
    (quantize, dict(rows=64), b"1 or 128"), (quantize, dict(K=60), b"multiple of 8"),
    (quantize, dict(K=62, dtype=F32), b"multiple of 4"), (quantize, dict(R=0), b"R=0"), (quantize, dict(dtype=2), b"dtype"),
    (quantize, dict(x=None), b"required"), (quantize, dict(s=None), b"required"), (quantize, dict(x=8), b"aligned"),
    (linear, dict(K=192), b"multiple of 128"), (linear, dict(N=60), b"multiple of 8"), (linear, dict(M=0), b"positive"),
    (linear, dict(K=16256), b"at most"), (linear, dict(epi=9), b"epilogue"), (linear, dict(epi=1, b=None), b"bias"),
    (linear, dict(epi=3, r=None), b"residual"), (linear, dict(dtype=-1), b"dtype"), (linear, dict(xq=None), b"required"),
    (linear, dict(xs=None), b"required"), (linear, dict(r=24), b"aligned"),
])
def test_refusals(call, kw, says):
    assert call(**kw) == _lib.NSW_ERR_INVALID
    assert says in _lib.lib().nsw_last_error(), _lib.lib().nsw_last_error()


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        ops.quantize_fp8(torch.zeros(4, 128))
    q, s = torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.linear_fp8(q, s, q, s)
