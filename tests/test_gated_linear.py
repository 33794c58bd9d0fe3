"""Refusals of the gated linear and the linear gradients that need no GPU."""
import pytest
import torch

from nsw import _lib, ops

BF16, F32 = _lib.NSW_DTYPE_BF16, _lib.NSW_DTYPE_F32
P = 16     # an aligned address that nothing reads
BIG = 1 << 50


def forward(M=4, H=48, K=64, act=0, dtype=BF16, x=P, b=P):
    return _lib.lib().nsw_gated_linear(x, P, b, P, M, H, K, act, dtype, None)


def backward(M=4, H=48, K=64, act=0, dtype=BF16, dh=P, ws=P, nbytes=BIG, dx=P):
    return _lib.lib().nsw_gated_linear_backward(dh, P, P, P, dx, P, P, M, H, K, act, dtype, ws, nbytes, None)


def linear(M=4, N=96, K=64, dtype=BF16, dy=P, ws=P, nbytes=BIG, db=P):
    return _lib.lib().nsw_linear_backward(dy, P, P, P, P, db, M, N, K, dtype, ws, nbytes, None)


@pytest.mark.parametrize("call,kw,says", [
    (forward, dict(H=40), b"multiple of 16"), (forward, dict(K=48), b"multiple of 32"),
    (forward, dict(K=24, dtype=F32), b"multiple of 16"), (forward, dict(M=0), b"positive"), (forward, dict(act=3), b"activation"),
    (forward, dict(dtype=9), b"dtype"), (forward, dict(x=None), b"required"), (forward, dict(x=8), b"aligned"),
    (forward, dict(b=8), b"aligned"), (forward, dict(H=1 << 20, K=1024), b"2 GiB"),
    (backward, dict(H=40), b"multiple of 16"), (backward, dict(K=48), b"K of 32"), (backward, dict(M=0), b"M=0"),
    (backward, dict(act=-1), b"activation"), (backward, dict(dh=None), b"required"), (backward, dict(ws=None), b"workspace"),
    (backward, dict(nbytes=1000), b"workspace"), (backward, dict(dx=8), b"aligned"), (backward, dict(dtype=5), b"dtype 5"),
    (linear, dict(N=80), b"multiples of 32"), (linear, dict(K=72, dtype=F32), b"multiples of 32"), (linear, dict(M=-1), b"M=-1"),
    (linear, dict(dy=None), b"required"), (linear, dict(ws=None), b"workspace"), (linear, dict(nbytes=8), b"workspace"),
    (linear, dict(db=4), b"aligned"),
])
def test_refusals(call, kw, says):
    assert call(**kw) == _lib.NSW_ERR_INVALID
    assert says in _lib.lib().nsw_last_error(), _lib.lib().nsw_last_error()


def test_workspace_sizes():
    L = _lib.lib()
    assert L.nsw_gated_linear_backward_workspace_size(100, 48, 64, BF16) >= 100 * 96 * 2
    assert L.nsw_gated_linear_backward_workspace_size(100, 40, 64, BF16) == 0
    assert L.nsw_linear_backward_workspace_size(100, 96, 64, BF16) > 0
    assert L.nsw_linear_backward_workspace_size(100, 96, 60, BF16) == 0


def test_nothing_asked_for():
    L = _lib.lib()
    assert L.nsw_gated_linear_backward(P, P, P, P, None, None, None, 4, 48, 64, 0, BF16, P, BIG, None) == _lib.NSW_OK


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 64), torch.zeros(96, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.gated_linear(x, w)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.linear_backward(torch.zeros(4, 96), x, w)
