"""Refusals of the residual norm that need no GPU: the C entry points check their
arguments before any launch, the tensor functions theirs before the library."""
import pytest
import torch

from nsw import _lib, ops

BF16, F32 = _lib.NSW_DTYPE_BF16, _lib.NSW_DTYPE_F32
P = 16     # an aligned address that nothing reads


def forward(rows=4, C=64, G=1, dtype=BF16, gate=P, norm=P, z=P, y=P, branch=P):
    return _lib.lib().nsw_residual_norm(branch, P, P, gate, norm, y, z, rows, C, G, 1.0, 1e-5, dtype, None)


def backward(rows=4, C=64, G=1, dtype=BF16, gate=P, norm=P, dz=P, dy=P, dgate=P, ws=P, nbytes=1 << 40, post=P, dpost=P):
    return _lib.lib().nsw_residual_norm_backward(dy, dz, P, P, post, gate, norm, P, P, dpost, dgate, P if norm else None,
                                                 rows, C, G, 1.0, 1e-5, dtype, ws, nbytes, None)


@pytest.mark.parametrize("call,kw,says", [
    (forward, dict(C=60), b"multiple of 8"), (forward, dict(C=62, dtype=F32), b"multiple of 4"),
    (forward, dict(C=8200), b"at most 8192"), (forward, dict(C=4100, dtype=F32), b"at most 4096"),
    (forward, dict(C=0), b"C=0"), (forward, dict(rows=-1), b"rows"), (forward, dict(rows=5, G=2), b"multiple of the gate"),
    (forward, dict(G=0), b"G=0"), (forward, dict(G=1 << 17, rows=1 << 17), b"at most 65536"), (forward, dict(G=2, gate=None), b"without a gate"), (forward, dict(dtype=7), b"dtype"),
    (forward, dict(norm=None), b"z is written"), (forward, dict(z=None), b"z is written"),
    (forward, dict(branch=None), b"required"), (forward, dict(y=24), b"aligned"),
    (backward, dict(C=60), b"multiple of 8"), (backward, dict(rows=5, G=2), b"multiple of the gate"),
    (backward, dict(dy=None, dz=None, norm=None), b"dy or dz"), (backward, dict(dz=None), b"go together"),
    (backward, dict(gate=None), b"not given"), (backward, dict(post=None), b"not given"),
    (backward, dict(ws=None), b"workspace"), (backward, dict(nbytes=64), b"workspace"), (backward, dict(ws=8), b"aligned"),
])
def test_refusals(call, kw, says):
    assert call(**kw) == _lib.NSW_ERR_INVALID
    assert says in _lib.lib().nsw_last_error()


def test_workspace_size():
    size = _lib.lib().nsw_residual_norm_backward_workspace_size
    assert size(4, 64, 1, BF16) >= 2 * 64 * 4
    assert size(129600, 1024, 2, BF16) % (2 * 2 * 1024 * 4) == 0      # whole partial rows for each of the two samples
    assert size(0, 64, 1, BF16) > 0
    assert size(4, 60, 1, BF16) == 0 and size(5, 64, 2, BF16) == 0


def test_no_rows_need_no_gpu():
    assert forward(rows=0, branch=None, y=None, z=None) == _lib.NSW_OK


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.residual_norm(x, x)
