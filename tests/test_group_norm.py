"""Refusals of the group norm that need no GPU: the C entry points check their arguments
before any launch, the tensor functions and the module theirs before the library."""
import pytest
import torch
from torch import nn

import nsw
from nsw import _lib, ops

BF16, F32 = _lib.NSW_DTYPE_BF16, _lib.NSW_DTYPE_F32
P = 16     # an aligned address that nothing reads


def forward(B=2, R=5, C=64, G=8, dtype=BF16, x=P, y=P, stats=P, w=P, eps=1e-5, act=_lib.NSW_ACT_SILU, ws=P, nbytes=1 << 40):
    return _lib.lib().nsw_group_norm(x, w, P, y, stats, B, R, C, G, eps, act, dtype, ws, nbytes, None)


def backward(B=2, R=5, C=64, G=8, dtype=BF16, dy=P, x=P, stats=P, dx=P, dw=P, act=_lib.NSW_ACT_SILU, ws=P, nbytes=1 << 40):
    return _lib.lib().nsw_group_norm_backward(dy, x, stats, P, P, dx, dw, P, B, R, C, G, act, dtype, ws, nbytes, None)


@pytest.mark.parametrize("call", [forward, backward])
@pytest.mark.parametrize("kw,says", [
    (dict(C=60, G=4), b"multiple of 8"), (dict(C=62, G=2, dtype=F32), b"multiple of 4"), (dict(C=4104), b"at most 4096"),
    (dict(C=2052, G=4, dtype=F32), b"at most 2048"), (dict(C=0), b"C=0"), (dict(G=0), b"groups"), (dict(G=7), b"groups"),
    (dict(G=128), b"groups"), (dict(B=-1), b"out of range"), (dict(B=1 << 20), b"out of range"), (dict(R=-1), b"out of range"),
    (dict(dtype=7), b"dtype"), (dict(act=9), b"activation"), (dict(x=None), b"required"), (dict(stats=None), b"required"),
    (dict(x=24), b"aligned"), (dict(ws=None), b"workspace"), (dict(ws=8), b"aligned"), (dict(nbytes=8), b"workspace"),
])
def test_refusals(call, kw, says):
    assert call(**kw) == _lib.NSW_ERR_INVALID
    assert says in _lib.lib().nsw_last_error()


@pytest.mark.parametrize("eps", [-1e-5, float("inf"), float("nan")])
def test_eps(eps):
    assert forward(eps=eps) == _lib.NSW_ERR_INVALID and b"eps" in _lib.lib().nsw_last_error()


def test_the_gated_linear_takes_no_missing_activation():
    assert _lib.lib().nsw_gated_linear(P, P, None, P, 4, 64, 64, _lib.NSW_ACT_NONE, BF16, None) == _lib.NSW_ERR_INVALID


def test_workspace_sizes():
    f, b = _lib.lib().nsw_group_norm_workspace_size, _lib.lib().nsw_group_norm_backward_workspace_size
    assert f(1, 1, 1024, 32, BF16) == 16                     # one workgroup a sample
    assert f(2, 64800, 1024, 32, BF16) % (2 * 32 * 8) == 0 and f(2, 64800, 1024, 32, BF16) > 2 * 32 * 8
    assert b(3, 5, 64, 8, F32) == 3 * 2 * 64 * 4
    assert f(1, 5, 60, 4, BF16) == 0 and b(1, 5, 64, 7, BF16) == 0


def test_no_rows_need_no_gpu():
    assert forward(B=0, x=None, y=None, stats=None) == _lib.NSW_OK
    assert forward(R=0, x=None, y=None, stats=None) == _lib.NSW_OK
    assert _lib.lib().nsw_group_norm_backward(None, None, None, None, None, None, None, None, 2, 0, 64, 8, 0, BF16, P, 1 << 20,
                                              None) == _lib.NSW_OK


def test_tensor_functions_refuse():
    x = torch.zeros(2, 4, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.group_norm(x, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.group_norm_backward(x, x, torch.zeros(2, 8, 2), 8)


def test_module():
    with pytest.raises(ValueError, match="groups"):
        nsw.GroupNorm(7, 64)
    m = nsw.GroupNorm(8, 64, act_layer=nn.Tanh)
    with pytest.raises(NotImplementedError, match="SiLU"):
        m.act_name
    with pytest.raises(ValueError, match="channels"):
        nsw.GroupNorm(8, 64)(torch.zeros(1, 2, 32))
    assert [nsw.GroupNorm(8, 64, act_layer=a).act_name for a in (None, nn.SiLU, nn.GELU, lambda: nn.GELU("tanh"))] == [
        "none", "silu", "gelu", "gelu_tanh"]
    assert sorted(nsw.GroupNorm(8, 64).state_dict()) == ["bias", "weight"] and not nsw.GroupNorm(8, 64, affine=False).state_dict()


def test_shapes_without_a_gpu():
    """The operator's shape function, as torch.compile asks it."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 3, 5, 64, dtype=torch.bfloat16)
        y, stats = torch.ops.nsw.group_norm(x, 8, None, None, "silu", 1e-5)
        assert y.shape == x.shape and y.dtype == x.dtype and stats.shape == (2, 8, 2) and stats.dtype == torch.float32
