"""Refusals of the position attention that need no GPU, its buckets, and the gradients of
the window maps' shapes: the C entry points check their arguments before any launch, the
tensor functions and modules theirs before the library."""
import math

import pytest
import torch

import nsw
from nsw import _lib, ops

BF16, F32 = _lib.NSW_DTYPE_BF16, _lib.NSW_DTYPE_F32
P = 16     # an aligned address that nothing reads


def tail(Bw, T, A, W, L, C, heads, scale, nb, H, Wi, s0, s1, dtype):
    return (Bw, T * A * W if L is None else L, C, heads, scale, nb, T, A, W, H, Wi, s0, s1, dtype)


def forward(Bw=4, T=1, A=3, W=5, L=None, C=64, heads=2, scale=0.2, nb=9, H=0, Wi=0, s0=0, s1=0, dtype=BF16, qkv=P, table=P,
            buckets=P, mask=None, nW=0, o=P, stats=P, **_):
    return _lib.lib().nsw_position_attention(qkv, table, buckets, mask, nW, o, stats,
                                             *tail(Bw, T, A, W, L, C, heads, scale, nb, H, Wi, s0, s1, dtype), None)


def backward(Bw=4, T=1, A=3, W=5, L=None, C=64, heads=2, scale=0.2, nb=9, H=0, Wi=0, s0=0, s1=0, dtype=BF16, qkv=P, table=P,
             buckets=P, mask=None, nW=0, o=P, stats=P, dtable=P, ws=P, nbytes=1 << 40):
    return _lib.lib().nsw_position_attention_backward(P, qkv, o, stats, table, buckets, mask, nW, P, dtable,
                                                      *tail(Bw, T, A, W, L, C, heads, scale, nb, H, Wi, s0, s1, dtype), ws, nbytes,
                                                      None)


@pytest.mark.parametrize("call", [forward, backward])
@pytest.mark.parametrize("kw,says", [
    (dict(dtype=7), b"dtype"), (dict(C=60), b"multiple of 8"), (dict(C=64, heads=3), b"heads"), (dict(heads=0), b"heads"),
    (dict(C=48, heads=2), b"head_dim=24"), (dict(C=512, heads=2), b"head_dim=256"), (dict(L=14), b"tokens of a window"),
    (dict(T=0), b"tokens of a window"), (dict(T=-1, A=-3, W=5), b"tokens of a window"), (dict(A=1, W=4097), b"displacements"),
    (dict(A=46, W=46), b"displacements"), (dict(nb=0), b"buckets"), (dict(nb=1 << 24), b"buckets"),
    (dict(scale=float("inf")), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(Bw=-1), b"Bw=-1"),
    (dict(mask=P, nW=3), b"multiple of the mask"), (dict(mask=P, nW=0), b"multiple of the mask"),
    (dict(s0=1, H=6, Wi=11), b"divisible"), (dict(s0=3, H=6, Wi=10), b"shift"), (dict(s1=-1, H=6, Wi=10), b"shift"),
    (dict(s0=1, H=6, Wi=15), b"image's 6 windows"), (dict(qkv=None), b"required"), (dict(table=None), b"required"),
    (dict(buckets=None), b"required"), (dict(o=None), b"required"), (dict(stats=None), b"required"), (dict(qkv=24), b"aligned"),
    (dict(stats=8), b"aligned"),
])
def test_refusals(call, kw, says):
    assert call(**kw) == _lib.NSW_ERR_INVALID
    assert says in _lib.lib().nsw_last_error(), _lib.lib().nsw_last_error()


@pytest.mark.parametrize("call", [forward, backward])
@pytest.mark.parametrize("kw", [dict(Bw=1 << 31), dict(Bw=1 << 30), dict(Bw=1 << 22, A=5, W=14), dict(C=1 << 18, heads=1 << 11),
                                dict(C=131072, heads=1024, A=1, W=4096)])
def test_sizes_past_a_launch_are_refused(call, kw):
    assert call(**kw) == _lib.NSW_ERR_INVALID


@pytest.mark.parametrize("kw", [dict(ws=None), dict(nbytes=64), dict(ws=8)])
def test_workspace_refusals(kw):
    assert backward(**kw) == _lib.NSW_ERR_INVALID and (b"workspace" in _lib.lib().nsw_last_error())


def test_workspace_size():
    size = _lib.lib().nsw_position_attention_backward_workspace_size
    n = size(400, 162, 1024, 16, 1, 9, 18, BF16)
    assert n % (16 * 4) == 0 and n >= 16 * (162 * 162 + 17 * 35) * 4     # sums by pair, then by displacement
    assert size(0, 15, 64, 2, 1, 3, 5, F32) > 0
    assert size(4, 14, 64, 2, 1, 3, 5, F32) == 0 and size(4, 15, 60, 2, 1, 3, 5, F32) == 0


def test_no_windows_need_no_gpu():
    assert forward(Bw=0, qkv=None, o=None, stats=None, table=None, buckets=None) == _lib.NSW_OK
    assert backward(Bw=0, dtable=None, ws=None, nbytes=0) == _lib.NSW_OK


def test_tensor_functions_refuse():
    qkv, table = torch.zeros(4, 15, 192), torch.zeros(45, 2)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.position_attention(qkv, 2, 0.2, table, torch.zeros(45, dtype=torch.int32), (1, 3, 5))


# ------------------------------------------------------------------- buckets ---

def test_each_displacement_its_own_bucket():
    b, n = nsw.position_buckets((2, 3, 5))
    assert n == 3 * 5 * 9 == ops.window_displacements((2, 3, 5)) and torch.equal(b, torch.arange(n, dtype=torch.int32))


@pytest.mark.parametrize("n", [2, 5, 40, 300])
def test_wide_buckets(n):
    """32 buckets: distances 0..7 one by one, then eight steps to 128, all beyond in the last; either sign."""
    b, count = nsw.position_buckets((1, 1, n), 32, 128)
    assert count == 32 and b.dtype == torch.int32 and b.shape == (2 * n - 1,)
    for i, d in enumerate(range(-(n - 1), n)):
        far = abs(d)
        want = far if far < 8 else 8 + min(7, math.floor(8 * math.log(far / 8) / math.log(16) + 1e-9))
        assert b[i] == want + (16 if d > 0 else 0), d


def test_bucket_borders():
    """Distances at a border fall into the bucket that begins there: 8 * 16^(k / 8) is whole at 8, 16, 32, 64, 128."""
    b, _ = nsw.position_buckets((1, 1, 200), 32, 128)
    at = lambda d: int(b[199 - d])
    assert [at(8), at(15), at(16), at(31), at(32), at(63), at(64), at(127), at(128), at(199)] == [8, 9, 10, 11, 12, 13, 14, 15, 15, 15]


def test_buckets_of_several_axes():
    b, n = nsw.position_buckets((1, 3, 20), 8, 16)
    assert n == 64 and b.shape == (5 * 39,) and int(b.min()) == 0 and int(b.max()) < 64
    one, _ = nsw.position_buckets((1, 1, 20), 8, 16)
    assert torch.equal(b.view(5, 39)[2], one)               # no step along the first of the two


@pytest.mark.parametrize("kw", [dict(num_buckets=3), dict(num_buckets=2), dict(num_buckets=32, max_distance=8)])
def test_bucket_refusals(kw):
    with pytest.raises(ValueError):
        nsw.position_buckets((1, 1, 9), **kw)
    with pytest.raises(ValueError):
        nsw.position_buckets((1, 0, 9))


def test_modules():
    with pytest.raises(ValueError, match="8192"):
        nsw.RelativePositionBias(2, (1, 46, 46))
    with pytest.raises(ValueError, match="heads"):
        nsw.PositionWindowAttention(64, 3, (3, 5))
    with pytest.raises(ValueError, match="divisible"):
        nsw.PositionAttentionBranch(64, 2, (10, 10), (3, 5))
    m = nsw.PositionAttentionBranch(64, 2, (6, 10), (3, 5), 2, (1, 2), num_groups=8)
    assert sorted(m.state_dict()) == ["attn.biasproj.bias", "attn.biasqkv.bias", "attn.position.table", "attn.proj.weight",
                                      "attn.qkv.weight", "norm.bias", "norm.weight"]
    assert m.attn.position.table.shape == (3 * 5 * 9, 2) and m.bfloat16().attn.position.buckets.dtype == torch.int32
    with pytest.raises(ValueError, match="expected"):
        m(torch.zeros(1, 1, 6, 10, 64))


def test_shapes_without_a_gpu():
    """The operators' shape functions, as torch.compile asks them, and the window maps' gradients."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    n = torch.ops.nsw
    with FakeTensorMode():
        qkv, table = torch.empty(4, 15, 192, dtype=torch.bfloat16), torch.empty(45, 2, dtype=torch.bfloat16)
        b = torch.empty(45, dtype=torch.int32)
        o, stats = n.position_attention(qkv, 2, 0.2, table, b, [1, 3, 5], None, [])
        assert o.shape == (4, 15, 64) and o.dtype == qkv.dtype and stats.shape == (4, 2, 15, 2 + 4) and stats.dtype == torch.float32
        dqkv, dtable = n.position_attention_backward(o, qkv, o, stats, 2, 0.2, table, b, [1, 3, 5], None, [], [True, False])
        assert dqkv.shape == qkv.shape and dtable.shape == (0,)
        x = torch.empty(2, 1, 6, 10, 8, requires_grad=True)
        n.window_reverse_roll(n.roll_window_partition(x, [3, 5], [1, 2]), [3, 5], [6, 10], [1, 2]).sum().backward()
        assert x.grad.shape == x.shape
        x.grad = None
        n.window_reverse(n.window_partition(x, [3, 5]), [3, 5], [6, 10]).sum().backward()
        assert x.grad.shape == x.shape
