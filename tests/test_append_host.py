"""dsa_cache_append's and dsa_cache.append's refusals, made on the host before any HIP call (these run without a GPU)."""

import ctypes

import pytest
import torch

from trnrt_amd import _lib
from trnrt_amd.kernels import dsa_cache

P = 256  # never dereferenced


def kind(**kw):
    base = dict(x=P, x_row=576, norm_weight=None, norm_bias=None, cache=P, scale=P, x_fp32=0, width=576, rope_at=512,
                interleaved=1, norm_fp32=0, norm_width=0, cache_bf16=0, eps=1e-6, fp8_max=448.0)
    return _lib.AppendRows(**{**base, **kw})


def call(kinds=None, n=None, table=P, ctx=P, cu=P, pos=None, freq=P, axes=None, T=10, B=2, R=32, n_axes=1, mp=4, ps=64, np_=9):
    kinds = [kind()] if kinds is None else kinds
    arr = (_lib.AppendRows * max(len(kinds), 1))(*kinds)
    return _lib.lib().dsa_cache_append(arr, len(kinds) if n is None else n, table, ctx, cu, pos, freq, axes, T, B, R, n_axes,
                                       1.0, mp, ps, np_, None)


def test_refusals():
    for kw in (dict(n=0), dict(table=None), dict(ctx=None), dict(freq=None), dict(T=-1), dict(B=-1), dict(mp=0), dict(ps=0),
               dict(np_=0), dict(R=0), dict(pos=P, n_axes=3), dict(pos=P, n_axes=0), dict(cu=None, T=11)):
        assert call(**kw) == _lib.DSA_EINVAL, kw
    for kw in (dict(kinds=[kind()] * 5), dict(T=(1 << 24) + 1), dict(R=30), dict(pos=P, n_axes=5, axes=bytes(32))):
        assert call(**kw) == _lib.DSA_EUNSUPPORTED, kw
    for kw in (dict(x=None), dict(cache=None), dict(x_row=575), dict(width=0), dict(x=264), dict(cache=264), dict(x_row=577),
               dict(rope_at=520), dict(fp8_max=0.0), dict(fp8_max=449.0), dict(fp8_max=float("nan")), dict(cache_bf16=1),
               dict(norm_bias=P), dict(norm_weight=P), dict(norm_weight=P, norm_width=584), dict(norm_weight=264, norm_width=8),
               dict(norm_weight=P, norm_width=512, eps=-1.0), dict(norm_weight=P, norm_width=512, eps=float("nan"))):
        assert call([kind(**kw)]) == _lib.DSA_EINVAL, kw
    for kw in (dict(width=572), dict(width=1032, x_row=1032), dict(rope_at=508), dict(norm_weight=P, norm_width=12)):
        assert call([kind(**kw)]) == _lib.DSA_EUNSUPPORTED, kw
    assert call(T=0, table=None) == _lib.DSA_OK and call(B=0, T=0) == _lib.DSA_OK


def test_packed_layout():
    """append packs dsa_append_rows by itself: the same bytes as the structure's."""
    k = kind(x=1 << 40, x_row=-5, norm_weight=7, norm_bias=9, cache=11, scale=13, norm_fp32=1, norm_width=3, cache_bf16=1)
    assert dsa_cache._KIND.size == ctypes.sizeof(k)
    packed = dsa_cache._KIND.pack(1 << 40, -5, 7, 9, 11, 13, 0, 576, 512, 1, 1, 3, 1, 1e-6, 448.0)
    assert packed[:84] == bytes(k)[:84]  # (then 4 bytes of padding)


def test_host_tensors_raise():
    z = torch.zeros(64, 576, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="GPU only"):
        dsa_cache.append(dsa_cache.Rows(torch.zeros(1, 576), z), torch.zeros(1, 1, dtype=torch.int32),
                         torch.zeros(1, dtype=torch.int32), 64)
    with pytest.raises(ValueError, match="no rows"):
        dsa_cache.append([], torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 64)
