"""dsa_expand_latent's and dsa_expanded_mla's refusals, made on the host before any HIP call (these run without a GPU)."""

import ctypes

import pytest
import torch

from trnrt_amd import _lib
from trnrt_amd.kernels import dsa_expand

P = ctypes.c_void_p(256)  # never dereferenced


def test_expand_refusals():
    def call(kv=P, w=P, k=P, rope=P, B=2, total=10, H=16, D=576, mp=4, ps=64, pages=100):
        return _lib.lib().dsa_expand_latent(kv, P, P, P, w, k, P, rope, B, total, H, D, mp, ps, pages, None)

    for kw in (dict(B=-1), dict(total=-1), dict(H=0), dict(mp=0), dict(ps=0), dict(pages=0), dict(kv=None), dict(w=None),
               dict(k=None), dict(rope=None)):
        assert call(**kw) == _lib.DSA_EINVAL, kw
    assert call(D=640) == _lib.DSA_EUNSUPPORTED
    assert call(pages=1 << 26) == _lib.DSA_EUNSUPPORTED  # 2^32 slots
    assert call(total=1 << 30, H=1 << 10) == _lib.DSA_EUNSUPPORTED  # more workgroups than a launch takes
    assert call(total=0, kv=None) == _lib.DSA_OK and call(B=0) == _lib.DSA_OK
    odd = ctypes.c_void_p(264)  # not a multiple of 16
    for kw in (dict(kv=odd), dict(w=odd), dict(k=odd), dict(rope=odd)):
        assert call(**kw) == _lib.DSA_EINVAL, kw


def test_attend_refusals():
    def call(q=P, k=P, v=P, out=P, ws=None, size=0, B=2, Tq=10, Tk=10, H=16):
        return _lib.lib().dsa_expanded_mla(q, k, None, v, P, P, out, None, P, ws, size, B, Tq, Tk, H, 1, 0.1, None)

    for kw in (dict(B=-1), dict(Tq=-1), dict(Tk=-1), dict(H=0), dict(q=None), dict(k=None), dict(v=None), dict(out=None)):
        assert call(**kw) == _lib.DSA_EINVAL, kw
    assert call(Tq=1 << 30, H=1 << 10) == _lib.DSA_EUNSUPPORTED
    assert call(B=0) == _lib.DSA_OK and call(Tq=0, q=None) == _lib.DSA_OK
    need = _lib.lib().dsa_expanded_workspace_bytes
    odd = ctypes.c_void_p(264)  # not a multiple of 16
    for kw in (dict(q=odd), dict(k=odd), dict(v=odd), dict(out=odd)):
        assert call(**kw) == _lib.DSA_EINVAL, kw
    assert need(2, 10, 10, 16) == 0 and need(0, 10, 10, 16) == 0 and need(2, 10, -1, 16) == 0
    size = need(1, 10, 100000, 16)  # one query tile a head, the keys in splits
    assert size >= 2 * 16 * 256 * 130 * 4
    assert call(B=1, Tk=100000) == _lib.DSA_EWORKSPACE and call(B=1, Tk=100000, ws=P, size=size - 1) == _lib.DSA_EWORKSPACE
    assert call(B=1, Tk=100000, ws=odd, size=size) == _lib.DSA_EWORKSPACE


def test_host_tensors_raise():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        dsa_expand.expand(torch.zeros(64, 576, dtype=torch.uint8), None, torch.zeros(1, 1, dtype=torch.int32), i, 1, 64,
                          torch.zeros(1, 256, 512, dtype=torch.bfloat16))
    z = torch.zeros(1, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU only"):
        dsa_expand.attend(z, z, None, z, i, i, 0.1)
