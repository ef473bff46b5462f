"""dsa_expanded_mla_spans' refusals, made on the host before any HIP call (these run without a GPU)."""

import ctypes

import pytest
import torch

from trnrt_amd import _lib
from trnrt_amd.kernels import dsa_expand

P = ctypes.c_void_p(256)  # never dereferenced


def test_refusals():
    def call(q=P, k=P, out=P, cap=0.0, ws=None, size=0, B=2, Tq=10, Tk=10, H=16):
        return _lib.lib().dsa_expanded_mla_spans(q, k, None, P, P, P, None, None, None, cap, out, None, P, ws, size, B, Tq, Tk,
                                                 H, 1, 0.1, None)

    for kw in (dict(cap=-1.0), dict(cap=1e-31), dict(cap=float("inf")), dict(cap=1e31), dict(cap=float("nan")), dict(q=None), dict(k=None), dict(out=None),
               dict(B=-1), dict(H=0), dict(q=ctypes.c_void_p(264))):
        assert call(**kw) == _lib.DSA_EINVAL, kw
    assert call(Tq=1 << 30, H=1 << 10) == _lib.DSA_EUNSUPPORTED
    assert call(B=1, Tk=100000) == _lib.DSA_EWORKSPACE
    assert call(B=0) == _lib.DSA_OK and call(Tq=0, q=None) == _lib.DSA_OK


def test_host_tensors_raise():
    z, i = torch.zeros(1, 1, 128, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        dsa_expand.attend(z, z, None, z, i, i, 0.1, first=i[:1], softcap=5.0)
