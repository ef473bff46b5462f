"""dsa_dense_mla's refusals, made on the host before any HIP call (these run without a GPU)."""

import ctypes

import pytest
import torch

from trnrt_amd import _lib
from trnrt_amd.kernels import dsa_dense

P = ctypes.c_void_p(256)  # never dereferenced


def test_refusals():
    lib = _lib.lib()
    ws = lib.dsa_dense_workspace_bytes(1, 64)
    assert ws >= 2 * 256 * 64 * 514 * 4 and lib.dsa_dense_workspace_bytes(0, 64) == 0
    assert lib.dsa_dense_workspace_bytes(1, 16) < ws and lib.dsa_dense_workspace_bytes(1 << 20, 1 << 20) == 0

    def call(q=P, out=P, outf=None, wsp=P, size=ws, B=2, S=1, H=64, D=576, mp=4, ps=64, pages=100):
        return lib.dsa_dense_mla(q, P, P, P, P, out, outf, P, wsp, size, B, S, H, D, mp, ps, pages, 0.1, None)

    for kw in (dict(B=-1), dict(S=0), dict(H=0), dict(mp=0), dict(ps=0), dict(pages=0), dict(q=None), dict(out=None)):
        assert call(**kw) == _lib.DSA_EINVAL, kw
    assert call(D=640) == _lib.DSA_EUNSUPPORTED
    assert call(pages=1 << 26) == _lib.DSA_EUNSUPPORTED  # 2^32 slots
    assert call(B=1 << 20, S=64) == _lib.DSA_EUNSUPPORTED  # more rows than a launch has threads for
    assert call(wsp=None) == _lib.DSA_EWORKSPACE
    assert call(size=2 * 256 * 64 * 514 * 4 - 1) == _lib.DSA_EWORKSPACE
    assert call(B=0, q=None) == _lib.DSA_OK
    odd = ctypes.c_void_p(264)  # not a multiple of 16
    assert call(q=odd) == _lib.DSA_EINVAL and call(out=odd) == _lib.DSA_EINVAL
    assert call(wsp=odd) == _lib.DSA_EWORKSPACE


def test_host_tensors_raise():
    with pytest.raises(RuntimeError, match="GPU only"):
        dsa_dense.attend(torch.zeros(1, 16, 576), torch.zeros(64, 576, dtype=torch.uint8), torch.ones(64),
                         torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), 64, 0.1)
