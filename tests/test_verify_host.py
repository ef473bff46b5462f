"""dsa_verify's refusals, made on the host before any HIP call (these run without a GPU)."""

import ctypes

import pytest
import torch

from trnrt_amd import _lib
from trnrt_amd.kernels import dsa_verify

P = ctypes.c_void_p(256)  # never dereferenced


def test_refusals():
    need = _lib.lib().dsa_verify_workspace_bytes

    def call(logits=P, row=1000, draft=P, probs=None, probs_row=1000, cu=P, u=P, v=P, temperature=P, tokens=P, accepted=P,
             logp=P, ws=P, size=None, N=10, V=1000, B=2):
        return _lib.lib().dsa_verify(logits, 0, row, draft, probs, 1, probs_row, cu, u, v, temperature, tokens, accepted, logp,
                                     ws, need(N, V, B) if size is None else size, N, V, B, None)

    for kw in (dict(logits=None), dict(row=999), dict(draft=None), dict(probs=P, probs_row=999), dict(cu=None), dict(u=None),
               dict(v=None), dict(temperature=None), dict(tokens=None), dict(accepted=None), dict(logp=None), dict(N=-1),
               dict(V=0), dict(B=-1)):
        assert call(**kw) == _lib.DSA_EINVAL, kw
    assert call(N=1 << 24, V=1 << 20, row=1 << 20) == _lib.DSA_EUNSUPPORTED
    assert call(B=1 << 25) == _lib.DSA_EUNSUPPORTED
    assert call(ws=None) == _lib.DSA_EWORKSPACE and call(size=need(10, 1000, 2) - 256) == _lib.DSA_EWORKSPACE
    assert call(ws=ctypes.c_void_p(264)) == _lib.DSA_EWORKSPACE
    assert call(B=0, cu=None) == _lib.DSA_OK
    assert need(-1, 10, 1) == 0 and need(1, 0, 1) == 0 and need(1, 1, -1) == 0 and need(0, 10, 1) > 0


def test_host_tensors_raise():
    f, i = torch.zeros(1), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        dsa_verify.verify(torch.zeros(1, 5), i, torch.tensor([0, 1], dtype=torch.int32), f, f, f)


def test_rows_of_too_many_logits_are_refused():
    """Past 2^30 logits a row an index would pass 2^31: nothing is launched, and there is no size of a workspace."""
    need, call = _lib.lib().dsa_verify_workspace_bytes, _lib.lib().dsa_verify
    for V in ((1 << 30) + 1, (1 << 31) - 2048, (1 << 31) - 1):
        assert need(1, V, 1) == 0
        for f32 in (0, 1):
            st = call(P, f32, V, P, None, 0, 0, P, P, P, P, P, P, P, P, ctypes.c_size_t(1 << 40), 1, V, 1, None)
            assert st == _lib.DSA_EUNSUPPORTED
    assert need(1, 1 << 30, 1) > 0
