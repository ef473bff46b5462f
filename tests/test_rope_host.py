"""dsa_rope_rotate's and dsa_rope.rotate's refusals, made on the host before any HIP call (these run without a GPU)."""

import ctypes

import pytest
import torch

from trnrt_amd import _lib
from trnrt_amd.kernels import dsa_rope

P = ctypes.c_void_p(256)  # never dereferenced


def test_refusals():
    def call(x=P, pos=P, freq=P, axes=None, out=P, T=4, H=2, R=32, n_axes=1):
        return _lib.lib().dsa_rope_rotate(x, 0, 64 * H, 64, pos, freq, axes, out, 64 * H, 64, T, H, R, n_axes, 1, 1.0, 0, None)

    for kw in (dict(x=None), dict(pos=None), dict(freq=None), dict(out=None), dict(T=-1), dict(H=0), dict(R=0), dict(n_axes=0),
               dict(n_axes=3), dict(axes=bytes([0] * 31 + [3]), n_axes=3), dict(axes=bytes([1] * 32))):
        assert call(**kw) == _lib.DSA_EINVAL, kw
    for kw in (dict(R=257), dict(n_axes=5), dict(T=(1 << 22) + 1), dict(H=(1 << 16) + 1)):
        assert call(**kw) == _lib.DSA_EUNSUPPORTED, kw
    assert call(T=0, x=None) == _lib.DSA_OK


def test_axis_map():
    pos = torch.zeros(3, 5, dtype=torch.int32)
    assert dsa_rope.axis_map([0, 1, 2, 0], pos, 4, 5, "x")[1:] == (3, bytes([0, 1, 2, 0]))
    assert dsa_rope.axis_map(None, pos[0], 4, 5, "x")[1:] == (1, None)
    assert dsa_rope.axis_map(None, None, 4, 5, "x") == (None, 1, None)
    for axes, p in (([0, 1], pos), ([0, 1, 2, 3], pos), (None, pos), ([0, 1, 0, 1], None), ([0, 0, 0, -1], pos),
                    (None, pos[0][:4]), (None, pos[None]), (None, pos[0].float())):
        with pytest.raises(ValueError):
            dsa_rope.axis_map(axes, p, 4, 5, "x")


def test_host_tensors_raise():
    with pytest.raises(RuntimeError, match="GPU only"):
        dsa_rope.rotate(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32), torch.ones(4))


def test_rows_of_outputs_that_overlap():
    """Against every pair of rows; the wrapper refuses outputs whose rows share values (two workgroups would write them)."""
    def slowly(T, H, row, head, W):
        at = sorted(t * row + h * head for t in range(T) for h in range(H))
        return all(b - a >= W for a, b in zip(at, at[1:]))

    for T in (0, 1, 2, 3, 5):
        for H in (1, 2, 4):
            for row in (0, 1, 3, 4, 5, 8, 9, 12, 13, 16, 20):
                for head in (0, 2, 4, 6, 8, 10, 12, 16, 21):
                    for W in (2, 4):
                        assert dsa_rope.rows_apart(T, H, row, head, W) == slowly(T, H, row, head, W), (T, H, row, head, W)
    assert dsa_rope.rows_apart(8192, 64, 64 * 192, 192, 64) and dsa_rope.rows_apart(1 << 22, 65536, 64, 64 << 22, 64)
    assert not dsa_rope.rows_apart(8192, 64, 63 * 64, 64, 64)
