"""Rotary positions on gfx950, of one axis or of several (time, height, width: prompts with images and video), for the
queries of the attention (64 of their 576 or 192 columns) and of the indexer (64 of 128); dsa_cache.append rotates the keys.

    rotate(x, positions, inv_freq)    (y0, y1) = factor (x0 cos - x1 sin, x1 cos + x0 sin), pair i by p[axis(i)] inv_freq[i]

The angles are exact to fp32 at any position (the product is taken in 64 bits), the rotation is in fp32 and rounded once. The
HIP kernel is in csrc/dsa_rope.hip.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from .. import _lib
from . import _common as C

MAX_FREQUENCIES = 256
MAX_AXES = 4


def axis_map(axes: Sequence[int] | None, positions: torch.Tensor | None, R: int, T: int, what: str) -> tuple:
    """(positions as int32, number of axes, each frequency's axis as bytes or None) of positions [T] or [axes, T]."""
    if axes is not None:
        if len(axes) != R:
            raise ValueError(f"{what}: {len(axes)} axes for {R} frequencies")
        axes = bytes(axes)
    if positions is None:
        if axes is not None and any(axes):
            raise ValueError(f"{what}: several axes need their positions")
        return None, 1, None
    n = 1 if positions.dim() == 1 else positions.shape[0]
    if positions.dim() not in (1, 2) or positions.shape[-1] != T or n < 1:
        raise ValueError(f"{what}: positions {tuple(positions.shape)} for {T} tokens, expected [T] or [axes, T]")
    if n > 1 and axes is None:
        raise ValueError(f"{what}: {n} axes of positions, but not which frequency is of which (axes)")
    if axes is not None and R and max(axes) >= n:
        raise ValueError(f"{what}: axis {max(axes)} of {n}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: positions of {positions.dtype}, expected int32 (or int64)")
    return C.as_i32(positions), n, axes


def rows_apart(T: int, H: int, row: int, head: int, width: int) -> bool:
    """Whether no two of T x H rows of `width` values, `row` and `head` values apart, share one."""
    if row >= head * (H - 1) + width and (head >= width or H < 2):
        return True  # (a token's heads, then the next token's)
    (n, a), (m, b) = sorted(((T, row), (H, head)), key=lambda x: x[1] if x[0] > 1 else 0)
    if T < 1 or (n < 2 or a >= width) and (m < 2 or b >= a * (n - 1) * (n > 1) + width):
        return True  # (one dimension's rows within a step of the other: every ordinary layout)
    if (n > 1 and a < width) or (m > 1 and b < width):
        return False
    (k, c), (l, d) = sorted(((n, a), (m, b)))  # (fewer rows first)
    for i in range(1, k):  # i steps of it against the nearest numbers of steps of the other
        j = min(i * c // d, l - 1)
        if i * c - j * d < width or (j + 1 < l and (j + 1) * d - i * c < width):
            return False
    return True


def rotate(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, axes: Sequence[int] | None = None,
           interleaved: bool = True, factor: float = 1.0, inverse: bool = False,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """x [T, H, 2R] or [T, 2R] (bf16 or fp32; a view of the rope columns of wider rows will do) rotated by positions [T], or
    [axes, T] with axes the axis of each of the R frequencies inv_freq [R] fp32; positions int32 (int64 ones within its
    range). interleaved: the pairs are columns (2i, 2i + 1), else (i, i + R). factor multiplies the result; inverse turns back
    (with factor, that is the gradient of rotate). out: a tensor or view of x's shape and type to write, x itself for a
    rotation in place (no other overlap); None for a new one."""
    dev = C.on_gpu(x, positions, inv_freq, out)
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"dsa_rope.rotate: x of {x.dtype}, expected bfloat16 or float32")
    C.need(inv_freq, "inv_freq", torch.float32, (None,))
    R = inv_freq.shape[0]
    if x.dim() not in (2, 3) or R < 1 or x.shape[-1] != 2 * R:
        raise ValueError(f"dsa_rope.rotate: x {tuple(x.shape)}, expected [T, H, {2 * R}] or [T, {2 * R}]")
    T, H = x.shape[0], x.shape[1] if x.dim() == 3 else 1
    if H < 1:
        raise ValueError(f"dsa_rope.rotate: x {tuple(x.shape)} has no heads")
    pos, n_axes, which = axis_map(axes, positions, R, T, "dsa_rope.rotate")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.dtype is not x.dtype or out.shape != x.shape:
        raise ValueError(f"dsa_rope.rotate: out {tuple(out.shape)} of {out.dtype} for x {tuple(x.shape)} of {x.dtype}")
    xs, os = x.stride(), out.stride()
    if xs[-1] != 1:
        x = x.contiguous()
        xs = x.stride()
    if os[-1] != 1 or not rows_apart(T, H, os[0], os[1] if H > 1 else 0, 2 * R):
        raise ValueError(f"dsa_rope.rotate: out with strides {os}: its columns must lie side by side, no row over another")
    st = C.call(dev, _lib.lib().dsa_rope_rotate, x.data_ptr(), x.dtype is torch.float32, xs[0], xs[1] if H > 1 else 0,
                pos.data_ptr(), inv_freq.data_ptr(), which, out.data_ptr(), os[0], os[1] if H > 1 else 0, T, H, R, n_axes,
                bool(interleaved), factor, bool(inverse))
    _lib.check(st, "dsa_rope.rotate")
    return out
