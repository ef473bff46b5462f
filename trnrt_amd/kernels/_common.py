"""Argument checks shared by the operator wrappers: device tensors only (the HIP path is the only path), the
dtypes and layouts the C ABI expects, and the current HIP stream."""

from __future__ import annotations

import threading

import torch

FP8 = torch.float8_e4m3fn  # OCP e4m3fn: gfx950's FP8 and the reference's CPU cache dtype (model_runner.py:54-70)


def on_gpu(*ts: torch.Tensor | None) -> torch.device:
    """The common GPU device of the tensors; RuntimeError for host tensors (there is no CPU path)."""
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(
                "trnrt_amd DSA kernels run on the GPU only (libdsa_gfx950.so); got a tensor on " + str(t.device)
            )
        d = t.device
        if dev is None:
            dev = d
        elif d != dev:
            raise ValueError(f"tensors on different devices: {dev} and {d}")
    if dev is None:
        raise ValueError("no tensor arguments")
    return dev


def stream_ptr(device: torch.device) -> int:
    # (the handle alone: a torch.cuda.Stream around it costs more of the host's time than most of a wrapper's checks)
    index = device.index
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


def call(device: torch.device, fn, *args) -> int:
    """fn(*args, stream): a C entry point on device's current stream, with device the current one (a launch goes to the
    current device, whichever the tensors are on)."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(device):
        return fn(*args, stream_ptr(device))


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def need(t: torch.Tensor, name: str, dtype: torch.dtype | tuple, shape: tuple | None = None) -> torch.Tensor:
    """t itself if it has the dtype (one of), shape (None entries free) and is contiguous; ValueError otherwise."""
    if t.dtype is not dtype and (not isinstance(dtype, tuple) or t.dtype not in dtype):
        dts = dtype if isinstance(dtype, tuple) else (dtype,)
        raise ValueError(f"{name}: dtype {t.dtype}, expected {' or '.join(map(str, dts))}")
    if shape is not None and t.shape != shape:  # (unequal also where an entry is free)
        if t.dim() != len(shape) or any(s is not None and s != d for s, d in zip(shape, t.shape)):
            raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {shape}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    return t


def as_bf16(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.bfloat16 and t.is_contiguous() else t.to(torch.bfloat16).contiguous()


def as_i32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def as_f32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


def aligned(t: torch.Tensor) -> torch.Tensor:
    """t itself if it starts at a multiple of 16 bytes (a view may not), else a copy that does."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def given(workspace: torch.Tensor, what: str) -> torch.Tensor:
    """A caller's workspace; ValueError where its bytes are not one range."""
    if not workspace.is_contiguous():
        raise ValueError(f"{what}: the workspace must be contiguous")
    return workspace


def rows_of(t: torch.Tensor, width: int) -> torch.Tensor:
    """A contiguous tensor as rows [n, width] (itself where it is that already)."""
    return t if t.dim() == 2 else t.reshape(-1, width)


def flat(t: torch.Tensor) -> torch.Tensor:
    return t if t.dim() == 1 else t.reshape(-1)


def fp8_bytes(t: torch.Tensor, name: str) -> torch.Tensor:
    """The e4m3fn cache as a contiguous tensor (float8_e4m3fn or its uint8 bit pattern)."""
    if t.dtype not in (FP8, torch.uint8):
        raise ValueError(f"{name}: dtype {t.dtype}, expected float8_e4m3fn (or its uint8 bits)")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    return t


# Zero-filled workspaces kept per (device, stream, use, host thread) and reused by the functional surfaces when the caller
# passes none: every call leaves the regions that must start at zero at zero again, so one zero fill serves every later
# call of the thread on the same stream (its calls on one stream never overlap; each stream has its own, and each thread,
# since a call of several launches lets another thread's in between). A call needing more grows it: a new zero-filled
# buffer on the same stream (the old one returns to torch's stream-ordered allocator). They outlive their threads, as a
# graph may have recorded one.
_WORKSPACES: dict = {}


def cached_workspace(device: torch.device, nbytes: int, use: str) -> torch.Tensor:
    """A zero-filled uint8 device buffer of at least nbytes for `use` on the current stream of `device`, this host
    thread's."""
    key = (device.index if device.index is not None else torch.cuda.current_device(), stream_ptr(device), use,
           threading.get_ident())
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = zeroed_workspace(max(int(nbytes), 256), device)
        _WORKSPACES[key] = ws
    return ws


class _Scratch(threading.local):  # (a thread's own buffers, let go with it)
    def __init__(self):
        self.kept: dict = {}


_SCRATCH = _Scratch()


def scratch(device: torch.device, nbytes: int, use: str) -> torch.Tensor:
    """A uint8 device buffer of at least nbytes that a call writes before it reads: the one that this host thread keeps for
    `use` on the current stream (another thread's launches may come between those of a call), and in a graph capture one
    of the graph's own memory (a graph that kept the stream's would replay into it after a later call had let it go for a
    larger one, or beside another graph's replay)."""
    n = max(int(nbytes), 256)
    if torch._C._cuda_isCurrentStreamCapturing():
        return torch.empty(n, dtype=torch.uint8, device=device)
    key = (device.index if device.index is not None else torch.cuda.current_device(), stream_ptr(device), use)
    ws = _SCRATCH.kept.get(key)
    if ws is None or ws.numel() < n:
        ws = _SCRATCH.kept[key] = torch.empty(n, dtype=torch.uint8, device=device)
    return ws


def zeroed_workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """A new uint8 device buffer of nbytes (a multiple of 256) zero-filled by the library's dsa_workspace_clear on the
    current stream, which also records it as zero, so its first call does not fill it again."""
    from .. import _lib

    n = (int(nbytes) + 255) // 256 * 256
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    _lib.check(_lib.lib().dsa_workspace_clear(ws.data_ptr(), n, stream_ptr(device)), "dsa_workspace_clear")
    return ws
