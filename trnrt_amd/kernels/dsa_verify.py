"""Verification of drafted tokens on gfx950: which of a speculative step's drafts the target takes, and the token after them,
from given random numbers. The step before it is dsa_dense.attend of the drafted tokens; after it the sequences' lengths go
back by the drafts that were not taken, whose cached rows the next dsa_cache.append writes over.

    verify(logits, draft, cu, u, v, temperature, draft_probs=q)    tokens, accepted, logp

With p = softmax(logits / temperature), a draft x of row j is taken iff u[j] q(x) < p(x), up to the first that is not; the
next token is drawn from max(p - q, 0) of that row (from p of the last row, once all are taken) by v: what comes out is
distributed as the target's own samples are. Tokens and counts are those of 64-bit probabilities, sums and comparisons (a
probability of no more than 2^-1022 of the row's largest is 0), and do not vary from run to run; logp is off by 2^-17 at most
beside its rounding. The HIP kernels are in csrc/dsa_verify.hip.
"""

from __future__ import annotations

import torch

from .. import _lib
from . import _common as C

_TYPES = (torch.bfloat16, torch.float32)


def _rows(t: torch.Tensor, name: str, shape: tuple) -> tuple[torch.Tensor, int]:
    """The rows, copied where a row's values do not lie side by side or rows overlap, and their stride."""
    if t.dtype not in _TYPES:
        raise ValueError(f"dsa_verify: {name} of {t.dtype}, expected bfloat16 or float32")
    if t.shape != shape:
        raise ValueError(f"dsa_verify: {name} {tuple(t.shape)}, expected {tuple(shape)}")
    N, V = shape
    row, col = t.stride()
    if (col != 1 and V > 1) or (row < V and N > 1):
        t = t.clone(memory_format=torch.contiguous_format)
    return t, max(t.stride(0), V)  # (a single row's stride says nothing)


def verify(logits: torch.Tensor, draft: torch.Tensor, cu: torch.Tensor, u: torch.Tensor, v: torch.Tensor,
           temperature: torch.Tensor, *, draft_probs: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(tokens [N] int32, accepted [B] int32, logp [N] fp32) of B sequences whose rows of logits [N, V] (bf16 or fp32, rows
    may be views) are cu[b] .. cu[b + 1] - 1 (cu [B + 1] int32 on the device). Every row but a sequence's last has a drafted
    token draft [N] int32 (the last rows' entries are not used), drawn from draft_probs [N, V] (bf16 or fp32), or certain
    (None: greedy or n-gram drafts). u [N] and v [B] fp32 in [0, 1), temperature [B] fp32 (0: the largest logit, the first
    of equals, is taken and comes next). tokens: a sequence's taken drafts, then its next token, then -1; accepted: how many
    were taken; logp: each token's log probability under the target (at temperature 1 for 0; 0 where tokens is -1). A draft
    outside [0, V) is not taken (draft and cu may be int64: values past int32's ends are these); a row without a logit above -infinity takes none and gives -1. Rows in no sequence are not
    written. workspace: dsa_verify_workspace_bytes(N, V, B) bytes, or None for one kept per stream and host thread (a
    captured graph has its own)."""
    dev = C.on_gpu(logits, draft, cu, u, v, temperature, draft_probs, workspace)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"dsa_verify: logits {tuple(logits.shape)}, expected [N, V]")
    N, V = logits.shape
    logits, l_row = _rows(logits, "logits", logits.shape)
    q, q_row = (None, 0) if draft_probs is None else _rows(draft_probs, "draft_probs", logits.shape)
    if cu.dim() != 1 or cu.numel() < 1:
        raise ValueError(f"dsa_verify: cu {tuple(cu.shape)}, expected [B + 1]")
    B = cu.numel() - 1
    cu = C.whole(cu, "cu")
    draft = C.need(C.whole(draft, "draft"), "draft", torch.int32, (N,))
    u, v = C.need(u, "u", torch.float32, (N,)), C.need(v, "v", torch.float32, (B,))
    temperature = C.need(C.as_f32(temperature), "temperature", torch.float32, (B,))
    tokens, accepted = draft.new_empty(N), draft.new_empty(B)
    logp = u.new_empty(N)
    lib = _lib.lib()
    if workspace is not None:
        ws = C.given(workspace, "dsa_verify")
    else:
        ws = C.scratch(dev, int(lib.dsa_verify_workspace_bytes(N, V, B)), "verify")
    st = C.call(dev, lib.dsa_verify, logits.data_ptr(), logits.dtype is torch.float32, l_row, draft.data_ptr(),
                C.ptr(q), q is not None and q.dtype is torch.float32, q_row, cu.data_ptr(),
                u.data_ptr(), v.data_ptr(), temperature.data_ptr(), tokens.data_ptr(), accepted.data_ptr(),
                logp.data_ptr(), ws.data_ptr(), ws.numel() * ws.element_size(), N, V, B)
    _lib.check(st, "dsa_verify")
    return tokens, accepted, logp
