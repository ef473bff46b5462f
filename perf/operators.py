"""The work asked of the latent attention without a selection and of the page operations under it.

Five families, each with its range (see draw()):

- dense: dsa_dense.attend, absorbed latent attention of a decode batch (one new token a sequence, or the S tokens of a
  speculative step) over every cached token of the paged FP8 latent cache.
- expand: dsa_expand.expand, the keys and values of every head from the cached latent rows.
- expanded: dsa_expand.attend, a prefill's attention over expanded keys and values, ragged batches, causal.
- fork: dsa_pages.fork and then dsa_pages.release of the children: n samples of running sequences, begun and ended.
- compact: dsa_pages.compact, the live pages of a fragmented pool moved to its front.

With `own` false each family runs in its plain form: elementary torch operations in 32 bits, rounded once at the end.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
PAGE = 64
DV = 512  # latent width (the value of the absorbed form)
DH = 128  # expanded key (without rope) and value width of a head
NEG = -1e30  # lse of a query that sees nothing


def listed() -> list[dict]:
    return [
        # one sequence of a short conversation on a tensor-parallel shard: the smallest call, all latency
        dict(name="dense-1x4k-h16", family="dense", B=1, S=1, L=4096, low=4096, H=16, D=576),
        # a small batch at 32K, 64 heads
        dict(name="dense-8x32k-h64", family="dense", B=8, S=1, L=32768, low=32768, H=64, D=576),
        # a serving batch of conversations of all lengths
        dict(name="dense-48-ragged-h64", family="dense", B=48, S=1, L=32768, low=500, H=64, D=576),
        # a speculative step of 4 tokens, all 128 heads on one GPU, NoPE latent rows, odd batch
        dict(name="dense-13-spec4-h128", family="dense", B=13, S=4, L=12345, low=2000, H=128, D=512),
        # three short prompts on a tensor-parallel shard
        dict(name="expand-1001-h16", family="expand", B=3, P=1001, H=16, D=576),
        # a prefill batch's contexts, 64 heads
        dict(name="expand-16k-h64", family="expand", B=4, P=16384, H=64, D=576),
        # five short prompts on a tensor-parallel shard: latency
        dict(name="expanded-5-short-h16", family="expanded", B=5, N=333, low=20, cached=0, H=16, D=576, causal=True),
        # one long prompt, 64 heads: the largest call
        dict(name="expanded-8k-h64", family="expanded", B=1, N=8192, low=8192, cached=0, H=64, D=576, causal=True),
        # two more samples of each of four short conversations
        dict(name="fork-8-4k", family="fork", B=4, n=8, L=4096, low=1000, pages=320, D=576),
        # four samples of each of 32 sequences, tables of 512 pages
        dict(name="fork-128-32k", family="fork", B=32, n=128, L=32768, low=500, pages=10000, D=576),
        # a small pool after some sequences ended
        dict(name="compact-300", family="compact", B=6, pages=300, live=0.7, D=576),
        # a large pool, a little more than half of it live
        dict(name="compact-12k", family="compact", B=64, pages=12345, live=0.6, D=512),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng: random.Random) -> dict:
    """One more case of the listed ones' ranges; none costs more than the largest listed one."""
    family = rng.choice(["dense", "dense", "dense", "expand", "expanded", "expanded", "fork", "compact"])
    D = rng.choice([576, 576, 512])
    if family == "dense":
        B, S, H = _log(rng, 1, 96), rng.choice([1, 1, 1, 2, 4, 7]), rng.choice([8, 16, 16, 32, 64, 64, 128])
        L = _log(rng, 1, min(1 << 19, (1 << 20) / B, (1 << 26) / (B * S * H)))
        return dict(family=family, B=B, S=S, L=L, low=L if rng.random() < 0.3 else max(1, int(L * rng.random())), H=H,
                    D=D)
    if family == "expand":
        H = rng.choice([8, 16, 32, 64, 128])
        P = _log(rng, 1, (1 << 20) / H)
        return dict(family=family, B=_log(rng, 1, min(P, 16)), P=P, H=H, D=D)
    if family == "expanded":
        H = rng.choice([8, 16, 32, 64, 128])
        N = _log(rng, 1, 8192)
        cached = 0 if rng.random() < 0.5 else _log(rng, 1, 16384)
        causal = rng.random() < 0.85
        most = (1 << 31) // H  # pairs of tokens, all heads: the largest listed case's
        while N * (N + 2 * cached) > most:
            N, cached = (N + 1) // 2, cached // 2
        room = most // (N * (N + 2 * cached))
        return dict(family=family, B=_log(rng, 1, min(room, 8)), N=N, low=max(1, int(N * rng.random())), cached=cached,
                    H=H, D=D, causal=causal)
    if family == "fork":
        B, L = _log(rng, 1, 64), _log(rng, 1, 32768)
        n = _log(rng, 1, 256)
        return dict(family=family, B=B, n=n, L=L, low=max(1, int(L * rng.random())),
                    pages=B * math.ceil(L / PAGE) // 2 + n + _log(rng, 1, 2000) + 8, D=D)
    return dict(family=family, B=_log(rng, 1, 128), pages=_log(rng, 16, 12000), live=rng.uniform(0.1, 0.95), D=D)


# -- what a program has in hand before the call ------------------------------------------------------------------


def _lengths(n: int, low: int, high: int, seed: int) -> list[int]:
    """n lengths, U[low, high], one of them the longest: the same ones for every seed (so that shapes follow from the
    case alone), in another order."""
    rng = random.Random(n * 1000003 + high)
    x = [high] + [rng.randint(low, high) for _ in range(n - 1)]
    random.Random(seed).shuffle(x)
    return x


def _i32(x) -> torch.Tensor:
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _latent(slots: int, D: int, g: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """An FP8 latent cache as a program stores it: rows of N(0, 1) times a spread of magnitudes, a scale per token."""
    cache = torch.empty(slots, D, dtype=torch.float8_e4m3fn, device=DEV)
    scale = torch.empty(slots, dtype=torch.float32, device=DEV)
    for s in range(0, slots, 1 << 18):
        n = min(1 << 18, slots - s)
        x = torch.randn(n, D, generator=g, device=DEV) * torch.exp(0.3 * torch.randn(n, 1, generator=g, device=DEV))
        sc = x.abs().amax(-1).clamp(min=1e-30) / 448.0
        cache[s:s + n] = (x / sc[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        scale[s:s + n] = sc
    return cache, scale


def _tables(lengths: list[int], g: torch.Generator) -> tuple[torch.Tensor, int]:
    """Each sequence's pages, a random permutation of 1 .., and the pool's size (page 0 is the null page)."""
    npg = [math.ceil(n / PAGE) for n in lengths]
    table = torch.zeros(len(lengths), max(npg), dtype=torch.int32, device=DEV)
    perm = (torch.randperm(sum(npg), generator=g, device=DEV) + 1).to(torch.int32)
    at = 0
    for b, n in enumerate(npg):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, 1 + sum(npg)


def _cu(lengths: list[int]) -> torch.Tensor:
    return torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), _i32(lengths).cumsum(0, dtype=torch.int32)])


def _prepare_dense(case: dict, seed: int, g: torch.Generator) -> dict:
    B, S, H, D = case["B"], case["S"], case["H"], case["D"]
    lengths = _lengths(B, case["low"], case["L"], seed)
    table, pages = _tables(lengths, g)
    kv, kv_scale = _latent(pages * PAGE, D, g)
    q = (torch.randn(B, S, H, D, generator=g, device=DEV) * 1.5).to(torch.bfloat16)
    return dict(q=q, kv=kv, kv_scale=kv_scale, table=table, ctx_len=_i32(lengths), lengths=lengths)


def _split(total: int, n: int, seed: int) -> list[int]:
    """total in n parts of one at least."""
    g = torch.Generator().manual_seed(seed)
    cuts = sorted((torch.randperm(total - 1, generator=g)[:n - 1] + 1).tolist())
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _prepare_expand(case: dict, seed: int, g: torch.Generator) -> dict:
    lengths = _split(case["P"], case["B"], seed)
    table, pages = _tables(lengths, g)
    kv, kv_scale = _latent(pages * PAGE, case["D"], g)
    w = (torch.randn(case["H"], 2 * DH, DV, generator=g, device=DEV) * DV ** -0.5).to(torch.bfloat16)
    return dict(kv=kv, kv_scale=kv_scale, table=table, cu=_cu(lengths), lengths=lengths, w=w)


def _prepare_expanded(case: dict, seed: int, g: torch.Generator) -> dict:
    nq = _lengths(case["B"], case["low"], case["N"], seed)
    nk = [n + case["cached"] for n in nq]
    H, rope = case["H"], case["D"] - DV
    q = (torch.randn(sum(nq), H, DH + rope, generator=g, device=DEV) * 1.5).to(torch.bfloat16)
    k = torch.randn(sum(nk), H, DH, generator=g, device=DEV).to(torch.bfloat16)
    v = torch.randn(sum(nk), H, DH, generator=g, device=DEV).to(torch.bfloat16)
    kr = torch.randn(sum(nk), rope, generator=g, device=DEV).to(torch.bfloat16) if rope else None
    return dict(q=q, k=k, kr=kr, v=v, cu_q=_cu(nq), cu_k=_cu(nk), nq=nq, nk=nk)


def _caches(pages: int, D: int, g: torch.Generator) -> list[torch.Tensor]:
    """A layer's caches as bytes: latent rows and scales, indexer rows and scales, and for NoPE rows (the pooled
    indexer) the pool keys."""
    slots = pages * PAGE
    widths = [D, 4, 128, 4] if D == 576 else [D, 4, 256, 4, 64]
    return [torch.randint(0, 256, (slots, w), dtype=torch.uint8, generator=g, device=DEV) for w in widths]


def _prepare_fork(case: dict, seed: int, g: torch.Generator) -> dict:
    B, pages = case["B"], case["pages"]
    lengths = _lengths(B, case["low"], case["L"], seed)
    npg = [math.ceil(n / PAGE) for n in lengths]
    room = pages - 1 - case["n"]
    table = torch.zeros(B, max(npg), dtype=torch.int32, device=DEV)
    perm = (torch.randperm(pages - 1, generator=g, device=DEV) + 1).to(torch.int32)
    at = 0
    for b, n in enumerate(npg):  # where the pool is too small for all, the later sequences share earlier ones' pages
        if at + n > room:
            at = 0
        n = min(n, room)
        lengths[b] = min(lengths[b], n * PAGE)
        table[b, :n] = perm[at:at + n]
        at += n
    ref = torch.zeros(pages, dtype=torch.int32, device=DEV)
    for b in range(B):
        ref.index_add_(0, table[b, :math.ceil(lengths[b] / PAGE)].long(),
                       torch.ones(math.ceil(lengths[b] / PAGE), dtype=torch.int32, device=DEV))
    parents = torch.randint(0, B, (case["n"],), generator=g, device=DEV).to(torch.int32)
    return dict(ref=ref, table=table, ctx_len=_i32(lengths), parents=parents, ctx_child=_i32(lengths)[parents.long()],
                caches=_caches(pages, case["D"], g))


def _prepare_compact(case: dict, seed: int, g: torch.Generator) -> dict:
    B, pages = case["B"], case["pages"]
    live = max(1, int(case["live"] * (pages - 1)))
    ids = (torch.randperm(pages - 1, generator=g, device=DEV)[:live] + 1).to(torch.int32)
    width = math.ceil(live / B) + 2
    table = torch.zeros(B, width, dtype=torch.int32, device=DEV)
    per = math.ceil(live / B)
    for b in range(B):
        own_pages = ids[b * per:(b + 1) * per]
        table[b, :len(own_pages)] = own_pages
        if b:  # the first pages of a shared prompt
            shared = ids[:2]
            table[b, len(own_pages):len(own_pages) + len(shared)] = shared
    ref = torch.bincount(table.flatten().long(), minlength=pages).to(torch.int32)
    ref[0] = 0
    return dict(ref=ref, table=table, caches=_caches(pages, case["D"], g))


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    make = dict(dense=_prepare_dense, expand=_prepare_expand, expanded=_prepare_expanded, fork=_prepare_fork,
                compact=_prepare_compact)[case["family"]]
    return dict(make(case, seed, g), case=case)


# -- one pass ----------------------------------------------------------------------------------------------------


def _slots(table_row: torch.Tensor, n: int) -> torch.Tensor:
    t = torch.arange(n, device=DEV)
    return table_row[t // PAGE].long() * PAGE + t % PAGE


def _plain_dense(s: dict) -> tuple:
    B, S, H, D = s["q"].shape
    scale = 192 ** -0.5
    out = torch.zeros(B, S, H, DV, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((B, S, H), NEG, device=DEV)
    for b, n in enumerate(s["lengths"]):
        at = _slots(s["table"][b], n)
        K = s["kv"][at].float() * s["kv_scale"][at][:, None]
        sc = (s["q"][b].float().view(S * H, D) @ K.T).view(S, H, n) * scale
        seen = n - S + 1 + torch.arange(S, device=DEV)
        sc.masked_fill_((torch.arange(n, device=DEV) >= seen[:, None])[:, None], -math.inf)
        m = sc.amax(-1, keepdim=True).clamp(min=-1e38)
        p = torch.exp(sc - m)
        l = p.sum(-1)
        o = (p.view(S * H, n) @ K[:, :DV]).view(S, H, DV) / l.clamp(min=1e-38)[..., None]
        any_ = (seen > 0)[:, None].expand(S, H)
        out[b] = torch.where(any_[..., None], o, 0.0).to(torch.bfloat16)
        lse[b] = torch.where(any_, m[..., 0] + torch.log(l), NEG)
    return out, lse


def _plain_expand(s: dict) -> tuple:
    at = torch.cat([_slots(s["table"][b], n) for b, n in enumerate(s["lengths"])])
    c = s["kv"][at].float() * s["kv_scale"][at][:, None]
    H = s["w"].shape[0]
    kv = (c[:, :DV] @ s["w"].float().view(H * 2 * DH, DV).T).view(-1, H, 2 * DH).to(torch.bfloat16)
    kr = c[:, DV:].to(torch.bfloat16) if c.shape[1] > DV else None
    return kv[..., :DH].contiguous(), kr, kv[..., DH:].contiguous()


def _plain_expanded(s: dict) -> tuple:
    Tq, H, dq = s["q"].shape
    scale = 192 ** -0.5
    out = torch.zeros(Tq, H, DH, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((Tq, H), NEG, device=DEV)
    q0 = k0 = 0
    for nq, nk in zip(s["nq"], s["nk"]):
        seen = nk - nq + 1 + torch.arange(nq, device=DEV) if s["case"]["causal"] else torch.full((nq,), nk, device=DEV)
        hidden = torch.arange(nk, device=DEV) >= seen[:, None]
        step = max(1, (1 << 28) // (nq * nk))  # heads at once
        for h in range(0, H, step):
            q = s["q"][q0:q0 + nq, h:h + step].float().transpose(0, 1).contiguous()
            k = s["k"][k0:k0 + nk, h:h + step].float().permute(1, 2, 0).contiguous()
            sc = q[..., :DH].contiguous() @ k
            if dq > DH:
                sc += q[..., DH:].contiguous() @ s["kr"][k0:k0 + nk].float().T.contiguous()
            sc = (sc * scale).masked_fill_(hidden, -math.inf)
            m = sc.amax(-1, keepdim=True).clamp(min=-1e38)
            p = torch.exp(sc - m)
            l = p.sum(-1)
            v = s["v"][k0:k0 + nk, h:h + step].float().transpose(0, 1).contiguous()
            o = p @ v / l.clamp(min=1e-38)[..., None]
            out[q0:q0 + nq, h:h + step] = torch.where((seen > 0)[:, None], o, 0.0).to(torch.bfloat16).transpose(0, 1)
            lse[q0:q0 + nq, h:h + step] = torch.where(seen > 0, m[..., 0] + torch.log(l), NEG).T
        q0 += nq
        k0 += nk
    return out, lse


def _plain_fork(s: dict) -> tuple:
    ref, table, lens, parents = s["ref"], s["table"], s["ctx_len"], s["parents"].long()
    width = table.shape[1]
    full = lens[parents] // PAGE
    part = lens[parents] % PAGE > 0
    free = (ref[1:] == 0).nonzero().flatten() + 1
    rank = part.long().cumsum(0) - 1
    fits = ~part | (rank < len(free))
    page = torch.where(part & fits, free[rank.clamp(0, max(len(free) - 1, 0))] if len(free) else rank, 0)
    col = torch.arange(width, device=DEV)
    child = torch.where(col < full[:, None], table[parents], 0)
    child = torch.where((col == full[:, None]) & part[:, None], page[:, None].int(), child)
    child = torch.where(fits[:, None], child, 0)
    ref.index_add_(0, child.flatten().long(), (child.flatten() > 0).int())
    move = part & fits
    src, dst = table[parents, full.clamp(max=width - 1)][move].long(), page[move]
    for c in s["caches"]:
        v = c.view(-1, PAGE, c.shape[1])
        v[dst] = v[src]
    pages = torch.where(fits, page, -1).int()
    # and the children end
    held = torch.where(col < ((s["ctx_child"] + PAGE - 1) // PAGE)[:, None], child, 0).flatten().long()
    ref.index_add_(0, held, -(held > 0).int())
    ref.clamp_(min=0)
    return child, pages, ref, s["caches"]


def _plain_compact(s: dict) -> tuple:
    ref, table = s["ref"], s["table"]
    live = ref > 0
    live[0] = False
    n = int(live.sum())
    ids = torch.arange(ref.shape[0], device=DEV)
    movers = ids[live & (ids > n)]
    holes = ids[~live & (ids > 0) & (ids <= n)]
    remap = torch.where(live, ids, 0)
    remap[movers] = holes
    new_ref = torch.zeros_like(ref)
    new_ref[remap[live]] = ref[live]
    for c in s["caches"]:
        v = c.view(-1, PAGE, c.shape[1])
        v[holes] = v[movers]
    return remap[table.long()].int(), new_ref, remap.int(), s["caches"]


def _own_pass(s: dict, family: str) -> tuple:
    from trnrt_amd.kernels import dsa_dense, dsa_expand, dsa_pages

    if family == "dense":
        return dsa_dense.attend(s["q"], s["kv"], s["kv_scale"], s["table"], s["ctx_len"], PAGE, 192 ** -0.5, lse=True)
    if family == "expand":
        return dsa_expand.expand(s["kv"], s["kv_scale"], s["table"], s["cu"], sum(s["lengths"]), PAGE, s["w"])
    if family == "expanded":
        return dsa_expand.attend(s["q"], s["k"], s["kr"], s["v"], s["cu_q"], s["cu_k"], 192 ** -0.5,
                                 causal=s["case"]["causal"], lse=True)
    if family == "fork":
        child, pages = dsa_pages.fork(s["ref"], s["table"], s["ctx_len"], s["parents"], s["caches"], PAGE)
        dsa_pages.release(s["ref"], child, s["ctx_child"], PAGE)
        return child, pages, s["ref"], s["caches"]
    table, ref, remap = dsa_pages.compact(s["ref"], s["table"], s["caches"], PAGE)
    return table, ref, remap, s["caches"]


def run(state: dict):
    family = state["case"]["family"]
    if own:
        out = _own_pass(state, family)
    else:
        out = dict(dense=_plain_dense, expand=_plain_expand, expanded=_plain_expanded, fork=_plain_fork,
                   compact=_plain_compact)[family](state)
    return [x for x in out if x is not None]


# -- what a pass cannot do without -------------------------------------------------------------------------------


def _page_bytes(D: int) -> int:
    return PAGE * (sum([D, 4, 128, 4]) if D == 576 else sum([D, 4, 256, 4, 64]))


def _mean(case: dict, n: int, low: int, high: int) -> float:
    return high + (n - 1) * (low + high) / 2


def work(case: dict) -> dict:
    f, D = case["family"], case["D"]
    if f == "dense":
        t, M = _mean(case, case["B"], case["low"], case["L"]), case["S"] * case["H"]
        return dict(bytes=t * (D + 4 + 4 / PAGE) + case["B"] * M * (2 * D + 2 * DV + 4), flops=2 * t * M * (D + DV))
    if f == "expand":
        P, H = case["P"], case["H"]
        return dict(bytes=P * (D + 4) + H * 2 * DH * DV * 2 + P * H * 2 * DH * 2 + P * (D - DV) * 2,
                    flops=2 * P * DV * H * 2 * DH)
    if f == "expanded":
        B, H, dq, c = case["B"], case["H"], DH + D - DV, case["cached"]
        q = _mean(case, B, case["low"], case["N"])
        per = q / B
        pairs = B * (per * c + (per * (per + 1) / 2 if case["causal"] else per * per))
        return dict(bytes=q * H * (2 * dq + 2 * DH + 4) + (q + B * c) * (H * 2 * DH * 2 + (D - DV) * 2),
                    flops=2 * pairs * H * (dq + DH))
    if f == "fork":
        table = case["n"] * math.ceil(case["L"] / PAGE) * 4
        return dict(bytes=case["n"] * 2 * _page_bytes(D) + 3 * table + 4 * case["pages"], flops=0)
    moved = case["live"] * (1 - case["live"]) * case["pages"]
    return dict(bytes=moved * 2 * _page_bytes(D) + 12 * case["pages"] + 8 * case["live"] * case["pages"], flops=0)


# -- the same from the definitions, in 64 bits -------------------------------------------------------------------


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    f = case["family"]
    d = torch.float64
    if f == "dense":
        outs, lses = [], []
        S, H = case["S"], case["H"]
        for b, n in enumerate(s["lengths"]):
            pos = torch.arange(n, device=DEV)
            slot = s["table"][b].to(torch.int64)[pos // PAGE] * PAGE + pos % PAGE
            rows = s["kv"][slot].to(d) * s["kv_scale"][slot].to(d).unsqueeze(1)
            for i in range(S):
                see = n - S + i + 1
                if see < 1:
                    outs.append(torch.zeros(H, DV, dtype=d, device=DEV))
                    lses.append(torch.full((H,), NEG, dtype=d, device=DEV))
                    continue
                z = torch.mm(s["q"][b, i].to(d), rows[:see].t()) / math.sqrt(192.0)
                norm = torch.logsumexp(z, 1)
                outs.append(torch.mm((z - norm.unsqueeze(1)).exp(), rows[:see, :DV]))
                lses.append(norm)
        return [torch.stack(outs).view(case["B"], S, H, DV), torch.stack(lses).view(case["B"], S, H)]
    if f == "expand":
        ks, vs, rs = [], [], []
        w = s["w"].to(d)
        for b, n in enumerate(s["lengths"]):
            pos = torch.arange(n, device=DEV)
            slot = s["table"][b].to(torch.int64)[pos // PAGE] * PAGE + pos % PAGE
            rows = s["kv"][slot].to(d) * s["kv_scale"][slot].to(d).unsqueeze(1)
            ks.append(torch.stack([torch.mm(rows[:, :DV], w[h, :DH].t().contiguous()) for h in range(case["H"])], 1))
            vs.append(torch.stack([torch.mm(rows[:, :DV], w[h, DH:].t().contiguous()) for h in range(case["H"])], 1))
            rs.append(rows[:, DV:])
        out = [torch.cat(ks), torch.cat(rs), torch.cat(vs)]
        return out if case["D"] > DV else [out[0], out[2]]
    if f == "expanded":
        H = case["H"]
        out = torch.zeros(sum(s["nq"]), H, DH, dtype=d, device=DEV)
        lse = torch.full((sum(s["nq"]), H), NEG, dtype=d, device=DEV)
        qa = ka = 0
        for nq, nk in zip(s["nq"], s["nk"]):
            for r0 in range(0, nq, 2048):  # rows of queries, so that the scores stay small
                r1 = min(nq, r0 + 2048)
                last = nk - nq + r1 if case["causal"] else nk
                for h in range(H):
                    key = s["k"][ka:ka + last, h].to(d)
                    if s["kr"] is not None:
                        key = torch.cat([key, s["kr"][ka:ka + last].to(d)], 1)
                    z = torch.mm(s["q"][qa + r0:qa + r1, h].to(d), key.t().contiguous()) / math.sqrt(192.0)
                    if case["causal"]:
                        z = z + torch.full_like(z, -math.inf).triu(nk - nq + r0 + 1)
                    norm = torch.logsumexp(z, 1)
                    out[qa + r0:qa + r1, h] = torch.mm((z - norm.unsqueeze(1)).exp(), s["v"][ka:ka + last, h].to(d))
                    lse[qa + r0:qa + r1, h] = norm
            qa += nq
            ka += nk
        return [out, lse]
    return None
