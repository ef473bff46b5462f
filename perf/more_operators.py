"""The work asked of what stands around the attention in a step over the paged caches.

Four families, each with its range (see draw()):

- rotate: dsa_rope.rotate, rotary positions of one or several axes (time, height, width) for queries.
- append: dsa_cache.append, new latent rows and indexer keys normed, rotated, quantised and put into the paged caches.
- spans: dsa_expand.attend with a range of keys for each query (prefixes, documents), scores capped by a tanh, or a bias
  that grows with the distance.
- verify: dsa_verify.verify, drafted tokens against the target's logits from given random numbers.

With `own` false each family runs in its plain form: elementary torch operations, in 32 bits (angles, probabilities and
their sums in 64), rounded once at the end.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
PAGE = 64
LATENT = 512
ROPE = 64
KEY = 128  # indexer key width
DH = 128  # expanded key (without rope) and value width of a head
EPS = 1e-6
FP8_MAX = 448.0
SCALE = 192 ** -0.5


def listed() -> list[dict]:
    return [
        # the attention queries' rope columns in a decode step of 8 sequences: the smallest call, all latency
        dict(name="rotate-8-h64", family="rotate", T=8, H=64, R=32, axes=1, wide=576, half=False, dtype="bf16",
             far=131072),
        # the rope columns of a prefill chunk with images and video in it, three axes
        dict(name="rotate-8k-h64-3axes", family="rotate", T=8192, H=64, R=32, axes=3, wide=192, half=False,
             dtype="bf16", far=16384),
        # a decode step of 8 sequences: one latent row and one indexer key each
        dict(name="append-8", family="append", B=8, low=1, new=1, cached=4096, D=576, key=128, axes=1, normed=False,
             dtype="bf16"),
        # a speculative step of 13 sequences, 5 new tokens each, the projections' rows as they come (normed on the way)
        dict(name="append-13-spec5-normed", family="append", B=13, low=5, new=5, cached=4096, D=576, key=128, axes=1,
             normed=True, dtype="bf16"),
        # a prefill batch with images, 16k new tokens at most
        dict(name="append-16k-normed-3axes", family="append", B=4, low=1000, new=8192, cached=2048, D=576, key=128,
             axes=3, normed=True, dtype="bf16"),
        # three short prompts that begin with an image (seen both ways), a tensor-parallel shard
        dict(name="spans-prefix-3-short-h16", family="spans", B=3, N=333, low=100, cached=0, H=16, D=576, mask="prefix",
             cap=0.0, slopes=False),
        # documents packed into one sequence, 32 heads
        dict(name="spans-documents-8k-h32", family="spans", B=1, N=8192, low=8192, cached=0, H=32, D=576,
             mask="documents", cap=0.0, slopes=False),
        # capped scores, two prompts with prefixes
        dict(name="spans-capped-4k-h32", family="spans", B=2, N=4096, low=2500, cached=0, H=32, D=576, mask="prefix",
             cap=50.0, slopes=False),
        # a chunk of a long prompt over what is cached before it, biased by distance, NoPE rows
        dict(name="spans-distance-2k-of-10k-h32", family="spans", B=1, N=2048, low=2048, cached=8192, H=32, D=512,
             mask="causal", cap=0.0, slopes=True),
        # one sequence with 3 tokens from an n-gram draft: latency
        dict(name="verify-1x4-32k", family="verify", B=1, low=3, drafts=3, V=32768, probs="none", dtype="bf16"),
        # drafts of all lengths, a vocabulary of odd size, 32-bit logits and draft probabilities
        dict(name="verify-13-ragged-100k", family="verify", B=13, low=0, drafts=7, V=100003, probs="fp32",
             dtype="fp32"),
        # a serving batch, 4 drafted tokens each
        dict(name="verify-64x5-128k", family="verify", B=64, low=4, drafts=4, V=131072, probs="fp32", dtype="bf16"),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng: random.Random) -> dict:
    """One more case of the listed ones' ranges; none costs more than the largest listed one."""
    family = rng.choice(["rotate", "append", "append", "spans", "spans", "spans", "verify", "verify"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if family == "rotate":
        R = rng.choice([16, 24, 32, 32, 64])
        H = rng.choice([1, 5, 8, 16, 64, 64, 128])
        return dict(family=family, T=_log(rng, 1, 16384 * 64 / H / R), H=H, R=R, axes=rng.choice([1, 1, 2, 3, 4]),
                    wide=2 * R + rng.choice([0, 64, 128, 512]), half=rng.random() < 0.4, dtype=dtype,
                    far=_log(rng, 10, 1 << 20))
    if family == "append":
        B = _log(rng, 1, 64)
        new = _log(rng, 1, 16384 / B)
        D = rng.choice([576, 576, 512])
        return dict(family=family, B=B, low=new if rng.random() < 0.3 else rng.randint(0, new), new=new,
                    cached=_log(rng, 1, 65536 / B), D=D, key=rng.choice([0, KEY, KEY]), axes=rng.choice([1, 1, 3]),
                    normed=rng.random() < 0.6, dtype=dtype)
    if family == "spans":
        H = rng.choice([8, 16, 32])
        N = _log(rng, 1, 6000)
        cached = 0 if rng.random() < 0.6 else _log(rng, 1, 8192)
        most = (1 << 31) // H  # pairs of tokens, all heads: the largest listed case's
        while N * (N + cached) > most:
            N, cached = (N + 1) // 2, cached // 2
        room = most // (N * (N + cached))
        return dict(family=family, B=_log(rng, 1, min(room, 6)), N=N, low=max(1, int(N * rng.random())), cached=cached,
                    H=H, D=rng.choice([576, 576, 512]), mask=rng.choice(["causal", "prefix", "documents"]),
                    cap=rng.choice([0.0, 0.0, 15.0, 30.0, 50.0]), slopes=rng.random() < 0.4)
    V = _log(rng, 1000, 200000)
    drafts = rng.choice([0, 1, 2, 3, 4, 5, 7])
    B = _log(rng, 1, min(64, 64 * 5 * 131072 / V / (drafts + 1)))
    return dict(family=family, B=B, low=rng.randint(0, drafts), drafts=drafts, V=V,
                probs=rng.choice(["none", "fp32", "fp32", "bf16"]), dtype=dtype)


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


def _cu(lengths: list[int]) -> torch.Tensor:
    return torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), _i32(lengths).cumsum(0, dtype=torch.int32)])


def _type(name: str) -> torch.dtype:
    return torch.bfloat16 if name == "bf16" else torch.float32


def _frequencies(R: int) -> torch.Tensor:
    return (10000.0 ** (-torch.arange(R, dtype=torch.float64) / R)).float().to(DEV)


def _axes(R: int, axes: int) -> list[int] | None:
    """The axis of each frequency: the axes in turn, so that each one has high and low frequencies."""
    return None if axes == 1 else [i % axes for i in range(R)]


def _prepare_rotate(case: dict, seed: int, g: torch.Generator) -> dict:
    T, H, R, wide = case["T"], case["H"], case["R"], case["wide"]
    dtype = _type(case["dtype"])
    q = torch.randn(T, H, wide, generator=g, device=DEV).to(dtype)  # a projection's output, its last columns to rotate
    into = torch.empty(T, H, wide, dtype=dtype, device=DEV)  # the attention's queries, their last columns to write
    shape = (T,) if case["axes"] == 1 else (case["axes"], T)
    pos = torch.randint(0, case["far"], shape, generator=g, device=DEV).to(torch.int32)
    return dict(x=q[..., wide - 2 * R:], out=into[..., wide - 2 * R:], pos=pos, freq=_frequencies(R),
                axes=_axes(R, case["axes"]))


def _prepare_append(case: dict, seed: int, g: torch.Generator) -> dict:
    B, D, key = case["B"], case["D"], case["key"]
    new = _lengths(B, case["low"], case["new"], seed)
    T = sum(new)
    ctx = [n + c for n, c in zip(new, _lengths(B, 0, case["cached"], seed + 1))]
    npg = [math.ceil(n / PAGE) for n in ctx]
    pages = 1 + sum(npg)
    perm = (torch.randperm(pages - 1, generator=g, device=DEV) + 1).to(torch.int32)
    width = max(npg)
    begin = torch.tensor([sum(npg[:b]) for b in range(B)], device=DEV)
    col = torch.arange(width, device=DEV)
    held = col < torch.tensor(npg, device=DEV)[:, None]
    table = torch.where(held, perm[(begin[:, None] + col).clamp(max=pages - 2)], 0).to(torch.int32)
    dtype = _type(case["dtype"])
    x = torch.randn(T, 1536 + D, generator=g, device=DEV) * torch.exp(0.3 * torch.randn(T, 1, generator=g, device=DEV))
    state = dict(cu=_cu(new), ctx_len=_i32(ctx), table=table, x=x.to(dtype)[:, 1536:], T=T,
                 kv=torch.zeros(pages * PAGE, D, dtype=torch.float8_e4m3fn, device=DEV),
                 kv_scale=torch.zeros(pages * PAGE, device=DEV), freq=_frequencies(ROPE // 2),
                 axes=_axes(ROPE // 2, case["axes"]), pos=None, key=None, norm=None, key_norm=None)
    if case["axes"] > 1:
        state["pos"] = torch.randint(0, 16384, (case["axes"], T), generator=g, device=DEV).to(torch.int32)
    if key:
        state["key"] = torch.randn(T, key, generator=g, device=DEV).to(dtype)
        state["k"] = torch.zeros(pages * PAGE, key, dtype=torch.float8_e4m3fn, device=DEV)
        state["k_scale"] = torch.zeros(pages * PAGE, device=DEV)
    if case["normed"]:
        state["norm"] = (1 + 0.2 * torch.randn(LATENT, generator=g, device=DEV)).to(torch.bfloat16)
        if key:
            state["key_norm"] = tuple((m + 0.2 * torch.randn(key, generator=g, device=DEV)).to(torch.bfloat16)
                                      for m in (1, 0))
    return state


def _document_lengths(n: int, seed: int) -> list[int]:
    """Documents of 1 to about n / 3 tokens that fill n: the same ones for every seed, in another order."""
    rng = random.Random(n)
    x = []
    while sum(x) < n:
        x.append(min(n - sum(x), _log(rng, 1, max(1, n / 3))))
    random.Random(seed).shuffle(x)
    return x


def _prefix(i: int, n: int) -> int:
    """Tokens of sequence i's prefix, of n."""
    return (n * (3 + i % 4) + 9) // 10


def _prepare_spans(case: dict, seed: int, g: torch.Generator) -> dict:
    nq = _lengths(case["B"], case["low"], case["N"], seed)
    nk = [n + case["cached"] for n in nq]
    H, rope = case["H"], case["D"] - LATENT
    q = (torch.randn(sum(nq), H, DH + rope, generator=g, device=DEV) * 1.5).to(torch.bfloat16)
    k = torch.randn(sum(nk), H, DH, generator=g, device=DEV).to(torch.bfloat16)
    v = torch.randn(sum(nk), H, DH, generator=g, device=DEV).to(torch.bfloat16)
    kr = torch.randn(sum(nk), rope, generator=g, device=DEV).to(torch.bfloat16) if rope else None
    first = last = None
    if case["mask"] == "prefix":  # the prefix's tokens see each other both ways, the others what comes before them
        last = torch.cat([(torch.arange(a, device=DEV) + b - a + 1).clamp(min=_prefix(i, b))
                          for i, (a, b) in enumerate(zip(nq, nk))]).to(torch.int32)
    elif case["mask"] == "documents":  # a token sees its own document
        first = []
        for a, b in zip(nq, nk):
            d = torch.tensor(_document_lengths(b, seed), device=DEV)
            first.append((d.cumsum(0) - d).repeat_interleave(d)[b - a:])
        first = torch.cat(first).to(torch.int32)
    slopes = torch.exp2(-8.0 * torch.arange(1, H + 1, device=DEV) / H) if case["slopes"] else None
    return dict(q=q, k=k, kr=kr, v=v, cu_q=_cu(nq), cu_k=_cu(nk), nq=nq, nk=nk, first=first, last=last, slopes=slopes)


def _prepare_verify(case: dict, seed: int, g: torch.Generator) -> dict:
    B, V = case["B"], case["V"]
    rows = [n + 1 for n in _lengths(B, case["low"], case["drafts"], seed)]
    N = sum(rows)
    target = torch.randn(N, V, generator=g, device=DEV) * 2.5
    target += 10 * (torch.rand(N, V, generator=g, device=DEV) < 20 / V)  # some tokens that matter
    logits = target.to(_type(case["dtype"]))
    temperature = torch.tensor([0.0 if b % 5 == 3 else 0.6 + 0.1 * (b % 7) for b in range(B)], device=DEV)
    seq = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(rows, device=DEV))
    other = target + 0.4 * torch.randn(N, V, generator=g, device=DEV)  # the draft's
    other /= temperature.clamp(min=0.3)[seq][:, None]
    probs = torch.softmax(other, -1)
    noise = -torch.log(torch.rand(N, V, generator=g, device=DEV).clamp(min=1e-30))
    draft = ((probs if case["probs"] != "none" else probs.square()) / noise).argmax(-1).to(torch.int32)
    if case["probs"] == "none":
        probs = None
    else:
        probs = probs.to(_type(case["probs"]))
    return dict(logits=logits, draft=draft, probs=probs, temperature=temperature, cu=_cu(rows), N=N,
                u=torch.rand(N, generator=g, device=DEV), v=torch.rand(B, generator=g, device=DEV))


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    make = dict(rotate=_prepare_rotate, append=_prepare_append, spans=_prepare_spans, verify=_prepare_verify)
    return dict(make[case["family"]](case, seed, g), case=case)


# -- one pass ----------------------------------------------------------------------------------------------------


def _turn(x: torch.Tensor, pos: torch.Tensor, freq: torch.Tensor, axes, half: bool) -> torch.Tensor:
    """The rows x [T, H, 2R] in 32 bits, rotated."""
    R = freq.shape[0]
    at = pos if axes is None else pos[torch.tensor(axes, device=DEV)].T
    phi = at.double().view(x.shape[0], -1) * freq.double()
    c, s = torch.cos(phi).float()[:, None], torch.sin(phi).float()[:, None]
    a, b = (x[..., :R], x[..., R:]) if half else (x[..., 0::2], x[..., 1::2])
    y = [a * c - b * s, b * c + a * s]
    return torch.cat(y, -1) if half else torch.stack(y, -1).flatten(-2)


def _plain_rotate(s: dict) -> tuple:
    s["out"].copy_(_turn(s["x"].float(), s["pos"], s["freq"], s["axes"], s["case"]["half"]))
    return (s["out"],)


def _plain_append(s: dict) -> tuple:
    T = s["T"]
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(s["cu"][1:], t, right=True)
    at = s["ctx_len"][b] - s["cu"][b + 1] + t
    slot = s["table"][b, at // PAGE].long() * PAGE + at % PAGE
    pos = at if s["pos"] is None else s["pos"]
    x = s["x"].float()
    if s["norm"] is not None:
        c = x[:, :LATENT]
        c = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + EPS) * s["norm"].float()
        x = torch.cat([c, x[:, LATENT:]], -1)
    if x.shape[1] > LATENT:
        x = torch.cat([x[:, :LATENT], _turn(x[:, None, LATENT:], pos, s["freq"], s["axes"], False)[:, 0]], -1)
    _put(s["kv"], s["kv_scale"], slot, x)
    if s["key"] is None:
        return s["kv"], s["kv_scale"]
    y = s["key"].float()
    if s["key_norm"] is not None:
        d = y - y.mean(-1, keepdim=True)
        y = d * torch.rsqrt(d.square().mean(-1, keepdim=True) + EPS)
        y = y * s["key_norm"][0].float() + s["key_norm"][1].float()
    if x.shape[1] > LATENT:
        y = torch.cat([_turn(y[:, None, :ROPE], pos, s["freq"], s["axes"], True)[:, 0], y[:, ROPE:]], -1)
    _put(s["k"], s["k_scale"], slot, y)
    return s["kv"], s["kv_scale"], s["k"], s["k_scale"]


def _put(cache: torch.Tensor, scale: torch.Tensor, slot: torch.Tensor, x: torch.Tensor) -> None:
    sc = x.abs().amax(-1).clamp(min=1e-30) / FP8_MAX
    code = (x / sc[:, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    cache.view(torch.uint8)[slot] = code.view(torch.uint8)
    scale[slot] = sc


def _plain_spans(s: dict) -> tuple:
    case, H = s["case"], s["q"].shape[1]
    nq, nk = (c[1:] - c[:-1] for c in (s["cu_q"], s["cu_k"]))
    iq, ik = torch.arange(max(s["nq"]), device=DEV), torch.arange(max(s["nk"]), device=DEV)
    real = iq < nq[:, None]
    row = torch.where(real, s["cu_q"][:-1, None] + iq, 0)  # [B, nq] padded, every sequence at once
    col = torch.where(ik < nk[:, None], s["cu_k"][:-1, None] + ik, 0)
    B, a, b = len(s["nq"]), len(iq), len(ik)

    def heads(x, at):
        return x[at].float().transpose(1, 2).contiguous().view(B * H, at.shape[1], -1)

    z = torch.bmm(heads(s["q"][..., :DH], row), heads(s["k"], col).transpose(1, 2).contiguous())
    if s["kr"] is not None:
        r = s["kr"][col].float()[:, None].expand(B, H, b, ROPE).reshape(B * H, b, ROPE)
        z += torch.bmm(heads(s["q"][..., DH:], row), r.transpose(1, 2).contiguous())
    z = z.view(B, H, a, b).mul_(SCALE)
    if case["cap"]:
        z.div_(case["cap"]).tanh_().mul_(case["cap"])
    place = (nk - nq)[:, None] + iq
    if s["slopes"] is not None:
        z -= s["slopes"].view(H, 1, 1) * (place[:, :, None] - ik).abs().float()[:, None]
    low = torch.zeros_like(place) if s["first"] is None else s["first"][row]
    high = place + 1 if s["last"] is None else s["last"][row]
    seen = (ik >= low[..., None]) & (ik < torch.minimum(high, nk[:, None])[..., None])
    z.masked_fill_(~seen[:, None], -math.inf)
    m = z.amax(-1, keepdim=True).clamp(min=-1e38)
    z.sub_(m).exp_()
    l = z.sum(-1)
    o = torch.bmm(z.view(B * H, a, b), heads(s["v"], col)).view(B, H, a, DH) / l[..., None]
    lse = m[..., 0] + torch.log(l)
    return o.transpose(1, 2)[real].to(torch.bfloat16), lse.transpose(1, 2)[real]


def _plain_verify(s: dict) -> tuple:
    cu, d, N, V = s["cu"].long(), s["draft"].long(), s["N"], s["logits"].shape[1]
    B = len(cu) - 1
    row = torch.arange(N, device=DEV)
    seq = torch.searchsorted(cu[1:], row, right=True)
    warm = s["temperature"][seq] > 0
    z = s["logits"].double() / torch.where(warm, s["temperature"][seq], 1.0).double()[:, None]
    m = z.amax(-1, keepdim=True)
    most = torch.where(z == m, torch.arange(V, device=DEV), V).amin(-1)  # the first of the largest
    p = torch.exp(z - m)
    whole = p.sum(-1, keepdim=True)
    p /= whole
    px = p.gather(1, d[:, None])[:, 0]
    qx = 1.0 if s["probs"] is None else s["probs"].gather(1, d[:, None])[:, 0].double()
    taken = torch.where(warm, s["u"].double() * qx < px, d == most) & (row < cu[seq + 1] - 1)
    stop = torch.full((B,), N, device=DEV).scatter_reduce_(0, seq, torch.where(taken, N, row), "amin")
    p, more = p[stop], stop < cu[1:] - 1
    if s["probs"] is None:
        r = torch.where(more[:, None] & (torch.arange(V, device=DEV) == d[stop][:, None]), 0.0, p)
    else:
        r = torch.where(more[:, None], (p - s["probs"][stop].double()).clamp(min=0), p)
    r = torch.where((r.sum(-1) > 0)[:, None], r, p)
    c = r.cumsum(-1)
    token = (c <= s["v"].double()[:, None] * c[:, -1:]).sum(-1)
    token = torch.where(s["temperature"] > 0, token, most[stop])
    out = torch.where(row < stop[seq], d, torch.where(row == stop[seq], token[seq], -1))
    logp = z.gather(1, out.clamp(min=0)[:, None])[:, 0] - m[:, 0] - torch.log(whole[:, 0])
    return out.int(), (stop - cu[:-1]).int(), torch.where(out < 0, 0.0, logp).float()


def _own_pass(s: dict, case: dict) -> tuple:
    from trnrt_amd.kernels import dsa_cache, dsa_expand, dsa_rope, dsa_verify

    if case["family"] == "rotate":
        return (dsa_rope.rotate(s["x"], s["pos"], s["freq"], axes=s["axes"], interleaved=not case["half"],
                                out=s["out"]),)
    if case["family"] == "append":
        roped = case["D"] > LATENT
        rows = [dsa_cache.Rows(s["x"], s["kv"], s["kv_scale"], rope_at=LATENT if roped else None, norm=s["norm"],
                               eps=EPS)]
        if s["key"] is not None:
            rows.append(dsa_cache.Rows(s["key"], s["k"], s["k_scale"], rope_at=0 if roped else None, interleaved=False,
                                       norm=s["key_norm"], eps=EPS))
        dsa_cache.append(rows, s["table"], s["ctx_len"], PAGE, cu_new=s["cu"], positions=s["pos"],
                         inv_freq=s["freq"] if roped else None, axes=s["axes"])
        return (s["kv"], s["kv_scale"]) if s["key"] is None else (s["kv"], s["kv_scale"], s["k"], s["k_scale"])
    if case["family"] == "spans":
        return dsa_expand.attend(s["q"], s["k"], s["kr"], s["v"], s["cu_q"], s["cu_k"], SCALE, causal=s["last"] is None,
                                 first=s["first"], last=s["last"], softcap=case["cap"], slopes=s["slopes"], lse=True)
    return dsa_verify.verify(s["logits"], s["draft"], s["cu"], s["u"], s["v"], s["temperature"], draft_probs=s["probs"])


def run(state: dict):
    case = state["case"]
    if own:
        return list(_own_pass(state, case))
    plain = dict(rotate=_plain_rotate, append=_plain_append, spans=_plain_spans, verify=_plain_verify)
    return list(plain[case["family"]](state))


# -- what a pass cannot do without -------------------------------------------------------------------------------


def work(case: dict) -> dict:
    f = case["family"]
    size = 2 if case.get("dtype") == "bf16" else 4
    if f == "rotate":
        n = case["T"] * case["H"] * 2 * case["R"]
        return dict(bytes=2 * n * size + 4 * case["T"] * case["axes"], flops=3 * n)
    if f == "append":
        T = sum(_lengths(case["B"], case["low"], case["new"], 0))
        W, kinds = case["D"] + case["key"], 1 + (case["key"] > 0)
        return dict(bytes=T * (W * (size + 1) + 4 * kinds + 4 * case["axes"]) + 4 * case["B"], flops=8 * T * W)
    if f == "spans":
        nq = _lengths(case["B"], case["low"], case["N"], 0)
        H, dq, pairs = case["H"], DH + case["D"] - LATENT, 0
        for i, n in enumerate(nq):
            c, k = case["cached"], n + case["cached"]
            if case["mask"] == "documents":
                at = 0
                for d in _document_lengths(k, 0):
                    new = max(0, min(d, at + d - c))  # of the document's tokens those that ask
                    pairs += new * d - new * (new - 1) // 2
                    at += d
            else:
                pairs += n * c + n * (n + 1) // 2
                if case["mask"] == "prefix":
                    both = max(0, _prefix(i, k) - c)  # queries of the prefix: what they see past themselves
                    pairs += both * (both - 1) // 2
        q = sum(nq)
        keys = q + case["B"] * case["cached"]
        return dict(bytes=q * H * (2 * dq + 2 * DH + 4) + keys * (H * 2 * DH * 2 + 2 * (dq - DH)),
                    flops=2 * pairs * H * (dq + DH))
    N = sum(n + 1 for n in _lengths(case["B"], case["low"], case["drafts"], 0))
    q = {"none": 0, "bf16": 2, "fp32": 4}[case["probs"]]
    return dict(bytes=(N * size + case["B"] * q) * case["V"] + 16 * N, flops=6 * N * case["V"])


# -- the same from the definitions, in 64 bits -------------------------------------------------------------------


def _rotated(x: torch.Tensor, angle: torch.Tensor, half: bool) -> torch.Tensor:
    """x [T, H, 2R] in 64 bits as complex numbers, turned by angle [T, R]."""
    R = angle.shape[1]
    pairs = x.reshape(*x.shape[:-1], 2, R).transpose(-1, -2) if half else x.reshape(*x.shape[:-1], R, 2)
    turned = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None]
    y = torch.view_as_real(turned)
    return (y.transpose(-1, -2) if half else y).reshape(x.shape)


def _angles(pos: torch.Tensor, freq: torch.Tensor, axes) -> torch.Tensor:
    own_axis = [0] * freq.shape[0] if axes is None else axes
    p = pos.reshape(-1, pos.shape[-1]).to(torch.float64)
    return torch.stack([p[a] * float(f) for a, f in zip(own_axis, freq.tolist())], 1)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    d = torch.float64
    if case["family"] == "rotate":
        return [_rotated(s["x"].to(d), _angles(s["pos"], s["freq"], s["axes"]), case["half"])]
    if case["family"] == "append":
        cu, ctx, table = s["cu"].tolist(), s["ctx_len"].tolist(), s["table"].to(torch.int64)
        slots, places = [], []
        for b in range(case["B"]):
            n = cu[b + 1] - cu[b]
            p = torch.arange(ctx[b] - n, ctx[b], device=DEV)
            slots.append(table[b][p // PAGE] * PAGE + p % PAGE)
            places.append(p)
        slot, place = torch.cat(slots), torch.cat(places)
        angle = _angles(place if s["pos"] is None else s["pos"], s["freq"], s["axes"])
        rows = s["x"].to(d)
        if s["norm"] is not None:
            part = rows[:, :LATENT]
            rows = torch.cat([part / torch.sqrt((part * part).sum(1, keepdim=True) / LATENT + EPS) * s["norm"].to(d),
                              rows[:, LATENT:]], 1)
        roped = case["D"] > LATENT
        if roped:
            rows = torch.cat([rows[:, :LATENT], _rotated(rows[:, LATENT:].unsqueeze(1), angle, False).squeeze(1)], 1)
        out = []
        for cache, scale, y, key in ((s["kv"], s["kv_scale"], rows, False),
                                     (s.get("k"), s.get("k_scale"), s["key"], True)):
            if y is None:
                continue
            y = y.to(d)
            if key and s["key_norm"] is not None:
                var, mean = torch.var_mean(y, 1, correction=0, keepdim=True)
                y = (y - mean) / torch.sqrt(var + EPS) * s["key_norm"][0].to(d) + s["key_norm"][1].to(d)
            if key and roped:
                y = torch.cat([_rotated(y[:, :ROPE].unsqueeze(1), angle, True).squeeze(1), y[:, ROPE:]], 1)
            step = torch.clamp(y.abs().max(1).values, min=1e-30) / FP8_MAX
            full, fs = cache.to(d), scale.to(d)
            full[slot] = y / step.unsqueeze(1)
            fs[slot] = step
            out += [full, fs]
        return out
    if case["family"] == "spans":
        H = case["H"]
        out = torch.zeros(sum(s["nq"]), H, DH, dtype=d, device=DEV)
        lse = torch.zeros(sum(s["nq"]), H, dtype=d, device=DEV)
        qa = ka = 0
        for nq, nk in zip(s["nq"], s["nk"]):
            t = torch.arange(nk, device=DEV)
            for r0 in range(0, nq, 2048):  # rows of queries, so that the scores stay small
                r1 = min(nq, r0 + 2048)
                p = torch.arange(nk - nq + r0, nk - nq + r1, device=DEV).unsqueeze(1)
                hide = t < s["first"][qa + r0:qa + r1].unsqueeze(1) if s["first"] is not None else t < 0
                hide = hide | ((t >= s["last"][qa + r0:qa + r1].unsqueeze(1)) if s["last"] is not None else t > p)
                for h in range(H):
                    key = s["k"][ka:ka + nk, h].to(d)
                    if s["kr"] is not None:
                        key = torch.cat([key, s["kr"][ka:ka + nk].to(d)], 1)
                    z = torch.mm(s["q"][qa + r0:qa + r1, h].to(d), key.t().contiguous()) / math.sqrt(192.0)
                    if case["cap"]:
                        z = case["cap"] * torch.tanh(z / case["cap"])
                    if s["slopes"] is not None:
                        z = z - float(s["slopes"][h]) * (p - t).abs()
                    z[hide] = -math.inf
                    norm = torch.logsumexp(z, 1)
                    out[qa + r0:qa + r1, h] = torch.mm((z - norm.unsqueeze(1)).exp(), s["v"][ka:ka + nk, h].to(d))
                    lse[qa + r0:qa + r1, h] = norm
            qa += nq
            ka += nk
        return [out, lse]
    cu, heat = s["cu"].tolist(), s["temperature"].tolist()
    logps = torch.zeros(s["N"], dtype=d, device=DEV)
    for b in range(case["B"]):
        for j in range(cu[b], cu[b + 1]):
            logs = torch.log_softmax(s["logits"][j].to(d) / (float(s["temperature"][b]) if heat[b] > 0 else 1.0), 0)
            x, p = int(s["draft"][j]), logs.exp()
            q = s["probs"][j].to(d) if s["probs"] is not None else None
            if j + 1 < cu[b + 1]:
                if heat[b] > 0:
                    taken = float(s["u"][j]) * (1.0 if q is None else float(q[x])) < float(p[x])
                else:
                    taken = int((logs == logs.max()).nonzero()[0]) == x
                if taken:
                    logps[j] = logs[x]
                    continue
                if q is None:
                    p[x] = 0
                else:
                    p = torch.relu(p - q)
            sums = torch.cumsum(p, 0)
            y = int((sums > float(s["v"][b]) * float(sums[-1])).nonzero()[0]) if heat[b] > 0 else int(
                (logs == logs.max()).nonzero()[0])
            logps[j] = logs[y]
            break
    return [None, None, logps]
