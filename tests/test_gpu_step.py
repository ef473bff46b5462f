"""The operators around the attention as a program uses them together: a prompt that begins with an image (append with several
axes, rotate, expand, attention with a prefix), and speculative steps over the same caches (append, rotate, dsa_dense.attend,
verify, the length back by what was not taken), eager and captured in a graph."""

import pytest
import torch

from tests._helpers import say
from tests.test_gpu_expand import cu_of, gather
from tests.test_gpu_rope import freqs
from tests.test_gpu_spans import compare, reference
from trnrt_amd.kernels import dsa_cache, dsa_dense, dsa_expand, dsa_rope, dsa_verify
from trnrt_amd.kernels.dsa_cache import Rows

pytestmark = pytest.mark.gpu
FP8, PS, H, SCALE = torch.float8_e4m3fn, 64, 4, 192 ** -0.5
AXES = [i % 3 for i in range(32)]


class Caches:
    def __init__(self, slots):
        self.kv, self.k = (torch.zeros(slots, w, dtype=FP8, device="cuda") for w in (576, 128))
        self.kvs, self.ks = torch.zeros(slots, device="cuda"), torch.zeros(slots, device="cuda")

    def append(self, rows, keys, table, ctx, freq, norm, **kw):
        dsa_cache.append([Rows(rows, self.kv, self.kvs, rope_at=512, norm=norm[0]),
                          Rows(keys, self.k, self.ks, rope_at=0, interleaved=False, norm=norm[1:])], table, ctx, PS,
                         inv_freq=freq, **kw)

    def all(self):
        return [self.kv.view(torch.uint8), self.k.view(torch.uint8), self.kvs, self.ks]


def norms(g):
    return [(1 + 0.1 * torch.randn(512, generator=g)).cuda(), (1 + 0.1 * torch.randn(128, generator=g)).cuda(),
            (0.1 * torch.randn(128, generator=g)).cuda()]


def test_prompt():
    """Two prompts whose images' tokens see each other both ways, against float64 attention over the rows in the cache."""
    say("step prompt")
    g = torch.Generator().manual_seed(1)
    lens, image = [150, 70], [90, 33]
    table = torch.tensor([[5, 2, 3], [1, 4, 0]], dtype=torch.int32)
    T = sum(lens)
    c = Caches(6 * PS)
    pos = torch.randint(0, 500, (3, T), generator=g).to(torch.int32).cuda()
    x = torch.randn(T, 576 + 1536, generator=g).bfloat16().cuda()
    keys = torch.randn(T, 128, generator=g).bfloat16().cuda()
    c.append(x[:, 1536:], keys, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), freqs(32), norms(g), cu_new=cu_of(lens).cuda(),
             positions=pos, axes=AXES)
    w = (torch.randn(H, 256, 512, generator=g) * 512 ** -0.5).bfloat16().cuda()
    k, kr, v = dsa_expand.expand(c.kv, c.kvs, table.cuda(), cu_of(lens).cuda(), T, PS, w)
    rows = gather(c.kv.cpu().view(torch.uint8), c.kvs.cpu(), table, lens, PS)
    assert ((kr.cpu().double() - rows[:, 512:]).abs() <= (2.0 ** -8 + 2.0 ** -23) * rows[:, 512:].abs()).all()
    q = torch.randn(T, H, 192, generator=g).bfloat16().cuda()
    dsa_rope.rotate(q[..., 128:], pos, freqs(32), axes=AXES, out=q[..., 128:])
    last = torch.cat([(torch.arange(n) + 1).clamp(min=m) for n, m in zip(lens, image)]).to(torch.int32).cuda()
    out, lse = dsa_expand.attend(q, k, kr, v, cu_of(lens).cuda(), cu_of(lens).cuda(), SCALE, causal=False, last=last)
    compare(out, lse, reference(q, k, kr, v, lens, lens, SCALE, False, None, last, 0.0, None))


@pytest.mark.parametrize("captured", [False, True])
def test_speculative_steps(captured):
    """Four steps of 3 drafted tokens in three sequences. The caches end as if the tokens taken alone had been appended, one
    at a time; a step's tokens are what verify gives for logits computed from float64 attention over the cache's own rows."""
    say("step speculative", captured)
    g = torch.Generator().manual_seed(2)
    B, S, V, steps = 3, 4, 40, 4
    table = torch.arange(1, 10).view(3, 3).to(torch.int32)
    old = [60, 1, 126]
    c, alone = Caches(10 * PS), Caches(10 * PS)
    freq, norm = freqs(32), norms(g)
    tb, ctx = table.cuda(), torch.tensor(old, dtype=torch.int32).cuda()
    start = torch.randn(sum(old), 576, generator=g).bfloat16().cuda(), torch.randn(sum(old), 128, generator=g).bfloat16().cuda()
    for x in (c, alone):
        x.append(*start, tb, ctx, freq, norm, cu_new=cu_of(old).cuda())
    head = (torch.randn(H * 512, V, generator=g) * 0.3).cuda()
    temperature = torch.tensor([0.8, 0.0, 1.3]).cuda()
    cu = torch.arange(0, B * S + 1, S, dtype=torch.int32).cuda()
    held = dict(x=torch.zeros(B * S, 576).bfloat16().cuda(), key=torch.zeros(B * S, 128).bfloat16().cuda(),
                q=torch.zeros(B * S, H, 192).bfloat16().cuda(), draft=torch.zeros(B * S, dtype=torch.int32).cuda(),
                probs=torch.zeros(B * S, V).cuda(), u=torch.zeros(B * S).cuda(), v=torch.zeros(B).cuda())
    place = torch.arange(S, dtype=torch.int32).cuda()

    def step():
        ctx.add_(S)
        c.append(held["x"], held["key"], tb, ctx, freq, norm)
        q = torch.empty(B * S, H, 576, dtype=torch.bfloat16, device="cuda")
        q[..., :512] = held["q"][..., :128].repeat(1, 1, 4)
        pos = (ctx[:, None] - S + place).reshape(-1)
        dsa_rope.rotate(held["q"][..., 128:], pos, freq, out=q[..., 512:])
        o, _ = dsa_dense.attend(q.view(B, S, H, 576), c.kv, c.kvs, tb, ctx, PS, SCALE)
        logits = o.view(B * S, H * 512).float() @ head
        got = dsa_verify.verify(logits, held["draft"], cu, held["u"], held["v"], temperature, draft_probs=held["probs"])
        ctx.sub_(S - 1 - got[1])
        return q, o, logits, got

    def fresh():
        for name, t in held.items():
            if name == "draft":
                t.copy_(torch.randint(0, V, t.shape, generator=g))
            elif name == "probs":
                t.copy_(torch.softmax(torch.randn(t.shape, generator=g), -1))
            elif name in "uv":
                t.copy_(torch.rand(t.shape, generator=g) * (0.3 if name == "u" else 1.0))  # (drafts that are often taken)
            else:
                t.copy_(torch.randn(t.shape, generator=g))

    graph = None
    if captured:
        fresh()
        at = ctx.clone()
        step()  # (torch's own kernels, once before the capture)
        ctx.copy_(at)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
    taken_any = 0
    for _ in range(steps):
        fresh()
        before = ctx.cpu()
        if captured:
            graph.replay()
        else:
            out = step()
        torch.cuda.synchronize()
        q, o, logits, (tokens, accepted, logp) = out
        again = dsa_verify.verify(logits, held["draft"], cu, held["u"], held["v"], temperature, draft_probs=held["probs"])
        assert all(torch.equal(a, b) for a, b in zip((tokens, accepted, logp), again))
        after, n = ctx.cpu(), accepted.cpu()
        assert torch.equal(after, before + 1 + n)
        taken_any += int(n.sum())
        for b in range(B):
            rows = gather(c.kv.cpu().view(torch.uint8), c.kvs.cpu(), table[b:b + 1], [int(before[b]) + S], PS)
            for i in range(S):
                m = int(before[b]) + i + 1
                p = torch.softmax(q[b * S + i].cpu().double() @ rows[:m].T * SCALE, -1)
                want, size = p @ rows[:m, :512], p @ rows[:m, :512].abs()
                # weights in two bf16 terms (2^-16) of scores that 576 fp32 sums have off by e, outputs rounded to bf16
                e = (q[b * S + i].cpu().double().abs() @ rows[:m].abs().T * SCALE).amax(-1, keepdim=True) * 576 * 2.0 ** -24
                tol = size * (2.0 ** -16 + 2 * e + 2.0 ** -20) * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
                assert ((o[b, i].cpu().double() - want).abs() <= tol).all()
            for i in range(1 + int(n[b])):  # the tokens that stay, one at a time
                alone.append(held["x"][b * S + i:][:1], held["key"][b * S + i:][:1], tb[b:b + 1],
                             torch.tensor([int(before[b]) + i + 1], dtype=torch.int32).cuda(), freq, norm)
    assert taken_any > 0
    for b in range(B):
        t = torch.arange(int(ctx[b]))
        slot = (table[b][t // PS].long() * PS + t % PS).cuda()
        for x, y in zip(c.all(), alone.all()):
            assert torch.equal(x[slot], y[slot])
