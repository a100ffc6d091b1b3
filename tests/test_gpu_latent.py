"""Latent attention against its definition in 64 bits (MI355X): writes, gathers,
the absorbed form over pages and the expanded form over dense rows.

Attention rounds its weights to the cache's type (half a step: u relative; their
sum is of the rounded ones) and the outputs, and sums in 32 bits: a score of n
products is off by less than 2 n 2^-24 times the sum of their magnitudes, and its
weight by as much relatively.  With weights p of values x, |error| <=
(u + 2 s) (sum p |x| + |out|) + u |out|, s the largest score's error.  Halves (fp16)
also lose what is below 2^-25 of 2^-7 of a row's largest weight: 2^-30 sum |x|.
"""
import math

import pytest
import torch

from stepquant_amd.kernels.kv_cache import BlockTables, KVCache
from stepquant_amd.kernels.latent_cache import LatentCache, expanded_attention
from stepquant_amd.kernels.rotary import Rotary
from tests.helpers import dev

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
U = {"bf16": 2. ** -8, "fp16": 2. ** -11}


def gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


def randn(g, *shape, dtype="bf16"):
    return torch.randn(*shape, generator=g, device=dev()).to(TYPES[dtype])


def attention64(q, k, v, seen, scale, u):
    """(out, bound) in 64 bits: q [n, d], k [j, d], v [j, e], seen [n, j]."""
    q, k, v = q.double(), k.double(), v.double()
    s = (q @ k.t().contiguous()) * scale
    size = (q.abs() @ k.abs().t().contiguous()) * abs(scale)
    off = 2 * (q.shape[1] + 4) * 2. ** -24 * torch.where(seen, size, 0.).amax(1, keepdim=True)
    # (of large scores the difference from the largest is rounded, too)
    off = off + 2. ** -22 * torch.where(seen, s.abs(), 0.).amax(1, keepdim=True)
    p = torch.softmax(s.masked_fill(~seen, -math.inf), 1)
    p = torch.where(seen.any(1, keepdim=True), p, 0.)
    out = p @ v
    spread = p @ v.abs() + out.abs()
    bound = (u + 2 * off) * spread + u * out.abs() + 2. ** -30 * (seen.double() @ v.abs()) + 1e-30
    return out, bound


class Batch:
    """Requests of (held, new) tokens over a latent cache, with the same rows kept dense."""

    def __init__(self, sizes, latent=512, dtype="bf16", P=64, heads=16, padding=0, seed=0, causal=True, size=1.):
        g = gen(seed)
        old, new = [o for o, _ in sizes], [n for _, n in sizes]
        blocks = [-(-(o + n) // P) for o, n in sizes]
        self.tables = BlockTables(len(sizes) + 2, 3 + sum(blocks), max(blocks) + 1, page_tokens=P)
        self.tables.free.copy_(torch.randperm(self.tables.pages - 1, generator=g, device=dev()) + 1)
        self.cache = LatentCache(self.tables.pages, latent, page_tokens=P, dtype=TYPES[dtype])
        # what earlier requests left in the pages is not seen
        self.cache.data[1:] = math.nan
        rows = torch.randperm(len(sizes) + 2, generator=g, device=dev())[:len(sizes)]
        self.dense = [randn(g, o + n, latent + 64, dtype=dtype) * size for o, n in sizes]
        plan = self.tables.plan(old, rows)
        held = torch.cat([x[:o] for x, o in zip(self.dense, old)])
        self.cache.append(held[:, :latent], held[:, latent:], plan)
        self.tables.commit(plan)
        tokens = sum(new) + padding
        self.plan = self.tables.plan(torch.tensor(new, device=dev()), rows, tokens=tokens, max_new=max(new), absorbed=heads,
                                     causal=causal)
        fresh = torch.cat([x[o:] for x, o in zip(self.dense, old)] + [randn(g, padding, latent + 64, dtype=dtype)])
        self.cache.append(fresh[:, :latent], fresh[:, latent:], self.plan)
        self.q = randn(g, tokens, heads, latent, dtype=dtype) * (3 * torch.rand(tokens, heads, 1, generator=g, device=dev())).to(TYPES[dtype])
        self.q_rope = randn(g, tokens, heads, 64, dtype=dtype)
        self.old, self.new, self.latent, self.dtype, self.causal, self.heads = old, new, latent, dtype, causal, heads

    def attend(self, scale=.05, **kw):
        return self.cache.attend(self.q, self.q_rope, self.plan, scale=scale, **kw)

    def check(self, y, scale=.05, skip=()):
        at = 0
        for i, (o, n) in enumerate(zip(self.old, self.new)):
            if i not in skip and n:
                x = self.dense[i]
                q = torch.cat([self.q[at:at + n], self.q_rope[at:at + n]], -1).flatten(0, 1)
                last = torch.arange(o, o + n, device=dev()) if self.causal else torch.full((n,), o + n - 1, device=dev())
                seen = torch.arange(o + n, device=dev())[None] <= last.repeat_interleave(self.heads)[:, None]
                out, bound = attention64(q, x, x[:, :self.latent], seen, scale, U[self.dtype])
                bad = ((y[at:at + n].flatten(0, 1).double() - out).abs() > bound) | ~torch.isfinite(y[at:at + n].flatten(0, 1))
                assert not bad.any(), (i, int(bad.sum()), bad.nonzero()[:4].tolist())
            at += n
        assert not y[at:].any()


# ---------------------------------------------------------------- pages
@pytest.mark.parametrize("latent,dtype,P,n,layout", [(512, "bf16", 64, 64, "half"), (256, "fp16", 128, 32, "interleaved"),
                                                     (512, "fp16", 192, 16, "half"), (256, "bf16", 64, 64, "interleaved")])
def test_appends_and_gathers(latent, dtype, P, n, layout):
    g = gen(latent + n)
    rotary = Rotary(n, layout=layout, base=1e5)
    tables = BlockTables(6, 40, 9, page_tokens=P)
    cache = LatentCache(40, latent, page_tokens=P, dtype=TYPES[dtype])
    dense = [torch.zeros(0, latent + 64, dtype=TYPES[dtype], device=dev()) for _ in range(5)]
    rows = torch.tensor([4, 0, 5, 2, 3], device=dev(), dtype=torch.int32)
    for step, new in enumerate(([P + 3, 0, 1, 2 * P, 65], [1] * 5, [P - 4, 70, 0, 1, 130])):
        tokens = sum(new) + step
        plan = tables.plan(torch.tensor(new, device=dev()), rows, tokens=tokens, max_new=max(new))
        whole = randn(g, tokens, latent + 72, dtype=dtype)  # rope keys start 16 bytes past the latents
        x, rope, q = whole[:, :latent], whole[:, latent + 8:], randn(g, tokens, 7, 64, dtype=dtype)
        got = cache.append(x, rope, plan, rotary=rotary, q=q)
        assert torch.equal(got, rotary.apply(q, plan.positions))
        fresh = torch.cat([x, rotary.apply(rope[:, None], plan.positions)[:, 0]], 1)
        at = 0
        for i, k in enumerate(new):
            dense[i] = torch.cat([dense[i], fresh[at:at + k]])
            at += k
        total = sum(len(d) for d in dense)
        for room in (None, total, total + 70, total - 7, 0):
            c, r, starts = cache.gather(plan, room)
            want = torch.cat(dense)
            room = total if room is None else room
            assert c.shape == (room, latent) and r.shape == (room, 64)
            assert torch.equal(torch.cat([c, r], 1)[:total], want[:room]) and not c[total:].any() and not r[total:].any()
            ends = torch.tensor([0] + [len(d) for d in dense]).cumsum(0).clamp(max=room)
            assert starts.tolist() == ends.tolist()
        tables.commit(plan)
    assert not cache.data[0].any()


def test_appends_without_a_rotary_and_in_place():
    g = gen(3)
    tables, cache = BlockTables(2, 8, 3), LatentCache(8, 256)
    plan = tables.plan([70, 5])
    x, whole = randn(g, 75, 320), randn(g, 75, 4, 192)
    assert cache.append(x[:, :256], x[:, 256:], plan) is None
    assert torch.equal(torch.cat(cache.gather(plan)[:2], 1), x)
    rotary = Rotary(64)
    want = rotary.apply(whole[..., 128:].contiguous(), plan.positions)
    kept = whole.clone()
    cache.append(x[:, :256], x[:, 256:], plan, rotary=rotary, q=whole[..., 128:], out=whole[..., 128:])
    assert torch.equal(whole[..., 128:], want) and torch.equal(whole[..., :128], kept[..., :128])


def test_requests_without_room():
    """A request that finds no room keeps its rows; its tokens are written nowhere."""
    tables, cache = BlockTables(3, 6, 3), LatentCache(6)
    g = gen(4)
    plan = tables.plan([100, 64])
    x = randn(g, 164, 576)
    cache.append(x[:, :512], x[:, 512:], plan)
    tables.commit(plan)
    before = cache.data.clone()
    plan = tables.plan([128, 1, 1], [2, 1, 0], absorbed=16, expanded=16)
    assert plan.granted.tolist() == [True, False, True]
    y = randn(g, 130, 576)
    cache.append(y[:, :512], y[:, 512:], plan)
    c, r, starts = cache.gather(plan)
    assert starts.tolist() == [0, 128, 192, 293]
    assert torch.equal(torch.cat([c, r], 1), torch.cat([y[:128], x[100:], x[:100], y[129:]]))
    changed = (cache.data != before).any(-1).any(-1).nonzero()[:, 0].tolist()
    assert sorted(changed) == sorted(tables.table[2, :2].tolist() + [int(tables.table[0, 1])])
    out = cache.attend(randn(g, 130, 16, 512), randn(g, 130, 16, 64), plan, scale=.1)
    assert not out[128].any() and out[:128].any(-1).all() and out[129].any(-1).all()
    k, v = randn(g, 293, 16, 128), randn(g, 293, 16, 128)
    out = expanded_attention(randn(g, 130, 16, 192), k, v, r, plan, starts)
    assert not out[128].any() and out[:128].any(-1).all() and out[129].any(-1).all()


def test_pages_are_copied():
    cache = LatentCache(5)
    cache.data[1:3] = randn(gen(5), 2, 64, 576)
    cache.copy(torch.tensor([1, 2], device=dev()), torch.tensor([4, 3], device=dev()))
    assert torch.equal(cache.data[3:], cache.data[1:3].flip(0)) and cache.nbytes == 5 * 64 * 576 * 2


# ---------------------------------------------------------------- absorbed
@pytest.mark.parametrize("latent", [512, 256])
@pytest.mark.parametrize("heads,sizes,dtype,P", [
    (16, [(0, 1)], "bf16", 64), (1, [(63, 1), (64, 1), (0, 1)], "fp16", 64), (16, [(999, 1)], "fp16", 64),
    (20, [(15, 1), (130, 1), (4000, 1), (1, 1)], "bf16", 128), (32, [(513, 1)] * 7 + [(0, 1)], "bf16", 64),
    (64, [(2000, 1), (77, 1)], "fp16", 192), (128, [(700, 1), (3, 1), (1500, 1)], "bf16", 64),
    (3, [(50, 1)] * 40, "bf16", 64), (5, [(300, 2), (0, 3), (64, 1)], "bf16", 64), (16, [(1000, 5), (65, 4), (2, 5)], "fp16", 64),
    (33, [(120, 3)], "bf16", 128), (8, [(0, 100), (500, 33)], "fp16", 64), (16, [(9000, 1)], "bf16", 4096),
    (7, [(30000, 1), (100, 1)], "bf16", 64), (16, [(5, 0), (70, 1), (0, 2)], "bf16", 64)])
def test_absorbed_attention(heads, sizes, dtype, P, latent):
    print(f"case {heads} heads, {sizes[:4]}, {dtype}, pages of {P}, {latent}", flush=True)
    b = Batch(sizes, latent, dtype, P, heads, padding=len(sizes) % 3)
    y = b.attend()
    b.check(y)
    assert torch.equal(y, b.attend())


@pytest.mark.parametrize("heads,sizes", [(16, [(70, 6), (0, 9)]), (40, [(129, 3), (1, 1)])])
def test_absorbed_attention_of_all_keys(heads, sizes):
    b = Batch(sizes, heads=heads, causal=False)
    b.check(b.attend())


@pytest.mark.parametrize("scale,size", [(-.07, 1.), (0., 1.), (3., 4.), (1e-3, 100.), (40., 30.)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scores_of_any_size(scale, size, dtype):
    b = Batch([(300, 1), (20, 2), (0, 1)], dtype=dtype, size=size, heads=24)
    b.check(b.attend(scale=scale), scale=scale)


def test_many_requests_of_unequal_lengths():
    sizes = [(int(3000 * (i * .618 % 1) ** 4), 1) for i in range(300)]
    b = Batch(sizes, 256, heads=9)
    b.check(b.attend())


def test_queries_of_any_layout():
    b = Batch([(200, 2), (70, 1)], heads=12)
    want = b.attend()
    t, h = b.q.shape[:2]
    both = torch.cat([b.q, b.q_rope], -1)
    b.q, b.q_rope = both[..., :512], both[..., 512:]
    out = torch.empty_like(want)
    assert b.attend(out=out) is out and torch.equal(out, want)
    b.q = b.q.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    odd = torch.zeros(t, h, 67, dtype=torch.bfloat16, device=dev())
    odd[..., 3:] = b.q_rope
    b.q_rope = odd[..., 3:]
    assert torch.equal(b.attend(), want)


@pytest.mark.parametrize("heads", [4, 16, 40])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_numbers_that_are_none_reach_only_the_rows_that_see_them(heads, value):
    """A draft's later token, and other requests' tokens, hold infinities and NaN."""
    b = Batch([(61, 4), (190, 3), (0, 1)], heads=heads)
    clean = b.attend()
    bad = torch.cat([x[o:] for x, o in zip(b.dense, b.old)])
    bad[2, 7], bad[2, 530], bad[6, :] = value, value, value
    b.cache.append(bad[:, :512], bad[:, 512:], b.plan)
    y = b.attend()
    for t in (0, 1, 4, 5, 7):
        assert torch.equal(y[t], clean[t]), t
    if not math.isinf(value):
        assert torch.isnan(y[2:4]).all() and torch.isnan(y[6]).all()


def test_values_near_the_largest():
    b = Batch([(130, 1)], dtype="fp16", heads=16)
    big = b.dense[0].sign() * 65504
    big[:, 512:] = b.dense[0][:, 512:]
    plan = b.plan
    flat = b.cache.data.view(-1, 576)
    page = b.tables.table[plan.rows[0], torch.arange(131, device=dev()) // 64].long() * 64 + torch.arange(131, device=dev()) % 64
    flat[page] = big
    b.dense[0] = big
    b.q.zero_()
    b.check(b.attend(scale=.1), scale=.1)


# ---------------------------------------------------------------- expanded
class Prompts:
    def __init__(self, sizes, heads=4, D=128, dtype="bf16", padding=0, causal=True, seed=0, extra=0, shared=True):
        g = gen(seed)
        old, new = [o for o, _ in sizes], [n for _, n in sizes]
        blocks = [-(-(o + n) // 64) for o, n in sizes]
        self.tables = BlockTables(len(sizes), 2 + sum(blocks), max(max(blocks), 1))
        if any(old):
            plan = self.tables.plan(old)
            self.tables.commit(plan)
        tokens = sum(new) + padding
        self.plan = self.tables.plan(new, tokens=tokens, expanded=heads, causal=causal)
        total = sum(old) + sum(new)
        kv = randn(g, total + extra, heads, 2 * D, dtype=dtype)
        self.k, self.v = (kv[..., :D], kv[..., D:]) if shared else (kv[..., :D].contiguous(), kv[..., D:].contiguous())
        self.rope = randn(g, total + extra, 64, dtype=dtype)
        self.q = randn(g, tokens, heads, D + 64, dtype=dtype) * (3 * torch.rand(tokens, heads, 1, generator=g, device=dev())).to(TYPES[dtype])
        self.starts = torch.tensor([0] + [o + n for o, n in sizes], device=dev()).cumsum(0).int()
        self.old, self.new, self.dtype, self.causal, self.heads = old, new, dtype, causal, heads

    def attend(self, **kw):
        return expanded_attention(self.q, self.k, self.v, self.rope, self.plan, self.starts, **kw)

    def check(self, y, scale=None, limit=None):
        at = 0
        scale = self.q.shape[-1] ** -.5 if scale is None else scale
        for i, (o, n) in enumerate(zip(self.old, self.new)):
            s0, s1 = self.starts[i:i + 2].tolist()
            for h in range(self.heads if n else 0):
                k = torch.cat([self.k[s0:s1, h], self.rope[s0:s1]], -1)
                last = torch.arange(o, o + n, device=dev()) if self.causal else torch.full((n,), o + n - 1, device=dev())
                seen = torch.arange(s1 - s0, device=dev())[None] <= last[:, None]
                out, bound = attention64(self.q[at:at + n, h], k, self.v[s0:s1, h], seen, scale, U[self.dtype])
                got = y[at:at + n, h]
                bad = ((got.double() - out).abs() > bound) | ~torch.isfinite(got)
                assert not bad.any(), (i, h, int(bad.sum()), bad.nonzero()[:4].tolist())
            at += n
        assert not y[at:].any()


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("heads,sizes,dtype,causal", [
    (4, [(0, 1)], "bf16", True), (1, [(0, 63), (0, 64), (0, 65)], "fp16", True), (2, [(0, 1000)], "bf16", True),
    (3, [(5, 1), (0, 300), (700, 20), (64, 0), (1, 255)], "bf16", True), (16, [(1000, 257)], "fp16", True),
    (5, [(0, 31)] * 9, "bf16", True), (2, [(100, 513), (0, 2)], "bf16", False), (8, [(3000, 1), (0, 1)], "bf16", True)])
def test_expanded_attention(heads, sizes, dtype, causal, D):
    print(f"case {heads} heads of {D}, {sizes[:4]}, {dtype}, causal {causal}", flush=True)
    p = Prompts(sizes, heads, D, dtype, padding=len(sizes) % 3, causal=causal, extra=3 * (heads == 2), shared=heads != 3)
    y = p.attend()
    p.check(y)
    assert torch.equal(y, p.attend())


@pytest.mark.parametrize("scale", [-.2, 0., 30.])
def test_expanded_scores_of_any_size(scale):
    for dtype in ("bf16", "fp16"):
        p = Prompts([(40, 200)], dtype=dtype)
        p.check(p.attend(scale=scale), scale)


def test_prompts_over_their_own_rows_need_no_starts():
    p = Prompts([(0, 100), (0, 7), (0, 260)])
    want = p.attend()
    assert torch.equal(expanded_attention(p.q, p.k, p.v, p.rope, p.plan), want)
    out = torch.empty_like(want)
    assert p.attend(out=out) is out and torch.equal(out, want)
    # rows of any order, and such as start off 16 bytes
    p.q = p.q.permute(1, 2, 0).contiguous().permute(2, 0, 1)
    odd = torch.zeros(367, 65, dtype=torch.bfloat16, device=dev())
    odd[:, 1:] = p.rope
    p.rope, p.v = odd[:, 1:], p.v.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    assert torch.equal(p.attend(), want)


def test_rows_that_are_not_there_are_not_seen():
    """Starts that give a request fewer rows than its tokens would see, or none."""
    p = Prompts([(100, 70), (0, 30), (0, 40)], heads=2)
    p.starts = torch.tensor([0, 90, 90, 400], device=dev(), dtype=torch.int32)
    y = p.attend()
    assert not y[70:100].any()
    k = torch.cat([p.k[:90, 0], p.rope[:90]], -1)
    out, bound = attention64(p.q[:70, 0], k, p.v[:90, 0], torch.ones(70, 90, dtype=torch.bool, device=dev()), 192 ** -.5, U["bf16"])
    assert ((y[:70, 0].double() - out).abs() <= bound).all()
    seen = torch.arange(150, device=dev())[None] <= torch.arange(40, device=dev())[:, None]
    k = torch.cat([p.k[90:240, 1], p.rope[90:240]], -1)
    out, bound = attention64(p.q[100:140, 1], k, p.v[90:240, 1], seen, 192 ** -.5, U["bf16"])
    assert ((y[100:140, 1].double() - out).abs() <= bound).all()


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_expanded_numbers_that_are_none_reach_only_the_rows_that_see_them(value):
    p = Prompts([(30, 300), (0, 50)], heads=2)
    clean = p.attend()
    kv = torch.cat([p.k, p.v], -1)
    kv[30 + 170, 0, 128 + 5] = value         # a value of the first request's token 170
    kv[330 + 20, 1, 3] = value               # a key of the second's token 20
    p.k, p.v = kv[..., :128], kv[..., 128:]
    y = p.attend()
    assert torch.equal(y[:170], clean[:170]) and torch.equal(y[:, 1][:320], clean[:, 1][:320])
    assert torch.equal(y[300:, 0], clean[300:, 0])
    assert not torch.isfinite(y[170:300, 0, 5]).any()
    if not math.isinf(value):
        assert torch.isnan(y[320:, 1]).all()


# ---------------------------------------------------------------- together
def test_both_forms_agree():
    """The same prompt chunk absorbed, and gathered, expanded and attended."""
    g = gen(9)
    heads, D, W = 6, 128, 512
    up = torch.randn(heads, 2 * D, W, generator=g, device=dev(), dtype=torch.float64) * W ** -.5
    rotary = Rotary(64, layout="interleaved", base=1e4)
    tables, cache = BlockTables(3, 60, 20), LatentCache(60)
    for step, new in enumerate(([400, 3, 70], [130, 1, 65], [1, 1, 1])):
        tokens = sum(new)
        plan = tables.plan(new, absorbed=heads, expanded=heads)
        q = randn(g, tokens, heads, D + 64)
        cache.append(randn(g, tokens, W), randn(g, tokens, 64), plan, rotary=rotary, q=q[..., D:], out=q[..., D:])
        c, r, starts = cache.gather(plan)
        kv = torch.matmul(c.double()[:, None, None], up.transpose(1, 2)[None]).squeeze(2).to(torch.bfloat16)
        a = expanded_attention(q, kv[..., :D], kv[..., D:], r, plan, starts)
        absorbed = torch.matmul(q[..., :D].double()[:, :, None], up[None, :, :D]).squeeze(2).to(torch.bfloat16)
        y = cache.attend(absorbed, q[..., D:], plan, scale=(D + 64) ** -.5)
        b = torch.matmul(y.double()[:, :, None], up[:, D:].transpose(1, 2)[None]).squeeze(2)
        # both round keys or queries, weights and outputs to 8 bits: some 2^-8 each of vectors of like size
        assert (a.double() - b).norm() < 8 * 2. ** -8 * b.norm(), step
        tables.commit(plan)


@pytest.mark.parametrize("heads", [16, 32, 128])
def test_a_step_replays(heads):
    """Plan, append with turned rope keys and queries, absorbed attention and commit in a graph."""
    g = gen(6)
    lengths = [60, 1, 64, 500, 127]
    rotary = Rotary(64, base=1e6)
    latent, rope = randn(g, 7, 512), randn(g, 7, 64)
    q, q_rope = randn(g, 7, heads, 512), randn(g, 7, heads, 64)
    counts = torch.ones(5, dtype=torch.int32, device=dev())
    first = randn(g, sum(lengths), 576)

    def fresh():
        tables, cache = BlockTables(5, 40, 12), LatentCache(40)
        plan = tables.plan(lengths)
        cache.append(first[:, :512], first[:, 512:], plan)
        tables.commit(plan)
        return tables, cache

    def step(tables, cache):
        plan = tables.plan(counts, tokens=7, max_new=1, absorbed=heads)
        turned = cache.append(latent, rope, plan, rotary=rotary, q=q_rope)
        y = cache.attend(q, turned, plan, scale=.05)
        tables.commit(plan)
        return y

    a, b = fresh(), fresh()
    want = [step(*b).clone() for _ in range(8)]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        y = step(*a)
    for w in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w) and not y[5:].any()
    assert torch.equal(a[1].data, b[1].data) and a[0].lens.tolist() == [n + 8 for n in lengths]


def test_prompts_replay():
    g = gen(7)
    x, q = randn(g, 300, 576), randn(g, 300, 4, 192)
    up = randn(g, 512, 4 * 256)
    counts = torch.tensor([200, 90], device=dev(), dtype=torch.int32)

    def step(tables, cache):
        plan = tables.plan(counts, tokens=300, max_new=200, expanded=4)
        cache.append(x[:, :512], x[:, 512:], plan)
        c, r, starts = cache.gather(plan, 900)
        kv = (c @ up).unflatten(1, (4, 256))
        y = expanded_attention(q, kv[..., :128], kv[..., 128:], r, plan, starts)
        tables.commit(plan)
        return y

    a, b = ((BlockTables(2, 40, 20), LatentCache(40)) for _ in range(2))
    want = [step(*b).clone() for _ in range(3)]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x[:, :512] @ up  # the library sets itself up
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            y = step(*a)
    for w in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y[:290], w[:290]) and not y[290:].any()


def test_plans_lay_out_several_kinds():
    """The 8-bit cache's layers, and both forms of latent ones, by one plan."""
    g = gen(8)
    tables = BlockTables(2, 20, 8)
    kv, cache = KVCache(20, 2, 128), LatentCache(20)
    plan = tables.plan([150, 70], heads=(4, 2), window=(0, 33), absorbed=8, expanded=8)
    k, v, q = randn(g, 220, 2, 128), randn(g, 220, 2, 128), randn(g, 220, 4, 128)
    kv.append(k, v, plan)
    x = randn(g, 220, 576)
    cache.append(x[:, :512], x[:, 512:], plan)
    ql, qr = randn(g, 220, 8, 512), randn(g, 220, 8, 64)
    got = kv.attend(q, plan), kv.attend(q, plan, window=33), cache.attend(ql, qr, plan, scale=.05)
    one = tables.plan([150, 70], heads=(4, 2), window=(0, 33))
    assert torch.equal(kv.attend(q, one), got[0]) and torch.equal(kv.attend(q, one, window=33), got[1])
    two = tables.plan([150, 70], absorbed=8)
    assert torch.equal(cache.attend(ql, qr, two, scale=.05), got[2])


def test_refusals():
    tables, cache = BlockTables(3, 10, 4), LatentCache(10)
    x = torch.zeros(5, 576, dtype=torch.bfloat16, device=dev())
    q, r = (torch.zeros(5, 16, n, dtype=torch.bfloat16, device=dev()) for n in (512, 64))
    plan = tables.plan([3, 2], absorbed=16, expanded=16)
    other = BlockTables(3, 10, 4, page_tokens=128).plan([3, 2], absorbed=16)
    more = BlockTables(3, 11, 4).plan([3, 2], absorbed=16)
    a = lambda l=x[:, :512], k=x[:, 512:], p=plan, **kw: (lambda: cache.append(l, k, p, **kw))
    rotary = Rotary(64)
    calls = [a(x[:, :256]), a(k=x[:, 500:]), a(x[:4, :512]), a(x[:, :512].half()), a(p=other), a(p=more), a(q=r), a(out=r),
             a(rotary=Rotary(80)), a(rotary=rotary, out=r), a(rotary=rotary, q=r[:4]), a(rotary=rotary, q=r.half()),
             a(rotary=rotary, q=r[0]), a(rotary=rotary, q=r, out=q),
             lambda: cache.gather(plan, -1), lambda: cache.gather(other), lambda: tables.plan([1], absorbed=0),
             lambda: tables.plan([1], absorbed=5000), lambda: tables.plan([1], expanded=-1),
             lambda: tables.plan([1], heads=(2, 1), window=(0, 1, 2), absorbed=2, expanded=2),
             lambda: cache.attend(q, r, tables.plan([3, 2]), scale=1.), lambda: cache.attend(q, r, tables.plan([3, 2], expanded=16), scale=1.),
             lambda: cache.attend(q[:, :8], r, plan, scale=1.), lambda: cache.attend(q, r[:, :8], plan, scale=1.),
             lambda: cache.attend(q[..., :256], r, plan, scale=1.), lambda: cache.attend(q.half(), r.half(), plan, scale=1.),
             lambda: cache.attend(q, r, plan, scale=math.inf), lambda: cache.attend(q, r, plan, scale=1., out=q[:4]),
             lambda: cache.attend(q, r, plan, scale=1., out=q.half()), lambda: cache.attend(q, r, other, scale=1.)]
    kv = torch.zeros(5, 16, 128, dtype=torch.bfloat16, device=dev())
    e = lambda q=torch.zeros(5, 16, 192, dtype=torch.bfloat16, device=dev()), k=kv, v=kv, r=x[:, :64], p=plan, **kw: (
        lambda: expanded_attention(q, k, v, r, p, **kw))
    calls += [e(kv), e(k=kv[:4]), e(v=kv[..., :96]), e(v=kv.float()), e(r=x[:4, :64]), e(r=x[:, :32]), e(k=kv.half()), e(p=tables.plan([3, 2])),
              e(starts=plan.cu.long()), e(starts=plan.cu[:2]), e(scale=math.nan), e(out=kv[:, :8]), e(v=kv[0])]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            print("no refusal:", i)
    assert expanded_attention(torch.zeros(5, 16, 192, dtype=torch.bfloat16, device=dev()), kv[:0], kv[:0], x[:0, :64], plan).any() == False  # noqa: E712
    none = tables.plan([0, 0], tokens=0, absorbed=16, expanded=16)
    assert cache.attend(q[:0], r[:0], none, scale=1.).shape == (0, 16, 512)
    assert cache.append(x[:0, :512], x[:0, 512:], none) is None
    assert expanded_attention(torch.zeros(0, 16, 192, dtype=torch.bfloat16, device=dev()), kv, kv, x[:, :64], none).shape == (0, 16, 128)
