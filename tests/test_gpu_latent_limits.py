"""Where latent attention could go wrong (MI355X): keys cut between workgroups,
many requests and heads, pages behind 2^32 bytes, rows far apart, other streams,
several graphs, nothing to do.  Tolerances as in ``test_gpu_latent``."""
import math

import pytest
import torch

from stepquant_amd import _native as N
from stepquant_amd.kernels.kv_cache import BlockTables, KVCache
from stepquant_amd.kernels.latent_cache import LatentCache, expanded_attention
from stepquant_amd.kernels.rotary import Rotary
from tests.helpers import dev
from tests.test_gpu_latent import U, Batch, Prompts, attention64, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,few", [(4, None), (24, None), (24, 1), (40, None), (40, 1), (128, None), (128, 1)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_cut_keys_with_numbers_that_are_none(heads, few, value, monkeypatch):
    """The last of a draft's tokens holds them: one part of its rows' keys is not finite.
    ``few``: sets of 64 and 128 rows where plans would take 32."""
    if few:
        monkeypatch.setattr(BlockTables, "latent_few_work", few)
    b = Batch([(3000, 4), (900, 2)], heads=heads)
    clean = b.attend()
    b.check(clean)
    bad = torch.cat([x[o:] for x, o in zip(b.dense, b.old)])
    bad[3] = value
    b.cache.append(bad[:, :512], bad[:, 512:], b.plan)
    y = b.attend()
    keep = [0, 1, 2, 4, 5]
    assert torch.equal(y[keep], clean[keep])
    assert not torch.isfinite(y[3]).any()


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_expanded_cut_keys_with_numbers_that_are_none(value):
    p = Prompts([(6000, 100), (0, 20)], heads=2)
    clean = p.attend()
    p.check(clean)
    kv = torch.cat([p.k, p.v], -1)
    kv[6050, 0, 128 + 9] = value  # a value of the chunk's token 50
    kv[6070, 1, 0] = math.nan     # a key of its token 70
    p.k, p.v = kv[..., :128], kv[..., 128:]
    y = p.attend()
    assert torch.equal(y[:50, 0], clean[:50, 0]) and torch.equal(y[:70, 1], clean[:70, 1]) and torch.equal(y[100:], clean[100:])
    assert not torch.isfinite(y[50:100, 0, 9]).any() and torch.isnan(y[70:100, 1]).all()


@pytest.mark.parametrize("heads,sizes", [(64, [(70, 1), (0, 2), (3, 1)]), (128, [(200, 1), (0, 1)]), (20, [(300, 4), (61, 3)]),
                                         (128, [(3000, 1)]), (110, [(5, 1), (64, 2)])])
def test_sets_that_the_work_decides(heads, sizes, monkeypatch):
    """Little work runs in sets of 32 rows, the same work in others where the choice is
    taken away: both are right, and of masks and padding alike."""
    few = BlockTables.latent_few_work
    for most in (few, 1):
        monkeypatch.setattr(BlockTables, "latent_few_work", most)
        for causal in (True, False):
            b = Batch(sizes, heads=heads, padding=2, causal=causal, latent=256 if heads == 64 else 512)
            fields = N.KV_SCHEDULE.unpack(b.plan.latent["absorbed"].packed)
            starts, workers = (fields[2] - b.plan._ints.data_ptr()) // 4, fields[5]
            assert int(b.plan._ints[starts + workers + 1]) == (32 if most == few else 128 if heads > 96 else 64)
            b.check(b.attend())


def test_more_requests_than_lanes():
    sizes = [((i * 37) % 90, (i * 5) % 4) for i in range(150)] + [(300, 70)]
    p = Prompts(sizes, heads=2, padding=3)
    p.check(p.attend())
    b = Batch([(o, n) for o, n in sizes if n], heads=8, latent=256)
    b.check(b.attend())


def test_heads_from_one_to_the_most():
    b = Batch([(70, 2), (0, 1)], heads=1)
    b.check(b.attend())
    b = Batch([(70, 1)], heads=4096, latent=256)
    b.check(b.attend())


@pytest.mark.parametrize("causal", [True, False])
def test_masks_over_cut_keys(causal):
    b = Batch([(2500, 7), (64, 1), (0, 3)], heads=12, causal=causal, latent=256)
    b.check(b.attend())
    p = Prompts([(4100, 33), (0, 64)], heads=2, causal=causal)
    p.check(p.attend())


def test_pages_behind_4_gib():
    """60,000 pages of 64 tokens of 1152 bytes; the requests have the last of them."""
    pages = 60000
    cache = LatentCache(pages)
    assert cache.nbytes > 1 << 32
    g = gen(4)
    x = randn(g, 400, 576)
    for turned in (False, True):
        tables = BlockTables(2, pages, 8)
        if turned:  # (pages are given out from one end of these)
            tables.free.copy_(tables.free.flip(0))
        plan = tables.plan([300, 100], absorbed=4)
        cache.append(x[:, :512], x[:, 512:], plan)
        c, r, _ = cache.gather(plan)
        assert torch.equal(torch.cat([c, r], 1), x)
        used = plan.slots // 64
        q, q_rope = randn(g, 400, 4, 512), randn(g, 400, 4, 64)
        y = cache.attend(q, q_rope, plan, scale=.05)
        seen = torch.arange(300, device=dev())[None] <= torch.arange(300, device=dev())[:, None]
        out, bound = attention64(torch.cat([q, q_rope], -1)[:300, 2], x[:300], x[:300, :512], seen, .05, U["bf16"])
        assert ((y[:300, 2].double() - out).abs() <= bound).all()
        if int(used.max()) > 58255:
            return
    raise AssertionError("no page behind 4 GiB was given out")


def test_rows_far_apart():
    """Keys and values with rows of 2^24 elements and more between them are copied."""
    p = Prompts([(0, 5)], heads=1)
    want = p.attend()
    wide = torch.zeros(4 * (1 << 24) + 256, dtype=torch.bfloat16, device=dev())
    k, v = wide.as_strided((5, 1, 128), (1 << 24, 128, 1)), wide.as_strided((5, 1, 128), (1 << 24, 128, 1), 128)
    k.copy_(p.k), v.copy_(p.v)
    p.k, p.v = k, v
    assert torch.equal(p.attend(), want)


def test_other_streams():
    """A step whose calls are made on a stream of their own, beside work on the first."""
    g = gen(11)
    rotary = Rotary(64)
    x, q, q_rope = randn(g, 500, 576), randn(g, 500, 8, 512), randn(g, 500, 8, 64)
    kv, eq = randn(g, 500, 2, 256), randn(g, 500, 2, 192)

    def run():
        tables, cache = BlockTables(3, 20, 12), LatentCache(20)
        plan = tables.plan([400, 30, 70], absorbed=8, expanded=2)
        turned = cache.append(x[:, :512], x[:, 512:], plan, rotary=rotary, q=q_rope)
        y = cache.attend(q, turned, plan, scale=.05)
        c, r, starts = cache.gather(plan, 500)
        return turned, y, expanded_attention(eq, kv[..., :128], kv[..., 128:], r, plan, starts)

    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    a = torch.randn(2048, 2048, device=dev())
    for _ in range(3):
        b = a @ a
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = run()
        for w, y in zip(want, got):
            side.synchronize()
            assert torch.equal(w, y)
        del b


@pytest.mark.parametrize("few", [None, 1])
def test_two_graphs_in_turn(few, monkeypatch):
    """Two graphs of one pool, whose workspaces share memory, replayed in turn and beside eager calls."""
    if few:
        monkeypatch.setattr(BlockTables, "latent_few_work", few)
    a, b = Batch([(2000, 1), (700, 1)], heads=16, seed=1), Batch([(1500, 3)], heads=128, seed=2)
    want = a.attend(), b.attend()
    pool, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in (a, b):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], pool=pool, stream=side):
                outs.append(x.attend())
    torch.cuda.current_stream().wait_stream(side)
    for k in (0, 1, 1, 0, 1, 0):
        graphs[k].replay()
        assert torch.equal(outs[k], want[k])
        assert torch.equal(b.attend(), want[1])


def test_nothing_to_do():
    tables, cache = BlockTables(3, 8, 3), LatentCache(8, 256)
    rotary = Rotary(64)
    empty = torch.empty(0, 256, dtype=torch.bfloat16, device=dev())
    plan = tables.plan([0, 0], absorbed=4, expanded=4)
    q = cache.append(empty, empty[:, :64], plan, rotary=rotary, q=empty[:, :64].reshape(0, 2, 64))
    assert q.shape == (0, 2, 64)
    assert cache.attend(empty.reshape(0, 4, 256), empty[:, :64].reshape(0, 4, 64), plan, scale=.1).shape == (0, 4, 256)
    c, r, starts = cache.gather(plan)
    assert c.shape == (0, 256) and r.shape == (0, 64) and not starts.any()
    y = expanded_attention(empty[:, :192].reshape(0, 1, 192).expand(0, 4, 192), empty.reshape(0, 2, 128)[:, :1].expand(0, 4, 128),
                           empty.reshape(0, 2, 128)[:, :1].expand(0, 4, 128), r, plan, starts)
    assert y.shape == (0, 4, 128)
    assert rotary.apply(empty.reshape(0, 4, 64), torch.empty(0, dtype=torch.int64, device=dev())).shape == (0, 4, 64)
    # rows to answer, and nothing that they see
    plan = tables.plan([0, 0], tokens=3, absorbed=4, expanded=4)
    g = gen(0)
    out = torch.full((3, 4, 256), 7., dtype=torch.bfloat16, device=dev())
    assert not cache.attend(randn(g, 3, 4, 256), randn(g, 3, 4, 64), plan, scale=.1, out=out).any()
    y = expanded_attention(randn(g, 3, 4, 192), randn(g, 0, 4, 128), randn(g, 0, 4, 128), randn(g, 0, 64), plan)
    assert y.shape == (3, 4, 128) and not y.any()


def test_keys_turned_from_rows_that_are_copied():
    """Queries whose strides are not whole 16 bytes are copied, and the copy lives until it is read."""
    g = gen(12)
    rotary = Rotary(32, layout="interleaved")
    tables, cache, kv = BlockTables(2, 40, 20), LatentCache(40, 256), KVCache(40, 2, 64)
    plan = tables.plan([900, 300])
    odd = torch.zeros(1200, 3, 65, dtype=torch.bfloat16, device=dev())
    odd[..., 1:] = randn(g, 1200, 3, 64)
    q = odd[..., 1:]
    want = rotary.apply(q.contiguous(), plan.positions)
    x = randn(g, 1200, 320)
    assert torch.equal(rotary.apply(q, plan.positions), want)
    assert torch.equal(cache.append(x[:, :256], x[:, 256:], plan, rotary=rotary, q=q), want)
    assert torch.equal(kv.append(x[:, :128], x[:, 128:256], plan, rotary=rotary, q=q), want)


def test_queries_beside_more_workgroups_than_they_need():
    """2048 KV heads and 8200 rows of padding launch over 2^24 workgroups for keys, and as
    many for the queries, which are turned once all the same."""
    heads, tokens = 2048, 8200
    tables, kv, rotary = BlockTables(4096, 4, 1), KVCache(4, heads, 64), Rotary(16)
    counts = torch.zeros(4096, dtype=torch.int32, device=dev())
    counts[5] = 3
    plan = tables.plan(counts, tokens=tokens, max_new=3)
    assert plan.max_tiles * heads >= 1 << 24
    k = torch.ones(tokens, 1, 64, dtype=torch.bfloat16, device=dev()).expand(tokens, heads, 64)
    q = randn(gen(1), tokens, 9, 64)
    want = rotary.apply(q, plan.positions)
    assert not torch.equal(want, q)
    assert kv.append(k, k, plan, rotary=rotary, q=q, out=q) is not None
    assert torch.equal(q, want)
