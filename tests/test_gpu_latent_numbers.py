"""Latent attention where latents, values or scores are infinite, or next to what
their types hold, and where operands are missing (MI355X).  Tolerances as in ``test_gpu_latent``."""
import math

import pytest
import torch

from stepquant_amd import _native as N
from stepquant_amd.kernels.kv_cache import BlockTables
from stepquant_amd.kernels.latent_cache import LatentCache, expanded_attention
from stepquant_amd.kernels.rotary import Rotary
from tests.helpers import dev
from tests.test_gpu_latent import U, Batch, Prompts, attention64

pytestmark = pytest.mark.gpu


def rewrite(b, edit):
    """The new tokens of a batch, edited and appended again."""
    x = torch.cat([d[o:] for d, o in zip(b.dense, b.old)])
    edit(x)
    b.cache.append(x[:, :b.latent], x[:, b.latent:], b.plan)
    at = 0
    for d, o, n in zip(b.dense, b.old, b.new):
        d[o:] = x[at:at + n]
        at += n


# ---------------------------------------------------------------- infinite latents
@pytest.mark.parametrize("heads,sizes,few", [(1, [(61, 4), (190, 3)], None), (4, [(61, 4), (0, 1)], None), (16, [(61, 4), (190, 3)], None),
                                             (40, [(61, 4), (9, 1)], 1), (128, [(61, 4), (9, 1)], 1), (16, [(3000, 4), (9, 1)], None),
                                             (128, [(3000, 4), (9, 1)], 1)])
@pytest.mark.parametrize("latent,dtype", [(512, "bf16"), (256, "fp16")])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_infinite_latents_reach_the_rows_that_see_them(value, latent, dtype, heads, sizes, few, monkeypatch):
    """Of a key whose score is -infinity the weight is 0 and the value infinite: no
    number in that dim, in tiles that all rows see and in others alike."""
    if few:
        monkeypatch.setattr(BlockTables, "latent_few_work", few)
    for sign in (1, -1):
        b = Batch(sizes, latent, dtype, heads=heads)
        b.q[..., 7] = sign
        clean = b.attend()
        b.check(clean)
        rewrite(b, lambda x: x[2, 7].fill_(value))
        y = b.attend()
        assert torch.equal(y[:2], clean[:2]) and torch.equal(y[4:], clean[4:])
        assert not torch.isfinite(y[2:4, :, 7]).any(), sign


@pytest.mark.parametrize("heads", [1, 16, 40, 128])
def test_infinite_latents_in_turn(heads):
    """Tiles with and without them after one another, of requests that share workgroups."""
    sizes = [(61, 4), (64, 4), (200, 3), (30, 2), (95, 5)] * 12
    b = Batch(sizes, heads=heads, latent=256)
    b.q[..., 7] = 1
    b.tables._cus = 2
    b.plan = b.tables.plan(b.new, b.plan.rows, absorbed=heads)
    clean = b.attend()
    b.check(clean)
    first = torch.tensor([0] + b.new[:-1]).cumsum(0)
    at = [(int(first[i]) + 1 + i % 2, i) for i in range(len(sizes)) if i % 3 == 0]
    at = [(t, i) for t, i in at if t < int(first[i]) + b.new[i]]

    def edit(x):
        x[[t for t, _ in at], 7] = -math.inf

    rewrite(b, edit)
    y = b.attend()
    seeing = torch.zeros(len(y), dtype=torch.bool, device=dev())
    for t, i in at:
        seeing[t:int(first[i]) + b.new[i]] = True
    assert torch.equal(y[~seeing], clean[~seeing]) and not torch.isfinite(y[seeing][..., 7]).any()


@pytest.mark.parametrize("heads", [1, 16, 128])
@pytest.mark.parametrize("old", [61, 640, 3000])
def test_infinite_rope_keys_whose_scores_are_minus_infinity_weigh_nothing(heads, old):
    b = Batch([(old, 4)], heads=heads)
    b.q_rope[..., 3] = 1
    rewrite(b, lambda x: x[2, 512 + 3].fill_(-math.inf))
    y = b.attend()
    keep = torch.ones(old + 4, dtype=torch.bool, device=dev())
    keep[old + 2] = False
    for t in range(4):
        q = torch.cat([b.q[t], b.q_rope[t]], -1)
        seen = ((torch.arange(old + 4, device=dev()) <= old + t) & keep)[None].expand(heads, -1)
        x = torch.where(keep[:, None], b.dense[0], 0.)
        out, bound = attention64(q, x, x[:, :512], seen, .05, U["bf16"])
        assert ((y[t].double() - out).abs() <= bound).all(), t


# ---------------------------------------------------------------- large and small values
def large(x, size):
    """Values of ``size`` with one sign a dim."""
    g = torch.Generator(device=dev()).manual_seed(3)
    sign = torch.where(torch.rand(x.shape[-1], generator=g, device=dev()) < .5, -1., 1.)
    return ((.3 + .7 * torch.rand(x.shape, generator=g, device=dev())) * sign * size).to(x.dtype)


@pytest.mark.parametrize("heads,sizes,few", [(16, [(2000, 1), (3, 1)], None), (24, [(2000, 1)], None), (40, [(2000, 2)], 1),
                                             (128, [(2000, 1), (0, 1)], 1), (128, [(200, 1)], None)])
@pytest.mark.parametrize("size", [3.3e38, 1e33, 1e-25])
@pytest.mark.parametrize("workgroups", [None, 2])
def test_sums_of_latents_of_any_size(workgroups, size, heads, sizes, few, monkeypatch):
    """Outputs are finite where latents are; queries that are 0 leave scores to the rope keys."""
    if few:
        monkeypatch.setattr(BlockTables, "latent_few_work", few)
    b = Batch(sizes, heads=heads)
    for d, i in zip(b.dense, b.plan.rows.tolist()):
        d[:, :512] = large(d[:, :512], size)
        n = torch.arange(len(d), device=dev())
        b.cache.data.view(-1, 576)[b.tables.table[i, n // 64].long() * 64 + n % 64] = d
    b.q.zero_()
    if workgroups:  # few, so that each of them has many keys
        b.tables._cus = workgroups
        b.plan = b.tables.plan(b.new, b.plan.rows, absorbed=heads)
    y = b.attend(scale=.3)
    assert (y[0] != 0).all()
    b.check(y, scale=.3)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sizes", [[(0, 300)], [(3000, 40), (0, 7)], [(2000, 700)]])
@pytest.mark.parametrize("size", [3.3e38, 1e33, 1e-25])
def test_sums_of_expanded_values_of_any_size(D, sizes, size):
    p = Prompts(sizes, heads=2, D=D, shared=False)
    p.v = large(p.v, size)
    y = p.attend()
    assert (y[:1] != 0).all()
    p.check(y)


# ---------------------------------------------------------------- scores
@pytest.mark.parametrize("heads,sizes,few", [(1, [(61, 4), (0, 1)], None), (16, [(61, 2), (0, 1)], None), (40, [(61, 2), (0, 1)], 1),
                                             (16, [(3000, 4), (0, 2)], None), (128, [(3000, 1), (5, 1)], 1), (128, [(3000, 1)], None)])
def test_rows_whose_scores_are_all_minus_infinity(heads, sizes, few, monkeypatch):
    """Not a number, as the definition has it: only rows that see nothing are zero."""
    if few:
        monkeypatch.setattr(BlockTables, "latent_few_work", few)
    b = Batch(sizes, heads=heads, padding=2)
    for d, i in zip(b.dense, b.plan.rows.tolist()):
        d[:, 512] = -1
        n = torch.arange(len(d), device=dev())
        b.cache.data.view(-1, 576)[b.tables.table[i, n // 64].long() * 64 + n % 64] = d
    y = b.attend()
    b.check(y)
    clean = y.clone()
    b.q_rope[0, 0, 0] = math.inf
    b.q_rope[-2:, :, 0] = math.inf
    y = b.attend()
    assert torch.isnan(y[0, 0]).all() and not y[-2:].any()
    assert torch.equal(y[0, 1:], clean[0, 1:]) and torch.equal(y[1:], clean[1:])


@pytest.mark.parametrize("sizes", [[(0, 70)], [(6000, 100)], [(0, 1000)]])
def test_expanded_rows_whose_scores_are_all_minus_infinity(sizes):
    p = Prompts(sizes, heads=2, padding=3)
    p.rope[:, 5] = -1
    clean = p.attend()
    p.check(clean)
    p.q[[0, 40, 69], 1, 128 + 5] = math.inf
    p.q[-3:, :, 128 + 5] = math.inf
    y = p.attend()
    keep = torch.ones(len(y), 2, dtype=torch.bool, device=dev())
    keep[[0, 40, 69], 1] = False
    assert torch.isnan(y[~keep]).all() and torch.equal(y[keep], clean[keep]) and not y[-3:].any()


@pytest.mark.parametrize("heads", [1, 16, 128])
def test_parts_whose_scores_are_all_minus_infinity(heads):
    """Keys cut between workgroups, some of which see no finite score."""
    b = Batch([(3000, 1)], heads=heads)
    b.q_rope[..., 0] = 1
    d, n = b.dense[0], torch.arange(3001, device=dev())
    d[:2000, 512] = -math.inf
    b.cache.data.view(-1, 576)[b.tables.table[b.plan.rows[0], n // 64].long() * 64 + n % 64] = d
    y = b.attend()
    out, bound = attention64(torch.cat([b.q[0], b.q_rope[0]], -1), d[2000:], d[2000:, :512],
                             torch.ones(heads, 1001, dtype=torch.bool, device=dev()), .05, U["bf16"])
    assert ((y[0].double() - out).abs() <= bound).all()


def test_a_scale_of_nothing_takes_the_mean_of_scores_of_any_size():
    for sizes in ([(0, 100)], [(3000, 60)]):
        p = Prompts(sizes, heads=2)
        p.q = (p.q.float() * 1e18).to(torch.bfloat16)
        p.k, p.rope = (p.k.float() * 1e18).to(torch.bfloat16), (p.rope.float() * 1e18).to(torch.bfloat16)
        p.check(p.attend(scale=0.), 0.)


@pytest.mark.parametrize("scale", [1.9e38, -1.9e38])
def test_the_largest_scales_of_queries_of_nothing(scale):
    b = Batch([(100, 2), (0, 1)], heads=20)
    b.q.zero_(), b.q_rope.zero_()
    b.check(b.attend(scale=scale), scale=scale)
    p = Prompts([(0, 100)], heads=2)
    p.q.zero_()
    p.check(p.attend(scale=scale), scale)


# ---------------------------------------------------------------- keys that are not there
@pytest.mark.parametrize("causal", [True, False])
def test_requests_that_held_tokens_need_starts(causal):
    """Without starts keys are the new tokens' alone: no numbers for requests that held
    others before, the plan's own answer for the rest, zero past them."""
    p = Prompts([(0, 100), (5, 70), (0, 300), (3000, 1), (1, 40)], heads=3, padding=2, causal=causal)
    fresh = torch.cat([torch.arange(int(s) + o, int(s) + o + n) for s, o, n in zip(p.starts, p.old, p.new)]).to(dev())
    p.k, p.v, p.rope = p.k[fresh], p.v[fresh], p.rope[fresh]
    # (by the same plan: another may cut keys elsewhere and round otherwise)
    alone = expanded_attention(p.q, p.k, p.v, p.rope, p.plan, p.plan.cu.clone())
    y = expanded_attention(p.q, p.k, p.v, p.rope, p.plan)
    at = 0
    for o, n in zip(p.old, p.new):
        if o:
            assert torch.isnan(y[at:at + n]).all(), (o, n)
        else:
            assert torch.equal(y[at:at + n], alone[at:at + n]), (o, n)
        at += n
    assert not y[at:].any()


def test_requests_that_held_tokens_without_any_rows():
    p = Prompts([(0, 4), (9, 3)], heads=2, padding=1)
    y = expanded_attention(p.q, p.k[:0], p.v[:0], p.rope[:0], p.plan)
    assert not y[:4].any() and torch.isnan(y[4:7]).all() and not y[7:].any()
    assert not expanded_attention(p.q, p.k[:0], p.v[:0], p.rope[:0], p.plan, p.starts).any()


def test_rows_beside_an_append_of_no_tokens():
    """Rows that the C entry is given are turned, whatever it appends."""
    rotary, cache = Rotary(64), LatentCache(4, 256)
    x = torch.randn(7, 3, 64, device=dev()).to(torch.bfloat16)
    positions = torch.arange(5, 12, device=dev(), dtype=torch.int32)
    out = torch.zeros_like(x)
    rows = N.RotaryRows(x=x.data_ptr(), out=out.data_ptr(), positions=positions.data_ptr(), tokens=7, x_stride=192,
                        x_head_stride=64, out_stride=192, out_head_stride=64, heads=3, head_dim=64, dtype=N.BF16,
                        positions_dtype=N.I32)
    stream = torch.cuda.current_stream().cuda_stream
    assert N.lib().sq_latent_append(cache._latent, N.LatentAppend(tokens=0), rotary._desc, rows, stream) == 0
    assert torch.equal(out, rotary.apply(x, positions)) and not cache.data.any()


@pytest.mark.parametrize("heads,sizes,few", [(16, [(300, 1), (0, 2)], None), (40, [(300, 2), (5, 1)], 1), (128, [(300, 1)], 1), (24, [(5000, 3)], None),
                                             (128, [(5000, 1), (70, 1)], 1)])
def test_absorbed_outputs_may_take_the_place_of_queries(heads, sizes, few, monkeypatch):
    if few:
        monkeypatch.setattr(BlockTables, "latent_few_work", few)
    b = Batch(sizes, heads=heads, padding=1)
    want = b.attend()
    assert torch.equal(b.attend(out=b.q), want) and torch.equal(b.q, want)


def test_expanded_outputs_over_values_are_refused():
    p = Prompts([(0, 100)], heads=2, shared=False)
    for out in (p.v, p.k):
        with pytest.raises(ValueError, match="overlap"):
            p.attend(out=out)
