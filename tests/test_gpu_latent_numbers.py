"""Latent attention where latents, values or scores are infinite, or next to what
their types hold (MI355X).  Tolerances as in ``test_gpu_latent``."""
import math

import pytest
import torch

from stepquant_amd.kernels.kv_cache import BlockTables
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
