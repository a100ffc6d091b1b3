"""Rotary positions, by themselves and on the way into the 8-bit KV cache,
against the formula in 64 bits on the host (MI355X).

An angle is off by 1.2e-7 (its 32-bit fraction and the product with 2 pi), sine
and cosine by 1.2e-7 more (series and roundings), each of their products with
the magnitude and with an element by 2^-24: |a| + |b| times the magnitude times
4e-7 in all, and half a step of the output's type.
"""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from stepquant_amd.kernels.kv_cache import BlockTables, KVCache
from stepquant_amd.kernels.rotary import Rotary, frequencies
from tests.helpers import dev

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF_STEP = {"bf16": 2. ** -8, "fp16": 2. ** -11, "fp32": 2. ** -24}
ERROR = 4e-7


def turned(x, positions, f, layout, magnitude):
    """(rows in 64 bits, the sum of magnitudes of each pair) of ``x`` [tokens, heads, dim]."""
    x, n = x.double().cpu().numpy(), 2 * len(f)
    turns = np.asarray(f, np.float64)
    # positions times frequencies modulo a turn, with more bits than the product in 64
    angle = np.array([[math.fmod(int(p) * float(w), 2 * math.pi) for w in turns] for p in positions])
    c, s = magnitude * np.cos(angle)[:, None], magnitude * np.sin(angle)[:, None]
    y, size = x.copy(), np.zeros_like(x)
    i = np.arange(n // 2)
    ia, ib = (i, i + n // 2) if layout == "half" else (2 * i, 2 * i + 1)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = (np.abs(a) + np.abs(b)) * abs(magnitude)
    still = np.asarray(positions) < 0
    y[still], size[still] = x[still], 0
    return y, size


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,heads,dim,n", [(1, 1, 64, 64), (1, 16, 256, 64), (7, 3, 128, 128), (33, 5, 72, 16),
                                                (130, 2, 80, 48), (300, 32, 128, 128), (513, 128, 64, 64),
                                                (2, 1, 1024, 1024), (41, 9, 136, 96)])
def test_rows_turn(tokens, heads, dim, n, dtype, layout):
    print(f"case {tokens} x {heads} x {dim}, {n} turned, {dtype}, {layout}", flush=True)
    g = torch.Generator().manual_seed(tokens * 7 + n)
    x = torch.randn(tokens, heads, dim, generator=g).to(TYPES[dtype])
    positions = torch.randint(0, 200000, (tokens,), generator=g, dtype=torch.int64 if heads & 1 else torch.int32)
    if tokens > 5:
        positions[3] = -1
    r = Rotary(n, layout=layout, base=5e5, scaling="yarn", factor=4., original=4096)
    got = r.apply(x.to(dev()), positions.to(dev()))
    f, magnitude = frequencies(n, base=5e5, scaling="yarn", factor=4., original=4096)
    want, size = turned(x, positions.tolist(), f.tolist(), layout, magnitude)
    # (the host's angle itself is good to 2^-53 of 200000 rad)
    limit = size * (ERROR + 1e-10) + np.abs(want) * HALF_STEP[dtype] + 1e-7 * (dtype == "fp16")
    limit[..., n:] = 0
    bad = np.abs(got.double().cpu().numpy() - want) > limit
    assert got.shape == x.shape and got.is_contiguous() and not bad.any(), np.argwhere(bad)[:5]


def test_far_positions():
    """Positions of up to 63 bits: the host's turns are exact fractions, with pi to 49 digits."""
    inverse = torch.tensor([1, 3, 5, 7, 11, 13, 17, 19], dtype=torch.float64) / 64 * 2 * math.pi
    r = Rotary(16, inverse=inverse)
    positions = torch.tensor([0, 1, 64, 2 ** 31 - 1, 2 ** 31 + 5, 2 ** 38 + 3])
    x = torch.randn(6, 2, 16, generator=torch.Generator().manual_seed(0))
    got = r.apply(x.to(dev()), positions.to(dev())).double().cpu().numpy()
    turn = 2 * Fraction("3.1415926535897932384626433832795028841971693993751")
    angle = np.array([[float(int(p) * Fraction(w) / turn % 1) * 2 * math.pi for w in inverse.tolist()] for p in positions.tolist()])
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = x[..., :8].double().numpy(), x[..., 8:].double().numpy()
    want = np.concatenate([a * c - b * s, a * s + b * c], -1)
    size = np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)
    # a frequency is off by 2^-65 of a turn a position
    off = 2 * math.pi * positions.double().numpy()[:, None, None] * 2. ** -65
    assert not (np.abs(got - want) > size * (ERROR + off) + 1e-7 * np.abs(want)).any()
    # what is past 2^63 / f turns wraps to the same angle: no position is out of range
    top = r.apply(x.to(dev()), torch.full((6,), 2 ** 63 - 1, device=dev()))
    assert torch.isfinite(top).all() and torch.allclose(top.norm(), x.norm().to(dev()), rtol=1e-6)


@pytest.mark.parametrize("heads", [1, 40])
def test_rows_in_place_and_strided(heads):
    g = torch.Generator(device=dev()).manual_seed(2)
    r = Rotary(64, layout="interleaved")
    whole = torch.randn(700, heads, 192, generator=g, device=dev()).to(torch.bfloat16)
    positions = torch.arange(700, device=dev(), dtype=torch.int32) - 3
    want = r.apply(whole[..., 128:].contiguous(), positions)
    kept = whole.clone()
    assert r.apply(whole[..., 128:], positions, out=whole[..., 128:]).data_ptr() == whole.data_ptr() + 256
    assert torch.equal(whole[..., 128:], want) and torch.equal(whole[..., :128], kept[..., :128])
    # another order of dims, rows and heads that start off 16 bytes, repeated rows
    other = kept.permute(1, 0, 2).contiguous().permute(1, 0, 2)[..., 128:]
    assert torch.equal(r.apply(other, positions), want)
    odd = torch.zeros(700, heads, 67, dtype=torch.bfloat16, device=dev())
    odd[..., 3:] = kept[..., 128:]
    assert torch.equal(r.apply(odd[..., 3:], positions), want)
    one = r.apply(kept[5:6, :, 128:].expand(700, heads, 64), positions)
    assert torch.equal(one[5], want[5]) and torch.equal(one[0], kept[5, :, 128:])
    with pytest.raises(ValueError):
        r.apply(odd[..., 3:], positions, out=odd[..., 3:])
    with pytest.raises(ValueError):
        r.apply(kept[..., 128:], positions, out=torch.empty(64, dtype=torch.bfloat16, device=dev()).expand(700, heads, 64))
    gaps = torch.full((1400,), 9, dtype=torch.int64, device=dev())
    gaps[::2] = positions
    assert torch.equal(r.apply(kept[..., 128:], gaps[::2]), want)


def test_values_that_are_not_numbers_stay_in_their_pair():
    r = Rotary(32)
    x = torch.ones(4, 2, 48, device=dev())
    x[1, 0, 3], x[2, 1, 40], x[3, 0, 20] = math.nan, math.inf, math.inf
    y = r.apply(x, torch.tensor([5, 5, -1, 7], device=dev()))
    bad = (~torch.isfinite(y)).nonzero().tolist()
    assert bad == [[1, 0, 3], [1, 0, 19], [2, 1, 40], [3, 0, 4], [3, 0, 20]]


def test_refusals():
    r = Rotary(64)
    x, p = torch.zeros(3, 2, 128, device=dev()), torch.zeros(3, dtype=torch.int32, device=dev())
    for bad in (lambda: r.apply(x[0], p), lambda: r.apply(x, p[:2]), lambda: r.apply(x, p.float()),
                lambda: r.apply(x.double(), p), lambda: r.apply(x.cpu(), p), lambda: r.apply(x, p.cpu()),
                lambda: r.apply(x[..., :56], p), lambda: r.apply(x[..., :100], p),
                lambda: r.apply(x, p, out=x.half()), lambda: r.apply(x, p, out=x[:2]),
                lambda: r.apply(x[:, :0], p)):
        with pytest.raises(ValueError):
            bad()
    assert r.apply(x[:0], p[:0]).shape == (0, 2, 128)


# ---------------------------------------------------------------- on the way into the cache
def quarters(n, layout):
    """Frequencies of whole quarter turns, at which turning is exact (radians in 64 bits are not)."""
    r = Rotary(n, layout=layout)
    r.turns.copy_(torch.tensor([(i % 4 << 62) - (i % 4 >> 1 << 64) for i in range(n // 2)]))
    return r


def quarter_turned(x, positions, n, layout):
    y = x.clone()
    i = torch.arange(n // 2)
    ia, ib = (i, i + n // 2) if layout == "half" else (2 * i, 2 * i + 1)
    a, b = x[..., ia], x[..., ib]
    q = ((positions[:, None].cpu() * (i % 4)) % 4).to(x.device)[:, None]
    y[..., ia] = torch.where(q == 0, a, torch.where(q == 1, -b, torch.where(q == 2, -a, b)))
    y[..., ib] = torch.where(q == 0, b, torch.where(q == 1, a, torch.where(q == 2, -b, -a)))
    return torch.where((positions >= 0)[:, None, None], y, x)


@pytest.mark.parametrize("storage", ["int8", "fp8"])
@pytest.mark.parametrize("dim,n,P,layout,dtype", [(64, 64, 64, "half", "bf16"), (128, 32, 64, "interleaved", "fp16"),
                                                  (128, 128, 256, "half", "fp16"), (256, 64, 64, "half", "bf16"),
                                                  (256, 256, 128, "interleaved", "bf16"), (64, 48, 512, "half", "bf16")])
def test_appends_that_turn_are_appends_of_turned_keys(dim, n, P, layout, dtype, storage):
    """At whole quarter turns every bit is that of the two calls one after the other."""
    print(f"case {dim} dims, {n} turned, pages of {P}, {layout}, {dtype}, {storage}", flush=True)
    g = torch.Generator(device=dev()).manual_seed(dim + n)
    r = quarters(n, layout)
    tables = BlockTables(5, 60, 12, page_tokens=P)
    caches = [KVCache(60, 3, dim, page_tokens=P, storage=storage) for _ in range(2)]
    for step, new in enumerate(([P + 5, 1, 2 * P, 0, 70], [1, 1, 1, 1, 1], [P - 7, 63, 0, 2, 1], [1, 0, 3, 0, 130])):
        tokens = sum(new) + step
        k, v = (torch.randn(tokens, 3, dim, generator=g, device=dev()).to(TYPES[dtype]) * (1 + step) for _ in range(2))
        q = torch.randn(tokens, 6, dim, generator=g, device=dev()).to(TYPES[dtype])
        plan = tables.plan(torch.tensor(new, device=dev()), tokens=tokens, max_new=max(new))
        want = quarter_turned(q, plan.positions, n, layout)
        got = caches[0].append(k, v, plan, rotary=r, q=q)
        assert torch.equal(got, want) and torch.equal(r.apply(q, plan.positions), want)
        caches[1].append(quarter_turned(k, plan.positions, n, layout), v, plan)
        assert torch.equal(caches[0].data, caches[1].data)
        tables.commit(plan)


@pytest.mark.parametrize("storage", ["int8", "fp8"])
@pytest.mark.parametrize("dim,n,layout", [(64, 64, "half"), (128, 128, "interleaved"), (256, 64, "half")])
def test_codes_of_turned_keys(dim, n, layout, storage):
    """Codes are within half a step of the keys that were turned in 64 bits."""
    g = torch.Generator().manual_seed(dim)
    P, top = 64, 127. if storage == "int8" else 448.
    tables, cache = BlockTables(3, 20, 5, page_tokens=P), KVCache(20, 2, dim, page_tokens=P, storage=storage)
    r = Rotary(n, layout=layout, base=1e4)
    plan = tables.plan([150, 1, 64])
    k = torch.randn(215, 2, dim, generator=g).to(torch.bfloat16)
    assert cache.append(k.to(dev()), k.to(dev()), plan, rotary=r) is None
    got, values = (x.double().cpu().numpy() for x in cache.decode(plan.pages, plan.filled))
    plain = KVCache(20, 2, dim, page_tokens=P, storage=storage)
    plain.append(k.to(dev()), k.to(dev()), plan)
    assert np.array_equal(values, plain.decode(plan.pages, plan.filled)[1].double().cpu().numpy())
    want, size = turned(k, plan.positions.tolist(), frequencies(n)[0].tolist(), layout, 1.)
    row = 0
    for tile, (page, count) in enumerate(zip(plan.pages.tolist(), plan.filled.tolist())):
        if not count:
            continue
        w, s = want[row:row + count], size[row:row + count]
        row += count
        for h in range(2):
            peak = np.abs(w[:, h]).max()
            x = np.abs(w[:, h])
            # half a step: of the code, or of an e4m3 number (2^-4 of it, 2^-10 of the code below 2^-6)
            step = np.full_like(x, .5 / top * peak) if storage == "int8" else np.maximum(x * 2. ** -4, 2. ** -10 / top * peak)
            # the peak's own error moves every value by as much, the quotient by 2^-23 of a code of up to `top`
            limit = step * (1 + 1e-5) + ERROR * (s[:, h] + s[:, h].max()) + 2. ** -22 * peak
            assert (np.abs(got[tile, :count, h] - w[:, h]) <= limit).all(), (tile, h)
    assert row == 215


def test_appends_that_turn_refuse():
    tables, cache = BlockTables(2, 8, 3), KVCache(8, 2, 64)
    plan = tables.plan([3, 4], heads=(4, 2))
    k, q = torch.zeros(7, 2, 64, dtype=torch.bfloat16, device=dev()), torch.zeros(7, 4, 64, dtype=torch.bfloat16, device=dev())
    r = Rotary(64)
    for kw in (dict(q=q), dict(out=q), dict(rotary=r, out=q), dict(rotary=Rotary(128), q=q), dict(rotary=r, q=q[:6]),
               dict(rotary=r, q=q[..., :32]), dict(rotary=r, q=q, out=q[:, :2]), dict(rotary=r, q=q.double())):
        with pytest.raises(ValueError):
            cache.append(k, k, plan, **kw)
    y = cache.append(k, k, plan, rotary=r, q=q.flatten(1), out=q)
    assert y.data_ptr() == q.data_ptr()
    none = tables.plan([0, 0], tokens=0)
    assert cache.append(k[:0], k[:0], none, rotary=r, q=q[:0]).shape == (0, 4, 64)


def test_a_step_that_turns_replays():
    """Plan, append with turned keys and queries, attention: a captured step against the same step launched."""
    P, requests = 64, 5
    r = Rotary(64, base=1e6)
    g = torch.Generator(device=dev()).manual_seed(4)
    k, v = (torch.randn(requests, 2, 128, generator=g, device=dev()).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(requests, 8, 128, generator=g, device=dev()).to(torch.bfloat16)
    counts = torch.ones(requests, dtype=torch.int32, device=dev())

    def fresh():
        tables, cache = BlockTables(requests, 40, 7, page_tokens=P), KVCache(40, 2, 128, page_tokens=P)
        plan = tables.plan([60, 64, 1, 130, 3])
        old = torch.randn(258, 2, 128, generator=torch.Generator(device=dev()).manual_seed(5), device=dev()).half()
        cache.append(old, old, plan, rotary=r)
        tables.commit(plan)
        return tables, cache

    def step(tables, cache):
        plan = tables.plan(counts, tokens=requests, max_new=1, heads=(8, 2))
        turned_q = cache.append(k, v, plan, rotary=r, q=q)
        y = cache.attend(turned_q, plan)
        tables.commit(plan)
        return turned_q, y

    a, b = fresh(), fresh()
    want = [tuple(x.clone() for x in step(*b)) for _ in range(6)]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        y = step(*a)
    for w in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y[0], w[0]) and torch.equal(y[1], w[1])
    assert torch.equal(a[1].data, b[1].data) and a[0].lens.tolist() == b[0].lens.tolist()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("dim,n,layout", [(72, 16, "half"), (256, 64, "half"), (200, 128, "interleaved"), (64, 64, "half")])
@pytest.mark.parametrize("tokens,heads", [(3, 2), (600, 9), (5000, 11)])
def test_dims_that_do_not_turn_are_copied(tokens, heads, dim, n, layout, dtype):
    """By threads of their own; the same rows in place, where they stay, and by the cache's launch."""
    g = torch.Generator(device=dev()).manual_seed(dim + tokens)
    x = torch.randn(tokens, heads, dim, generator=g, device=dev()).to(TYPES[dtype])
    pos = torch.randint(-2, 70000, (tokens,), generator=g, device=dev())
    rotary = Rotary(n, layout=layout, base=3e4)
    y, z = rotary.apply(x, pos), x.clone()
    assert torch.equal(y[..., n:], x[..., n:]) and torch.equal(y[pos < 0], x[pos < 0])
    assert rotary.apply(z, pos, out=z) is z and torch.equal(y, z)
    wide = torch.zeros(tokens, heads + 1, dim + 8, dtype=x.dtype, device=dev())
    out = wide[:, :heads, 8:]
    rotary.apply(x, pos, out=out)
    assert torch.equal(out, y) and not wide[:, heads].any() and not wide[..., :8].any()


def test_rows_in_place_have_one_layout():
    rotary = Rotary(16)
    x = torch.zeros(64, dtype=torch.bfloat16, device=dev())
    a, b = x.as_strided((2, 2, 16), (32, 16, 1)), x.as_strided((2, 2, 16), (16, 32, 1))
    with pytest.raises((ValueError, RuntimeError)):
        rotary.apply(a, torch.zeros(2, dtype=torch.int64, device=dev()), out=b)
