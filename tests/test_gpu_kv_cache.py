"""Block tables, quantising writes and attention of the 8-bit KV cache against
plain implementations in 64 bits on the host (MI355X).

Tolerances follow from the arithmetic: a code is within half a step of its
value (plus 2^-15 of a step for the 32-bit quotient); attention rounds its
probabilities to half precision (2^-11 relative, 2^-25 absolute below 2^-14),
sums in 32 bits, and rounds the output once.
"""
import math

import numpy as np
import pytest
import torch

from stepquant_amd import _native as N
from stepquant_amd.kernels.kv_cache import BlockTables, KVCache
from tests.helpers import dev

pytestmark = pytest.mark.gpu

TOP = {"int8": 127., "fp8": 448.}


def rng(*seed):
    return np.random.default_rng(seed)


# ---------------------------------------------------------------- block tables
def plan_oracle(table, lens, free, counters, rows, new, tokens, P, max_new):
    table, B, width = table.copy(), len(rows), table.shape[1]
    head, tail = counters
    most = min(tokens, tokens // P + 2 * B)
    out = dict(cu=[0], slots=[-1] * tokens, positions=[-1] * tokens, lens=[], granted=[], pages=[], filled=[])
    end = asked = taken = 0
    for r, n in zip(rows, new):
        start, end = end, end + n
        out["cu"].append(min(end, tokens))
        known = 0 <= r < table.shape[0]
        old = int(lens[r]) if known else 0
        had, blocks = -(-old // P), -(-(old + n) // P)
        fits = known and n <= max_new and blocks <= width and end <= tokens
        need = blocks - had if fits else 0
        first, asked = asked, asked + need
        ok = fits and (need == 0 or asked <= tail - head)
        out["granted"].append(ok)
        out["lens"].append(old + n if ok else old)
        if not ok:
            continue
        if need:
            taken = asked
        for j in range(need):
            table[r, had + j] = free[(head + first + j) % len(free)]
        for i in range(n):
            pos = old + i
            out["slots"][start + i] = int(table[r, pos // P]) * P + pos % P
            out["positions"][start + i] = pos
        if n:
            for b in range(old // P, blocks):
                out["pages"].append(int(table[r, b]))
                out["filled"].append(min(P, old + n - b * P))
    for k in ("pages", "filled"):
        out[k] += [0] * (most - len(out[k]))
    out["counters"] = [head + taken, tail]
    return out, table


def check_plan(tables, rows, new, **kw):
    before = [x.cpu().numpy() for x in (tables.table, tables.lens, tables.free)]
    counters = tables.counters.tolist()
    host_rows = rows.tolist() if isinstance(rows, torch.Tensor) else rows
    plan = tables.plan(new, rows, **kw)
    counts = new.tolist() if isinstance(new, torch.Tensor) else new
    want, table = plan_oracle(*before, counters, host_rows, counts, plan.tokens, tables.page_tokens,
                              kw.get("max_new", max(counts)))
    for name, w in want.items():
        got = getattr(plan, name).tolist()
        assert got == w, (name, [(i, a, b) for i, (a, b) in enumerate(zip(got, w)) if a != b][:5])
    assert np.array_equal(tables.table.cpu().numpy(), table)
    assert tables.lens.tolist() == before[1].tolist() and tables.counters.tolist() == counters
    return plan


@pytest.mark.parametrize("batch,P,most,dtype", [(1, 64, 1, torch.int32), (1, 64, 3000, torch.int64), (7, 128, 300, torch.int32),
                                                (64, 64, 1, torch.int64), (513, 64, 70, torch.int32),
                                                (1300, 192, 5, torch.int64), (4096, 64, 3, torch.int32)])
def test_plans_follow_each_other(batch, P, most, dtype):
    print(f"case {batch} requests, pages of {P}, up to {most} tokens", flush=True)
    g = rng(batch, P)
    requests = batch + 5
    tables = BlockTables(requests, 2 + requests * (2 + 4 * most // P), 3 + 4 * most // P, page_tokens=P)
    tables.free.copy_(torch.from_numpy(g.permutation(tables.pages - 1).astype(np.int32) + 1))
    for step in range(4):
        rows = torch.from_numpy(g.permutation(requests)[:batch]).to(dev(), dtype)
        new = torch.from_numpy(g.integers(0 if step else 1, most + 1, batch)).to(dev(), dtype)
        pad = int(g.integers(0, 4))
        plan = check_plan(tables, rows, new, tokens=int(new.sum()) + pad, max_new=most)
        assert plan.granted.all()
        tables.commit(plan)
        assert torch.equal(tables.lens[rows.long()], plan.lens)
        if step == 2:
            gone = rows[:batch // 2 + 1]
            held = [p for r in gone.tolist() for p in tables.table[r, :-(-int(tables.lens[r]) // P)].tolist()]
            tail = int(tables.counters[1])
            # a row named twice gives its pages back once
            tables.release(torch.cat([gone, gone[:1]]))
            assert int(tables.counters[1]) == tail + len(held)
            ring = tables.free.cpu().numpy()
            back = [int(ring[(tail + i) % len(ring)]) for i in range(len(held))]
            assert sorted(back) == sorted(held) and not tables.lens[gone.long()].any()
            assert not tables.table[gone.long()].any()
    # no page is lost or held twice
    head, tail = tables.counters.tolist()
    ring = tables.free.cpu().numpy()
    pages = [int(ring[i % len(ring)]) for i in range(head, tail)]
    for r in range(requests):
        pages += tables.table[r, :-(-int(tables.lens[r]) // P)].tolist()
    assert sorted(pages) == list(range(1, tables.pages))


def test_plans_refuse_what_has_no_room():
    tables = BlockTables(8, 12, 4, page_tokens=64)
    # rows: the third is too long for its table's row, the fourth does not exist
    plan = check_plan(tables, [0, 1, 2, 9, 3, -1], [100, 64, 300, 5, 1, 2])
    assert plan.granted.tolist() == [True, True, False, False, True, False]
    tables.commit(plan)
    # 7 pages are left: the third request passes them, and from there on only
    # tokens that need no page get room
    plan = check_plan(tables, [4, 5, 6, 0, 7, 1], [256, 190, 128, 28, 1, 1])
    assert plan.granted.tolist() == [True, True, False, True, False, False]
    tables.commit(plan)
    assert tables.lens.tolist() == [128, 64, 0, 1, 256, 190, 0, 0]
    # more rows than the call has, and more tokens than max_new
    new = torch.tensor([5, 3], device=dev())
    plan = check_plan(tables, [3, 5], new, tokens=6, max_new=5)
    assert plan.granted.tolist() == [True, False] and plan.cu.tolist() == [0, 5, 6]
    plan = check_plan(tables, [3, 5], new, tokens=9, max_new=4)
    assert plan.granted.tolist() == [False, False]
    # nothing new, and no packed rows at all
    plan = check_plan(tables, [3, 5], [0, 0])
    assert plan.granted.all() and plan.tokens == 0
    tables.commit(plan)


# ---------------------------------------------------------------- writes
def e4m3(y):
    m, e = np.frexp(np.abs(y))
    unit = np.exp2(np.maximum(e - 1, -6) - 3.)
    return np.rint(y / unit) * unit, unit


def page_parts(cache):
    """(codes as the numbers they are [pages, heads, 2, P, D], peaks [pages, heads, 2]) on the host."""
    raw = cache.data.cpu()
    codes = 2 * cache.heads * cache.page_tokens * cache.dim
    c = raw[:, :codes].reshape(-1, cache.heads, 2, cache.page_tokens, cache.dim).contiguous()
    c = c.numpy().astype(np.int16) - 128 if cache.storage == "int8" else c.view(torch.float8_e4m3fn).float().numpy()
    peaks = raw[:, codes:codes + 8 * cache.heads].contiguous().view(torch.float32).reshape(-1, cache.heads, 2).numpy()
    return c.astype(np.float64), peaks


def check_append(cache, k, v, plan):
    """One append against the definition, from the pages as they were."""
    P, top = cache.page_tokens, TOP[cache.storage]
    codes, peaks = page_parts(cache)
    cache.append(k, v, plan)
    got, got_peaks = page_parts(cache)
    slots = plan.slots.cpu().numpy()
    touched = {}
    for t, s in enumerate(slots):
        if s >= 0:
            touched.setdefault(int(s) // P, []).append((int(s) % P, t))
    for part, x in enumerate((k, v)):
        x = x.reshape(plan.tokens, cache.heads, cache.dim).double().cpu().numpy()
        for page, tokens in touched.items():
            start, rows = tokens[0][0], [t for _, t in tokens]
            new = x[rows].transpose(1, 0, 2)
            with np.errstate(invalid="ignore"):
                peak = np.maximum(np.abs(new).max((1, 2)), 2. ** -60)
                if start:
                    peak = np.maximum(peak, peaks[page, :, part])
            np.testing.assert_array_equal(got_peaks[page, :, part], peak.astype(np.float32))
            for h in range(cache.heads):
                c = got[page, h, part]
                if not np.isfinite(peak[h]):
                    assert not c[:start + len(rows)].any()
                    continue
                y = new[h] / peak[h] * top
                near(c[start:start + len(rows)], y, cache.storage)
                if start and peak[h] == peaks[page, h, part]:
                    np.testing.assert_array_equal(c[:start], codes[page, h, part, :start])
                elif start:
                    y = codes[page, h, part, :start] * (float(peaks[page, h, part]) / peak[h])
                    near(c[:start], y, cache.storage)
                np.testing.assert_array_equal(c[start + len(rows):], codes[page, h, part, start + len(rows):])
    left = [p for p in range(cache.pages) if p not in touched]
    np.testing.assert_array_equal(got[left], codes[left])


def near(code, y, storage):
    step = 1. if storage == "int8" else e4m3(y)[1]
    assert (np.abs(code - y) <= step * (.5 + 2. ** -15)).all()


def make(batch, heads, dim, P, storage, tokens_each):
    blocks = -(-tokens_each // P) + 1
    tables = BlockTables(batch, 1 + batch * blocks, blocks, page_tokens=P)
    g = rng(batch, heads, dim, P)
    tables.free.copy_(torch.from_numpy(g.permutation(tables.pages - 1).astype(np.int32) + 1))
    return tables, KVCache(tables.pages, heads, dim, page_tokens=P, storage=storage)


def values(g, shape, dtype, spread=.5):
    x = g.standard_normal(shape) * np.exp(spread * g.standard_normal((shape[0], 1, 1)))
    return torch.from_numpy(x).to(dev(), dtype)


@pytest.mark.parametrize("heads,dim,P,storage,dtype", [
    (1, 64, 64, "int8", torch.bfloat16), (3, 64, 512, "fp8", torch.float16), (2, 128, 64, "int8", torch.float16),
    (2, 128, 192, "fp8", torch.bfloat16), (5, 256, 64, "int8", torch.bfloat16), (2, 256, 128, "fp8", torch.float16),
    (1, 128, 256, "int8", torch.bfloat16)])
def test_appends_quantise_block_by_block(heads, dim, P, storage, dtype):
    print(f"case {heads} heads of {dim}, pages of {P}, {storage}", flush=True)
    tables, cache = make(3, heads, dim, P, storage, 2 * P + 40)
    g = rng(heads, dim, P)
    for new in ([1, 0, P], [1, P - 1, 1], [3, 7, P // 2 + 5], [P, 1, 0], [0, 1, 1]):
        plan = tables.plan(new)
        # a fused projection's row: keys and values are views of it
        row = values(g, (plan.tokens, 3 * heads, dim), dtype)
        check_append(cache, row[:, heads:2 * heads], row.flatten(1)[:, 2 * heads * dim:], plan)
        tables.commit(plan)


def test_appends_of_extreme_values():
    tables, cache = make(5, 1, 64, 64, "int8", 100)
    big, tiny = 3e38, 1e-38
    for step in range(2):
        plan = tables.plan([4] * 5)
        x = torch.randn((20, 1, 64), generator=torch.Generator().manual_seed(step))
        x[0:4] = 0
        x[4:8] *= tiny
        x[8:12] = x[8:12].clamp(-1, 1) * big
        if step:
            x[13, 0, 5] = math.nan
            x[17, 0, 6] = -math.inf
        x = x.to(dev(), torch.bfloat16)
        check_append(cache, x, -x, plan)
        tables.commit(plan)
    k, v = cache.decode(plan.pages, plan.filled)
    for b, bad in enumerate([False, False, False, True, True]):
        assert bool(k[b, :8].isnan().all()) == bad and bool(v[b, :8].isnan().all()) == bad
        assert not k[b, 8:].any() and not v[b, 8:].any()
    assert not k[0].any()


@pytest.mark.parametrize("storage,dtype", [("int8", torch.float32), ("fp8", torch.bfloat16), ("int8", torch.float16)])
def test_decode_gives_the_values_that_codes_stand_for(storage, dtype):
    tables, cache = make(2, 2, 128, 64, storage, 150)
    plan = tables.plan([130, 1])
    x = values(rng(4), (131, 2, 128), torch.bfloat16)
    cache.append(x, x * .5, plan)
    codes, peaks = page_parts(cache)
    want = torch.from_numpy(codes * (peaks / np.float32(TOP[storage])).astype(np.float64)[..., None, None])
    k, v = cache.decode(plan.pages, plan.filled, dtype=dtype)
    assert k.shape == (plan.pages.numel(), 64, 2, 128) and k.dtype == dtype
    unit = {torch.float32: 2. ** -24, torch.bfloat16: 2. ** -8, torch.float16: 2. ** -11}[dtype]
    for i, (p, n) in enumerate(zip(plan.pages.tolist(), plan.filled.tolist())):
        for part, got in enumerate((k, v)):
            w = want[p, :, part].transpose(0, 1)[:n]
            got = got[i].double().cpu()
            assert not got[n:].any()
            assert ((got[:n] - w).abs() <= w.abs() * (unit + 2. ** -22) + 2. ** -25 * (dtype == torch.float16)).all()
    # all tokens of a page; pages that do not exist
    k, _ = cache.decode([int(plan.pages[0]), 0, -3, cache.pages], dtype=torch.float32)
    assert torch.equal(k[0].cpu(), cache.decode(plan.pages[:1], [64])[0][0].cpu()) and not k[1:].any()


def test_copy_moves_a_part_filled_page():
    tables, cache = make(2, 2, 64, 64, "int8", 64)
    plan = tables.plan([10, 0])
    x = values(rng(5), (10, 2, 64), torch.bfloat16)
    cache.append(x, x, plan)
    page = int(plan.pages[0])
    other = 1 + page % (cache.pages - 1)
    cache.copy([page], [other])
    assert torch.equal(cache.data[page], cache.data[other])


# ---------------------------------------------------------------- attention
def attend_oracle(cache, table, held, old, q, q0, n, scale, causal, window):
    """Rows [n, q_heads, dim] in 64 bits and their error bounds."""
    codes, peaks = cache
    P, D = codes.shape[3], codes.shape[4]
    ids = table[:-(-held // P)]
    x = (codes[ids] * peaks[ids][..., None, None]).transpose(2, 1, 0, 3, 4).reshape(2, codes.shape[1], -1, D)[:, :, :held]
    Hq = q.shape[1]
    out, bound = np.zeros((n, Hq, D)), np.zeros((n, Hq, 1))
    for t in range(n):
        pos = old + t
        lo = max(0, pos - window + 1) if window else 0
        hi = pos + 1 if causal else held
        if hi <= lo:
            continue
        for h in range(Hq):
            k, v = x[:, h * codes.shape[1] // Hq, lo:hi]
            qr = q[q0 + t, h]
            s = k @ qr * scale
            p = np.exp(s - s.max())
            out[t, h] = p @ v / p.sum()
            size = np.abs(v).max()
            # scores: products and sums in 32 bits, scaled a few times
            ds = (D + 8) * 2. ** -24 * scale * (np.abs(k) @ np.abs(qr)).max()
            m = hi - lo
            bound[t, h] = size * (2. ** -11 + m * 2. ** -25 + 2 * ds + (m + 64) * 2. ** -23)
    return out, bound


def check_attend(tables, cache, plan, rows, old, new, q, *, causal=True, window=0, scale=None, out=None, **kw):
    got = cache.attend(q, plan, scale=scale, out=out, **kw) if out is None else out
    codes, peaks = page_parts(cache)
    parts = codes, peaks.astype(np.float64) / TOP[cache.storage]
    table = tables.table.cpu().numpy()
    x, y = q.double().cpu().numpy(), got.double().cpu().numpy()
    assert got.shape == x.shape and got.dtype == q.dtype
    unit = 2. ** -8 if q.dtype == torch.bfloat16 else 2. ** -11
    at = 0
    for r, o, n in zip(rows, old, new):
        want, bound = attend_oracle(parts, table[r], o + n, o, x, at, n, scale or cache.dim ** -.5, causal, window)
        err = np.abs(y[at:at + n] - want)
        tol = bound + np.abs(want) * unit * (1 + 2. ** -9) + 2. ** -25
        assert (err <= tol).all(), (r, o, n, float((err / tol).max()), np.argwhere(err > tol)[:4].tolist())
        at += n
    assert not y[at:].any()
    return got


CASES = [  # heads, KV heads, dim, page, storage, dtype, cached, new, padding, causal, window
    (1, 1, 64, 64, "int8", "bf16", [0], [1], 0, True, 0),
    (4, 4, 64, 64, "fp8", "fp16", [0, 62, 63, 64, 700], [1, 1, 1, 1, 1], 2, True, 0),
    (8, 2, 128, 64, "int8", "bf16", [1, 63, 129, 1000, 5000], [1, 1, 1, 1, 1], 0, True, 0),
    (8, 1, 128, 128, "fp8", "bf16", [127, 128, 4099], [1, 1, 1], 3, True, 0),
    (16, 2, 256, 64, "int8", "fp16", [999, 3, 64], [1, 1, 1], 0, True, 0),
    (32, 1, 256, 128, "fp8", "bf16", [517], [1], 0, True, 0),
    (14, 2, 64, 192, "int8", "bf16", [400, 191], [1, 2], 0, True, 0),
    (20, 4, 128, 64, "int8", "bf16", [333, 0, 64], [5, 3, 1], 1, True, 0),
    (6, 2, 64, 64, "fp8", "bf16", [90, 7, 2000], [7, 130, 33], 5, True, 0),
    (12, 4, 128, 64, "int8", "fp16", [0, 65], [200, 63], 0, True, 0),
    (4, 2, 256, 64, "int8", "bf16", [10, 0], [65, 129], 0, True, 0),
    (4, 1, 256, 128, "fp8", "fp16", [300], [70], 0, True, 0),
    (64, 1, 128, 64, "int8", "bf16", [100], [9], 0, True, 0),
    (8, 2, 128, 64, "int8", "bf16", [1000, 40, 5], [1, 1, 1], 0, True, 100),
    (8, 2, 128, 64, "fp8", "bf16", [700, 0], [90, 150], 2, True, 64),
    (8, 2, 64, 64, "int8", "fp16", [300], [17], 0, True, 1),
    (4, 2, 128, 64, "int8", "bf16", [129, 0, 1], [30, 64, 2], 3, False, 0),
    (2, 2, 64, 256, "fp8", "bf16", [1025], [1], 0, False, 0),
    (4, 1, 256, 64, "int8", "bf16", [500, 0], [40, 90], 1, True, 70),
    (8, 2, 256, 64, "fp8", "bf16", [130, 1], [20, 50], 0, False, 0),
    (32, 1, 256, 64, "int8", "fp16", [700, 31], [1, 1], 1, True, 0),
    (3, 3, 128, 192, "int8", "bf16", [100], [37], 0, True, 0),
    (40, 2, 128, 64, "fp8", "bf16", [257, 90], [1, 1], 0, True, 33),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_attention(case):
    print(f"case {case}", flush=True)
    Hq, H, D, P, storage, dt, old, new, pad, causal, window = case
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16}[dt]
    g = rng(Hq, H, D, sum(old))
    tables, cache = make(len(old) + 2, H, D, P, storage, max(o + n for o, n in zip(old, new)))
    # pages that nobody holds: codes and peaks of an earlier user's, NaN among them
    cache.data.copy_(torch.from_numpy(g.integers(0, 256, cache.data.shape, dtype=np.uint8)))
    if storage == "fp8":
        # e4m3's NaN is never written by an append
        cache.data[(cache.data & 127) == 127] -= 1
    cache.data[:, 2 * H * P * D:2 * H * P * D + 8 * H] = 255
    rows = g.permutation(len(old) + 2)[:len(old)].tolist()
    first = tables.plan(old, rows)
    cache.append(values(g, (first.tokens, H, D), dtype), values(g, (first.tokens, H, D), dtype), first)
    tables.commit(first)
    tokens = sum(new) + pad
    plan = tables.plan(new, rows, tokens=tokens, heads=(Hq, H), causal=causal, window=window)
    cache.append(values(g, (tokens, H, D), dtype), values(g, (tokens, H, D), dtype), plan)
    # rows of a fused projection, some of them looking at few keys
    q = values(g, (tokens, Hq + 2 * H, D), dtype, 1.)[:, :Hq]
    got = check_attend(tables, cache, plan, rows, old, new, q, causal=causal, window=window)
    again = cache.attend(q, plan)
    assert torch.equal(got, again)
    # after the commit the plan still holds
    tables.commit(plan)
    assert torch.equal(got, cache.attend(q.flatten(1), plan))


@pytest.fixture(params=[(0, 0), (1 << 14, 1)], ids=["256", "256-decided"])
def sets_of_256(request, monkeypatch):
    """Sets of 256 rows, which short prompts would not get: asked for, or as the plan decides."""
    monkeypatch.setattr(BlockTables, "few_rows", request.param[0])
    monkeypatch.setattr(BlockTables, "few_work", request.param[1])


@pytest.mark.parametrize("case", [c for c in CASES if max(c[7]) * (c[0] // c[1]) > 64],
                         ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_attention_in_sets_of_256(case, sets_of_256):
    test_attention(case)


def filled(old, new, Hq=8, H=2, D=128, P=64, storage="int8", seed=0, **kw):
    g = rng(seed, Hq, D)
    tables, cache = make(len(old), H, D, P, storage, max(o + n for o, n in zip(old, new)))
    first = tables.plan(old)
    cache.append(values(g, (first.tokens, H, D), torch.bfloat16), values(g, (first.tokens, H, D), torch.bfloat16), first)
    tables.commit(first)
    plan = tables.plan(new, heads=(Hq, H), **kw)
    cache.append(values(g, (plan.tokens, H, D), torch.bfloat16), values(g, (plan.tokens, H, D), torch.bfloat16), plan)
    return tables, cache, plan, values(g, (plan.tokens, Hq, D), torch.bfloat16)


@pytest.mark.parametrize("Hq,H,D,storage,window", [(4, 2, 64, "int8", 0), (2, 1, 128, "fp8", 0), (8, 1, 64, "fp8", 50)])
def test_many_requests_of_unequal_lengths(Hq, H, D, storage, window):
    """More sets of rows than workgroups for them: shares with several sets, cut
    at both ends."""
    g = rng(Hq, H, D)
    old = [int(x) for x in np.exp(g.uniform(0, np.log(900), 230))]
    new = [int(x) for x in g.integers(1, 3, 230)]
    print(f"case {Hq} over {H} heads of {D}, {sum(old)} tokens held", flush=True)
    tables, cache, plan, q = filled(old, new, Hq=Hq, H=H, D=D, storage=storage, window=window)
    check_attend(tables, cache, plan, list(range(230)), old, new, q, window=window)


@pytest.mark.parametrize("Hq,H,D,old,new,causal", [(8, 1, 64, [0], [1100], True), (4, 2, 128, [900, 70], [333, 400], True),
                                                   (2, 1, 256, [64], [520], False), (4, 1, 256, [333], [300], True)])
def test_prompts_of_many_sets_of_rows(Hq, H, D, old, new, causal):
    print(f"case {Hq} over {H} heads of {D}, {new} over {old}", flush=True)
    tables, cache, plan, q = filled(old, new, Hq=Hq, H=H, D=D, causal=causal)
    check_attend(tables, cache, plan, list(range(len(old))), old, new, q, causal=causal)


@pytest.mark.parametrize("D,new", [(128, 1), (128, 5), (64, 40), (256, 30)])
@pytest.mark.parametrize("scale", [-.1, 0., 3.])
def test_scales_of_any_sign(D, new, scale):
    old = [90]
    tables, cache, plan, q = filled(old, [new], D=D, H=1, Hq=8)
    out = cache.attend(q, plan, scale=scale)
    codes, peaks = page_parts(cache)
    parts = codes, peaks.astype(np.float64) / TOP["int8"]
    x = q.double().cpu().numpy()
    want, bound = attend_oracle(parts, tables.table.cpu().numpy()[0], 90 + new, 90, x, 0, new, scale, True, 0)
    if scale <= 0:  # the oracle's bound takes the scale's size
        bound = attend_oracle(parts, tables.table.cpu().numpy()[0], 90 + new, 90, x, 0, new, abs(scale), True, 0)[1]
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= bound + np.abs(want) * 2. ** -8 * (1 + 2. ** -9) + 2. ** -25).all()


def test_requests_come_and_go():
    """Pages that were released serve other requests, whose blocks start afresh."""
    g = rng(21)
    tables, cache = BlockTables(4, 12, 6), KVCache(12, 2, 64)
    held = [0, 0, 0, 0]
    for step in range(14):
        rows = g.permutation(4)[:int(g.integers(1, 5))].tolist()
        new = [int(x) for x in g.integers(0, 120, len(rows))]
        plan = tables.plan(new, rows, heads=(4, 2))
        x = values(g, (plan.tokens, 2, 64), torch.bfloat16, 1.)
        y = values(g, (plan.tokens, 2, 64), torch.bfloat16, 1.)
        check_append(cache, x, y, plan)
        ok = plan.granted.tolist()
        q = values(g, (plan.tokens, 4, 64), torch.bfloat16)
        out = cache.attend(q, plan)
        at = 0
        for r, n, good in zip(rows, new, ok):
            if not good:
                assert not out[at:at + n].any()
            at += n
        if all(ok) and plan.tokens:
            check_attend(tables, cache, plan, rows, [held[r] for r in rows], new, q, out=out)
        tables.commit(plan)
        for r, n, good in zip(rows, new, ok):
            held[r] += n if good else 0
        assert tables.lens.tolist() == held
        gone = [r for r in range(4) if held[r] and g.random() < (.9 if not all(ok) else .25)]
        tables.release(gone) if gone else None
        for r in gone:
            held[r] = 0


def test_rows_that_kernels_do_not_take_are_copied():
    old, new = [100], [3]
    tables, cache, plan, q = filled(old, new)
    want = cache.attend(q, plan)
    wide = torch.empty((3, 8, 130), dtype=q.dtype, device=dev())
    wide[..., 1:129] = q
    assert torch.equal(cache.attend(wide[..., 1:129], plan), want)
    assert torch.equal(cache.attend(q.transpose(1, 2).contiguous().transpose(1, 2), plan), want)
    k = values(rng(30), (3, 2, 128), torch.bfloat16)
    cache.append(k, k, plan)
    want = cache.data.clone()
    cache.append(k.transpose(0, 1).contiguous().transpose(0, 1), k[:, :, :].clone().flatten(1), plan)
    assert torch.equal(cache.data, want)


def test_starts_that_kernels_do_not_take_are_copied():
    tables, cache, plan, q = filled([70], [3])
    want = cache.attend(q, plan)
    k = values(rng(31), (3, 2, 128), torch.bfloat16)
    cache.append(k, k, plan)
    data, want = cache.data.clone(), cache.attend(q, plan)

    def moved(x):
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
        return y.copy_(x)

    assert moved(q).is_contiguous() and moved(q).data_ptr() % 16
    assert torch.equal(cache.attend(moved(q), plan), want)
    cache.append(moved(k), moved(k), plan)
    assert torch.equal(cache.data, data)


def test_plans_without_tokens():
    tables, cache = make(2, 2, 128, 64, "int8", 64)
    plan = tables.plan([0, 0], heads=(8, 2))
    none = torch.empty((0, 8, 128), dtype=torch.bfloat16, device=dev())
    cache.append(none[:, :2], none[:, :2], plan)
    assert cache.attend(none, plan).shape == cache.attend(none.flatten(1), plan).shape == (0, 8, 128)
    tables.commit(plan)
    assert tables.lens.tolist() == [0, 0] and plan.granted.tolist() == [True, True]
    tables.release([])
    assert cache.decode([])[0].shape == (0, 64, 2, 128)
    assert tables.counters.tolist() == [0, tables.pages - 1]


def test_a_plan_lives_on_for_another_stream():
    tables, cache, plan, q = filled([130], [2])
    want = cache.attend(q, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = cache.attend(q, plan)
    plan.record_stream(side)
    del plan
    tables.plan([5], heads=(8, 2))
    side.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5, 90])
def test_values_of_very_different_sizes(D, new):
    """Blocks of values of 0, 2^-30, 2^20 and between, each looked at by some rows:
    none is lost beside another one's size, in the outputs or in the sums."""
    Hq, sizes = 4, [2. ** -30, 1., 0., 2. ** 20, 2. ** -12, 2. ** -6]
    print(f"case {new} new tokens of {D} dims", flush=True)
    g = rng(41, D, new)
    old = 64 * len(sizes)
    tables, cache = make(1, 1, D, 64, "int8", old + new)
    k, v = g.standard_normal((old + new, 1, D)) * .1, g.standard_normal((old + new, 1, D))
    sharp = (40. * D ** .5) ** .5
    for b, size in enumerate(sizes):
        v[64 * b:64 * (b + 1)] *= size
        k[64 * b:64 * (b + 1), :, b] += sharp
    q = g.standard_normal((new, Hq, D)) * .1
    for t in range(new):
        for h in range(Hq):
            # a block, two of them alike, or none
            i = (t * Hq + h + D // 64) % 8
            q[t, h, :6] += sharp * np.eye(6)[i % 6] if i < 6 else sharp / 2 * (i == 6) * np.array([0, 1, 1, 0, 0, 0])
    x = [torch.tensor(a, dtype=torch.bfloat16, device=dev()) for a in (k, v, q)]
    plan = tables.plan([old])
    cache.append(x[0][:old], x[1][:old], plan)
    tables.commit(plan)
    plan = tables.plan([new], heads=(Hq, 1))
    cache.append(x[0][old:], x[1][old:], plan)
    got = cache.attend(x[2], plan).double().cpu().numpy()
    codes, peaks = page_parts(cache)
    unit = peaks.astype(np.float64) / 127.
    ids = tables.table.cpu().numpy()[0]
    keys, vals = ((codes[ids] * unit[ids][..., None, None]).transpose(2, 1, 0, 3, 4).reshape(2, -1, D))
    peak = np.repeat(peaks[ids].reshape(len(ids), -1)[:, 1].astype(np.float64), 64)
    queries = x[2].double().cpu().numpy()
    for t in range(new):
        n = old + t + 1
        for h in range(Hq):
            s = keys[:n] @ queries[t, h] * D ** -.5
            p = np.exp(s - s.max())
            p /= p.sum()
            want, size = p @ vals[:n], p @ np.abs(vals[:n])
            ds = (D + 8) * 2. ** -24 * D ** -.5 * (np.abs(keys[:n]) @ np.abs(queries[t, h])).max()
            # halves of weights and of the sum's terms (2^-17 of the largest at least), and
            # of products too small for a half beside the row's largest product
            tol = size * (2. ** -10 + n * 2. ** -17 + 2 * ds + (n + 64) * 2. ** -23) + n * 2. ** -24 * (p * peak[:n]).max()
            tol += np.abs(want) * 2. ** -8 * (1 + 2. ** -9)
            err = np.abs(got[t, h] - want)
            assert (err <= tol).all(), (t, h, float((err / tol).max()))


@pytest.mark.parametrize("D,new", [(64, 1), (64, 90), (128, 20), (128, 90), (256, 5), (256, 90)])
def test_scores_beyond_fractions(D, new):
    """Scores of 10^8 and more: the largest takes the row, nothing overflows."""
    old, Hq = 300, 4
    print(f"case {new} new tokens of {D} dims", flush=True)
    g = rng(43, D, new)
    tables, cache = make(1, 1, D, 64, "int8", old + new)
    big = [torch.from_numpy(np.clip(2e4 * g.standard_normal((old + new, h, D)), -6e4, 6e4)).to(dev(), torch.float16)
           for h in (1, Hq)]
    v = values(g, (old + new, 1, D), torch.float16)
    plan = tables.plan([old])
    cache.append(big[0][:old], v[:old], plan)
    tables.commit(plan)
    plan = tables.plan([new], heads=(Hq, 1))
    cache.append(big[0][old:], v[old:], plan)
    q = big[1][old:]
    got = cache.attend(q, plan).double().cpu().numpy()
    codes, peaks = page_parts(cache)
    ids = tables.table.cpu().numpy()[0]
    x = (codes[ids] * (peaks.astype(np.float64) / 127.)[ids][..., None, None]).transpose(2, 1, 0, 3, 4).reshape(2, -1, D)
    clear = 0
    for t in range(new):
        for h in range(Hq):
            s = x[0][:old + t + 1] @ q[t, h].double().cpu().numpy() * D ** -.5
            best, other = np.sort(s)[[-1, -2]]
            assert np.abs(got[t, h]).max() <= np.abs(x[1]).max() * 1.001
            # 32-bit sums of D products: a gap of twice their error leaves one key
            if best - other > 2 * ((D + 8) * 2. ** -24 * np.abs(s).max() * D ** .5 + 100):
                clear += 1
                want = x[1][s.argmax()]
                assert (np.abs(got[t, h] - want) <= np.abs(want) * 2. ** -10 + 2. ** -24).all(), (t, h)
    assert clear >= new


@pytest.mark.parametrize("D", [64, 128, 256])
def test_sizes_and_scores_in_sets_of_256(D, sets_of_256):
    test_values_of_very_different_sizes(D, 90)
    test_scores_beyond_fractions(D, 90)
    for scale in (-.1, 0., 3.):
        test_scales_of_any_sign(D, 40, scale)


@pytest.mark.parametrize("storage", ["int8", "fp8"])
def test_a_bad_block_in_sets_of_256(storage, sets_of_256):
    test_a_bad_block_reaches_only_rows_that_see_it(storage)


def test_prompts_of_many_sets_in_sets_of_256(sets_of_256):
    test_prompts_of_many_sets_of_rows(4, 2, 128, [900, 70], [333, 400], True)
    test_prompts_of_many_sets_of_rows(2, 1, 256, [64], [520], False)


def test_a_graph_follows_the_lengths():
    """Chunks of 40 tokens, captured once: the plan takes sets of 32 rows while the
    requests are short and of 256 when they have grown."""
    H, Hq, D, n = 2, 16, 128, 40
    g = rng(47)
    tables, cache = make(1, H, D, 64, "int8", 18 * n + 1)
    new, rows = torch.tensor([n], dtype=torch.int32, device=dev()), torch.zeros(1, dtype=torch.int32, device=dev())
    q, k, v = (torch.empty((n, h, D), dtype=torch.bfloat16, device=dev()) for h in (Hq, H, H))
    tables.few_work = n * Hq * 6  # (tiles of the chunk's middle: up to five)
    warm = tables.plan(new, rows, tokens=n, max_new=n, heads=(Hq, H))
    for t in (q, k, v):
        t.zero_()
    cache.append(k, v, warm)
    cache.attend(q, warm)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            plan = tables.plan(new, rows, tokens=n, max_new=n, heads=(Hq, H))
            cache.append(k, v, plan)
            out = cache.attend(q, plan)
            tables.commit(plan)
    for i in range(18):
        for t in (q, k, v):
            t.copy_(values(g, t.shape, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        check_attend(tables, cache, plan, [0], [n * i], [n], q, out=out)
    assert tables.lens.tolist() == [18 * n]


def test_refused_requests_give_zero():
    tables, cache = make(2, 2, 64, 64, "int8", 64)
    plan = tables.plan([3, 200, 5], [0, 1, 1], heads=(4, 2), causal=False)
    assert plan.granted.tolist() == [True, False, True]
    x = values(rng(7), (208, 2, 64), torch.bfloat16)
    cache.append(x, x, plan)
    out = cache.attend(values(rng(8), (208, 4, 64), torch.bfloat16), plan)
    assert out[:3].any() and not out[3:203].any() and out[203:].any()


@pytest.mark.parametrize("storage", ["int8", "fp8"])
def test_a_bad_block_reaches_only_rows_that_see_it(storage):
    old, new = [0, 200], [200, 1]
    tables, cache, plan, q = filled(old, new, storage=storage)
    clean = cache.attend(q, plan)
    # the values of the request's third block, and the keys of its last
    page, last = tables.table[0, 2], tables.table[0, 3]
    codes = 2 * 2 * 64 * 128
    peaks = cache.data[:, codes:codes + 16].clone().view(torch.float32)
    peaks[page, 1] = math.nan
    peaks[last, 2] = math.nan
    cache.data[:, codes:codes + 16] = peaks.view(torch.uint8)
    out = cache.attend(q, plan)
    assert torch.equal(out[:128], clean[:128]) and torch.equal(out[200:], clean[200:])
    assert out[128:, :4][:72].isnan().all() and torch.equal(out[128:192, 4:], clean[128:192, 4:])
    assert not torch.isfinite(out[192:200, 4:]).all(-1).any()


def test_bad_and_extreme_queries_keep_to_their_rows():
    old, new = [700, 0], [3, 1]
    tables, cache, plan, q = filled(old, new)
    clean = cache.attend(q, plan)
    q[0, 1, 3] = math.nan
    q[2, 5, 0] = math.inf
    q[1, 2] = 0
    q[1, 3] *= 1e-30
    q[1, 4] = q[1, 4] * 2. ** -40
    out = cache.attend(q, plan)
    assert out[0, 1].isnan().all() and not torch.isfinite(out[2, 5]).any()
    same = torch.ones((4, 8), dtype=torch.bool)
    for t, h in ((0, 1), (2, 5), (1, 2), (1, 3), (1, 4)):
        same[t, h] = False
    assert torch.equal(out[same.to(dev())], clean[same.to(dev())])
    ok = q.clone()
    ok[0, 1, 3] = 0
    ok[2, 5, 0] = 0
    check_attend(tables, cache, plan, [0, 1], old, new, ok)
    # one key far above the rest: a softmax of one
    check_attend(tables, cache, plan, [0, 1], old, new, ok * 200)


def test_pages_past_32_bit_offsets():
    """Pages that start beyond 2^32 bytes."""
    pages = 70000
    cache = KVCache(pages, 4, 128)
    assert cache.page_bytes * (pages - 8) > 1 << 32
    tables = BlockTables(1, pages, 5)
    tables.free.copy_(torch.arange(pages - 1, 0, -1, dtype=torch.int32))
    g = rng(9)
    plan = tables.plan([250], heads=(8, 4))
    cache.append(values(g, (250, 4, 128), torch.bfloat16), values(g, (250, 4, 128), torch.bfloat16), plan)
    q = values(g, (250, 8, 128), torch.bfloat16)
    got = cache.attend(q, plan)
    # the same tokens in the first pages of a small cache
    small_tables, small = BlockTables(1, 6, 5), KVCache(6, 4, 128)
    p2 = small_tables.plan([250], heads=(8, 4))
    for i in range(4):
        small.data[int(p2.pages[i])] = cache.data[int(plan.pages[i])]
    assert torch.equal(got, small.attend(q, p2))
    k, v = cache.decode(plan.pages, plan.filled)
    k2, v2 = small.decode(p2.pages, p2.filled)
    assert torch.equal(k, k2) and torch.equal(v, v2)


def test_table_entries_outside_the_cache_are_passed_over():
    old, new = [300], [2]
    tables, cache, plan, q = filled(old, new)
    want = cache.attend(q, plan)
    page = int(tables.table[0, 1])
    for bad in (0, -5, cache.pages, 1 << 30):
        tables.table[0, 1] = bad
        out = cache.attend(q, plan)
        assert torch.isfinite(out).all() and not torch.equal(out, want)
    tables.table[0, 1] = page
    assert torch.equal(cache.attend(q, plan), want)


def test_windows_of_one_plan_and_a_given_output():
    old, new = [500, 90], [1, 1]
    tables, cache, plan, q = filled(old, new, window=(0, 128))
    check_attend(tables, cache, plan, [0, 1], old, new, q)
    out = torch.empty_like(q)
    assert cache.attend(q, plan, window=128, scale=.05, out=out) is out
    check_attend(tables, cache, plan, [0, 1], old, new, q, window=128, scale=.05, out=out)


def test_another_stream_and_graph_replays():
    """The serving step: plan, append, attend, commit, captured once and
    replayed while the requests grow past their pages."""
    B, H, Hq, D = 3, 2, 8, 128
    g = rng(11)
    made = []
    for _ in range(2):
        tables, cache = make(B, H, D, 64, "int8", 300)
        first = tables.plan([62, 1, 120])
        x = values(rng(12), (183, H, D), torch.bfloat16)
        cache.append(x, x, first)
        tables.commit(first)
        made.append((tables, cache))
    new = torch.ones(B, dtype=torch.int32, device=dev())
    rows = torch.arange(B, device=dev())
    q, k, v = (torch.empty((B, n, D), dtype=torch.bfloat16, device=dev()) for n in (Hq, H, H))

    def step(tables, cache):
        plan = tables.plan(new, rows, tokens=B, max_new=1, heads=(Hq, H))
        cache.append(k, v, plan)
        out = cache.attend(q, plan)
        tables.commit(plan)
        return plan, out

    (eager_tables, eager), (tables, cache) = made
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            plan, out = step(tables, cache)
    for i in range(6):
        for t, n in ((q, Hq), (k, H), (v, H)):
            t.copy_(values(g, (B, n, D), torch.bfloat16))
        _, want = step(eager_tables, eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(tables.lens, eager_tables.lens) and torch.equal(cache.data, eager.data)
        with torch.cuda.stream(side):
            side_out = eager.attend(q, eager_tables.plan([0] * B, rows, tokens=B, heads=(Hq, H)))
        side.synchronize()
        assert not side_out.any()
    assert tables.lens.tolist() == [68, 7, 126]


def test_refusals():
    tables, cache, plan, q = filled([5], [2])
    k = torch.zeros((2, 2, 128), dtype=torch.bfloat16, device=dev())
    with pytest.raises(ValueError, match="bf16 or fp16"):
        cache.attend(q.float(), plan)
    with pytest.raises(ValueError, match="queries must be"):
        cache.attend(q[:1], plan)
    with pytest.raises(ValueError, match="window"):
        cache.attend(q, plan, window=5)
    with pytest.raises(ValueError, match="without heads"):
        cache.attend(q, tables.plan([2]))
    with pytest.raises(ValueError, match="KV heads"):
        cache.attend(q, tables.plan([2], heads=(8, 4)))
    with pytest.raises(ValueError, match="out must be"):
        cache.attend(q, plan, out=q.float())
    with pytest.raises(ValueError, match="one dtype"):
        cache.append(k, k.half(), plan)
    with pytest.raises(ValueError, match="keys must be"):
        cache.append(k[:, :1], k, plan)
    with pytest.raises(ValueError, match="device"):
        cache.append(k.cpu(), k, plan)
    with pytest.raises(ValueError, match="other pages"):
        KVCache(4, 2, 128, page_tokens=128).append(k, k, plan)
    with pytest.raises(ValueError, match="other block tables"):
        BlockTables(1, 4, 2).commit(plan)
    with pytest.raises(ValueError, match="tokens and max_new"):
        tables.plan(torch.ones(1, dtype=torch.int32, device=dev()))
    for bad in (dict(new=[-1]), dict(new=[]), dict(new=[1], rows=[0, 0]), dict(new=[1], window=4, causal=False),
                dict(new=[1], heads=(3, 2)), dict(new=[1], heads=(2, 2), window=-1), dict(new=[1], rows=[.5]),
                dict(new=[1] * 4097), dict(new=[1], window=(1, 2, 3, 4, 5), heads=(2, 2)), dict(new=[1], tokens=-1)):
        with pytest.raises(ValueError):
            tables.plan(**bad)
    with pytest.raises(ValueError):
        cache.decode([1], dtype=torch.int8)
    with pytest.raises(ValueError, match="integers"):
        cache.decode([1.5])
    with pytest.raises(ValueError, match="int32 or int64"):
        tables.plan(torch.tensor([1.]))
    with pytest.raises(TypeError):
        tables.plan([1.5])
    with pytest.raises(ValueError):
        cache.decode([1], [1, 2])
    with pytest.raises(ValueError):
        tables.release(list(range(4097)))
