"""The 8-bit KV cache at the ends of its number ranges, against plain
implementations in 64 bits on the host (MI355X).
"""
import numpy as np
import pytest
import torch

from stepquant_amd import _native as N
from stepquant_amd.kernels.kv_cache import BlockTables
from tests.helpers import dev
from tests.test_gpu_kv_cache import TOP, check_append, filled, make, page_parts, rng

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- writes
@pytest.mark.parametrize("storage", ["int8", "fp8"])
@pytest.mark.parametrize("sizes", [(1e37, 2e37, 3e38), (7e35, 8e35, 1e36, 1e38), (1., 1e30, 3e38), (1e-19, 3e38, 3.1e38)],
                         ids=lambda s: "-".join(map(str, s)))
def test_large_blocks_grow(storage, sizes):
    """Older codes are brought to a finite larger peak, whatever the peaks."""
    print(f"case {storage}, peaks {sizes}", flush=True)
    tables, cache = make(2, 2, 64, 64, storage, 64)
    g = rng(51, len(sizes))
    for size in sizes:
        plan = tables.plan([5, 1])
        x = [torch.from_numpy(g.uniform(-1, 1, (6, 2, 64)) * size).to(dev(), torch.bfloat16) for _ in range(2)]
        check_append(cache, *x, plan)
        tables.commit(plan)
    k, v = cache.decode(plan.pages, plan.filled)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()


# ---------------------------------------------------------------- attention
@pytest.fixture(params=[(0, 0), (1 << 14, 1)], ids=["256", "256-decided"])
def sets_of_256(request, monkeypatch):
    """Sets of 256 rows, which short prompts would not get: asked for, or as the plan decides."""
    monkeypatch.setattr(BlockTables, "few_rows", request.param[0])
    monkeypatch.setattr(BlockTables, "few_work", request.param[1])


def attended(k, v, q, storage="int8", workgroups=None):
    """One request of one KV head: the first keys held, the others new beside ``q``
    [new, heads, D].  (outputs, keys, values and their blocks' peaks as held, in 64 bits)"""
    n, D = k.shape
    new, Hq, _ = q.shape
    tables, cache = make(1, 1, D, 64, storage, n)
    if workgroups:  # few, so that each of them has many keys
        tables._cus = workgroups
    k, v = k.view(n, 1, D), v.view(n, 1, D)
    first = tables.plan([n - new])
    cache.append(k[:n - new], v[:n - new], first)
    tables.commit(first)
    plan = tables.plan([new], heads=(Hq, 1))
    cache.append(k[n - new:], v[n - new:], plan)
    got = cache.attend(q, plan).double().cpu().numpy()
    codes, peaks = page_parts(cache)
    ids = tables.table.cpu().numpy()[0, :-(-n // 64)]
    peaks = peaks[ids, 0].astype(np.float64)
    keys, vals = (codes[ids, 0] * (peaks / TOP[storage])[..., None, None]).transpose(1, 0, 2, 3).reshape(2, -1, D)[:, :n]
    return got, keys, vals, np.repeat(peaks[:, 1], 64)[:n]


def check_sums(got, keys, vals, peak, q):
    """Halves of weights (2^-11) in the products and in the sums, 32-bit sums, one
    rounding at the end.  A weight has all its bits down to 2^-20 of a row's
    largest and is within 2^-31 of that below (of the largest weight times a block's
    peak in the products)."""
    new, Hq, D = q.shape
    x, unit = q.double().cpu().numpy(), 2. ** -8 if q.dtype == torch.bfloat16 else 2. ** -11
    worst = 0.
    for t in range(new):
        n = len(keys) - new + t + 1
        s = x[t] @ keys[:n].T * D ** -.5
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        want, size = p @ vals[:n], p @ np.abs(vals[:n])
        ds = (D + 8) * 2. ** -24 * D ** -.5 * (np.abs(x[t]) @ np.abs(keys[:n]).T).max(1)[:, None]
        tol = size * (2. ** -10 + 2 * ds + (n / 16 + 64) * 2. ** -23) + np.abs(want) * unit * (1 + 2. ** -9)
        tol += n * 2. ** -31 * ((p * peak[:n]).max(1)[:, None] + np.abs(want)) + 2. ** -25
        worst = max(worst, float((np.abs(got[t] - want) / tol).max())) if np.isfinite(got[t]).all() else np.inf
    assert worst <= 1, worst


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5, 90])
@pytest.mark.parametrize("storage", ["int8", "fp8"])
def test_values_near_the_largest(D, new, storage):
    """Outputs are finite where values are, however many of them a row sums."""
    print(f"case {new} new tokens of {D} dims, {storage}", flush=True)
    g = rng(52, D, new)
    n = 2000 + new
    sign = np.where(g.random(D) < .5, -1., 1.)
    k = torch.from_numpy(g.standard_normal((n, D)) * .1).to(dev(), torch.bfloat16)
    v = torch.from_numpy(g.uniform(.3, 1, (n, D)) * sign * 3.3e38).to(dev(), torch.bfloat16)
    q = torch.from_numpy(g.standard_normal((new, 4, D))).to(dev(), torch.bfloat16)
    check_sums(*attended(k, v, q, storage), q)
    check_sums(*attended(k, v, q, storage, workgroups=1), q)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("storage", ["int8", "fp8"])
def test_values_near_the_largest_in_sets_of_256(D, storage, sets_of_256):
    test_values_near_the_largest(D, 90, storage)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5, 90])
@pytest.mark.parametrize("depth,first", [(18, 128.), (18, 8.), (23, 0.), (26, 0.)])
def test_many_small_weights_beside_a_large_one(D, new, depth, first):
    """20,000 keys at 2^-depth of a row's first one, whose values are ``first``
    times the others' or zero."""
    print(f"case {new} new tokens of {D} dims, 2^-{depth}, {first}", flush=True)
    g = rng(53, D, new, depth)
    n = 20000 + new
    k, v = g.standard_normal((n, D)) * .3, 1 + .3 * g.standard_normal((n, D))
    k[0, 0], v[0] = depth * np.log(2.), first * (1 + .1 * g.standard_normal(D))
    q = .02 * g.standard_normal((new, 4, D))
    q[..., 0] = D ** .5 * g.uniform(1, 1.05, (new, 4))
    k, v, q = (torch.from_numpy(a).to(dev(), torch.float16) for a in (k, v, q))
    check_sums(*attended(k, v, q, workgroups=1), q)


def check_winners(got, keys, vals, q):
    """Rows whose largest score is clear of the second by more than their error."""
    new, Hq, D = q.shape
    x, clear = q.double().cpu().numpy(), 0
    for t in range(new):
        n = len(keys) - new + t + 1
        for h in range(Hq):
            s = keys[:n] @ x[t, h] * D ** -.5
            other, best = np.sort(s)[-2:]
            if best - other > 2 * ((D + 8) * 2. ** -24 * np.abs(s).max() * D ** .5 + 100):
                clear += 1
                want = vals[s.argmax()]
                tol = np.abs(want) * (2. ** -8 * (1 + 2. ** -9) + 2. ** -10) + np.abs(want).max() * 2. ** -22
                assert (np.abs(got[t, h] - want) <= tol).all(), (t, h, got[t, h][:4], want[:4])
    assert clear >= new


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5, 90])
def test_scores_past_2_30_and_values_of_any_size(D, new):
    """Where 32 bits hold no difference of 100 between scores, blocks' value
    peaks still come out as they are."""
    print(f"case {new} new tokens of {D} dims", flush=True)
    g = rng(54, D, new)
    n = 320 + new
    sizes = np.repeat([2. ** 40, 2. ** -20, 2. ** 100, 1., 2. ** -50, 2. ** 17, 2. ** 10], 64)[:n]
    k, q = 1e5 * g.standard_normal((n, D)), 1e5 * g.standard_normal((new, 4, D))
    v = g.standard_normal((n, D)) * sizes[:, None]
    k, v, q = (torch.from_numpy(a).to(dev(), torch.bfloat16) for a in (k, v, q))
    got, keys, vals, _ = attended(k, v, q)
    assert np.isfinite(got).all()
    check_winners(got, keys, vals, q)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_past_2_30_in_sets_of_256(D, sets_of_256):
    test_scores_past_2_30_and_values_of_any_size(D, 90)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("depth,first", [(18, 128.), (18, 8.), (23, 0.), (26, 0.)])
def test_many_small_weights_in_sets_of_256(D, depth, first, sets_of_256):
    test_many_small_weights_beside_a_large_one(D, 90, depth, first)


def unit_rows(plan, window=0):
    """Rows of a unit as the plan kernel stored them."""
    fields = N.KV_SCHEDULE.unpack(plan.schedules[window].packed)
    return int(plan._ints[(fields[2] - plan._ints.data_ptr()) // 4 + fields[5] + 1])


def test_the_plan_decides_by_its_lengths():
    """One captured plan takes sets of 32 rows while a request is short, of 256 when it has grown."""
    n, Hq, H = 40, 16, 2
    tables = BlockTables(1, 20, 18)
    tables.few_work = n * Hq * 6  # (five tiles up to the chunk's middle, and one)
    new, rows = torch.tensor([n], dtype=torch.int32, device=dev()), torch.zeros(1, dtype=torch.int32, device=dev())
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        plan = tables.plan(new, rows, tokens=n, max_new=n, heads=(Hq, H))
        tables.commit(plan)
    seen = []
    for i in range(18):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(unit_rows(plan))
    assert seen == [32 if (n * i + n // 2) // 64 + 1 <= 6 else 256 for i in range(18)] and len(set(seen)) == 2


def test_sets_of_256_are_those(sets_of_256):
    """What the tests in sets of 256 rows run, whether asked for or decided."""
    for Hq, D, new in ((8, 128, 90), (4, 256, 90), (4, 64, 90)):
        assert unit_rows(filled([200], [new], Hq=Hq, H=1, D=D)[2]) == 256
    assert unit_rows(filled([200], [new], Hq=4, H=1, D=64, window=50)[2], 50) == 256


def test_row_counts_by_the_longest_request():
    for Hq, H, new, rows in ((4, 4, [16, 1], 16), (8, 1, [2, 1], 16), (8, 1, [3], 32), (8, 1, [8, 2], 32), (8, 1, [9], 32),
                             (8, 1, [2100], 256)):
        print(f"case {Hq} over {H}, {new}", flush=True)
        assert unit_rows(filled([0] * len(new), new, Hq=Hq, H=H)[2]) == rows


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_bad_block_of_any_head_size(D, bad, sets_of_256):
    """Rows that see none of a block hold, whatever its peaks are; the others' come out as NaN."""
    print(f"case {D} dims, {bad}", flush=True)
    tables, cache, plan, q = filled([0], [200], D=D)
    clean = cache.attend(q, plan)
    codes = 2 * 2 * 64 * D
    for block, part in ((2, 1), (2, 0), (1, 1), (1, 0)):
        kept = cache.data.clone()
        peaks = cache.data[:, codes:codes + 16].clone().view(torch.float32)
        peaks[tables.table[0, block], part] = bad
        cache.data[:, codes:codes + 16] = peaks.view(torch.uint8)
        # as appends write such a block: codes of zero
        cache.data[tables.table[0, block], 64 * D * part:64 * D * (part + 1)] = 128
        out = cache.attend(q, plan)
        assert out[64 * block:, :4].isnan().all()
        # (other rows of a wave may raise their units at other tiles: outputs differ by a rounding)
        for a, b in ((out[:64 * block], clean[:64 * block]), (out[:, 4:], clean[:, 4:])):
            torch.testing.assert_close(a, b, rtol=2. ** -7, atol=2. ** -9)
        cache.data.copy_(kept)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5, 90])
@pytest.mark.parametrize("size,keys_size", [(1e32, 1e-30), (1e32, 1e-16), (3e38, 1e-17), (2. ** -108, 2. ** 108),
                                            (2. ** -120, 2. ** 120), (2. ** -126, 1.)])
def test_queries_of_any_size(D, new, size, keys_size):
    print(f"case {new} new tokens of {D} dims, queries of {size}, keys of {keys_size}", flush=True)
    g = rng(55, D, new)
    n = 320 + new
    k, q = g.standard_normal((n, D)) * keys_size, np.clip(g.standard_normal((new, 4, D)) / 4, -1, 1) * size
    v = g.standard_normal((n, D))
    k, v, q = (torch.from_numpy(a).to(dev(), torch.bfloat16) for a in (k, v, q))
    got, keys, vals, peak = attended(k, v, q)
    if size * keys_size > 2 and keys.any():  # (keys below 2^-60 are zero as held)
        check_winners(got, keys, vals, q)
    else:
        check_sums(got, keys, vals, peak, q)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size,keys_size", [(1e32, 1e-30), (3e38, 1e-17), (2. ** -120, 2. ** 120)])
def test_queries_of_any_size_in_sets_of_256(D, size, keys_size, sets_of_256):
    test_queries_of_any_size(D, 90, size, keys_size)
