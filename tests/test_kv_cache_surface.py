"""Host-side surface of the 8-bit KV cache on the CPU: struct layouts and refusals."""
import ctypes
import os
import subprocess

import pytest
import torch

from stepquant_amd import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"sq_kv_cache": N.KVCache, "sq_kv_tables": N.KVTables, "sq_kv_schedule": N.KVSchedule,
           "sq_kv_plan_args": N.KVPlan, "sq_kv_append_args": N.KVAppend, "sq_kv_attend_args": N.KVAttend}


def test_structs_match_header_layout(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "stepquant_hip.h"', "int main(void) {"]
    for name, cls in STRUCTS.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {field} %zu\\n", offsetof({name}, {field}));' for field, _ in cls._fields_]
    lines += [f'  printf("limits {n} %d\\n", SQ_KV_{n});' for n in ("INT8", "FP8", "MAX_REQUESTS", "MAX_SCHEDULES")]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;\n}"]))
    subprocess.run(["gcc", "-std=c99", "-I", f"{ROOT}/include", "-o", str(exe), str(src)], check=True)
    seen = {}
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, value = line.split()
        seen[name, field] = int(value)
    for name, cls in STRUCTS.items():
        assert seen[name, "size"] == ctypes.sizeof(cls), name
        for field, _ in cls._fields_:
            assert seen[name, field] == getattr(cls, field).offset, (name, field)
    assert (seen["limits", "INT8"], seen["limits", "FP8"]) == (N.KV_INT8, N.KV_FP8)
    assert (seen["limits", "MAX_REQUESTS"], seen["limits", "MAX_SCHEDULES"]) == (N.KV_MAX_REQUESTS, N.KV_MAX_SCHEDULES)


def _cache(**kw):
    a = dict(data=4096, page_bytes=32896, num_pages=4, heads=2, dim=128, page_tokens=64, storage=N.KV_INT8)
    return N.KVCache(**{**a, **kw})


def _tables(**kw):
    a = dict(table=16, lens=16, free_pages=16, counters=16, requests=4, capacity=3, width=2, page_tokens=64)
    return N.KVTables(**{**a, **kw})


def _schedule(**kw):
    a = dict(units=16, merges=16, starts=16, max_units=4 + 2 + 1 + 256, max_merges=256, max_workers=256, max_partials=512,
             q_heads=8, kv_heads=2, rows=16, causal=1, window=0, slots=512, min_tiles=1, merge_rows=16)
    return N.KVSchedule(**{**a, **kw})


def _plan(schedule=None, **kw):
    a = {n: 16 for n in ("rows", "counts", "cu", "slots", "positions", "lens", "granted", "pages", "filled", "tiles",
                         "counters")}
    a.update(tokens=16, batch=2, max_tiles=4, rows_dtype=N.I32, counts_dtype=N.I64, n_schedules=1, max_count=16)
    p = N.KVPlan(**{**a, **kw})
    p.schedules[0] = schedule or _schedule()
    return p


@pytest.mark.parametrize("cache,code", [
    (dict(data=None), -22), (dict(data=4100), -22), (dict(dim=96), -23), (dict(heads=0), -23),
    (dict(page_tokens=48), -23), (dict(page_tokens=320), -23), (dict(storage=2), -24), (dict(num_pages=0), -22),
    (dict(page_bytes=32768), -22), (dict(page_bytes=32888), -22)])
def test_caches_are_checked_before_any_launch(cache, code):
    L = N.lib()
    assert L.sq_kv_decode(_cache(**cache), None, None, 1, None, None, N.F32, None) == code
    assert L.sq_kv_append(_cache(**cache), N.KVAppend(), None) == code
    assert L.sq_kv_attend(_cache(**cache), N.KVAttend(), None) == code


@pytest.mark.parametrize("tables,plan,schedule", [
    (dict(table=None), {}, {}), (dict(requests=0), {}, {}), (dict(capacity=1 << 31), {}, {}), (dict(page_tokens=0), {}, {}),
    ({}, dict(rows=None), {}), ({}, dict(granted=None), {}), ({}, dict(rows_dtype=N.F32), {}), ({}, dict(batch=0), {}),
    ({}, dict(batch=4097), {}), ({}, dict(tokens=-1), {}), ({}, dict(max_tiles=3), {}), ({}, dict(n_schedules=5), {}),
    ({}, dict(max_count=-1), {}), ({}, {}, dict(units=None)), ({}, {}, dict(q_heads=7)), ({}, {}, dict(rows=48)),
    ({}, {}, dict(window=3, causal=0)), ({}, {}, dict(window=-1)), ({}, {}, dict(slots=0)), ({}, {}, dict(max_units=262)),
    ({}, {}, dict(max_merges=6)), ({}, {}, dict(max_partials=511)), ({}, {}, dict(max_workers=255)),
    ({}, {}, dict(slots=4097)), ({}, {}, dict(starts=None)), ({}, {}, dict(cut_tiles=-1)), ({}, {}, dict(min_tiles=0)),
    ({}, {}, dict(merge_rows=15)), ({}, {}, dict(merge_rows=17)), ({}, {}, dict(few_work=-1)),
    ({}, {}, dict(few_work=9, few_min_tiles=1)), ({}, {}, dict(few_work=9, rows=256, few_min_tiles=0)),
    ({}, {}, dict(few_work=9, rows=256, few_min_tiles=1, few_cut_tiles=-1)),
    # (room for sets of 256 rows only)
    ({}, {}, dict(few_work=9, rows=256, few_min_tiles=1, max_units=1 + 3 + 256))])
def test_plans_are_checked_before_any_launch(tables, plan, schedule):
    rc = N.lib().sq_kv_plan(_tables(**tables), _plan(_schedule(**schedule), **plan), None)
    assert rc in (-22, -23) and b"kv " in N.lib().sq_last_error()
    with pytest.raises(ValueError):
        N.check(rc, "plan")


def _attend(schedule=None, **kw):
    a = dict(q=16, out=16, workspace=16, table=16, requests=2, tokens=16, q_stride=1024, q_head_stride=128, width=4,
             dtype=N.BF16, scale=1., schedule=schedule or _schedule())
    return N.KVAttend(**{**a, **kw})


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(q=8), dict(out=24), dict(workspace=None), dict(table=None), dict(width=0), dict(requests=0),
    dict(dtype=N.F32), dict(q_stride=1020), dict(q_stride=-1024), dict(q_head_stride=4), dict(tokens=-1),
    dict(schedule=_schedule(kv_heads=4, q_heads=8, max_units=400)), dict(schedule=_schedule(max_units=1)),
    dict(schedule=_schedule(rows=7))])
def test_attention_is_checked_before_any_launch(kw):
    assert N.lib().sq_kv_attend(_cache(), _attend(**kw), None) in (-22, -23)


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=24), dict(k_stride=12), dict(v_head_stride=-8), dict(dtype=N.F32),
                                dict(max_tiles=-1), dict(tiles=None)])
def test_appends_are_checked_before_any_launch(kw):
    a = dict(k=16, v=16, pages=16, filled=16, tiles=16, tokens=4, k_stride=256, k_head_stride=128, v_stride=256,
             v_head_stride=128, max_tiles=4, dtype=N.F16)
    assert N.lib().sq_kv_append(_cache(), N.KVAppend(**{**a, **kw}), None) == -22


def test_releases_are_checked_before_any_launch():
    L = N.lib()
    assert L.sq_kv_release(_tables(), None, N.I32, 1, None) == -22
    assert L.sq_kv_release(_tables(), 16, N.F32, 1, None) == -22
    assert L.sq_kv_release(_tables(), 16, N.I32, 4097, None) == -22
    assert L.sq_kv_release(_tables(), None, N.I32, 0, None) == 0


def test_python_surface_refuses_without_a_device():
    from stepquant_amd.kernels.kv_cache import BlockTables, KVCache
    with pytest.raises(ValueError, match="GPU"):
        KVCache(4, 2, 128, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        BlockTables(4, 9, 2, device="cpu")
    for kw in (dict(head_dim=96), dict(page_tokens=48), dict(storage="int4"), dict(kv_heads=0), dict(pages=0),
               dict(head_dim=256, page_tokens=192)):
        with pytest.raises(ValueError):
            KVCache(**{**dict(pages=4, kv_heads=2, head_dim=128, device="cpu"), **kw})
    for a in ((0, 4, 1), (1, 1, 1), (1, 4, 0), (1, 1 << 31, 1), (1, 4, 1 << 26)):
        with pytest.raises(ValueError):
            BlockTables(*a, device="cpu")
    with pytest.raises(ValueError):
        BlockTables(1, 4, 1, page_tokens=32, device="cpu")


def _host_objects(cache_pages=6, table_pages=6):
    """A cache and a plan of tables without their device memory, for checks before any launch."""
    from types import SimpleNamespace
    from stepquant_amd.kernels.kv_cache import KVCache
    cpu = torch.device("cpu")
    cache = KVCache.__new__(KVCache)
    cache.pages, cache.heads, cache.dim, cache.page_tokens, cache.device = cache_pages, 2, 128, 64, cpu
    return cache, SimpleNamespace(tokens=3, schedules={}, tables=SimpleNamespace(pages=table_pages, page_tokens=64, device=cpu))


def test_plans_of_more_pages_than_the_cache_has_are_refused():
    """Their tokens would be left out of the cache without an error."""
    cache, plan = _host_objects(cache_pages=5)
    k = torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="6 pages, the cache has 5"):
        cache.append(k, k, plan)
    with pytest.raises(ValueError, match="6 pages, the cache has 5"):
        cache.attend(k, plan)
    cache, plan = _host_objects(cache_pages=7)
    cache._check_plan(plan)


def _host_tables():
    from stepquant_amd.kernels.kv_cache import BlockTables
    tables = BlockTables.__new__(BlockTables)
    tables.device, tables.page_tokens, tables._cus, tables._layouts = torch.device("cpu"), 64, 256, {}
    return tables


@pytest.mark.parametrize("kw", [
    dict(window=1 << 31, heads=(8, 2)), dict(window=(0, 1 << 40), heads=(8, 2)), dict(window=-1, heads=(8, 2)),
    dict(heads=(1 << 33, 1 << 32)), dict(heads=(1 << 30, 1)), dict(tokens=1 << 30), dict(tokens=1 << 70, max_new=1),
    dict(rows=[1 << 70]), dict(new=[1 << 70]), dict(new=[1 << 40], rows=[0])], ids=str)
def test_numbers_past_the_kernels_types_are_refused_by_plan(kw):
    with pytest.raises(ValueError):
        _host_tables().plan(**{**dict(new=[5]), **kw})


@pytest.mark.parametrize("scale", [1e39, -1e39, float("inf"), float("nan"), 3e38])
def test_scales_past_32_bits_are_refused(scale):
    from types import SimpleNamespace
    cache, plan = _host_objects()
    plan.schedules = {0: SimpleNamespace(q_heads=2, kv_heads=2, floats=4, packed=b"")}
    with pytest.raises(ValueError, match="scale"):
        cache.attend(torch.zeros((3, 2, 128), dtype=torch.bfloat16), plan, scale=scale)


def test_pages_are_integers_of_any_width():
    cache, _ = _host_objects()
    for dtype in (torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16):
        assert cache._numbers(torch.tensor([1, 2, 100], dtype=dtype)).tolist() == [1, 2, 100]
    assert cache._numbers([3, -7, 1 << 40]).tolist() == [3, -1, 0x7fffffff]
    with pytest.raises(ValueError):
        cache._numbers([1 << 70])


@pytest.mark.parametrize("new,tokens,heads", [([1], 1, (8, 2)), ([2], 2, None), ([5, 0, 0], 5, (4, 4)), ([90] * 3, 300, (8, 1)),
                                              ([1] * 256, 256, (32, 8))])
def test_parts_of_a_plan_start_on_their_boundaries(new, tokens, heads, monkeypatch):
    calls, tables = [], _host_tables()
    tables._at = 0
    monkeypatch.setattr(N, "kv_entry", lambda name: lambda at, args, stream: calls.append(args) or 0)
    monkeypatch.setattr(N, "raw_stream", lambda: 0)
    plan = tables.plan(new, tokens=tokens, heads=heads, window=(0, 64))
    a = N.KVPlan.from_buffer_copy(calls[0])
    assert a.tiles % 8 == 0 and a.slots % 8 == 0 and a.counters % 8 == 0
    spans = [(a.cu, len(new) + 1), (a.positions, tokens), (a.lens, len(new)), (a.granted, -(-len(new) // 4)),
             (a.pages, a.max_tiles), (a.filled, a.max_tiles), (a.tiles, 2 * a.max_tiles)]
    for s in a.schedules[:a.n_schedules]:
        assert s.units % 32 == 0 and s.merges % 32 == 0
        spans += [(s.units, 8 * s.max_units), (s.merges, 8 * s.max_merges), (s.starts, s.max_workers + 2)]
    # each within the plan's memory, none over another one
    spans = sorted((start, start + 4 * n) for start, n in spans)
    assert all(x[1] <= y[0] for x, y in zip(spans, spans[1:]))
    base = plan._ints.data_ptr()
    assert spans[0][0] >= base and spans[-1][1] <= base + 4 * plan._ints.numel()
    for name, at in (("cu", a.cu), ("positions", a.positions), ("lens", a.lens), ("granted", a.granted), ("pages", a.pages),
                     ("filled", a.filled), ("slots", a.slots), ("counters", a.counters)):
        assert getattr(plan, name).data_ptr() == at, name
    assert plan.granted.numel() == len(new) and plan.pages.numel() == plan.filled.numel() == a.max_tiles


def test_misaligned_outputs_are_refused():
    L = N.lib()
    assert L.sq_kv_plan(_tables(), _plan(tiles=20), None) == -22
    assert L.sq_kv_decode(_cache(), 16, None, 1, 16, 24, N.F32, None) == -22
    assert L.sq_kv_decode(_cache(), 16, None, 1, 20, 16, N.BF16, None) == -22
    assert L.sq_kv_attend(_cache(), _attend(workspace=24), None) == -22
