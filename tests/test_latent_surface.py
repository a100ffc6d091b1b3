"""Latent attention without a GPU: struct layouts and refusals."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

from stepquant_amd import _native as N
from stepquant_amd.kernels.latent_cache import LatentCache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"sq_latent_cache": N.LatentCache, "sq_latent_append_args": N.LatentAppend,
           "sq_latent_gather_args": N.LatentGather, "sq_latent_attend_args": N.LatentAttend,
           "sq_expanded_attend_args": N.ExpandedAttend}
PACKED = {"sq_latent_append_args": N.LATENT_APPEND, "sq_latent_gather_args": N.LATENT_GATHER,
          "sq_latent_attend_args": N.LATENT_ATTEND, "sq_expanded_attend_args": N.EXPANDED_ATTEND}


def test_structs_match_header_layout(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "stepquant_hip.h"', "int main(void) {"]
    for name, cls in STRUCTS.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {field} %zu\\n", offsetof({name}, {field}));' for field, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;\n}"]))
    subprocess.run(["gcc", "-std=c99", "-I", f"{ROOT}/include", "-o", str(exe), str(src)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, value = line.split()
        cls = STRUCTS[name]
        assert int(value) == (ctypes.sizeof(cls) if field == "size" else getattr(cls, field).offset), (name, field)
    for name, packed in PACKED.items():
        assert packed.size == ctypes.sizeof(STRUCTS[name]), name


@pytest.mark.parametrize("kw", [dict(latent_dim=128), dict(rope_dim=32), dict(page_tokens=48), dict(page_tokens=0),
                                dict(page_tokens=4160), dict(dtype=torch.float32), dict(pages=0), dict(device="cpu")])
def test_caches_refuse_before_the_gpu(kw):
    with pytest.raises(ValueError):
        LatentCache(**{"pages": 4, **kw})


def _cache(**kw):
    return N.LatentCache(**{**dict(data=4096, num_pages=4, latent=512, rope=64, page_tokens=64, dtype=N.BF16), **kw})


def _schedule(**kw):
    a = dict(units=16, merges=16, starts=16, max_units=600, max_merges=256, max_workers=256, max_partials=512, q_heads=8,
             kv_heads=1, rows=16, causal=1, window=0, slots=256, min_tiles=1, merge_rows=16)
    return N.KVSchedule(**{**a, **kw})


BAD_CACHES = [dict(data=None), dict(data=4100), dict(latent=384), dict(rope=32), dict(page_tokens=32),
              dict(page_tokens=8192), dict(dtype=N.F32), dict(num_pages=0)]


@pytest.mark.parametrize("cache", BAD_CACHES)
def test_caches_are_checked_before_any_launch(cache):
    L, c = N.lib(), _cache(**cache)
    assert L.sq_latent_append(c, N.LatentAppend(tokens=1), None, None, None) in (-22, -23, -24)
    assert L.sq_latent_gather(c, N.LatentGather(), None) in (-22, -23, -24)
    assert L.sq_latent_attend(c, N.LatentAttend(tokens=1), None) in (-22, -23, -24)
    assert b"latent cache" in L.sq_last_error()


@pytest.mark.parametrize("kw", [dict(latent=None), dict(rope=24), dict(slots=None), dict(tokens=-1), dict(latent_stride=508),
                                dict(rope_stride=-64), dict(tokens=1 << 28)])
def test_appends_are_checked_before_any_launch(kw):
    a = dict(latent=16, rope=16, slots=16, positions=16, tokens=4, latent_stride=512, rope_stride=64)
    assert N.lib().sq_latent_append(_cache(), N.LatentAppend(**{**a, **kw}), None, None, None) == -22


def test_appends_refuse_rotations_that_do_not_fit():
    L = N.lib()
    rotary = lambda **kw: N.Rotary(**{**dict(turns=16, dim=64, magnitude=1.), **kw})
    rows = lambda **kw: N.RotaryRows(**{**dict(x=16, out=16, positions=16, tokens=4, x_stride=512, x_head_stride=64,
                                               out_stride=512, out_head_stride=64, heads=8, head_dim=64, dtype=N.BF16,
                                               positions_dtype=N.I32), **kw})
    a = dict(latent=16, rope=16, slots=16, positions=16, tokens=4, latent_stride=512, rope_stride=64)
    call = lambda r, q, **kw: L.sq_latent_append(_cache(), N.LatentAppend(**{**a, **kw}), r, q, None)
    assert call(rotary(dim=80), None) == -23 and call(rotary(turns=None), None) == -22
    assert call(rotary(), None, positions=None) == -22 and call(None, rows()) == -22
    assert call(rotary(), rows(dtype=N.F16)) == -22 and call(rotary(), rows(x=None)) == -22
    assert call(rotary(), rows(tokens=1 << 28)) == -22


@pytest.mark.parametrize("kw", [dict(rows=None), dict(lens=None), dict(table=None), dict(starts=None), dict(batch=0),
                                dict(batch=4097), dict(requests=0), dict(width=0), dict(rows_out=-1), dict(latent=None),
                                dict(rope=24), dict(rows_dtype=N.F32), dict(rows_out=1 << 31)])
def test_gathers_are_checked_before_any_launch(kw):
    a = dict(rows=16, lens=16, table=16, latent=16, rope=16, starts=16, requests=4, rows_out=100, batch=3, width=5,
             rows_dtype=N.I32)
    assert N.lib().sq_latent_gather(_cache(), N.LatentGather(**{**a, **kw}), None) == -22


@pytest.mark.parametrize("kw", [dict(q=None), dict(q_rope=8), dict(out=24), dict(workspace=None), dict(workspace=8),
                                dict(table=None), dict(requests=0), dict(width=0), dict(tokens=-1), dict(q_stride=4100),
                                dict(q_head_stride=-512), dict(rope_stride=12), dict(rope_head_stride=-8),
                                dict(scale=math.inf), dict(scale=math.nan)] +
                         [dict(schedule=_schedule(**s)) for s in (
                             dict(kv_heads=2), dict(rows=256), dict(rows=7), dict(window=5), dict(units=None),
                             dict(max_units=3), dict(slots=0), dict(max_partials=511),
                             dict(rows=256, few_work=9, few_min_tiles=1))])
def test_absorbed_attention_is_checked_before_any_launch(kw):
    a = dict(q=16, q_rope=16, out=16, workspace=16, table=16, requests=2, tokens=16, q_stride=4096, q_head_stride=512,
             rope_stride=512, rope_head_stride=64, width=4, scale=1., schedule=_schedule())
    assert N.lib().sq_latent_attend(_cache(), N.LatentAttend(**{**a, **kw}), None) in (-22, -23)


@pytest.mark.parametrize("kw", [dict(q=None), dict(k=8), dict(v=None), dict(rope=24), dict(out=8), dict(cu=None),
                                dict(starts=None), dict(tokens=-1), dict(rows=-1), dict(dim=96), dict(dtype=N.F32),
                                dict(batch=0), dict(batch=4097), dict(q_stride=12), dict(k_head_stride=-128),
                                dict(v_stride=4), dict(rope_stride=-64), dict(scale=math.inf), dict(workspace=None), dict(workspace=8),
                                dict(k_stride=1 << 24)] +
                         [dict(schedule=_schedule(**{**dict(kv_heads=8, rows=256), **s})) for s in (
                             dict(kv_heads=4), dict(rows=16), dict(window=5), dict(units=None), dict(max_units=3))])
def test_expanded_attention_is_checked_before_any_launch(kw):
    a = dict(q=16, k=16, v=16, rope=16, out=16, workspace=16, cu=16, starts=16, tokens=16, rows=16, q_stride=1536, q_head_stride=192,
             k_stride=1024, k_head_stride=128, v_stride=1024, v_head_stride=128, rope_stride=64, batch=2, dim=128,
             dtype=N.F16, scale=1., schedule=_schedule(kv_heads=8, rows=256))
    assert N.lib().sq_expanded_attend(N.ExpandedAttend(**{**a, **kw}), None) in (-22, -23)


def test_attention_of_the_8_bit_cache_refuses_latent_schedules():
    cache = N.KVCache(data=4096, page_bytes=16512, num_pages=4, heads=1, dim=128, page_tokens=64, storage=N.KV_INT8)
    a = N.KVAttend(q=16, out=16, workspace=16, table=16, requests=2, tokens=16, q_stride=1024, q_head_stride=128, width=4,
                   dtype=N.BF16, scale=1., schedule=_schedule(rows=64))
    assert N.lib().sq_kv_attend(cache, a, None) == -23
