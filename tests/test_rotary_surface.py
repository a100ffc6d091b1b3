"""Rotary positions without a GPU: frequencies, struct layouts and refusals."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

from stepquant_amd import _native as N
from stepquant_amd.kernels.rotary import Rotary, frequencies

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"sq_rotary": N.Rotary, "sq_rotary_rows": N.RotaryRows}


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
    assert N.ROTARY_ROWS.size == ctypes.sizeof(N.RotaryRows)


def test_frequencies_by_their_formulas():
    f, m = frequencies(64, base=1e6)
    assert m == 1 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1e6 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-14)
    g, _ = frequencies(64, base=1e6, scaling="linear", factor=4.)
    assert torch.equal(g, f / 4)
    g, _ = frequencies(64, base=1e6, scaling="base", factor=4.)
    assert g[0] == 1 and math.isclose(g[-1], f[-1] / 4, rel_tol=1e-12)
    turns = 8192 * f / (2 * math.pi)
    g, m = frequencies(64, base=1e6, scaling="yarn", factor=8., original=8192)
    assert math.isclose(m, .1 * math.log(8) + 1)
    kept = torch.isclose(g, f, rtol=1e-12)
    # (the borders are whole pairs: the fast one rounded down, the slow one up)
    assert kept[turns > 32 * 1.6].all() and torch.isclose(g, f / 8, rtol=1e-12)[turns < 1 / 1.6].all()
    assert ((g <= f * (1 + 1e-12)) & (g >= f / 8 * (1 - 1e-12))).all() and not kept.all()
    assert frequencies(64, scaling="yarn", factor=1., original=64)[1] == 1.
    g, m = frequencies(64, base=1e6, scaling="bands", factor=8., original=8192)
    for i, n in enumerate(turns.tolist()):
        keep = min(1, max(0, (n - 1) / 3))
        assert math.isclose(g[i], f[i] * keep + f[i] / 8 * (1 - keep), rel_tol=1e-12)
    assert m == 1


@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=7), dict(dim=8, base=1.), dict(dim=8, factor=0.),
                                dict(dim=8, scaling="other"), dict(dim=8, scaling="yarn", factor=2.),
                                dict(dim=8, scaling="bands", original=0), dict(dim=2, scaling="base", factor=2.),
                                dict(dim=8, scaling="yarn", original=64, fast=1., slow=2.),
                                dict(dim=8, scaling="bands", original=64, low=0.), dict(dim=8, factor=math.inf)])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        frequencies(**kw)


@pytest.mark.parametrize("kw", [dict(dim=24), dict(dim=0), dict(dim=1040), dict(dim=16, layout="quarters"),
                                dict(dim=16, inverse=[0.] * 7), dict(dim=16, inverse=[math.inf] + [0.] * 7),
                                dict(dim=16, inverse=[0.] * 8, base=100.), dict(dim=16, magnitude=math.nan),
                                dict(dim=16, device="cpu")])
def test_rotaries_refuse_before_the_gpu(kw):
    with pytest.raises(ValueError):
        Rotary(**kw)


def _rotary(**kw):
    return N.Rotary(**{**dict(turns=16, dim=64, interleaved=0, magnitude=1.), **kw})


def _rows(**kw):
    return N.RotaryRows(**{**dict(x=16, out=16, positions=16, tokens=3, x_stride=512, x_head_stride=128, out_stride=512,
                                  out_head_stride=128, heads=4, head_dim=128, dtype=N.BF16, positions_dtype=N.I32), **kw})


BAD_ROTARY = [dict(turns=None), dict(turns=12), dict(dim=8), dict(dim=0), dict(dim=1040), dict(magnitude=math.inf),
              dict(magnitude=math.nan)]
BAD_ROWS = [dict(x=None), dict(out=None), dict(positions=None), dict(tokens=-1), dict(x=24), dict(out=24), dict(heads=0),
            dict(head_dim=56), dict(head_dim=132), dict(dtype=N.I32), dict(positions_dtype=N.F32), dict(x_stride=508),
            dict(x_head_stride=-128), dict(out_stride=-512), dict(out_head_stride=12), dict(x=16, out=16, out_stride=1024)]


@pytest.mark.parametrize("rotary,rows", [(r, {}) for r in BAD_ROTARY] + [({}, r) for r in BAD_ROWS])
def test_calls_are_checked_before_any_launch(rotary, rows):
    L = N.lib()
    assert L.sq_rotary_apply(_rotary(**rotary), _rows(**rows), None) in (-22, -23)
    assert b"rotary" in L.sq_last_error()
    cache = N.KVCache(data=4096, page_bytes=32896, num_pages=4, heads=2, dim=128, page_tokens=64, storage=N.KV_INT8)
    a = N.KVAppend(k=16, v=16, pages=16, filled=16, tiles=16, tokens=4, k_stride=256, k_head_stride=128, v_stride=256,
                   v_head_stride=128, max_tiles=4, dtype=N.F16)
    assert L.sq_kv_append_rotary(cache, a, 16, _rotary(**rotary), _rows(**rows), None) in (-22, -23)


def test_launches_on_another_device_are_refused(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 40 + device, raising=False)
    assert N.stream_on(torch.device("cuda", 1)) == 41
    with pytest.raises(ValueError, match="cuda:0.*cuda:1"):
        N.stream_on(torch.device("cuda", 0))


def test_appends_refuse_rotations_that_do_not_fit():
    L = N.lib()
    cache = N.KVCache(data=4096, page_bytes=16512, num_pages=4, heads=2, dim=64, page_tokens=64, storage=N.KV_INT8)
    a = N.KVAppend(k=16, v=16, pages=16, filled=16, tiles=16, tokens=4, k_stride=128, k_head_stride=64, v_stride=128,
                   v_head_stride=64, max_tiles=4, dtype=N.F16)
    assert L.sq_kv_append_rotary(cache, a, 16, _rotary(dim=80), None, None) == -23
    assert L.sq_kv_append_rotary(cache, a, None, _rotary(), None, None) == -22
    assert L.sq_kv_append_rotary(cache, a, 16, None, None, None) == -22
    assert L.sq_kv_append_rotary(cache, a, 16, _rotary(), _rows(tokens=1 << 27, head_dim=64), None) == -22
    a.k = None
    assert L.sq_kv_append_rotary(cache, a, 16, _rotary(), None, None) == -22
