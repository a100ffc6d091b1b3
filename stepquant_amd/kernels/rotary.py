"""Rotary positions, on one MI355X GPU.

The softmax-attention layers between recurrent ones turn the pairs of their
queries' and keys' first ``dim`` dims by an angle that grows with the token's
position (no reference counterpart: the reference leaves these layers to its host engine).
``Rotary.apply`` turns queries, or keys that are not cached; keys that go into
a cache are turned on the way there (``KVCache.append``, ``LatentCache.append``
with ``rotary``), their queries in the same launch.

Pair i turns by position * f_i, f_i = base ** (-2 i / dim) before any scaling
for contexts longer than those trained on:

* ``linear``: f_i / factor, as if positions were closer together;
* ``base``: base * factor ** (dim / (dim - 2)) in place of the base, so that the
  slowest pair is stretched by ``factor`` and the fastest not at all;
* ``yarn``: pairs that turn more than ``fast`` times in ``original`` positions
  stay, those that turn fewer than ``slow`` times are stretched by ``factor``,
  with a straight ramp over the pairs between; cosines and sines are
  multiplied by 0.1 ln(factor) + 1;
* ``bands``: f_i stays above ``high`` turns in ``original`` positions, is
  stretched below ``low``, and is mixed between by its number of turns.
"""
from __future__ import annotations

import ctypes
import math
from fractions import Fraction

import torch

from .. import _native as N

_TURN = 2 * Fraction("3.1415926535897932384626433832795028841971693993751")
_LAYOUTS = {"half": 0, "interleaved": 1}


def frequencies(dim, *, base=10000., scaling=None, factor=1., original=None, fast=32., slow=1., low=1., high=4.):
    """(f_i [dim / 2] in radians a position, fp64 on the host; the magnitude)."""
    if dim <= 0 or dim % 2 or not base > 1 or not 0 < factor < math.inf:
        raise ValueError("frequencies need an even number of dims, a base above 1 and a positive factor")
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    if scaling == "base":
        if dim < 4:
            raise ValueError("scaling the base needs at least 4 dims")
        return (base * factor ** (dim / (dim - 2))) ** (-i / dim), 1.
    f = float(base) ** (-i / dim)
    if scaling is None:
        return f, 1.
    if scaling == "linear":
        return f / factor, 1.
    if scaling not in ("yarn", "bands"):
        raise ValueError("scaling must be None, linear, base, yarn or bands")
    if original is None or original <= 0:
        raise ValueError(f"{scaling} needs the number of positions trained on")
    if scaling == "yarn":
        if not 0 < slow < fast:
            raise ValueError("yarn needs 0 < slow < fast")
        # the pair that turns so many times in `original` positions
        pair = lambda turns: dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        first, last = max(0, math.floor(pair(fast))), min(dim - 1, math.ceil(pair(slow)))
        ramp = ((i / 2 - first) / max(last - first, .001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, .1 * math.log(factor) + 1 if factor > 1 else 1.
    if not 0 < low < high:
        raise ValueError("bands need 0 < low < high")
    keep = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
    return f * keep + f / factor * (1 - keep), 1.


class Rotary:
    """Turns the first ``dim`` dims of heads (a multiple of 16, at most 1024).

    ``layout`` says which dims are a pair: ``half`` (i, i + dim / 2) or
    ``interleaved`` (2 i, 2 i + 1).  The frequencies are those of
    ``frequencies(dim, ...)``, or ``inverse`` [dim / 2] in radians a position;
    ``magnitude`` multiplies cosines and sines (default: the scaling's).
    """

    def __init__(self, dim, *, layout="half", inverse=None, magnitude=None, device="cuda", **scaling):
        if layout not in _LAYOUTS:
            raise ValueError("layout must be half or interleaved")
        if not 0 < dim <= 1024 or dim % 16:
            raise ValueError("dim must be a multiple of 16, at most 1024")
        if inverse is None:
            inverse, natural = frequencies(dim, **scaling)
        elif scaling:
            raise ValueError("frequencies are given, or made from a base")
        else:
            inverse, natural = torch.as_tensor(inverse).detach().to("cpu", torch.float64), 1.
        if inverse.shape != (dim // 2,) or not bool(torch.isfinite(inverse).all()):
            raise ValueError(f"there are {dim // 2} finite frequencies")
        magnitude = natural if magnitude is None else float(magnitude)
        if not abs(magnitude) < 3e38:
            raise ValueError("magnitude must be finite, below 3e38")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("rotary positions require a GPU (cuda) device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.dim, self.layout, self.magnitude, self.inverse = dim, layout, magnitude, inverse
        # turns a position, a 64-bit fraction of a turn
        turns = [round(Fraction(x) / _TURN % 1 * 2 ** 64) % 2 ** 64 for x in inverse.tolist()]
        turns = [x - (1 << 64) if x >> 63 else x for x in turns]
        self.turns = torch.tensor(turns, dtype=torch.int64, device=self.device)
        self._desc = N.Rotary(turns=self.turns.data_ptr(), dim=dim, interleaved=_LAYOUTS[layout], magnitude=magnitude)
        self._at = ctypes.addressof(self._desc)

    def _rows(self, x, positions, positions_dtype, out):
        """(packed sq_rotary_rows, out, the rows that are read) of ``x`` [tokens, heads, head_dim]."""
        dtype = N.FLOATS.get(x.dtype)
        if dtype is None:
            raise ValueError("rows must be fp32, bf16 or fp16")
        if x.device != self.device:
            raise ValueError("rows must be on the rotary's device")
        tokens, heads, dim = x.shape
        if dim < self.dim or dim % 8 or not 0 < heads <= 65536 or dim > 65536:
            raise ValueError(f"rows must have heads of at least {self.dim} dims, a multiple of 8")
        whole = 3 if dtype == N.F32 else 7
        off = lambda y, s: s[2] != 1 or (s[0] | s[1]) & whole or y.data_ptr() % 16
        strides = x.stride()
        copied = tokens and off(x, strides)
        if out is None:
            out = x.new_empty((tokens, heads, dim)) if copied or not x.is_contiguous() else torch.empty_like(x)
            os, oh = heads * dim, dim
        else:
            if out.dim() == 2 and out.shape == (tokens, heads * dim) and out.stride(1) == 1:
                out = out.unflatten(1, (heads, dim))
            if out.shape != x.shape or out.dtype != x.dtype or out.device != self.device:
                raise ValueError("out must be like the rows")
            os, oh, _ = out.stride()
            if tokens and (off(out, out.stride()) or (tokens > 1 and os == 0) or (heads > 1 and oh == 0)):
                raise ValueError("out must have heads that are contiguous inside, and strides and a start of whole 16 bytes")
        if copied:
            x = x.clone(memory_format=torch.contiguous_format)
            strides = x.stride()
        return N.ROTARY_ROWS.pack(x.data_ptr(), out.data_ptr(), positions, tokens, strides[0], strides[1], os, oh, heads,
                                  dim, dtype, positions_dtype), out, x

    def apply(self, x, positions, *, out=None):
        """``x`` [tokens, heads, head_dim] (fp32, bf16 or fp16) turned to
        ``positions`` [tokens] (int32 or int64), of any size; rows at negative
        positions stay as they are, and so do dims past the first ``dim``.  Angles are off
        by 1.2e-7 rad at most, and by position * 2^-65 of a turn more.

        The result is new and contiguous, or ``out`` (like ``x``, which it may be;
        otherwise they do not overlap).  Heads are contiguous inside; rows and heads
        of ``x`` may have any strides (copied where they are not whole 16 bytes).
        """
        if x.dim() != 3:
            raise ValueError("rows must be [tokens, heads, head_dim]")
        if positions.dtype not in N.INTS or positions.shape != x.shape[:1] or positions.device != self.device:
            raise ValueError("positions must be int32 or int64, one a token, on the rotary's device")
        if not positions.is_contiguous():
            positions = positions.contiguous()
        rows, out, x = self._rows(x, positions.data_ptr(), N.INTS[positions.dtype], out)
        if x.shape[0]:
            rc = N.kv_entry("sq_rotary_apply")(self._at, rows, N.stream_on(self.device))
            if rc:
                N.check(rc, "rotary")
        return out
