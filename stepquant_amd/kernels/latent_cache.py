"""Latent attention on one MI355X GPU: keys and values of all heads from one
shared vector a token.

The softmax-attention layers of models that compress their keys and values (no
reference counterpart: the reference leaves them to its host engine).  A token
holds its latent c (256 or 512 dims) and a rope key r (64 dims) that all
heads share; head h's keys are [K_h c, r] and its values V_h c, with projections
K_h [dim, latent] and V_h [dim, latent] of the model.  The pages, requests and plans are those of
``BlockTables``.  Two forms of the same attention:

* absorbed (``LatentCache.attend``), for single tokens and drafts: with queries
  K_h^T q the latents themselves are the keys, and the values of all heads; each
  is read once.  The model applies V_h to the outputs.
* expanded (``LatentCache.gather`` and ``expanded_attention``), for prompts: the
  model expands the gathered latents into keys and values of every head by one
  matrix product each, a third of the absorbed form's arithmetic a pair.

    plan = tables.plan(new, rows, tokens=T, max_new=1, absorbed=32)
    q_rope = cache.append(latent, rope, plan, rotary=rotary, q=q_rope)
    y = cache.attend(q_latent, q_rope, plan, scale=192 ** -.5)   # [T, 32, latent]
    tables.commit(plan)

All calls are asynchronous on the current stream and can be captured in HIP
graphs (``plan`` and ``gather`` with sizes given).
"""
from __future__ import annotations

import ctypes

import torch

from .. import _native as N
from .kv_cache import TILE, _device
from .pool import PackedStatePool

_HALVES = {torch.bfloat16: N.BF16, torch.float16: N.F16}
ROPE = 64


def _whole(x):
    """``x`` with a last dim that is contiguous and other strides and a start of whole 16 bytes (a copy where it has not)."""
    s = x.stride()
    if s[-1] != 1 or (s[0] | s[-2]) & 7 or x.data_ptr() % 16:  # (of two or three dims)
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _near(x):
    """The same, with rows fewer than 2^24 elements apart."""
    return _whole(x) if x.stride(0) < 1 << 24 else x.clone(memory_format=torch.contiguous_format)


def _scale(scale):
    scale = float(scale)
    if not abs(scale) < 2e38:  # (kernels multiply it by log2 e)
        raise ValueError("scale must be finite, below 2e38")
    return scale


def _range(x):
    at = x.data_ptr()
    return at, at + (1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride()))) * x.element_size() if x.numel() else at


def _output(out, shape, like, *operands, in_place=None):
    """``out``, or a new tensor; it lies over no operand, but may be ``in_place``."""
    if out is None:
        return torch.empty_like(like) if like.shape == shape and like.is_contiguous() else like.new_empty(shape)
    if out.shape != shape or out.dtype != like.dtype or out.device != like.device or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise ValueError(f"out must be contiguous {list(shape)} of the queries' type")
    if in_place is not None and (in_place.data_ptr() != out.data_ptr() or not in_place.is_contiguous()):
        operands += in_place,
    start, end = _range(out)
    for x in operands:
        first, last = _range(x)
        if first < last and first < end and start < last:
            raise ValueError("out overlaps an operand")
    return out


class LatentCache:
    """One attention layer's latents and rope keys in ``pages`` pages of ``page_tokens`` tokens.

    ``data`` [pages, page_tokens, latent_dim + 64] of ``dtype`` (bf16 or fp16):
    a token's latent and its rope key.  ``latent_dim`` is 256 or 512 and
    ``page_tokens`` a multiple of 64, at most 4096.  A plan's block tables have
    the same ``page_tokens`` and no more pages.
    """

    def __init__(self, pages, latent_dim=512, rope_dim=ROPE, *, page_tokens=64, dtype=torch.bfloat16, device="cuda"):
        if latent_dim not in (256, 512) or rope_dim != ROPE:
            raise ValueError("latent_dim must be 256 or 512, rope_dim 64")
        if not 0 < page_tokens <= 4096 or page_tokens % TILE:
            raise ValueError(f"page_tokens must be a positive multiple of {TILE}, at most 4096")
        if dtype not in _HALVES:
            raise ValueError("latents are held in bf16 or fp16")
        if not 0 < pages <= 0x7fffffff:
            raise ValueError("pages must be a positive 32-bit number")
        self.device = _device(device)
        self.pages, self.latent_dim, self.rope_dim = pages, latent_dim, rope_dim
        self.page_tokens, self.dtype = page_tokens, dtype
        self.data = torch.zeros((pages, page_tokens, latent_dim + rope_dim), dtype=dtype, device=self.device)
        self._latent = N.LatentCache(data=self.data.data_ptr(), num_pages=pages, latent=latent_dim, rope=rope_dim,
                                     page_tokens=page_tokens, dtype=_HALVES[dtype])
        self._at = ctypes.addressof(self._latent)
        self._words = torch.empty(0, dtype=torch.float32, device=self.device)  # workspaces are made like it
        # page copies read only these
        self.page_bytes = 2 * page_tokens * (latent_dim + rope_dim)
        self._desc = N.Pool(data=self.data.data_ptr(), page_bytes=self.page_bytes, num_slots=pages)

    @property
    def nbytes(self):
        return self.data.numel() * 2

    def wait(self):
        """Writes are made on the caller's stream: nothing to wait for."""

    def copy(self, source, destination):
        """Copies whole pages (a request that starts as another one's copy)."""
        PackedStatePool.copy(self, source, destination)

    def _check_plan(self, plan):
        tables = plan.tables
        if tables.page_tokens != self.page_tokens or tables.device != self.device:
            raise ValueError("the plan's block tables have other pages than the cache")
        if tables.pages > self.pages:
            raise ValueError(f"the plan's block tables give out {tables.pages} pages, the cache has {self.pages}")

    def _like(self, x, shape, what):
        if x.dtype != self.dtype or x.device != self.device:
            raise ValueError(f"{what} must have the cache's type and device")
        if x.shape != shape:
            raise ValueError(f"{what} must be {list(shape)}")
        return _whole(x)

    def append(self, latent, rope, plan, *, rotary=None, q=None, out=None):
        """Writes the plan's new latents [tokens, latent_dim] and rope keys
        [tokens, 64] (the cache's type) to their pages.

        ``rotary`` (a ``Rotary`` of at most 64 dims) turns the rope keys to the
        plan's positions on the way; then ``q``, rows [tokens, heads, dim] such as the same
        tokens' rope queries, are turned in the same launch and returned, in ``out``
        where it is given (which may be ``q``, and lies over no latent or rope key: they
        are read meanwhile).  Rows without a slot come back as they are.
        """
        self._check_plan(plan)
        latent = self._like(latent, (plan.tokens, self.latent_dim), "latents")
        rope = self._like(rope, (plan.tokens, self.rope_dim), "rope keys")
        if rotary is None:
            if q is not None or out is not None:
                raise ValueError("queries are turned by a rotary")
        elif rotary.device != self.device or rotary.dim > self.rope_dim:
            raise ValueError("the rotary is on another device, or turns more dims than a rope key has")
        rows = None
        if q is not None:
            if q.dim() != 3 or q.shape[0] != plan.tokens or q.dtype != self.dtype:
                raise ValueError(f"queries must be [{plan.tokens}, heads, dim], the plan's tokens, of the cache's type")
            rows, out, q = rotary._rows(q, plan._positions, N.I32, out)
        elif out is not None:
            raise ValueError("out is where queries go")
        if not plan.tokens:
            return out
        args = N.LATENT_APPEND.pack(latent.data_ptr(), rope.data_ptr(), plan._slots, plan._positions, plan.tokens,
                                    latent.stride(0), rope.stride(0))
        rc = N.kv_entry("sq_latent_append")(self._at, args, None if rotary is None else rotary._at, rows, N.stream_on(self.device))
        if rc:
            N.check(rc, "latent append")
        return out

    def gather(self, plan, tokens=None):
        """All that the plan's requests hold once its tokens are appended, request
        after request: latents [tokens, latent_dim], rope keys [tokens, 64] and
        ``starts`` [B + 1], the first row of each request.

        ``tokens`` is the number of rows to make room for; rows past the last are
        zero, and starts end at ``tokens``.  Without it the plan's lengths are
        read back.
        """
        self._check_plan(plan)
        if tokens is None:
            tokens = int(plan.lens.sum())
        tokens = int(tokens)
        if not 0 <= tokens <= 0x7fffffff:
            raise ValueError("tokens must be a non-negative 32-bit number")
        latent = self.data.new_empty((tokens, self.latent_dim))
        rope = self.data.new_empty((tokens, self.rope_dim))
        starts = plan._ints.new_empty((plan.batch + 1,))
        t = plan.tables
        args = N.LATENT_GATHER.pack(plan.rows.data_ptr(), plan._lens, t.table.data_ptr(), latent.data_ptr(),
                                    rope.data_ptr(), starts.data_ptr(), t.requests, tokens, plan.batch, t.max_blocks,
                                    N.INTS[plan.rows.dtype], 0)
        rc = N.kv_entry("sq_latent_gather")(self._at, args, N.stream_on(self.device))
        if rc:
            N.check(rc, "latent gather")
        return latent, rope, starts

    def attend(self, q, q_rope, plan, *, scale, out=None):
        """Absorbed attention of the plan's new tokens over all that their requests hold.

        ``q`` [tokens, heads, latent_dim] are the queries times the keys' projection,
        ``q_rope`` [tokens, heads, 64] their rope part, of the cache's type, after
        ``append`` of the same plan (made with ``absorbed=heads``); the result is
        like ``q``, each row the weighted mean of the latents that its token sees (as
        the plan's ``causal`` says), zero where it sees none.  ``scale`` is that of
        the heads' own dims, which the latents do not tell.  ``out`` may be ``q``.

        What a token does not see does not reach it.  One that sees a latent that is
        infinite or NaN has NaN in that dim, or, near where some token's sight ends, in all.
        Scores are held in 32 bits: a head with one above their range, or with none but
        -infinity, is NaN.
        """
        self._check_plan(plan)
        s = plan.latent.get("absorbed")
        if s is None:
            if plan.tokens:
                raise ValueError("the plan was made without absorbed heads")
            if q.dim() != 3 or q.shape[0] or q.shape[2] != self.latent_dim:
                raise ValueError(f"queries must be [0, heads, {self.latent_dim}]")
            return _output(out, q.shape, q)
        q = self._like(q, (plan.tokens, s.q_heads, self.latent_dim), "queries")
        q_rope = self._like(q_rope, (plan.tokens, s.q_heads, self.rope_dim), "rope queries")
        scale, out = _scale(scale), _output(out, q.shape, q, q_rope, in_place=q)
        ws = self._words.new_empty((s.floats * (self.latent_dim + 2),))
        t = plan.tables
        args = N.LATENT_ATTEND.pack(q.data_ptr(), q_rope.data_ptr(), out.data_ptr(), ws.data_ptr(), t.table.data_ptr(),
                                    t.requests, plan.tokens, *q.stride()[:2], *q_rope.stride()[:2], t.max_blocks, scale,
                                    s.packed)
        rc = N.kv_entry("sq_latent_attend")(self._at, args, N.stream_on(self.device))
        if rc:
            N.check(rc, "latent attend")
        return out


def expanded_attention(q, k, v, rope, plan, starts=None, *, scale=None, out=None):
    """Expanded attention of the plan's new tokens over keys and values of every head.

    ``q`` [tokens, heads, dim + 64] (the rope part last), ``k`` and ``v``
    [rows, heads, dim] with ``dim`` 64 or 128, ``rope`` [rows, 64], one type
    (bf16 or fp16); the plan was made with ``expanded=heads``.  ``starts`` [B + 1]
    (int32) says where each request's rows begin, as ``LatentCache.gather``
    returns it; default: the plan's ``cu``, keys and values of the new tokens alone, for
    requests that held none before (others are NaN: they would see keys that are not there).
    Each token sees its request's rows up to its own position (all of them in a
    plan that is not ``causal``); the result is [tokens, heads, dim], zero where a
    token sees none.  ``scale`` defaults to ``(dim + 64) ** -0.5``.  ``out`` lies over no operand.

    What a token does not see does not reach it.  One that sees a value that is
    infinite or NaN has NaN in that dim, or, within 64 keys of where some token's
    sight ends, in all.  Scores are held in 32 bits: a head with one above their range,
    or with none but -infinity, is NaN.
    """
    tables = plan.tables
    if v.dim() != 3 or v.shape[2] not in (64, 128) or v.dtype not in _HALVES or v.device != tables.device:
        raise ValueError("values must be [rows, heads, 64 or 128], bf16 or fp16, on the plan's device")
    rows, heads, dim = v.shape
    for x, shape, what in ((q, (plan.tokens, heads, dim + ROPE), "queries"), (k, v.shape, "keys"),
                           (rope, (rows, ROPE), "rope keys")):
        if x.dtype != v.dtype or x.device != v.device or x.shape != shape:
            raise ValueError(f"{what} must be {list(shape)}, of the values' type and device")
    if starts is None:
        starts_at = plan._cu
    elif starts.dtype != torch.int32 or starts.shape != (plan.batch + 1,) or starts.device != v.device \
            or not starts.is_contiguous():
        raise ValueError("starts must be contiguous int32, one more than requests")
    else:
        starts_at = starts.data_ptr()
    scale = _scale((dim + ROPE) ** -.5 if scale is None else scale)
    out = _output(out, (plan.tokens, heads, dim), q, q, k, v, rope)
    s = plan.latent.get("expanded")
    if s is None or s.q_heads != heads:
        if plan.tokens:
            raise ValueError(f"the plan was made without expanded={heads}")
        return out
    if not rows:  # (none is read)
        k = v = v.new_empty((1, heads, dim))
        rope = rope.new_empty((1, ROPE))
    q, k, v, rope = _whole(q), _near(k), _near(v), _near(rope)
    ws = torch.empty(s.floats * (dim + 2), dtype=torch.float32, device=v.device)
    args = N.EXPANDED_ATTEND.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), rope.data_ptr(), out.data_ptr(), ws.data_ptr(), plan._cu,
                                  starts_at, plan.tokens, rows, *q.stride()[:2], *k.stride()[:2], *v.stride()[:2],
                                  rope.stride(0), plan.batch, dim, _HALVES[v.dtype], scale, s.packed)
    rc = N.kv_entry("sq_expanded_attend")(args, N.stream_on(v.device))
    if rc:
        N.check(rc, "expanded attention")
    return out
