"""Attention over keys and values held in 8 bits in pages, on one MI355X GPU.

The softmax-attention layers between the recurrent layers that the state
pools serve, where keys and values have one head size of 64, 128 or 256 (no
reference counterpart: the reference leaves them to its host engine).  Three pieces, used in turn by one model step:

* ``BlockTables`` gives requests their pages.  ``plan`` turns the number of
  new tokens of each request into block tables, slot maps and the attention
  layers' split of work, on the GPU, without reading anything back;
  ``commit`` takes the plan over; ``release`` returns requests' pages.
* ``KVCache`` holds one layer's keys and values: ``append`` quantises the
  plan's new tokens into their pages, ``decode`` gives pages back dense.
* ``KVCache.attend`` is attention of the plan's new tokens over everything
  that their requests hold.

A block of ``page_tokens`` tokens shares one peak per KV head for its keys and
one for its values.  ``int8`` codes stand for code * peak / 127, ``fp8`` codes
(e4m3) for code * peak / 448; a token that raises the peak of a block that
already holds tokens brings their codes to it (one more rounding).  A block
that is given an infinity or a NaN reads as NaN.

All calls are asynchronous on the current stream and can be captured in HIP
graphs (``plan`` with device tensors, ``tokens`` and ``max_new``).
"""
from __future__ import annotations

import ctypes
from operator import index

import torch

from .. import _native as N
from .pool import PackedStatePool

_STORAGE = {"int8": N.KV_INT8, "fp8": N.KV_FP8}
_HALVES = {torch.bfloat16: N.BF16, torch.float16: N.F16}
TILE = 64  # keys of one attention tile


def _device(device):
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("the KV cache requires a GPU (cuda) device")
    return torch.device("cuda", torch.cuda.current_device()) if device.index is None else device


class KVPlan:
    """New tokens of a batch of requests, as ``BlockTables.plan`` lays them out.

    ``cu`` [B + 1] first packed row of each request; ``slots`` [tokens]
    page * page_tokens + offset (-1: none); ``positions`` [tokens] position in
    the request (-1: none); ``lens`` [B] tokens held afterwards; ``granted``
    [B] whether the request's tokens found room; ``pages`` the pages that new
    tokens fall into (0 past the last) and ``filled`` the tokens that each then
    holds; ``counters`` the tables' counters afterwards.
    """

    __slots__ = ("tables", "rows", "counts", "tokens", "batch", "max_tiles", "schedules", "_args", "_ints", "_longs",
                 "_sizes", "_append", "_views")

    def _view(self, i):
        # views are made when they are asked for: a step's kernels need none
        views = self._views
        if views is None:
            counters, slots = self._longs.split((2, self.tokens))
            views = self._ints.split_with_sizes(self._sizes)
            self._views = views = (views[1], slots, *views[2:4], views[4].view(torch.bool)[:self.batch], *views[5:7],
                                   counters)
        return views[i]

    cu = property(lambda self: self._view(0))
    slots = property(lambda self: self._view(1))
    positions = property(lambda self: self._view(2))
    lens = property(lambda self: self._view(3))
    granted = property(lambda self: self._view(4))
    pages = property(lambda self: self._view(5))
    filled = property(lambda self: self._view(6))
    counters = property(lambda self: self._view(7))

    def record_stream(self, stream):
        """The plan's memory is also used on ``stream`` (not only on the one it was made on)."""
        for x in (self._ints, self._longs, self.rows, self.counts):
            x.record_stream(stream)


class _Schedule:
    """One kind of attention layer's split of a plan (``sq_kv_schedule``)."""

    __slots__ = ("packed", "q_heads", "kv_heads", "floats")


class BlockTables:
    """Pages of up to ``requests`` requests of up to ``max_blocks`` blocks.

    ``table`` [requests, max_blocks], ``lens`` [requests], ``free`` (a ring of
    page numbers) and ``counters`` (pages taken from it and given to it so far)
    live on the GPU.  Page 0 is the padding page and is never given out.
    """

    def __init__(self, requests, pages, max_blocks, *, page_tokens=64, device="cuda"):
        if requests <= 0 or max_blocks <= 0 or pages < 2:
            raise ValueError("block tables need requests, blocks and at least 2 pages")
        if page_tokens <= 0 or page_tokens % TILE:
            raise ValueError(f"page_tokens must be a positive multiple of {TILE}")
        if max(requests, pages) > 0x7fffffff or max_blocks * page_tokens > 0x7fffffff:
            raise ValueError("requests, pages and tokens of a request must be 32-bit numbers")
        self.device = _device(device)
        self.requests, self.pages, self.max_blocks, self.page_tokens = requests, pages, max_blocks, page_tokens
        dev = self.device
        self.table = torch.zeros((requests, max_blocks), dtype=torch.int32, device=dev)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.free = torch.arange(1, pages, dtype=torch.int32, device=dev)
        self.counters = torch.tensor([0, pages - 1], dtype=torch.int64, device=dev)
        self._desc = N.KVTables(table=self.table.data_ptr(), lens=self.lens.data_ptr(),
                                free_pages=self.free.data_ptr(), counters=self.counters.data_ptr(),
                                requests=requests, capacity=pages - 1, width=max_blocks, page_tokens=page_tokens)
        self._at = ctypes.addressof(self._desc)
        self._layouts = {}
        self._cus = torch.cuda.get_device_properties(dev).multi_processor_count

    def _index(self, x, what):
        if not isinstance(x, torch.Tensor):
            x = torch.as_tensor(x)
            x = x if x.numel() else x.long()
        if x.dim() != 1 or x.dtype not in N.INTS:
            raise ValueError(f"{what} must be one-dimensional int32 or int64")
        return x if x.device == self.device and x.is_contiguous() else x.to(self.device).contiguous()

    def plan(self, new, rows=None, *, tokens=None, max_new=None, heads=None, causal=True, window=0):
        """Room for ``new[b]`` tokens of the request in row ``rows[b]`` (default: row b).

        ``new`` and ``rows`` are lists or int32/int64 tensors, ``rows``
        distinct.  ``tokens`` is the number of packed rows (at least
        ``sum(new)``; rows past it are padding) and ``max_new`` the most new
        tokens of a request (requests past either are refused); both default to
        those of ``new`` where that is on the host and are required where it is
        on the GPU.  ``heads``
        (query heads, KV heads) also lays out the work of ``attend``: with
        ``causal`` each token sees its request's tokens up to itself, else all
        of them; ``window`` > 0 leaves it the last ``window`` of those.  A
        tuple of windows lays out several kinds of layers.

        Requests that find no room (``granted`` 0) keep their length; their
        tokens have no slot and their attention is zero.
        """
        if isinstance(new, torch.Tensor) and new.is_cuda:
            if tokens is None or max_new is None:
                raise ValueError("counts on the GPU need tokens and max_new")
        else:
            if isinstance(new, torch.Tensor):
                if new.dim() != 1 or new.dtype not in N.INTS:
                    raise ValueError("new must be one-dimensional int32 or int64")
                new = new.tolist()
            host = [index(x) for x in new]
            if any(x < 0 for x in host):
                raise ValueError("new tokens cannot be negative")
            tokens = sum(host) if tokens is None else tokens
            max_new = max(host, default=0) if max_new is None else max_new
            new = torch.tensor([min(x, 0x7fffffff) for x in host], dtype=torch.int64)
        counts = self._index(new, "new")
        batch = counts.numel()
        if rows is None:
            rows = torch.arange(batch, device=self.device)
        rows = self._index(rows, "rows")
        if rows.numel() != batch:
            raise ValueError("new and rows must have the same length")
        if not 0 < batch <= N.KV_MAX_REQUESTS:
            raise ValueError(f"a plan takes 1 to {N.KV_MAX_REQUESTS} requests")
        tokens, max_new = int(tokens), min(int(max_new), 0x7fffffff)
        if tokens < 0 or max_new < 0:
            raise ValueError("tokens and max_new cannot be negative")
        if tokens > 0x3fffffff:
            raise ValueError("a plan takes fewer than 2^30 tokens")
        windows = tuple(window) if isinstance(window, (tuple, list)) else (window,)
        if len(windows) > N.KV_MAX_SCHEDULES or len(set(windows)) < len(windows):
            raise ValueError(f"a plan takes at most {N.KV_MAX_SCHEDULES} windows, each once")
        if any(windows) and not causal:
            raise ValueError("a window needs causal attention")
        heads = None if heads is None else tuple(heads)
        key = (batch, tokens, max_new, heads, causal, windows)
        layout = self._layouts.get(key)
        if layout is None:
            if len(self._layouts) >= 64:
                self._layouts.clear()
            layout = self._layouts[key] = self._layout(batch, tokens, max_new, heads, bool(causal), windows)
        sizes, total, offsets, most, schedules = layout
        p = KVPlan()
        p.tables, p.rows, p.counts, p.tokens, p.batch, p.max_tiles, p._views = self, rows, counts, tokens, batch, most, None
        p._sizes = sizes
        p._ints = ints = torch.empty(total, dtype=torch.int32, device=self.device)
        p._longs = longs = torch.empty(2 + tokens, dtype=torch.int64, device=self.device)
        base, counters = ints.data_ptr(), longs.data_ptr()
        tiles, cu, positions, lens, granted, pages, filled = (base + x for x in offsets)
        p.schedules, packed = {}, b""
        for w, q_heads, kv_heads, floats, units, merges, starts, numbers in schedules:
            s = _Schedule()
            s.packed = N.KV_SCHEDULE.pack(base + units, base + merges, base + starts, *numbers)
            s.q_heads, s.kv_heads, s.floats = q_heads, kv_heads, floats
            p.schedules[w] = s
            packed += s.packed
        p._append = (pages, filled, tiles)
        p._args = args = N.KV_PLAN.pack(
            rows.data_ptr(), counts.data_ptr(), cu, counters + 16, positions, lens, granted, pages, filled, tiles, counters,
            tokens, batch, most, N.INTS[rows.dtype], N.INTS[counts.dtype], len(schedules), max_new,
            packed.ljust(N.KV_MAX_SCHEDULES * N.KV_SCHEDULE.size, b"\0"))
        rc = N.kv_entry("sq_kv_plan")(self._at, args, N.raw_stream())
        if rc:
            N.check(rc, "kv plan")
        return p

    # Rows of a set.  16: one workgroup.  32: two that read the same keys side by
    # side (32 rows of 8 heads of 128 dims, 160 requests of 4096 tokens: 477 us in
    # sets of 16, 318 so).  256: tiles that are converted once for 8 waves; that
    # pays past 64 rows (64 rows of 4 requests of 4000: 39.8 us, 30.1 in sets of 32;
    # of 160 requests 638 and 590; 96 rows of 160 requests 653 and 851).
    # Slots, the workgroups that run at a time: two on a CU up to 32 rows (three
    # would wait for one another: 64 requests of up to 8192, 116 us with two, 130
    # with one, 131 with three), one of 256 rows.
    # Least 64-key tiles of a workgroup where a set of rows is cut: two of 256 dims
    # are a step for each of four waves (1 request of 1000 tokens 13.3 us with 2,
    # 14.1 with 4, 16.7 with 8); other dims are alike from 1 to 8.
    min_tiles = {16: 2, 32: 2, 256: 4}
    # What partial results cost, in tiles: 64 requests of up to 8192 take 116 us
    # cut, 131 uncut; 160 of up to 4096 and 32 rows 223 us with 4 here, 210 with 8 to
    # 16, but 64 tokens over 1000 (256 dims) 36 us with 16, 28 with 12; prompts of up
    # to 2048 and 7 rows a token 77 us with 16, 58 with 24; a prompt of 8192 tokens
    # 543 us uncut, 709 cut (with 0 here).
    cut_tiles = {16: 4, 32: 12, 256: 24}
    # A tile is 2 us of a set of 256, and its start and end 10 more; a short prompt
    # ends sooner in sets of 32, all at a time (128 tokens of 32 heads over 500: 30 us
    # in sets of 256, 21 so; 64 of 256 dims over 1000: 94 and 28; but 64 over 8000 of
    # 128 dims 34 and 45).  So for up to `few_rows` query rows of all heads the plan
    # kernel, which knows the lengths, decides: sets of 32 where rows times the tiles
    # that they see are at most `few_work`.  It is one number for every head size,
    # which a plan is not told, and for sets of 256 cut or not, so near it the other
    # side can be ahead.  At 2^17.3, sets of 32 and of 256: 32 heads of 64 dims, 64
    # tokens 23.5 and 19.9 us, 256 tokens 20.4 and 40.8; of 128 dims 33.5 and 25.9,
    # 29.3 and 47.6; 16 heads of 256 dims 52 and 74, 56 and 76.  At 2^18: 28 and 24, 27
    # and 31; 41 and 33, 39 and 37; 67 and 65, 71 and 81.
    few_rows, few_work = 1 << 14, 3 << 16

    def _layout(self, batch, tokens, max_new, heads, causal, windows):
        """Where a plan's parts lie in its 32-bit words: (sizes of the parts, all
        words, byte offsets of the first seven, page entries, per window what
        ``sq_kv_schedule`` holds)."""
        most = min(tokens, tokens // self.page_tokens + 2 * batch)
        # (page entries' pairs of words first, on a boundary of theirs)
        sizes = [2 * most, batch + 1, tokens, batch, -(-batch // 4), most, most]
        schedules = []
        if heads is not None:
            q_heads, kv_heads = (int(x) for x in heads)
            if q_heads <= 0 or kv_heads <= 0 or q_heads % kv_heads:
                raise ValueError("query heads must be a positive multiple of KV heads")
            group = q_heads // kv_heads
            if q_heads > 0x7fffffff or tokens * group > 0x3fffffff:
                raise ValueError("heads, or tokens times the heads of a group, too many")
            if not all(0 <= int(w) <= 0x7fffffff for w in windows):
                raise ValueError("a window is a non-negative 32-bit number")
            rows = max_new * group
            rows = 16 if rows <= 16 else 32 if rows <= 64 else 256
            slots = 2 * self._cus if rows == 16 else self._cus
            few = rows == 256 and tokens * q_heads <= self.few_rows
            sets, cuts = -(-tokens * group // (32 if few else rows)) + batch + 1, max(1, slots // kv_heads)
            workers, joins = max(sets, cuts), min(sets, cuts)
            sizes.append(-sum(sizes) % 8)  # units and merges start on a boundary of their 32 bytes
            for w in windows if tokens else ():
                units = 4 * sum(sizes)
                merges = units + 32 * (sets + cuts)
                numbers = (sets + cuts, joins, workers, 2 * cuts, q_heads, kv_heads, rows, causal, int(w), slots,
                           self.min_tiles[rows], self.cut_tiles[rows], max(1, min(rows, max_new * group)),
                           self.few_work if few else 0, self.min_tiles[32], self.cut_tiles[32])
                schedules.append((int(w), q_heads, kv_heads, 2 * cuts * kv_heads * rows, units, merges,
                                  merges + 32 * joins, numbers))
                sizes.append(8 * (sets + cuts + joins) + (workers + 9) // 8 * 8)
        offsets = [4 * sum(sizes[:i]) for i in range(7)]
        return sizes, sum(sizes), offsets, most, schedules

    def commit(self, plan):
        """Takes a plan's lengths and pages over; plans made before it are void.

        The plan's ``rows`` are read again: a tensor of the caller's stays as it
        was for ``plan`` until then.
        """
        if plan.tables is not self:
            raise ValueError("the plan is of other block tables")
        rc = N.kv_entry("sq_kv_commit")(self._at, plan._args, N.raw_stream())
        if rc:
            N.check(rc, "kv commit")

    def release(self, rows):
        """Gives the pages of the requests in ``rows`` back; their rows are empty
        afterwards, and plans made before that name them are void."""
        rows = self._index(rows, "rows")
        if rows.numel() > N.KV_MAX_REQUESTS:
            raise ValueError(f"at most {N.KV_MAX_REQUESTS} rows at once")
        if rows.numel():
            N.check(N.lib().sq_kv_release(self._desc, N.ptr(rows), N.dtype_code(rows), rows.numel(),
                                          N.stream_handle()), "kv release")


class KVCache:
    """One attention layer's keys and values in ``pages`` pages of ``page_tokens`` tokens.

    ``data`` [pages, page_bytes] uint8: per head the keys' and the values'
    codes [page_tokens, head_dim], then per head their two fp32 peaks.
    ``head_dim`` is 64, 128 or 256 and ``page_tokens`` a multiple of 64, with
    at most 32,768 values of a head in a page.  A plan's block tables have the
    same ``page_tokens`` and no more pages.
    """

    def __init__(self, pages, kv_heads, head_dim, *, page_tokens=64, storage="int8", device="cuda"):
        if storage not in _STORAGE:
            raise ValueError("KV storage must be int8 or fp8")
        if head_dim not in (64, 128, 256):
            raise ValueError("head_dim must be 64, 128 or 256")
        if page_tokens <= 0 or page_tokens % TILE or page_tokens * head_dim > 32768:
            raise ValueError(f"page_tokens must be a positive multiple of {TILE} with page_tokens * head_dim <= 32768")
        if not 0 < kv_heads <= 4096 or not 0 < pages <= 0x7fffffff:
            raise ValueError("pages and kv_heads must be positive, kv_heads at most 4096")
        self.device = _device(device)
        self.pages, self.heads, self.dim, self.page_tokens, self.storage = pages, kv_heads, head_dim, page_tokens, storage
        codes = 2 * kv_heads * page_tokens * head_dim
        # whole 128-byte lines, so that every token's row starts on one
        self.page_bytes = -(-(codes + 8 * kv_heads) // 128) * 128
        self.data = torch.zeros((pages, self.page_bytes), dtype=torch.uint8, device=self.device)
        self._kv = N.KVCache(data=self.data.data_ptr(), page_bytes=self.page_bytes, num_pages=pages, heads=kv_heads,
                             dim=head_dim, page_tokens=page_tokens, storage=_STORAGE[storage])
        self._at = ctypes.addressof(self._kv)
        # page copies read only these
        self._desc = N.Pool(data=self.data.data_ptr(), page_bytes=self.page_bytes, num_slots=pages)

    @property
    def nbytes(self):
        return self.data.numel()

    def wait(self):
        """Writes are made on the caller's stream: nothing to wait for."""

    def copy(self, source, destination):
        """Copies whole pages, codes and peaks (a request that starts as another one's copy)."""
        PackedStatePool.copy(self, source, destination)

    def _rows(self, x, heads, tokens, what):
        """[tokens, heads, dim] with rows that the kernels take: bf16 or fp16,
        heads contiguous inside, strides of whole 16 bytes."""
        if x.dtype not in _HALVES:
            raise ValueError(f"{what} must be bf16 or fp16")
        if x.device != self.device:
            raise ValueError(f"{what} must be on the cache's device")
        if x.dim() == 2 and x.shape[1] == heads * self.dim:
            x = x.unflatten(1, (heads, self.dim))
        if x.shape != (tokens, heads, self.dim):
            raise ValueError(f"{what} must be [{tokens}, {heads}, {self.dim}], the plan's tokens")
        s0, s1, s2 = x.stride()
        if s2 != 1 or (s0 | s1) % 8 or s0 < 0 or s1 < 0 or x.data_ptr() % 16:
            x = x.clone(memory_format=torch.contiguous_format)
        return x

    def _check_plan(self, plan):
        tables = plan.tables
        if tables.page_tokens != self.page_tokens or tables.device != self.device:
            raise ValueError("the plan's block tables have other pages than the cache")
        if tables.pages > self.pages:
            raise ValueError(f"the plan's block tables give out {tables.pages} pages, the cache has {self.pages}")

    def append(self, k, v, plan):
        """Quantises the plan's new keys and values [tokens, kv_heads, head_dim]
        (or [tokens, kv_heads * head_dim]; bf16 or fp16) into their pages.

        Every page belongs to one request, as ``BlockTables`` gives them out: two
        requests that wrote to one page would race for its peaks.
        """
        self._check_plan(plan)
        k = self._rows(k, self.heads, plan.tokens, "keys")
        v = self._rows(v, self.heads, plan.tokens, "values")
        if k.dtype != v.dtype:
            raise ValueError("keys and values must have one dtype")
        if not plan.tokens:
            return
        (ks, kh, _), (vs, vh, _) = k.stride(), v.stride()
        args = N.KV_APPEND.pack(k.data_ptr(), v.data_ptr(), *plan._append, plan.tokens, ks, kh, vs, vh, plan.max_tiles,
                                _HALVES[k.dtype])
        rc = N.kv_entry("sq_kv_append")(self._at, args, N.raw_stream())
        if rc:
            N.check(rc, "kv append")

    def decode(self, pages, filled=None, *, dtype=torch.float32):
        """Keys and values [n, page_tokens, kv_heads, head_dim] of ``pages``,
        zero past the first ``filled`` tokens of each (default: all are taken)
        and for pages that the cache does not have (page 0 among them)."""
        if dtype not in N.FLOATS:
            raise ValueError("dense keys and values are fp32, bf16 or fp16")
        pages = self._numbers(pages)
        n = pages.numel()
        if filled is not None:
            filled = self._numbers(filled)
            if filled.numel() != n:
                raise ValueError("pages and filled must have the same length")
        shape = (n, self.page_tokens, self.heads, self.dim)
        k = torch.empty(shape, dtype=dtype, device=self.device)
        v = torch.empty(shape, dtype=dtype, device=self.device)
        if n:
            rc = N.kv_entry("sq_kv_decode")(self._at, pages.data_ptr(), 0 if filled is None else filled.data_ptr(), n,
                                            k.data_ptr(), v.data_ptr(), N.FLOATS[dtype], N.raw_stream())
            if rc:
                N.check(rc, "kv decode")
        return k, v

    def _numbers(self, x):
        if isinstance(x, torch.Tensor) and x.dtype == torch.int32 and x.dim() == 1 and x.device == self.device \
                and x.is_contiguous():
            return x
        x = torch.as_tensor(x)
        if x.numel() and (x.is_floating_point() or x.is_complex() or x.dtype == torch.bool):
            raise ValueError("pages and token counts must be integers")
        # (numbers that 32 bits do not hold are of no page)
        return x.long().clamp(-1, 0x7fffffff).to(device=self.device, dtype=torch.int32).reshape(-1).contiguous()

    def attend(self, q, plan, *, scale=None, window=None, out=None):
        """Attention of the plan's new tokens over all that their requests hold.

        ``q`` is [tokens, q_heads, head_dim] (or [tokens, q_heads * head_dim]),
        bf16 or fp16, after ``append`` of the same plan; the result has its
        shape (three-dimensional) and dtype.  ``scale`` defaults to
        ``head_dim ** -0.5``; ``window`` picks one of the plan's windows
        (default: the first).  Tokens that see no key get zero.
        """
        self._check_plan(plan)
        schedules = plan.schedules
        if not schedules and plan.tokens:
            raise ValueError("the plan was made without heads")
        if not plan.tokens:
            shape = (0, q.shape[-1] // self.dim, self.dim) if q.dim() == 2 else (0, *q.shape[1:])
            return q.new_empty(shape) if out is None else out
        if window is None:
            s = next(iter(schedules.values()))
        elif window in schedules:
            s = schedules[window]
        else:
            raise ValueError(f"the plan was made without the window {window}")
        if s.kv_heads != self.heads:
            raise ValueError(f"the plan was made for {s.kv_heads} KV heads")
        q = self._rows(q, s.q_heads, plan.tokens, "queries")
        scale = self.dim ** -.5 if scale is None else float(scale)
        if not abs(scale) < 3e38:
            raise ValueError("scale must be finite, below 3e38")
        if out is None:
            out = torch.empty((plan.tokens, s.q_heads, self.dim), dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != self.device or not out.is_contiguous() \
                or out.data_ptr() % 16:
            raise ValueError("out must be contiguous and like the queries")
        ws = torch.empty(s.floats * (self.dim + 2), dtype=torch.float32, device=self.device)
        t = plan.tables
        qs, qh, _ = q.stride()
        args = N.KV_ATTEND.pack(q.data_ptr(), out.data_ptr(), ws.data_ptr(), t.table.data_ptr(), t.requests, plan.tokens,
                                qs, qh, t.max_blocks, _HALVES[q.dtype], scale, 0, s.packed)
        rc = N.kv_entry("sq_kv_attend")(self._at, args, N.raw_stream())
        if rc:
            N.check(rc, "kv attend")
        return out
