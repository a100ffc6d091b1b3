"""Performance cases of the 8-bit paged KV cache: block tables and slot maps,
the quantising write with its read-back, and attention over the cached pages.

``run`` with ``own`` makes the calls of ``stepquant_amd.kernels.kv_cache``;
without it the same operators in elementary torch operations, 32 bits
throughout.  ``exact`` gives the outputs from the definitions in 64 bits.

A page holds ``page`` tokens of every KV head.  Each (page, head) has one peak
for its keys and one for its values, the largest magnitude among the block's
tokens; a value x is held as rint(x / peak * 127) (int8) or as the nearest
e4m3 number to x / peak * 448 (fp8).
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TOP = {"int8": 127., "fp8": 448.}
FLOOR = 2. ** -60  # the least peak of a block
SPARE = 7          # pages beyond those that a case fills


def _case(name, kind, **kw):
    case = dict(name=name, kind=kind, batch=1, q_heads=32, kv_heads=8, dim=128, page=64, storage="int8",
                dtype="bf16", context=0, new=1, ragged=False, padding=0, causal=True, window=0)
    case.update(kw)
    return case


def listed():
    return [
        # block tables of a full decode batch: every request grows by one token
        _case("plan_decode_b256", "plan", batch=256, context=32768, ragged=True),
        # block tables of a mixed batch of prompts, some continuing a cached prefix
        _case("plan_prompts_b48", "plan", batch=48, context=5000, new=2731, ragged=True, padding=13),
        # one decode step's keys and values into part-filled pages, which are read back
        _case("append_decode_b64", "append", batch=64, context=1500, ragged=True),
        # a long prompt's keys and values, handed back dense
        _case("append_prompt_t16384", "append", new=16384),
        # chunks of prompts of odd lengths on wide heads, into part-filled pages
        _case("append_fp8_ragged", "append", batch=5, kv_heads=2, dim=256, storage="fp8", dtype="fp16", context=333,
              new=1777, ragged=True),
        # one user's chat: a short context on wide heads, where latency counts
        _case("attend_decode_b1", "attend", q_heads=16, kv_heads=2, dim=256, context=999),
        # one long document: few rows, so the context is split
        _case("attend_decode_b1_long", "attend", context=131071),
        # a full decode batch with ragged contexts, padded as a captured graph is
        _case("attend_decode_b64", "attend", batch=64, context=8191, ragged=True, padding=3),
        # the largest decode batch, e4m3 pages of 128 tokens
        _case("attend_decode_b256_fp8", "attend", batch=256, context=4095, storage="fp8", page=128),
        # a small draft checked by the model: several tokens a request, one head a group, small heads
        _case("attend_draft_b32", "attend", batch=32, q_heads=16, kv_heads=16, dim=64, dtype="fp16", context=2048,
              new=5, ragged=True),
        # a long prompt over its own keys
        _case("attend_prompt_t8192", "attend", new=8192),
        # chunks of prompts over cached prefixes, wide heads, e4m3
        _case("attend_chunks_fp8", "attend", batch=4, q_heads=16, kv_heads=2, dim=256, storage="fp8", context=12000,
              new=701, ragged=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "append"] + ["attend"] * 5)
    q_heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 128), (16, 2, 256), (16, 16, 64), (24, 8, 128),
                                         (14, 2, 64), (8, 1, 128), (20, 4, 128), (32, 1, 256)])
    case = _case("", kind, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=rng.choice([64, 64, 128]),
                 storage=rng.choice(["int8", "fp8"]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                 ragged=rng.random() < .7, padding=rng.choice([0, 0, rng.randint(1, 9)]))
    heads = max(1, kv_heads * dim // 512)
    if kind == "plan":
        case["batch"] = _log(rng, 1, 512)
        case["context"] = _log(rng, 1, 32768)
        case["new"] = rng.choice([1, _log(rng, 1, max(2, 131072 // case["batch"]))])
    elif kind == "append":
        case["batch"] = _log(rng, 1, 64)
        case["context"] = rng.choice([0, _log(rng, 1, 2000)])
        case["new"] = rng.choice([1, _log(rng, 1, max(2, 16384 // case["batch"] // heads))])
    elif rng.random() < .6:  # one or a few tokens a request
        case["new"] = rng.choice([1, 1, 1, rng.randint(2, 8)])
        case["batch"] = _log(rng, 1, 256)
        case["context"] = _log(rng, 1, min(131072, 1048576 // case["batch"] // heads))
        case["window"] = rng.choice([0, 0, 0, 1024])
    else:
        case["batch"] = _log(rng, 1, 16)
        case["new"] = _log(rng, 9, 8192 // case["batch"])
        case["context"] = rng.choice([0, _log(rng, 1, 16384 // case["batch"])])
        case["window"] = rng.choice([0, 0, 0, 1024])
        case["causal"] = case["window"] > 0 or rng.random() < .85
    case.pop("name")
    return case


# ---------------------------------------------------------------- sizes
def _spread(most, n, ragged, least):
    """``n`` lengths: all ``most``, or spread over [least, most] with ``most`` first."""
    if not ragged:
        return [most] * n
    return [max(least, most - int(most * .9 * (i * .6180339887 % 1.))) for i in range(n)]


def _sizes(case):
    """(cached tokens, new tokens) of each request."""
    n = case["batch"]
    old = _spread(case["context"], n, case["ragged"], min(1, case["context"]))
    new = _spread(case["new"], n, case["ragged"], 1)
    return old, new[::-1]


def _blocks(tokens, page):
    return -(-tokens // page)


def _tiles(case):
    """How many page entries a plan has room for."""
    tokens = sum(_sizes(case)[1]) + case["padding"]
    return min(tokens, tokens // case["page"] + 2 * case["batch"])


def _visible(case):
    """(key, query) pairs that are seen, and the keys that any query sees."""
    pairs = keys = 0
    for o, n in zip(*_sizes(case)):
        w = case["window"] or o + n
        keys += min(o + n, w + n - 1) if case["causal"] else o + n
        if not case["causal"]:
            pairs += n * (o + n)
        else:
            pairs += sum(min(o + i + 1, w) for i in range(n)) if case["window"] else n * o + n * (n + 1) // 2
    return pairs, keys


def work(case):
    old, new = _sizes(case)
    tokens, n, P = sum(new) + case["padding"], case["batch"], case["page"]
    H, D = case["kv_heads"], case["dim"]
    if case["kind"] == "plan":
        grown = sum(_blocks(o + x, P) - _blocks(o, P) for o, x in zip(old, new))
        # lens, rows, new; free pages; slots and positions; the tables' and the plan's page entries; per request
        return {"bytes": 12 * n + 4 * grown + 12 * tokens + 4 * grown + 8 * _tiles(case) + 9 * n, "flops": 0}
    if case["kind"] == "append":
        values = 2 * sum(new) * H * D
        kept = 2 * H * D * sum(o % P for o in old)
        touched = 2 * H * D * P * _tiles(case)
        # keys and values; codes; the live codes of part-filled pages; the pages handed back dense
        return {"bytes": 2 * values + values + kept + 2 * touched, "flops": 6 * values}
    pairs, keys = _visible(case)
    q = tokens * case["q_heads"] * D
    return {"bytes": 4 * q + 2 * keys * H * D + 8 * H * _blocks(keys, P), "flops": 4 * D * case["q_heads"] * pairs}


# ---------------------------------------------------------------- inputs
def _rng(seed, part):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + part)


def _new_kv(case, seed, part, tokens):
    """Keys and values as a layer's projections give them: keys with channels
    of unequal size, both with unequal tokens."""
    g = _rng(seed, part)
    shape = (tokens, case["kv_heads"], case["dim"])
    dt = TYPES[case["dtype"]]
    channel = torch.exp(torch.randn(shape[1:], device="cuda", generator=_rng(seed, 1)) * .5)
    size = torch.exp(torch.randn((tokens, 1, 1), device="cuda", generator=g) * .2)
    k = (torch.randn(shape, device="cuda", generator=g) * channel * size).to(dt)
    v = (torch.randn(shape, device="cuda", generator=g) * size).to(dt)
    return k, v


def _tables(case, seed):
    """Room for the case's requests: rows in mixed order, free pages in the
    order in which earlier requests gave them back."""
    old, new = _sizes(case)
    P, n = case["page"], case["batch"]
    pages = 1 + sum(_blocks(o + x, P) for o, x in zip(old, new)) + SPARE
    width = max(_blocks(o + x, P) for o, x in zip(old, new)) + 1
    g = _rng(seed, 2)
    free = (torch.randperm(pages - 1, device="cuda", generator=g) + 1).to(torch.int32)
    rows = torch.randperm(n + 3, device="cuda", generator=g)[:n].to(torch.int32)
    return pages, width, free, rows


def _own_tables(case, seed):
    from stepquant_amd.kernels.kv_cache import BlockTables
    pages, width, free, rows = _tables(case, seed)
    tables = BlockTables(case["batch"] + 3, pages, width, page_tokens=case["page"])
    tables.free.copy_(free)
    return tables, rows


def _plain_tables(case, seed):
    pages, width, free, rows = _tables(case, seed)
    return dict(table=torch.zeros((case["batch"] + 3, width), dtype=torch.int32, device="cuda"), free=free,
                lens=torch.zeros(case["batch"] + 3, dtype=torch.int32, device="cuda"),
                counters=torch.tensor([0, pages - 1], dtype=torch.int64, device="cuda")), rows, pages


def prepare(case, seed):
    old, new = _sizes(case)
    tokens = sum(new) + case["padding"]
    counts = torch.tensor(new, dtype=torch.int32, device="cuda")
    state = dict(case=case, tokens=tokens, counts=counts, old=old, new=new)
    # requests fill their contexts a few at a time, as they came
    groups, size = [[]], 0
    for i, o in enumerate(old):
        if size + o > 65536 and groups[-1]:
            groups.append([])
            size = 0
        groups[-1].append(i)
        size += o
    values = case["kind"] != "plan"
    if own:
        from stepquant_amd.kernels.kv_cache import KVCache
        tables, rows = _own_tables(case, seed)
        if values:
            cache = KVCache(tables.pages, case["kv_heads"], case["dim"], page_tokens=case["page"],
                            storage=case["storage"])
        for i, group in enumerate(groups):
            plan = tables.plan([old[j] for j in group], rows[group[0]:group[-1] + 1])
            if values:
                cache.append(*_new_kv(case, seed, 10 + i, plan.tokens), plan)
            tables.commit(plan)
        state.update(tables=tables, rows=rows)
        if values:
            state.update(cache=cache, plan=tables.plan(
                counts, rows, tokens=tokens, max_new=max(new), heads=(case["q_heads"], case["kv_heads"]),
                causal=case["causal"], window=case["window"]))
    else:
        tables, rows, pages = _plain_tables(case, seed)
        if values:
            cache = _empty(case, pages)
        for i, group in enumerate(groups):
            count = torch.tensor([old[j] for j in group], dtype=torch.int32, device="cuda")
            total = sum(old[j] for j in group)
            plan = _plan(tables, rows[group[0]:group[-1] + 1], count, total, case["page"])
            if values:
                _append(cache, case, *_new_kv(case, seed, 10 + i, total), plan)
            _commit(tables, rows[group[0]:group[-1] + 1], plan)
        state.update(tables=tables, rows=rows)
        if values:
            state.update(cache=cache, plan=_plan(tables, rows, counts, tokens, case["page"]))
    if values:
        k, v = _new_kv(case, seed, 3, tokens)
        if case["kind"] == "append":
            state.update(k=k, v=v)
        else:
            if own:
                cache.append(k, v, state["plan"])
            else:
                _append(cache, case, k, v, state["plan"])
            q = torch.randn((tokens, case["q_heads"], case["dim"]), device="cuda", generator=_rng(seed, 4))
            # a few rows look at few keys, most at many
            size = torch.exp(torch.randn((tokens, case["q_heads"], 1), device="cuda", generator=_rng(seed, 5)) * .7)
            state["q"] = (q * size).to(TYPES[case["dtype"]])
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        if kind == "plan":
            plan = state["tables"].plan(state["counts"], state["rows"], tokens=state["tokens"],
                                        max_new=max(state["new"]), heads=(case["q_heads"], case["kv_heads"]))
            return [plan.cu, plan.slots, plan.positions, plan.lens, plan.granted, plan.pages, plan.filled,
                    plan.counters, state["tables"].table]
        if kind == "append":
            cache, plan = state["cache"], state["plan"]
            cache.append(state["k"], state["v"], plan)
            return list(cache.decode(plan.pages, plan.filled, dtype=TYPES[case["dtype"]]))
        return state["cache"].attend(state["q"], state["plan"])
    if kind == "plan":
        plan = _plan(state["tables"], state["rows"], state["counts"], state["tokens"], case["page"])
        return [plan["cu"], plan["slots"], plan["positions"], plan["lens"], plan["granted"], plan["pages"],
                plan["filled"], plan["counters"], state["tables"]["table"]]
    if kind == "append":
        _append(state["cache"], case, state["k"], state["v"], state["plan"])
        return _decode(state["cache"], case, state["plan"])
    return _attend(state)


def _plan(tables, rows, new, tokens, P):
    """Slots of the new tokens, and the pages that they fill, from the lengths."""
    table, lens, free, counters = tables["table"], tables["lens"], tables["free"], tables["counters"]
    n, width = rows.numel(), table.shape[1]
    rows, new = rows.long(), new.long()
    old = lens[rows].long()
    want = old + new
    had, blocks = (old + P - 1) // P, (want + P - 1) // P
    end = new.cumsum(0)
    fits = (blocks <= width) & (end <= tokens)
    need = torch.where(fits, blocks - had, 0)
    total = need.cumsum(0)
    head, tail = counters[0], counters[1]
    granted = fits & ((need == 0) | (total <= tail - head))
    taken = torch.where(granted & (need > 0), total, 0).amax()
    first = total - need
    after = torch.where(granted, want, old)
    cu = torch.cat([end.new_zeros(1), end]).clamp(max=tokens)
    # the pages that new tokens fall into, request by request
    touched = torch.where(granted & (new > 0), blocks - old // P, 0)
    ends = touched.cumsum(0)
    i = torch.arange(min(tokens, tokens // P + 2 * n), device=rows.device)
    b = torch.searchsorted(ends, i, right=True)
    used = b < n
    b = b.clamp(max=n - 1)
    block = torch.where(used, old[b] // P + i - (ends - touched)[b], 0)
    fresh = block >= had[b]
    at = (head + first[b] + block - had[b]) % free.numel()
    page = torch.where(fresh, free[at], table[rows[b], block])
    pages = torch.where(used, page, 0)
    filled = torch.where(used, (after[b] - block * P).clamp(max=P), 0)
    grown = used & fresh
    at = torch.where(grown, rows[b] * width + block, table.numel())
    flat = torch.cat([table.reshape(-1), table.new_zeros(1)])
    flat[at] = torch.where(grown, page, 0).to(torch.int32)
    table.copy_(flat[:-1].view_as(table))
    # the tokens
    t = torch.arange(tokens, device=rows.device)
    q = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    live = q < n
    q = q.clamp(max=n - 1)
    live = live & granted[q]
    pos = torch.where(live, old[q] + t - cu[q], -1)
    slot = torch.where(live, table[rows[q], torch.where(live, pos // P, 0)].long() * P + pos % P, -1)
    start = torch.where(used, (old[b] - block * P).clamp(min=0), 0)
    return dict(cu=cu.int(), slots=slot, positions=pos.int(), lens=after.int(), granted=granted, pages=pages.int(),
                filled=filled.int(), counters=torch.stack([head + taken, tail]), start=start,
                tile_of=ends - touched, old=old)


def _commit(tables, rows, plan):
    tables["lens"][rows.long()] = plan["lens"]
    tables["counters"].copy_(plan["counters"])


def _empty(case, pages):
    """Pages [pages, keys and values, tokens, heads, dim] of codes, and the blocks' peaks."""
    shape = (pages, 2, case["page"], case["kv_heads"], case["dim"])
    return dict(codes=torch.zeros(shape, dtype=torch.int8, device="cuda"),
                peaks=torch.full((pages, 2, case["kv_heads"]), FLOOR, device="cuda"))


def _round(x, storage):
    """Codes as the numbers they stand for."""
    return x.round() if storage == "int8" else x.to(torch.float8_e4m3fn).float()


def _hold(x, storage):
    return x.to(torch.int8) if storage == "int8" else x.to(torch.float8_e4m3fn).view(torch.int8)


def _held(codes, storage):
    return codes.float() if storage == "int8" else codes.view(torch.float8_e4m3fn).float()


def _append(cache, case, k, v, plan):
    """New tokens into their pages: the block's peak, the live codes brought to
    it where it grew, the new codes."""
    storage, P = case["storage"], case["page"]
    top = TOP[storage]
    pages = plan["pages"].long()
    n = pages.numel()
    live = plan["slots"] >= 0
    # each new token's page entry: the entries of a request are in block order
    of = torch.searchsorted(plan["cu"][1:].contiguous().long(), torch.arange(k.shape[0], device="cuda"), right=True)
    of = of.clamp(max=plan["old"].numel() - 1)
    tile = plan["tile_of"][of] + plan["positions"].long() // P - plan["old"][of] // P
    offset = plan["positions"].long() % P
    # the scratch entry past the last takes the tokens that have no page
    tile = torch.where(live, tile, n)
    offset = torch.where(live, offset, 0)
    for part, x in enumerate((k, v)):
        dense = torch.zeros((n + 1, P, *x.shape[1:]), device="cuda")
        dense[tile, offset] = x.float()
        dense = dense[:n]
        here = torch.arange(P, device="cuda")[None]
        fresh = (here >= plan["start"][:, None]) & (here < plan["filled"][:, None])
        kept = here < plan["start"][:, None]
        before = torch.where(plan["start"][:, None] > 0, cache["peaks"][pages, part], FLOOR)
        peak = torch.maximum(before, dense.abs().amax((1, 3))).clamp(min=FLOOR)
        at = peak[:, None, :, None]
        was = _held(cache["codes"][pages, part], storage)
        moved = _round(was * before[:, None, :, None] / at, storage)
        put = _round(dense / at * top, storage)
        codes = torch.where(fresh[..., None, None], put, torch.where(kept[..., None, None], moved, was))
        cache["codes"][pages, part] = _hold(codes, storage)
        cache["peaks"][pages, part] = peak


def _decode(cache, case, plan):
    """The touched pages as dense keys and values, zero past their tokens."""
    pages = plan["pages"].long()
    there = torch.arange(case["page"], device="cuda")[None] < plan["filled"][:, None]
    out = []
    for part in range(2):
        x = _held(cache["codes"][pages, part], case["storage"])
        x = x * (cache["peaks"][pages, part] / TOP[case["storage"]])[:, None, :, None]
        out.append(torch.where(there[..., None, None], x, 0.).to(TYPES[case["dtype"]]))
    return out


def _request_kv(cache, case, table, length, low):
    """Keys and values [heads, tokens from ``low`` on, dim] of one request in 32 bits."""
    P = case["page"]
    pages = table[low // P:_blocks(length, P)].long()
    out = []
    for part in range(2):
        x = _held(cache["codes"][pages, part], case["storage"])
        x = x * (cache["peaks"][pages, part] / TOP[case["storage"]])[:, None, :, None]
        x = x.reshape(-1, *x.shape[2:])[low % P:low % P + length - low]
        out.append(x.transpose(0, 1).contiguous())
    return out


def _attend(state):
    case, q = state["case"], state["q"]
    H, D = case["kv_heads"], case["dim"]
    G = case["q_heads"] // H
    out = torch.zeros_like(q)
    at = 0
    for i, (o, n) in enumerate(zip(state["old"], state["new"])):
        low = max(0, o - case["window"] + 1) if case["window"] else 0
        k, v = _request_kv(state["cache"], case, state["tables"]["table"][state["rows"][i].long()], o + n, low)
        j = torch.arange(low, o + n, device="cuda")
        kt = k.transpose(1, 2).contiguous()
        step = max(1, (1 << 28) // (case["q_heads"] * (o + n)))
        for t0 in range(0, n, step):
            t1 = min(n, t0 + step)
            x = q[at + t0:at + t1].float().view(t1 - t0, H, G, D).permute(1, 2, 0, 3).reshape(H, -1, D)
            s = torch.matmul(x, kt) * D ** -.5
            if case["causal"]:
                pos = torch.arange(o + t0, o + t1, device="cuda")[:, None]
                seen = j[None] <= pos
                if case["window"]:
                    seen = seen & (j[None] > pos - case["window"])
                s = s.view(H, G, t1 - t0, -1).masked_fill(~seen, -math.inf).view(H, G * (t1 - t0), -1)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            y = torch.matmul(p, v) / p.sum(-1, keepdim=True)
            y = y.view(H, G, t1 - t0, D).permute(2, 0, 1, 3).reshape(t1 - t0, H * G, D)
            out[at + t0:at + t1] = y.to(q.dtype)
        at += n
    return out


# ---------------------------------------------------------------- in 64 bits
def _e4m3(x):
    """Nearest e4m3 number, ties to even: 3 fraction bits, exponents from -6 up."""
    m, e = torch.frexp(x)
    unit = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return ((x / unit).round() * unit).clamp(-448, 448)


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    old, new, P, top = state["old"], state["new"], case["page"], TOP[case["storage"]]
    cache, table, rows = state["cache"], state["tables"]["table"].cpu(), state["rows"].cpu()
    held = lambda ids, part: _held(cache["codes"][ids, part], case["storage"]).double()
    if case["kind"] == "append":
        shape = (_tiles(case), P, case["kv_heads"], case["dim"])
        out = [torch.zeros(shape, dtype=torch.float64, device="cuda") for _ in range(2)]
        row = tile = 0
        for i, (o, n) in enumerate(zip(old, new)):
            done = 0
            while done < n:
                block, start = divmod(o + done, P)
                count = min(P - start, n - done)
                page = int(table[rows[i], block])
                for part, x in enumerate((state["k"], state["v"])):
                    x = x[row + done:row + done + count].double()
                    peak = x.abs().amax((0, 2)).clamp(min=FLOOR)
                    if start:
                        before = cache["peaks"][page, part].double()
                        peak = torch.maximum(peak, before)
                        y = held(page, part)[:start] * (before / peak)[:, None]
                        y = y.round() if top == 127 else _e4m3(y)
                        out[part][tile, :start] = y * (peak / top)[:, None]
                    y = x / peak[:, None] * top
                    y = y.round() if top == 127 else _e4m3(y)
                    out[part][tile, start:start + count] = y * (peak / top)[:, None]
                done += count
                tile += 1
            row += n
        return out
    q = state["q"].double()
    H, D = case["kv_heads"], case["dim"]
    out = torch.zeros_like(q)
    row = 0
    for i, (o, n) in enumerate(zip(old, new)):
        ids = table[rows[i], :_blocks(o + n, P)].long().cuda()
        kv = []
        for part in range(2):
            x = held(ids, part) * (cache["peaks"][ids, part].double() / top)[:, None, :, None]
            kv.append(x.flatten(0, 1)[:o + n])
        for h in range(case["q_heads"]):
            kh, vh = (x[:, h * H // case["q_heads"]].contiguous() for x in kv)
            for t0 in range(0, n, 2048):
                t1 = min(n, t0 + 2048)
                s = q[row + t0:row + t1, h] @ kh.t() / math.sqrt(D)
                if case["causal"]:
                    back = torch.arange(o + t0, o + t1, device="cuda")[:, None] - torch.arange(o + n, device="cuda")
                    hidden = back < 0
                    if case["window"]:
                        hidden |= back >= case["window"]
                    s[hidden] = -math.inf
                out[row + t0:row + t1, h] = torch.softmax(s, -1) @ vh
        row += n
    return out
