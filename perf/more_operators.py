"""Performance cases of what attention layers beside recurrent ones need besides
the 8-bit cache's own kernels: rotary positions, the quantising write with the
rotation on the way, and latent attention (one shared vector a token) over a
paged cache, absorbed for single tokens and drafts, expanded for prompts.

``run`` with ``own`` makes the calls of ``stepquant_amd.kernels``; without it
the same operators in elementary torch operations, 32 bits throughout (angles
in 64).  ``exact`` gives the outputs from the definitions in 64 bits.

Pair i of a head's first ``rotated`` dims turns by position * f_i, scaled by
``magnitude``; the pairs are (i, i + rotated / 2) in the half layout and
(2 i, 2 i + 1) in the interleaved one.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TOP = {"int8": 127., "fp8": 448.}
FLOOR = 2. ** -60  # the least peak of a block
SPARE = 7          # pages beyond those that a case fills
BASE = 1e6         # frequencies are BASE ** (-2 i / rotated) before any scaling
ORIGINAL = 8192    # positions that the unscaled frequencies were trained on


def _case(name, kind, **kw):
    case = dict(name=name, kind=kind, batch=1, q_heads=32, kv_heads=8, dim=128, rotated=128, layout="half", scaling="",
                factor=1., page=64, storage="int8", dtype="bf16", context=0, new=1, ragged=False, padding=0, causal=True,
                latent=512, far=0)
    case.update(kw)
    return case


def listed():
    return [
        # one token's queries of wide heads, a quarter of each rotated, where latency counts
        _case("rotary_token", "rotary", q_heads=16, dim=256, rotated=64, far=5000),
        # a prompt's queries at far positions of a stretched context
        _case("rotary_prompt_t16384", "rotary", new=16384, layout="interleaved", scaling="yarn", factor=16., far=100000),
        # one decode step: keys turned and quantised into part-filled pages, queries turned
        _case("append_rotary_decode_b64", "append", batch=64, context=1500, ragged=True),
        # prompts of odd lengths, wide heads with a quarter rotated, e4m3, some continuing a prefix
        _case("append_rotary_ragged_fp8", "append", batch=5, q_heads=16, kv_heads=2, dim=256, rotated=64, storage="fp8",
              dtype="fp16", context=333, new=3777, ragged=True),
        # one decode step of a latent layer: the shared vectors into the pages, rope keys and queries turned
        _case("latent_append_decode_b256", "latent_append", batch=256, rotated=64, context=500, ragged=True, padding=5),
        # chunks of prompts that continue prefixes: written, then everything gathered for the expansion
        _case("latent_gather_chunks", "gather", batch=6, q_heads=16, rotated=64, layout="interleaved", context=8000,
              new=1111, ragged=True),
        # one user's chat, 16 heads over a short context, where latency counts
        _case("absorbed_decode_b1", "absorbed", q_heads=16, context=999),
        # a full decode batch of ragged contexts, padded as a captured graph is
        _case("absorbed_decode_b64", "absorbed", batch=64, context=8191, ragged=True, padding=3),
        # every head on one GPU over long contexts
        _case("absorbed_decode_b32_h128", "absorbed", batch=32, q_heads=128, context=16383, ragged=True),
        # a small draft checked by the model: several tokens a request, a narrower latent
        _case("absorbed_draft_b32", "absorbed", batch=32, q_heads=16, latent=256, dtype="fp16", context=2048, new=5,
              ragged=True),
        # a long prompt over its own keys
        _case("expanded_prompt_t8192", "expanded", q_heads=16, new=8192),
        # chunks of prompts of odd lengths over gathered prefixes
        _case("expanded_chunks_b4", "expanded", batch=4, q_heads=16, context=12000, new=701, ragged=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "append", "append", "latent_append", "gather"] + ["absorbed"] * 4 +
                      ["expanded"] * 3)
    case = _case("", kind, page=rng.choice([64, 64, 128]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                 layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["", "linear", "yarn", "bands"]),
                 factor=rng.choice([2., 4., 8., 32.]), ragged=rng.random() < .7,
                 padding=rng.choice([0, 0, rng.randint(1, 9)]))
    if kind in ("rotary", "append"):
        q_heads, kv_heads, dim, rotated = rng.choice([(32, 8, 128, 128), (16, 2, 256, 64), (16, 16, 64, 64),
                                                      (24, 8, 128, 64), (14, 2, 64, 64), (20, 4, 128, 32)])
        case.update(q_heads=q_heads, kv_heads=kv_heads, dim=dim, rotated=rotated, storage=rng.choice(["int8", "fp8"]))
        most = 8192 // max(1, q_heads * dim // 4096)
        if kind == "rotary":
            case["far"] = rng.choice([0, _log(rng, 10, 1000000)])
            case["new"] = _log(rng, 1, most)
            case["dtype"] = rng.choice(["bf16", "fp16", "fp32"])
        else:
            case["batch"] = _log(rng, 1, 64)
            case["context"] = rng.choice([0, _log(rng, 1, 2000)])
            case["new"] = rng.choice([1, _log(rng, 1, max(2, most // case["batch"]))])
    else:
        case.update(q_heads=rng.choice([8, 16, 16, 20, 32, 64, 128]), rotated=64, latent=rng.choice([512, 512, 256]))
        if kind == "latent_append":
            case["batch"] = _log(rng, 1, 256)
            case["context"] = rng.choice([0, _log(rng, 1, 500)])
            case["new"] = rng.choice([1, _log(rng, 1, max(2, 8192 // case["batch"]))])
            case["q_heads"] = rng.choice([8, 16, 32])
        elif kind == "gather":
            case["batch"] = _log(rng, 1, 16)
            case["context"] = rng.choice([0, _log(rng, 1, 32768 // case["batch"])])
            case["new"] = _log(rng, 1, 8192 // case["batch"])
            case["q_heads"] = rng.choice([8, 16])
        elif kind == "absorbed":
            case["new"] = rng.choice([1, 1, 1, rng.randint(2, 6)])
            case["batch"] = _log(rng, 1, 128)
            most = min(65536, 400000 // case["batch"], 40000000 // (case["batch"] * case["q_heads"] * case["new"]))
            case["context"] = _log(rng, 1, max(2, most))
        else:
            case["q_heads"] = rng.choice([8, 16, 16, 12])
            case["dim"] = rng.choice([128, 128, 64])
            case["batch"] = _log(rng, 1, 8)
            case["new"] = _log(rng, 9, 6000 // case["batch"])
            case["context"] = rng.choice([0, _log(rng, 1, 8000 // case["batch"])])
            case["causal"] = rng.random() < .85
    case.pop("name")
    return case


# ---------------------------------------------------------------- sizes
def _spread(most, n, ragged, least):
    """``n`` lengths: all ``most``, or spread over [least, most] with ``most`` first."""
    if not ragged:
        return [most] * n
    return [max(least, most - int(most * .9 * (i * .6180339887 % 1.))) for i in range(n)]


def _sizes(case):
    """(held tokens, new tokens) of each request."""
    n = case["batch"]
    old = _spread(case["context"], n, case["ragged"], min(1, case["context"]))
    return old, _spread(case["new"], n, case["ragged"], 1)[::-1]


def _blocks(tokens, page):
    return -(-tokens // page)


def _tiles(case):
    """How many page entries a plan has room for."""
    tokens = sum(_sizes(case)[1]) + case["padding"]
    return min(tokens, tokens // case["page"] + 2 * case["batch"])


def work(case):
    old, new = _sizes(case)
    tokens, kind, H = sum(new) + case["padding"], case["kind"], case["q_heads"]
    size = 4 if case["dtype"] == "fp32" else 2
    held = sum(old) + sum(new)
    if kind == "rotary":
        x = tokens * H * case["dim"]
        return {"bytes": 2 * size * x + 4 * tokens, "flops": 3 * tokens * H * case["rotated"]}
    if kind == "append":
        KH, D, P = case["kv_heads"], case["dim"], case["page"]
        values = 2 * sum(new) * KH * D
        kept = 2 * KH * D * sum(o % P for o in old)
        touched = 2 * KH * D * P * _tiles(case)
        # keys and values, codes, live codes of part-filled pages, the pages handed back dense, the queries
        return {"bytes": 2 * values + values + kept + 3 * touched + 4 * tokens * H * D,
                "flops": 6 * values + 3 * tokens * (H + KH) * case["rotated"]}
    width = case["latent"] + 64
    if kind == "latent_append":
        return {"bytes": 4 * sum(new) * width + 4 * tokens * H * 64, "flops": 3 * tokens * (H + 1) * 64}
    if kind == "gather":
        return {"bytes": 4 * sum(new) * width + 4 * held * width + 4 * tokens * H * 64,
                "flops": 3 * tokens * (H + 1) * 64}
    pairs = sum(n * o + (n * (n + 1) // 2 if case["causal"] else n * n) for o, n in zip(old, new))
    if kind == "absorbed":
        return {"bytes": 2 * held * width + 2 * tokens * H * (width + case["latent"]),
                "flops": 2 * H * pairs * (width + case["latent"])}
    D = case["dim"]
    return {"bytes": 2 * held * (2 * H * D + 64) + 2 * tokens * H * (2 * D + 64), "flops": 2 * H * pairs * (2 * D + 64)}


# ---------------------------------------------------------------- inputs
def _rng(seed, part):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + part)


def _randn(seed, part, *shape):
    return torch.randn(shape, device="cuda", generator=_rng(seed, part))


def _uneven(case, seed, part, *shape):
    """Channels of unequal size (the same for all parts of a seed) and unequal rows."""
    channel = torch.exp(_randn(seed, 1, *shape[1:]) * .4)
    size = torch.exp(_randn(seed, part + 1, shape[0], *[1] * (len(shape) - 1)) * .2)
    return (_randn(seed, part, *shape) * channel * size).to(TYPES[case["dtype"]])


def _queries(case, seed, part, *shape):
    """Rows of which a few look at few keys, most at many."""
    return (_randn(seed, part, *shape) * torch.exp(_randn(seed, part + 1, *shape[:-1], 1) * .7)).to(TYPES[case["dtype"]])


def _frequencies(case):
    """f_i in 64 bits, and the magnitude."""
    n = case["rotated"]
    i = torch.arange(0, n, 2, dtype=torch.float64)
    f = BASE ** (-i / n)
    s = case["factor"]
    if case["scaling"] == "linear":
        return f / s, 1.
    if case["scaling"] == "yarn":  # pairs that turn fewer than once in ORIGINAL are stretched, more than 32 times not
        at = lambda turns: n * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(BASE))
        low, high = max(0, math.floor(at(32.))), min(n - 1, math.ceil(at(1.)))
        ramp = ((i / 2 - low) / max(high - low, .001)).clamp(0, 1)
        return f * (1 - ramp) + f / s * ramp, .1 * math.log(s) + 1
    if case["scaling"] == "bands":  # stretched below 1 turn in ORIGINAL, not above 4, mixed between
        keep = ((ORIGINAL * f / (2 * math.pi) - 1) / 3).clamp(0, 1)
        return f * keep + f / s * (1 - keep), 1.
    return f, 1.


def _own_rotary(case):
    from stepquant_amd.kernels.rotary import Rotary
    more = dict(linear=dict(factor=case["factor"]), yarn=dict(factor=case["factor"], original=ORIGINAL),
                bands=dict(factor=case["factor"], original=ORIGINAL)).get(case["scaling"], {})
    return Rotary(case["rotated"], base=BASE, layout=case["layout"], scaling=case["scaling"] or None, **more)


def _order(case, seed):
    """(pages, blocks of a table row, free pages in the order in which earlier requests gave them back, table rows)."""
    old, new = (torch.tensor(x) for x in _sizes(case))
    blocks = (old + new + case["page"] - 1) // case["page"]
    pages, n = 1 + int(blocks.sum()) + SPARE, case["batch"]
    free = (torch.randperm(pages - 1, device="cuda", generator=_rng(seed, 2)) + 1).to(torch.int32)
    rows = torch.randperm(n + 3, device="cuda", generator=_rng(seed, 3))[:n].to(torch.int32)
    return pages, int(blocks.max()) + 1, free, rows


def _table(case, seed):
    """The requests' pages [batch, blocks]: those of the held tokens are given out first."""
    P = case["page"]
    _, width, free, _ = _order(case, seed)
    old, new = (torch.tensor(x, device="cuda") for x in _sizes(case))
    had, all_ = (old + P - 1) // P, (old + new + P - 1) // P
    block = torch.arange(width, device="cuda")[None]
    at_old = (had.cumsum(0) - had)[:, None] + block
    grown = all_ - had
    at_new = had.sum() + (grown.cumsum(0) - grown)[:, None] + block - had[:, None]
    at = torch.where(block < had[:, None], at_old, at_new).clamp(max=free.numel() - 1)
    return torch.where(block < all_[:, None], free[at].long(), 0)


def _plan(table, old, new, tokens, P):
    """Slots and positions of packed new tokens, and the page entries that they fall into."""
    n = old.numel()
    end = new.cumsum(0)
    t = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(end, t, right=True)
    live = b < n
    b = b.clamp(max=n - 1)
    pos = torch.where(live, old[b] + t - (end - new)[b], -1)
    slot = torch.where(live, table[b, pos.clamp(min=0) // P] * P + pos % P, -1)
    touched = torch.where(new > 0, (old + new + P - 1) // P - old // P, 0)
    ends = touched.cumsum(0)
    i = torch.arange(min(tokens, tokens // P + 2 * n), device="cuda")
    e = torch.searchsorted(ends, i, right=True)
    used = e < n
    e = e.clamp(max=n - 1)
    block = torch.where(used, old[e] // P + i - (ends - touched)[e], 0)
    tile = (ends - touched)[b] + pos // P - old[b] // P
    return dict(old=old, new=new, lens=old + new, positions=pos, slots=slot, live=live, request=b, tile=tile,
                pages=torch.where(used, table[e, block], 0), end=end,
                filled=torch.where(used, (old + new)[e] - block * P, 0).clamp(max=P),
                start=torch.where(used, old[e] - block * P, 0).clamp(min=0))


def prepare(case, seed):
    kind, P, H = case["kind"], case["page"], case["q_heads"]
    old, new = _sizes(case)
    tokens = sum(new) + case["padding"]
    state = dict(case=case, tokens=tokens)
    if kind == "rotary":
        far = torch.randint(0, case["far"] + 1, (tokens,), device="cuda", generator=_rng(seed, 4))
        state["positions"] = (far + torch.arange(tokens, device="cuda")).to(torch.int32)
        state["x"] = _uneven(case, seed, 10, tokens, H, case["dim"])
        if own:
            state["rotary"] = _own_rotary(case)
        else:
            state["frequencies"], state["magnitude"] = _frequencies(case)
        return state
    counts = torch.tensor(new, dtype=torch.int32, device="cuda")
    before = sum(old)
    latent = kind != "append"
    W = case["latent"]
    shape = (W + 64,) if latent else (case["kv_heads"], case["dim"])
    if kind != "expanded":
        held = _uneven(case, seed, 10, before, *shape)
        fresh = _uneven(case, seed, 20, tokens, *shape)
        if not latent:
            held_v, state["v"] = _uneven(case, seed, 30, before, *shape), _uneven(case, seed, 40, tokens, *shape)
    if own:
        from stepquant_amd.kernels.kv_cache import BlockTables, KVCache
        from stepquant_amd.kernels.latent_cache import LatentCache
        pages, width, free, rows = _order(case, seed)
        tables = BlockTables(case["batch"] + 3, pages, width, page_tokens=P)
        tables.free.copy_(free)
        plan = tables.plan(old, rows)
        if kind == "append":
            state["cache"] = KVCache(pages, case["kv_heads"], case["dim"], page_tokens=P, storage=case["storage"])
            state["cache"].append(held, held_v, plan)
        elif kind != "expanded":
            state["cache"] = LatentCache(pages, W, 64, page_tokens=P, dtype=TYPES[case["dtype"]])
            state["cache"].append(held[:, :W], held[:, W:], plan)
        tables.commit(plan)
        forms = {kind: H} if kind in ("absorbed", "expanded") else {}
        plan = tables.plan(counts, rows, tokens=tokens, max_new=max(new), causal=case["causal"], **forms)
        state.update(tables=tables, plan=plan)
    else:
        table = _table(case, seed)
        zero = torch.zeros(case["batch"], dtype=torch.int64, device="cuda")
        was = torch.tensor(old, device="cuda")
        plan = _plan(table, was, counts.long(), tokens, P)
        state.update(table=table, plan=plan)
        pages = _order(case, seed)[0]
        filled = _plan(table, zero, was, before, P)
        if kind == "append":
            shape = (pages, 2, P, case["kv_heads"], case["dim"])
            state["cache"] = dict(codes=torch.zeros(shape, dtype=torch.int8, device="cuda"),
                                  peaks=torch.full((pages, 2, case["kv_heads"]), FLOOR, device="cuda"))
            _quantise(state["cache"], case, torch.stack([held, held_v], 1).float(), filled)
        elif kind != "expanded":
            state["cache"] = torch.zeros((pages, P, W + 64), dtype=TYPES[case["dtype"]], device="cuda")
            state["cache"].view(-1, W + 64)[filled["slots"]] = held
    if kind in ("append", "latent_append", "gather"):
        if own:
            state["rotary"] = _own_rotary(case)
        else:
            state["frequencies"], state["magnitude"] = _frequencies(case)
        state["q"] = _queries(case, seed, 50, tokens, H, 64 if latent else case["dim"])
        if latent:
            state.update(latent=fresh[:, :W], rope=fresh[:, W:], held=sum(old) + sum(new))
        else:
            state["k"] = fresh
    elif kind == "absorbed":
        if own:
            state["cache"].append(fresh[:, :W], fresh[:, W:], plan)
        else:
            live = plan["live"].nonzero()[:, 0]
            state["cache"].view(-1, W + 64)[plan["slots"][live]] = fresh[live]
        q = _queries(case, seed, 50, tokens, H, W + 64)
        state.update(q=q[..., :W].contiguous(), q_rope=q[..., W:].contiguous())
    else:
        D, total = case["dim"], before + sum(new)
        kv = _uneven(case, seed, 10, total, H, 2 * D)
        state.update(k=kv[..., :D], v=kv[..., D:], rope=_uneven(case, seed, 60, total, 64),
                     q=_queries(case, seed, 50, tokens, H, D + 64))
        lens = torch.tensor([0] + [o + n for o, n in zip(old, new)], device="cuda")
        state["starts"] = lens.cumsum(0).to(torch.int32)
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        if kind == "rotary":
            return state["rotary"].apply(state["x"], state["positions"])
        cache, plan = state.get("cache"), state["plan"]
        if kind == "append":
            q = cache.append(state["k"], state["v"], plan, rotary=state["rotary"], q=state["q"])
            return [q, *cache.decode(plan.pages, plan.filled, dtype=TYPES[case["dtype"]])]
        if kind == "latent_append":
            q = cache.append(state["latent"], state["rope"], plan, rotary=state["rotary"], q=state["q"])
            return [q, cache.data]
        if kind == "gather":
            q = cache.append(state["latent"], state["rope"], plan, rotary=state["rotary"], q=state["q"])
            return [q, *cache.gather(plan, tokens=state["held"])]
        if kind == "absorbed":
            return cache.attend(state["q"], state["q_rope"], plan, scale=192 ** -.5)
        from stepquant_amd.kernels.latent_cache import expanded_attention
        return expanded_attention(state["q"], state["k"], state["v"], state["rope"], plan, state["starts"])
    if kind == "rotary":
        return _rotate(state, state["x"].float(), state["positions"]).to(state["x"].dtype)
    if kind == "append":
        return _append(state)
    if kind == "latent_append":
        return [_latent_append(state), state["cache"]]
    if kind == "gather":
        return [_latent_append(state), *_gather(state)]
    return _absorbed(state) if kind == "absorbed" else _expanded(state)


def _rotate(state, x, positions):
    """``x`` [tokens, heads, dim] in 32 bits; rows at negative positions stay."""
    case, n = state["case"], state["case"]["rotated"]
    angle = positions.double().clamp(min=0)[:, None, None] * state["frequencies"].cuda()
    cos, sin = (angle.cos() * state["magnitude"]).float(), (angle.sin() * state["magnitude"]).float()
    y = x.clone()
    if case["layout"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        y[..., :n // 2], y[..., n // 2:n] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :n:2], x[..., 1:n:2]
        y[..., :n:2], y[..., 1:n:2] = a * cos - b * sin, a * sin + b * cos
    return torch.where((positions >= 0)[:, None, None], y, x)


def _round(x, storage):
    """Codes as the numbers they stand for."""
    return x.round() if storage == "int8" else x.to(torch.float8_e4m3fn).float()


def _hold(x, storage):
    return x.to(torch.int8) if storage == "int8" else x.to(torch.float8_e4m3fn).view(torch.int8)


def _held(codes, storage):
    return codes.float() if storage == "int8" else codes.view(torch.float8_e4m3fn).float()


def _quantise(cache, case, x, plan):
    """``x`` [tokens, keys and values, heads, dim] into pages: the block's peak,
    the live codes brought to it where it grew, the new codes."""
    storage, P, pages = case["storage"], case["page"], plan["pages"]
    n = pages.numel()
    # the scratch entry past the last takes the tokens that have no page
    tile = torch.where(plan["live"], plan["tile"], n)
    dense = torch.zeros((n + 1, P, *x.shape[1:]), device="cuda")
    dense[tile, plan["positions"].clamp(min=0) % P] = x
    dense = dense[:n].transpose(1, 2)
    here = torch.arange(P, device="cuda")[None]
    fresh = (here >= plan["start"][:, None]) & (here < plan["filled"][:, None])
    kept = here < plan["start"][:, None]
    fresh, kept = fresh[:, None, :, None, None], kept[:, None, :, None, None]
    before = torch.where(plan["start"][:, None, None] > 0, cache["peaks"][pages], FLOOR)
    peak = torch.maximum(before, torch.where(fresh, dense.abs(), 0.).amax((2, 4))).clamp(min=FLOOR)
    at = peak[:, :, None, :, None]
    was = _held(cache["codes"][pages], storage)
    moved = _round(was * (before[:, :, None, :, None] / at), storage)
    put = _round(dense / at * TOP[storage], storage)
    cache["codes"][pages] = _hold(torch.where(fresh, put, torch.where(kept, moved, was)), storage)
    cache["peaks"][pages] = peak


def _append(state):
    """The rotated queries, and the touched pages dense, zero past their tokens."""
    case, cache, plan = state["case"], state["cache"], state["plan"]
    dtype = TYPES[case["dtype"]]
    k = _rotate(state, state["k"].float(), plan["positions"])
    _quantise(cache, case, torch.stack([k, state["v"].float()], 1), plan)
    there = torch.arange(case["page"], device="cuda")[None] < plan["filled"][:, None]
    x = _held(cache["codes"][plan["pages"]], case["storage"])
    x = x * (cache["peaks"][plan["pages"]] / TOP[case["storage"]])[:, :, None, :, None]
    x = torch.where(there[:, None, :, None, None], x, 0.).to(dtype)
    return [_rotate(state, state["q"].float(), plan["positions"]).to(dtype), x[:, 0], x[:, 1]]


def _latent_append(state):
    case, cache, plan = state["case"], state["cache"], state["plan"]
    rope = _rotate(state, state["rope"].float()[:, None], plan["positions"])[:, 0].to(cache.dtype)
    x = torch.cat([state["latent"], rope], -1)
    # tokens without a slot go to the padding page and are cleared there
    slot = plan["slots"].clamp(min=0)
    cache.view(-1, x.shape[1])[slot] = torch.where(plan["live"][:, None], x, 0)
    return _rotate(state, state["q"].float(), plan["positions"]).to(cache.dtype)


def _gather(state):
    case, plan, W, P = state["case"], state["plan"], state["case"]["latent"], state["case"]["page"]
    end = plan["lens"].cumsum(0)
    t = torch.arange(state["held"], device="cuda")
    b = torch.searchsorted(end, t, right=True)
    pos = t - (end - plan["lens"])[b]
    x = state["cache"][state["table"][b, pos // P], pos % P]
    return x[:, :W], x[:, W:], torch.cat([end.new_zeros(1), end]).int()


def _padded(x, end, count, most):
    """Packed rows [tokens, ...] as [batch, most, ...] in 32 bits, with the rows' places."""
    at = (end - count)[:, None] + torch.arange(most, device="cuda")[None]
    return x[at.clamp(max=x.shape[0] - 1)].float()


def _softmax_rows(s, seen):
    s = s.masked_fill_(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _seen(state, keys):
    """[batch, new tokens, keys] which keys a request's token sees, and that padding rows see one."""
    plan, causal = state["plan"], state["case"]["causal"]
    j = torch.arange(keys, device="cuda")[None, None]
    i = torch.arange(int(state["case"]["new"]), device="cuda")[None, :, None]
    last = plan["old"][:, None, None] + i + 1 if causal else plan["lens"][:, None, None]
    return j < torch.minimum(last, plan["lens"][:, None, None])


def _absorbed(state):
    case, plan, W, P = state["case"], state["plan"], state["case"]["latent"], state["case"]["page"]
    most, H, N, B = max(case["context"] + case["new"], 1), case["q_heads"], case["new"], case["batch"]
    j = torch.arange(most, device="cuda")
    table = state["table"][:, (j // P).clamp(max=state["table"].shape[1] - 1)]
    there = (j[None] < plan["lens"][:, None])[..., None]
    keys = torch.where(there, state["cache"][table, (j % P)[None]].float(), 0.)
    q = _padded(torch.cat([state["q"], state["q_rope"]], -1), plan["end"], plan["new"], N)
    s = torch.matmul(q.view(B, N * H, W + 64), keys.transpose(1, 2)) * 192 ** -.5
    p = _softmax_rows(s.view(B, N, H, most), _seen(state, most)[:, :, None])
    y = torch.matmul(p.view(B, N * H, most), keys[..., :W].contiguous()).view(B, N, H, W)
    out = torch.zeros_like(state["q"])
    live = plan["live"]
    t = (plan["positions"] - plan["old"][plan["request"]]).clamp(min=0)
    return torch.where(live[:, None, None], y[plan["request"], t].to(out.dtype), out)


def _expanded(state):
    case, plan, D = state["case"], state["plan"], state["case"]["dim"]
    most, H, N, B = case["context"] + case["new"], case["q_heads"], case["new"], case["batch"]
    starts = state["starts"].long()
    place = lambda x: _padded(x, starts[1:], plan["lens"], most)
    k = torch.cat([place(state["k"]), place(state["rope"])[:, :, None].expand(B, most, H, 64)], -1)
    q = _padded(state["q"], plan["end"], plan["new"], N)
    s = torch.matmul(q.transpose(1, 2).contiguous(), k.permute(0, 2, 3, 1).contiguous()) * (D + 64) ** -.5
    p = _softmax_rows(s, _seen(state, most)[:, None])
    there = (torch.arange(most, device="cuda")[None] < plan["lens"][:, None])[..., None, None]
    v = torch.where(there, place(state["v"]), 0.)
    y = torch.matmul(p, v.transpose(1, 2).contiguous()).transpose(1, 2)
    out = torch.zeros((state["tokens"], H, D), dtype=state["q"].dtype, device="cuda")
    t = (plan["positions"] - plan["old"][plan["request"]]).clamp(min=0)
    return torch.where(plan["live"][:, None, None], y[plan["request"], t].to(out.dtype), out)


# ---------------------------------------------------------------- in 64 bits
def _e4m3(x):
    """Nearest e4m3 number, ties to even: 3 fraction bits, exponents from -6 up."""
    e = torch.frexp(x)[1]
    unit = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return ((x / unit).round() * unit).clamp(-448, 448)


def _turned(case, x, positions):
    """Pairs as complex numbers, multiplied by the turned unit."""
    f, magnitude = _frequencies(case)
    n = case["rotated"]
    x, head = x.double().clone(), x[..., :n].double()
    pairs = head.unflatten(-1, (2, n // 2)).transpose(-1, -2) if case["layout"] == "half" else head.unflatten(-1, (n // 2, 2))
    z = torch.view_as_complex(pairs.contiguous())
    z = z * torch.polar(torch.full_like(f, magnitude), positions.double().cpu()[:, None] * f).cuda()[:, None]
    pairs = torch.view_as_real(z)
    turned = (pairs.transpose(-1, -2) if case["layout"] == "half" else pairs).flatten(-2)
    live = (positions >= 0)[:, None, None]
    x[..., :n] = torch.where(live, turned, head)
    return x


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    kind, P = case["kind"], case["page"]
    if kind == "rotary":
        return _turned(case, state["x"], state["positions"])
    old, new = _sizes(case)
    plan, W, H, tokens = state["plan"], case["latent"], case["q_heads"], state["tokens"]
    ends = [sum(new[:i + 1]) for i in range(len(new))]
    positions = torch.full((tokens,), -1, dtype=torch.int64, device="cuda")
    for o, n, e in zip(old, new, ends):
        positions[e - n:e] = torch.arange(o, o + n, device="cuda")
    if kind in ("append", "latent_append", "gather"):
        q = _turned(case, state["q"], positions)
    if kind == "append":
        top, cache, table = TOP[case["storage"]], state["cache"], state["table"].cpu()
        out = [torch.zeros((_tiles(case), P, case["kv_heads"], case["dim"]), dtype=torch.float64, device="cuda")
               for _ in range(2)]
        sources, tile, row = (_turned(case, state["k"], positions), state["v"].double()), 0, 0
        for i, (o, n) in enumerate(zip(old, new)):
            done = 0
            while done < n:
                block, start = divmod(o + done, P)
                count = min(P - start, n - done)
                page = int(table[i, block])
                for part, x in enumerate(sources):
                    x = x[row + done:row + done + count]
                    peak = x.abs().amax((0, 2)).clamp(min=FLOOR)
                    if start:
                        before = cache["peaks"][page, part].double()
                        peak = torch.maximum(peak, before)
                        y = _held(cache["codes"][page, part], case["storage"]).double()[:start] * (before / peak)[:, None]
                        y = y.round() if top == 127 else _e4m3(y)
                        out[part][tile, :start] = y * (peak / top)[:, None]
                    y = x / peak[:, None] * top
                    y = y.round() if top == 127 else _e4m3(y)
                    out[part][tile, start:start + count] = y * (peak / top)[:, None]
                done += count
                tile += 1
            row += n
        return [q, *out]
    if kind in ("latent_append", "gather"):
        rope = _turned(case, state["rope"][:, None], positions)[:, 0]
        x = torch.cat([state["latent"].double(), rope], -1)
        data = state["cache"].double()
        live = positions >= 0
        data.view(-1, W + 64)[plan["slots"][live]] = x[live]
        if kind == "latent_append":
            return [q, data]
        rows = [data[state["table"][i, :_blocks(o + n, P)]].flatten(0, 1)[:o + n] for i, (o, n) in enumerate(zip(old, new))]
        rows = torch.cat(rows)
        return [q, rows[:, :W], rows[:, W:], None]
    width = W if kind == "absorbed" else case["dim"]
    out = torch.zeros((tokens, H, width), dtype=torch.float64, device="cuda")
    key = 0
    for i, (o, n, e) in enumerate(zip(old, new, ends)):
        if kind == "absorbed":
            x = state["cache"][state["table"][i, :_blocks(o + n, P)]].flatten(0, 1)[:o + n].double()
        for h in range(0, H, H if kind == "absorbed" and n < 64 else 1):
            if kind == "absorbed":
                heads = H if n < 64 else 1
                q = torch.cat([state["q"][e - n:e, h:h + heads], state["q_rope"][e - n:e, h:h + heads]], -1).double()
                k, v, scale = x, x[:, :W], math.sqrt(192)
            else:
                heads, span = 1, slice(key, key + o + n)
                q, scale = state["q"][e - n:e, h:h + 1].double(), math.sqrt(case["dim"] + 64)
                k, v = torch.cat([state["k"][span, h], state["rope"][span]], -1).double(), state["v"][span, h].double()
            for t0 in range(0, n, 2048):
                t1 = min(n, t0 + 2048)
                s = q[t0:t1].flatten(0, 1) @ k.t().contiguous() / scale
                if case["causal"]:
                    last = torch.arange(o + t0, o + t1, device="cuda").repeat_interleave(heads)[:, None]
                    s[torch.arange(o + n, device="cuda")[None] > last] = -math.inf
                out[e - n + t0:e - n + t1, h:h + heads] = (torch.softmax(s, -1) @ v).view(t1 - t0, heads, width)
        key += o + n
    return out
