"""A hybrid model's serving loop: recurrent layers over packed state pages and
softmax-attention layers over an 8-bit KV cache.

Random weights of a small model: blocks of three gated-delta layers
(``PackedStatePool``) and one attention layer (``KVCache``), residual
connections, no MLP and no vocabulary.  Prompts of unequal lengths are
prefilled in one call; then every request grows by one position a step, in a
HIP graph that plans its pages, runs the layers and commits the plan without
returning to the host.

    python examples/hybrid_serving.py --requests 16 --prompt 700 --steps 64
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from stepquant_amd.kernels.kv_cache import BlockTables, KVCache  # noqa: E402
from stepquant_amd.kernels.pool import PackedStatePool  # noqa: E402
from stepquant_amd.quantization import QuantizationPlan  # noqa: E402

DIM, PAGE = 128, 64


def normed(x):
    y = x.float()
    return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class Recurrent:
    """One gated-delta layer: q, k of ``heads / 2`` heads, v and gates of ``heads``."""

    def __init__(self, width, heads, slots, rng, dev):
        self.heads, self.keys = heads, heads // 2
        bits = torch.tensor([4, 6, 6, 8] * (heads // 4))[:, None].expand(heads, DIM).contiguous()
        plan = QuantizationPlan("gdn", bits.to(dev), torch.ones(heads, DIM, device=dev))
        self.pool = PackedStatePool(plan, slots, DIM)
        n = 2 * self.keys * DIM + heads * DIM
        draw = lambda *s: (torch.randn(*s, generator=rng, device=dev) * s[0] ** -.5).to(torch.bfloat16)
        self.qkv, self.gates, self.out = draw(width, n), draw(width, 2 * heads), draw(heads * DIM, width)
        self.a_log, self.dt_bias = torch.zeros(2, heads, device=dev, dtype=torch.bfloat16)

    def __call__(self, x, slots, cu=None):
        h = normed(x)
        q, k, v = (h @ self.qkv).split([self.keys * DIM, self.keys * DIM, self.heads * DIM], -1)
        a, b = (h @ self.gates).split(self.heads, -1)
        kw = dict(normalize=True, scale=DIM ** -.5, a_log=self.a_log, dt_bias=self.dt_bias)
        if cu is None:
            y = self.pool.step(q, k, v, a, b, slots, **kw)
        else:
            y = self.pool.extend(q, k, v, a, b, slots, cu, **kw)
        return x + y.reshape(x.shape[0], -1) @ self.out


class Attention:
    """One softmax-attention layer with grouped heads over its own 8-bit pages."""

    def __init__(self, width, q_heads, kv_heads, pages, storage, rng, dev):
        self.q_heads, self.kv_heads = q_heads, kv_heads
        self.cache = KVCache(pages, kv_heads, DIM, page_tokens=PAGE, storage=storage, device=dev)
        draw = lambda *s: (torch.randn(*s, generator=rng, device=dev) * s[0] ** -.5).to(torch.bfloat16)
        self.qkv, self.out = draw(width, (q_heads + 2 * kv_heads) * DIM), draw(q_heads * DIM, width)

    def __call__(self, x, plan):
        q, k, v = (normed(x) @ self.qkv).split([n * DIM for n in (self.q_heads, self.kv_heads, self.kv_heads)], -1)
        self.cache.append(k, v, plan)
        return x + self.cache.attend(q, plan).flatten(1) @ self.out


class Hybrid:
    def __init__(self, requests, tokens, blocks=2, width=1024, heads=8, q_heads=8, kv_heads=2, storage="int8", seed=0):
        dev = torch.device("cuda", torch.cuda.current_device())
        rng = torch.Generator(device=dev).manual_seed(seed)
        rows = -(-tokens // PAGE)
        self.heads = (q_heads, kv_heads)
        self.tables = BlockTables(requests, 1 + requests * rows, rows, page_tokens=PAGE, device=dev)
        # slot 0 of a state pool is the padding slot: request r has slot r + 1
        self.rows = torch.arange(requests, device=dev, dtype=torch.int32)
        self.slots = self.rows.long() + 1
        self.layers = []
        for _ in range(blocks):
            self.layers += [Recurrent(width, heads, requests + 1, rng, dev) for _ in range(3)]
            self.layers.append(Attention(width, q_heads, kv_heads, self.tables.pages, storage, rng, dev))
        for layer in self.layers:
            if isinstance(layer, Recurrent):
                layer.pool.clear(self.slots)

    def prefill(self, x, lengths):
        """``x`` [sum(lengths), width]: every request's prompt."""
        cu = torch.tensor([0] + lengths).cumsum(0)
        plan = self.tables.plan(lengths, self.rows, heads=self.heads)
        for layer in self.layers:
            x = layer(x, plan) if isinstance(layer, Attention) else layer(x, self.slots, cu)
        self.tables.commit(plan)
        return x

    def step(self, x, counts):
        """``x`` [requests, width]: one position of every request (``counts`` ones on the GPU)."""
        plan = self.tables.plan(counts, self.rows, tokens=x.shape[0], max_new=1, heads=self.heads)
        for layer in self.layers:
            x = layer(x, plan) if isinstance(layer, Attention) else layer(x, self.slots)
        self.tables.commit(plan)
        return x


def capture(model, x, counts):
    """(graph, output): ``model.step`` on ``x``, to be replayed; capturing runs nothing."""
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        y = model.step(x, counts)
    return graph, y


def serve(requests=16, prompt=700, steps=64, storage="int8", graph=True, seed=0, **sizes):
    """Prefills prompts of ``prompt`` tokens and less, then decodes; returns the
    prompts' outputs, the last step's, and the seconds of a step."""
    model = Hybrid(requests, prompt + steps + 1, storage=storage, seed=seed, **sizes)
    dev, width = model.slots.device, model.layers[0].qkv.shape[0]
    rng = torch.Generator(device=dev).manual_seed(seed + 1)
    lengths = [max(1, prompt - i * prompt // (2 * requests)) for i in range(requests)]
    first = model.prefill(torch.randn(sum(lengths), width, generator=rng, device=dev).to(torch.bfloat16), lengths)
    counts = torch.ones(requests, dtype=torch.int32, device=dev)
    ends = torch.tensor(lengths, device=dev).cumsum(0) - 1
    x = normed(model.step(normed(first[ends]), counts))  # the first step is always launched: libraries set themselves up
    if graph:
        replay, y = capture(model, x, counts)
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(steps):
        if graph:
            replay.replay()
        else:
            y = model.step(x, counts)
        x.copy_(normed(y))
    torch.cuda.synchronize()
    return first, x, (time.perf_counter() - start) / max(1, steps), model


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--requests", type=int, default=16)
    p.add_argument("--prompt", type=int, default=700, help="longest prompt")
    p.add_argument("--steps", type=int, default=64)
    p.add_argument("--storage", choices=["int8", "fp8"], default="int8")
    p.add_argument("--eager", action="store_true", help="launch every step instead of replaying a graph")
    a = p.parse_args()
    _, out, seconds, model = serve(a.requests, a.prompt, a.steps, a.storage, not a.eager)
    layers = len(model.layers)
    print(f"{a.requests} requests, {layers} layers: {seconds * 1e6:.0f} us a step, "
          f"{a.requests / seconds:.0f} tokens/s, outputs finite: {bool(torch.isfinite(out).all())}")
