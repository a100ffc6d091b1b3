"""The hybrid serving example with rotary positions and with latent attention
layers: steps in a graph against the same steps launched eagerly, and its
layers against plain attention in 64 bits (MI355X)."""
import math

import pytest
import torch

from tests.helpers import dev
from tests.test_gpu_hybrid_example import SMALL, example

pytestmark = pytest.mark.gpu


def turn(x, pos, half):
    """``x`` [tokens, heads, dim] at ``pos`` [tokens], base 10000, in 64 bits."""
    n = x.shape[-1] // 2
    t = pos.double()[:, None, None] * 10000. ** (-torch.arange(n, dtype=torch.float64, device=x.device) / n)
    a, b = (x[..., :n], x[..., n:]) if half else (x[..., 0::2], x[..., 1::2])
    y = [a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()]
    return torch.cat(y, -1) if half else torch.stack(y, -1).flatten(-2)


def attention(q, k, v, scale):
    """The last rows' [tokens, heads, dim] attention over [keys, heads, dim], causal."""
    n, new = k.shape[0], q.shape[0]
    s = torch.einsum("tgd,jgd->tgj", q, k) * scale
    hidden = torch.arange(n, device=q.device) > torch.arange(n - new, n, device=q.device)[:, None]
    return torch.einsum("tgj,jgd->tgd", torch.softmax(s.masked_fill(hidden[:, None], -math.inf), -1), v)


@pytest.mark.parametrize("kind", [dict(rotary=True), dict(latent=256), dict(latent=512)], ids=["rotary", "256", "512"])
def test_graph_steps_are_the_eager_ones(kind):
    m = example()
    dev()
    a = m.serve(steps=5, graph=True, **kind, **SMALL)
    b = m.serve(steps=5, graph=False, **kind, **SMALL)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.isfinite(a[1]).all()
    assert a[3].tables.lens.tolist() == b[3].tables.lens.tolist()
    for x, y in zip(a[3].layers, b[3].layers):
        if not isinstance(x, m.Recurrent):
            assert torch.equal(x.cache.data, y.cache.data)


@pytest.mark.parametrize("kind", [dict(rotary=True), dict(latent=256)], ids=["rotary", "latent"])
def test_steps_attend_over_prompts_and_steps(kind):
    m = example()
    model = m.Hybrid(2, 200, blocks=1, width=256, heads=4, q_heads=4, kv_heads=2, **kind)
    layer, latent = model.layers[-1], bool(model.latent)
    kept, errors = [[], []], []

    def call(x, plan, *held):
        y = type(layer).__call__(layer, x, plan, *held)
        h, cu = m.normed(x), plan.cu.tolist()
        for r in range(2):
            here = slice(cu[r], cu[r + 1])
            if latent:
                q = (h[here] @ layer.q).double().unflatten(1, (4, 192))
                c = (h[here] @ layer.down).double()
            else:
                q, c = ((h[here] @ layer.qkv).double().split([512, 512], -1))
                q = q.unflatten(1, (4, 128))
            kept[r].append(c)
            c = torch.cat(kept[r])
            at = torch.arange(c.shape[0], device=x.device)
            new = at[-q.shape[0]:]
            if latent:
                k, v = ((c[:, :256] @ w.double()).unflatten(1, (4, 128)) for w in (layer.keys, layer.values))
                rope = turn(c[:, None, 256:], at, False).expand(-1, 4, -1)
                q = torch.cat([q[..., :128], turn(q[..., 128:], new, False)], -1)
                o = attention(q, torch.cat([k, rope], -1), v, 192 ** -.5)
            else:
                k, v = (z.unflatten(1, (2, 128)).repeat_interleave(2, 1) for z in c.split(256, -1))
                o = attention(turn(q, new, True), turn(k, at, True), v, 128 ** -.5)
            want = o.flatten(1) @ layer.out.double()
            errors.append(float((y[here].double() - x[here].double() - want).norm() / want.norm()))
        return y

    model.layers[-1] = type("Checked", (type(layer),), {"__init__": lambda self: None, "__call__": lambda self, *a: call(*a)})()
    lengths = [70, 121]
    g = torch.Generator(device=dev()).manual_seed(3)
    x = model.prefill(torch.randn(191, 256, generator=g, device=dev()).to(torch.bfloat16), lengths)
    x = m.normed(x[[69, 190]])
    counts = torch.ones(2, dtype=torch.int32, device=dev())
    for _ in range(5):
        x = m.normed(model.step(x, counts))
    assert len(errors) == 12
    # 8-bit keys and values as without positions: .03.  Latents: half steps of 2^-8
    # of the result (a 2^-9 of the root mean square) for queries, latents, keys,
    # values, weights, outputs, their product, the sum that x is added to (x is of the
    # size of the result or up to eight times larger: 2^-6), in all below 8 * 2^-9 + 2^-6.
    assert max(errors) < (.032 if latent else .03), errors
