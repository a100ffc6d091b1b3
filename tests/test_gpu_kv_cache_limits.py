"""The 8-bit KV cache at the ends of its number ranges, against plain
implementations in 64 bits on the host (MI355X).
"""
import numpy as np
import pytest
import torch

from tests.helpers import dev
from tests.test_gpu_kv_cache import check_append, make, rng

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- writes
@pytest.mark.parametrize("storage", ["int8", "fp8"])
@pytest.mark.parametrize("sizes", [(1e37, 2e37, 3e38), (7e35, 8e35, 1e36, 1e38), (1., 1e30, 3e38), (1e-19, 3e38, 3.1e38)],
                         ids=lambda s: "-".join(map(str, s)))
def test_large_blocks_grow(storage, sizes):
    """Older codes are brought to a finite larger peak, whatever the peaks."""
    print(f"case {storage}, peaks {sizes}", flush=True)
    tables, cache = make(2, 2, 64, 64, storage, 64)
    g = rng(51, len(sizes))
    for size in sizes:
        plan = tables.plan([5, 1])
        x = [torch.from_numpy(g.uniform(-1, 1, (6, 2, 64)) * size).to(dev(), torch.bfloat16) for _ in range(2)]
        check_append(cache, *x, plan)
        tables.commit(plan)
    k, v = cache.decode(plan.pages, plan.filled)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()
