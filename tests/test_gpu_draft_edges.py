"""Edges of the drafted-token operators on the GPU: counts and scales at the ends of what they may be, caches that hold rows of
zeros, what a caller may change between two calls."""
import numpy as np
import pytest
import torch

import draftref as ref
from test_gpu_draft import BF16, DEV, F16, F32, assert_within, gen, half_step, held_rows, i64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("store", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("none", [0, -1, -64, -(1 << 32) + 5, -(1 << 62)])
def test_keep_of_no_rows_leaves_the_cache(store, none):
    """A count of zero or less keeps nothing: codes and scales of every layer are as they were, the other sequences' rows move.
    The path's storage goes on behind its rows with numbers that are slots of the cache, so a read behind a row would show."""
    from sparse_transformers_b200 import KVCache

    L, B, kv, rows, hd = 2, 3, 2, 400, 32
    cache = KVCache(B, kv, rows, hd, dtype=F16, store=store, layers=L, device=DEV)
    g = gen(1)
    for i in range(L):
        x = torch.randn(B, rows, kv, hd, generator=g, device=DEV).to(F16)
        cache.layer(i).append(x, -2 * x, torch.zeros(B, dtype=torch.long, device=DEV))
    held = [t for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale) if t is not None]
    was = [t.clone() for t in held]
    block = torch.arange(B * 300, device=DEV).view(B, 300) % 90 + 7
    start, counts = i64(3, 10, 20), i64(none, 4, none)
    cache.keep(start, block[:, :64], counts)
    for now, old in zip(held, was):
        want = old.clone()
        for i in range(4):
            want[:, 1, :, 10 + i] = old[:, 1, :, 10 + int(block[1, i])]
        assert torch.equal(now, want)
