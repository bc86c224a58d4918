"""Attention over the cache where blocks of a prompt meet windows and holes.

The oracles are those of test_operators.py.  Tolerances count roundings in the same way.
"""
import math

import pytest
import torch

from test_operators import BF, FP, Cache, attend, check_attend, gen, gpu, randn


# ---------------------------------------------------------------------------
# Prompts whose rows begin to see somewhere inside a block
# ---------------------------------------------------------------------------
def low_scores(cache, q, by):
    """All scores `by` lower, in nats: one element of every key is 127 * 0.05, and of every query what makes that of it."""
    d = q.shape[-1]
    cache.codes[0][..., 0] = 127
    cache.scales[0][..., 0] = torch.where(cache.scales[0][..., 0].isnan(), cache.scales[0][..., 0], 0.05)
    cache.values[0] = cache.codes[0].double() * cache.scales[0].double()
    q = q.clone()
    q[..., 0] = -by * math.sqrt(d) / (127 * 0.05)
    return q


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hq,hk,d", [(2, 2, 128), (2, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("window", [160, 256, 512])
@pytest.mark.parametrize("prefix", [128, 160, 192, 224, 37, 131])
def test_windows_that_begin_inside_a_block(dtype, hq, hk, d, window, prefix):
    """A row's first position may be the first of a step, behind one in which its neighbours see some and it sees none."""
    g = gen(window + prefix + hq)
    queries = [512, 300]
    cache = Cache(g, [queries[0] + prefix, queries[1] + 2 * prefix], hk, d, 32, "int8")
    q = randn(g, sum(queries), hq, d, dtype=dtype)
    out, lse = attend(q, cache, queries, max(queries), window=window)
    check_attend(out, q, cache, queries, lse, window=window)
    q = low_scores(cache, q, 40.0)
    out, lse = attend(q, cache, queries, max(queries), window=window)
    check_attend(out, q, cache, queries, lse, window=window)


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hq,hk", [(2, 2), (8, 2)])
@pytest.mark.parametrize("window", [None, 256])
@pytest.mark.parametrize("holes", [8, 16, 11])
def test_prompts_whose_first_pages_are_gone(dtype, hq, hk, window, holes):
    """Whole steps of positions without a page come first; what follows is seen by all."""
    g = gen(holes + hq)
    queries = [512]
    cache = Cache(g, [900], hk, 128, 16, "int8")
    cache.pages[0, :holes] = -1
    if window:
        cache.pages[0, 26: 26 + holes] = -1
    q = low_scores(cache, randn(g, 512, hq, 128, dtype=dtype), 40.0)
    out, lse = attend(q, cache, queries, 512, window=window)
    check_attend(out, q, cache, queries, lse, window=window)
