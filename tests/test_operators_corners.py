"""Attention over the cache where blocks of a prompt meet windows and holes, where scales of values lie far apart, and where
prompts are many blocks of few rows; verification of rows whose maximum rises all along.

The oracles are those of test_operators.py.  Tolerances count roundings in the same way.
"""
import math

import pytest
import torch

from gpuos_b200 import rowops as R
from test_operators import BF, DEV, F32, FP, TYPES, Cache, attend, c_attend, check_attend, gen, gpu, plain_attend, randn, refused


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


# ---------------------------------------------------------------------------
# Scales of values that a query does not see
# ---------------------------------------------------------------------------
def mixed(got, other, take):
    """Rows `take` of `got`, the others of `other`."""
    return torch.where(take.to(got.device)[:, None, None], got, other.to(got.device))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,groups,hq,hk", [(128, 1, 4, 1), (64, 1, 2, 2), (64, 2, 2, 1), (256, 1, 2, 1)])
@pytest.mark.parametrize("queries,longest", [(5, None), (40, 1), (400, None)])
@pytest.mark.parametrize("up", [16, 30, 90])
def test_scales_of_positions_that_are_not_seen(dtype, d, groups, hq, hk, queries, longest, up):
    """Scales of values 2^up larger at the last positions, and at some before the windows: queries that do not see them have
    their results as if they were not there, and those that do are dominated by them."""
    g = gen(d + queries + up)
    n, window = 700, 300
    cache = Cache(g, [n], hk, d, 16, "int8", groups)
    q = randn(g, queries, hq, d, dtype=dtype)
    j = torch.arange(n)
    at = (cache.pages[0, j // 16], j % 16)
    last = n - queries + torch.arange(queries)
    for where, how in ((slice(n - queries // 2, n), {}), (slice(0, n - window - queries // 2 + 1), {"window": window})):
        ordinary, values = cache.scales[1].clone(), cache.values[1]
        out, _ = attend(q, cache, [queries], longest, **how)
        cache.scales[1][at[0][where], at[1][where]] *= 2.0 ** up
        odd, _ = attend(q, cache, [queries], longest, **how)
        free = last < where.start if "window" not in how else last - window >= where.stop - 1
        assert 0 < int(free.sum()) < queries
        check_attend(mixed(odd, out, free), q, cache, [queries], **how)  # (cache.values are the ordinary ones)
        cache.values[1] = (cache.codes[1].double().unflatten(-1, (groups, -1)) * cache.scales[1].double()[..., None]).flatten(-2)
        want = plain_attend(q, cache, [queries], **how)[0]
        if float(want.abs().max()) < torch.finfo(dtype).max:
            check_attend(mixed(odd, want.to(dtype), ~free), q, cache, [queries], **how)
        cache.scales[1], cache.values[1] = ordinary, values


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [6, 300])
def test_scales_that_fall_by_much(dtype, queries):
    """The largest scales are seen first, in a window's first positions or by some rows only; small ones follow, and the other
    way round."""
    g = gen(queries)
    n = 900
    for window, steps in ((None, 0.5), (None, -0.5), (400, 0.1), (400, -0.1), (400, -0.5)):
        cache = Cache(g, [n], 2, 64, 16, "e4m3")
        j = torch.arange(n)
        cache.scales[1][cache.pages[0, j // 16], j % 16] = torch.exp2((j.float() - 450) * steps * 0.2)[:, None, None]
        cache.values[1] = torch.where(cache.scales[1].isnan(), 0.0, cache.codes[1].double() * cache.scales[1].double())
        q = randn(g, queries, 4, 64, dtype=dtype)
        out, lse = attend(q, cache, [queries], window=window)
        want = plain_attend(q, cache, [queries], window=window)[0]
        fits = (want.abs() < torch.finfo(dtype).max / 2).all(-1, keepdim=True)  # (the others are not numbers of this type)
        check_attend(torch.where(fits.to(DEV), out.double(), want.to(DEV)), q, cache, [queries], lse, window=window)


# ---------------------------------------------------------------------------
# Prompts that are taken few rows at a time: many blocks of a sequence, shared out over the GPU
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype,d,groups", [(F32, 64, 1), (BF, 64, 2), (FP, 256, 1), (BF, 256, 1)])
@pytest.mark.parametrize("hq,hk", [(16, 1), (6, 2)])
@pytest.mark.parametrize("queries", [[600, 700, 0, 300, 1], [1, 0, 520], [0, 1, 1, 640, 0, 0, 650, 5, 500], [1] * 130 + [400, 450] + [2] * 150])
@pytest.mark.parametrize("window", [None, 90])
def test_prompts_of_few_rows(dtype, d, groups, hq, hk, queries, window):
    """Sequences of many blocks beside one another, and beside single tokens and none."""
    g = gen(len(queries) + d)
    lengths = [n + int(torch.randint(0, 200 if len(queries) < 100 else 20, (1,), generator=g)) for n in queries]
    cache = Cache(g, lengths, hk, d, 64, "int8", groups)
    q = randn(g, sum(queries), hq, d, dtype=dtype)
    out, lse = attend(q, cache, queries, max(queries), window=window)
    check_attend(out, q, cache, queries, lse, window=window)


@gpu
def test_prompts_of_few_rows_cost_what_their_products_do():
    """2048 queries of 16 heads are 2048 blocks of 16 rows: finding each must not walk over the others.  Against 64 queries behind
    4096 positions, a (query, position) took 30 times as long where it did."""

    def per_product(queries, length):
        g = torch.Generator(device=DEV).manual_seed(1)
        codes = tuple(torch.randint(-127, 128, (length // 64, 64, 2, 128), generator=g, device=DEV, dtype=torch.int8) for _ in range(2))
        scales = tuple(torch.rand(length // 64, 64, 2, 1, generator=g, device=DEV) * 0.05 for _ in range(2))
        q = torch.randn(queries, 32, 128, generator=g, device=DEV)
        pages, n = torch.arange(length // 64, device=DEV)[None], torch.tensor([length], device=DEV)
        offsets, times = torch.tensor([0, queries], device=DEV), []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            R.attend(q, codes, scales, pages, n, offsets=offsets, longest=queries)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times) / (queries * (length - queries / 2))

    assert per_product(2048, 2048) < 6 * per_product(64, 4096 + 64)


# ---------------------------------------------------------------------------
# Verification of rows whose maximum rises all along
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("v,rise", [((1 << 24) - 1, 0.4), ((1 << 24) - 1, 6.0), (1 << 22, 1.0), (300001, 3.0)])
def test_verify_rising_rows(v, rise):
    """A thread's sum is brought to a new maximum at each of its steps, up to 256 times; random numbers next to p."""
    x = torch.stack((torch.linspace(0, rise, v), torch.zeros(v)))[None]
    drafts = torch.tensor([[v - 1 - v // 3]])
    p = x[0, 0].double().softmax(-1)[drafts[0, 0]]
    for by in (-2.0 ** -12, -2.0 ** -14, -2.0 ** -16, -2.0 ** -20, 2.0 ** -20, 2.0 ** -16, 2.0 ** -14, 2.0 ** -12):
        u = torch.tensor([[float(p * (1 + by)), 0.5]])
        got = R.verify(x.to(DEV), drafts.to(DEV), u.to(DEV))
        assert int(got.accepted) == int(u[0, 0].double() < p)


# ---------------------------------------------------------------------------
# Refusals (CPU)
# ---------------------------------------------------------------------------
def test_attend_refuses_scales_that_leave_32_bits():
    """Times log2(e) they would be infinite: 2.36e38 is the last that is not."""
    q, pages, lengths = torch.zeros(1, 2, 32), torch.zeros(1, 1).int(), torch.zeros(1).int()
    k, v, ks, vs = *(torch.zeros(1, 4, 1, 32, dtype=torch.int8) for _ in range(2)), *(torch.zeros(1, 4, 1, 1) for _ in range(2))
    for scale in (3e38, -3e38, 2.4e38, math.inf, -math.inf, math.nan):
        refused(c_attend(q, k, v, ks, vs, pages, lengths, None, torch.zeros(1, 2, 32), scale=scale), "scale")
