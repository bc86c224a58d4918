"""Attention over the cache, rows sorted by expert and verification of drafted tokens
(gpuos_b200.rowops; gpuos_attend, gpuos_order, gpuos_dispatch, gpuos_combine*, gpuos_verify behind it).

CPU tests: refusals of the entry points, before anything is launched.  GPU tests compare each operator with its
definition in 64 bits over types, layouts, strides, odd sizes, masks and padding, then all of them as one step.

Tolerances count roundings: half a step of the output's type, and what 32-bit sums and 16-bit weights may add, as
derived beside each check.
"""
import ctypes
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import gpuos_b200.cabi as C
from gpuos_b200 import rowops as R
from gpuos_b200 import scheduler as S

ROOT = Path(__file__).resolve().parents[1]
DEV = "cuda:0"
gpu = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF, FP, F32]
E4 = torch.float8_e4m3fn


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(dtype, exact):
    """Half a step at `exact`; below the normal numbers (of fp16: 2^-14) the step stays that of the least of them."""
    f = torch.finfo(dtype)
    return f.eps / 2 * exact.abs().clamp(min=f.smallest_normal)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=F32, by=1.0):
    return (torch.randn(*shape, generator=g) * by).to(dtype)


def ref(t):
    return None if t is None else ctypes.byref(C.tensor(t))


def arr(ts):
    return (C.Tensor * max(len(ts), 1))(*[C.tensor(t) for t in ts])


def refused(rc, text):
    assert rc == C.EINVAL
    assert text in C.lib().gpuos_last_error().decode(), C.lib().gpuos_last_error()


# ---------------------------------------------------------------------------
# Refusals (CPU): CPU tensors stand for device memory; nothing is launched.
# ---------------------------------------------------------------------------
def rows_of(choices, count, align):
    n = ctypes.c_int64()
    assert C.lib().gpuos_order_rows(choices, count, align, n) == C.OK
    return n.value


def c_order(experts, places, sources, offsets, counts, align=1):
    return C.lib().gpuos_order(ref(experts), align, ref(places), ref(sources), ref(offsets), ref(counts), None)


def test_order_refuses():
    i32 = torch.int32
    e, p, s, o, c = torch.zeros(6, 2).long(), torch.zeros(6, 2, dtype=i32), torch.zeros(12, dtype=i32), torch.zeros(5, dtype=i32), torch.zeros(4, dtype=i32)
    refused(c_order(e.float(), p, s, o, c), "int32 or int64")
    refused(c_order(e[0], p, s, o, c), "2 dims")
    refused(c_order(e, p[:5], s, o, c), "sizes of experts")
    refused(c_order(e, p.long(), s, o, c), "int32")
    refused(c_order(e, p, s[:11], o, c), "too small")
    refused(c_order(e, p, s, o, c, align=2), "too small")  # 12 + 4 rows
    refused(c_order(e, p, s, o, c, align=0), "align")
    refused(c_order(e, p, s, o, c, align=1 << 17), "align")
    refused(c_order(e, p, s, o[:4], c), "one more")
    refused(c_order(e, p, s, torch.zeros(1026, dtype=i32), torch.zeros(1025, dtype=i32)), "1024")
    refused(c_order(e, p, s, o[:1], c[:0]), "between 1 and 1024")
    refused(c_order(torch.zeros(6, 65).long(), torch.zeros(6, 65, dtype=i32), torch.zeros(390, dtype=i32), o, c), "64 choices")
    refused(c_order(e, p.t().contiguous().t(), s, o, c), "contiguous")
    refused(c_order(e, p, torch.zeros(24, dtype=i32)[::2], o, c), "contiguous")
    both = torch.zeros(12, dtype=i32)
    refused(c_order(e, both.view(6, 2), both, o, c), "overlap")
    assert rows_of(12, 4, 1) == 12
    assert rows_of(12, 4, 2) == 16
    assert rows_of(3, 100, 16) == 48
    assert rows_of(0, 4, 8) == 0
    n = ctypes.c_int64()
    refused(C.lib().gpuos_order_rows(5, 0, 8, n), "experts")
    refused(C.lib().gpuos_order_rows(5, 4, 0, n), "align")
    refused(C.lib().gpuos_order_rows(1 << 31, 4, 1, n), "choices")
    refused(C.lib().gpuos_order_rows(5, 4, 1, None), "NULL")


def test_rows_refuse():
    i32, L = torch.int32, C.lib()
    x, p, s, rows = torch.zeros(6, 8), torch.zeros(6, 2, dtype=i32), torch.zeros(12, dtype=i32), torch.zeros(12, 8)
    w, gw = torch.zeros(6, 2), torch.zeros(6, 2)

    def dispatch(x, p, s, r):
        return L.gpuos_dispatch(ref(x), ref(p), ref(s), ref(r), None)

    def combine(y, p, s, w, o):
        return L.gpuos_combine(ref(y), ref(p), ref(s), ref(w), ref(o), None)

    def grad(g, y, p, s, w, gy, gw):
        return L.gpuos_combine_grad(ref(g), ref(y), ref(p), ref(s), ref(w), ref(gy), ref(gw), None)

    refused(dispatch(x.long(), p, s, rows.long()), "float32, float16 or bfloat16")
    refused(dispatch(x.half(), p, s, rows), "one dtype")
    refused(dispatch(x[:5], p, s, rows), "tokens of places")
    refused(dispatch(x, p, s, rows[:11]), "row of sources")
    refused(dispatch(x, p, s, torch.zeros(12, 7)), "row of sources")
    refused(dispatch(x, p.long(), s, rows), "int32")
    refused(dispatch(torch.zeros(8, 6).t(), p, s, rows), "contiguous")
    refused(dispatch(x, p, s, torch.zeros(12, 16)[:, :8]), "rows must be contiguous")
    refused(dispatch(rows[:6], p, s, rows), "overlap")
    refused(combine(rows, p, s, w.half(), x), "float32")
    refused(combine(rows, p, s, w[:5], x), "sizes of places")
    refused(combine(rows[:11], p, s, w, x), "rows of sources")
    refused(combine(rows, p, s, w, x[:5]), "token of places")
    refused(combine(rows, p, s, w, rows[:6]), "overlap")
    refused(grad(x, rows, p, s, w, None, None), "neither")
    refused(grad(x, None, p, s, w, None, gw), "NULL")
    refused(grad(x, rows.half(), p, s, w, None, gw), "one dtype")
    refused(grad(x, rows, p, s, None, rows.clone(), gw), "NULL")
    refused(grad(x, rows, p, s, w, rows, gw), "overlap")
    refused(grad(x, rows, p, s, w, rows.clone(), w), "overlap")
    refused(grad(x, rows, p, s, w, rows.clone(), gw.half()), "float32")


def c_verify(x, d, u, q, tokens, accepted, t=1.0):
    return C.lib().gpuos_verify(ref(x), ref(d), ref(u), ref(q), ref(tokens), ref(accepted), t, None)


def test_verify_refuses():
    x, d, u, q = torch.zeros(3, 3, 10), torch.zeros(3, 2).long(), torch.zeros(3, 3), torch.zeros(3, 2, 10)
    o, a = torch.zeros(3, 3).long(), torch.zeros(3).long()
    refused(c_verify(x.long(), d, u, q, o, a), "float32, float16 or bfloat16")
    refused(c_verify(x[0], d, u, q, o, a), "3 dims")
    refused(c_verify(x[:, :, :0], d, u, None, o, a), "between 1")
    refused(c_verify(x[:, :0], d, u, None, o, a), "draft + 1")
    refused(c_verify(torch.zeros(1, 65, 2), d, u, None, o, a), "63")
    refused(c_verify(x.transpose(1, 2), d, u, q, o, a), "contiguous")
    for t in (-1.0, float("nan"), float("inf"), 1e-40, 1e31):
        refused(c_verify(x, d, u, q, o, a, t), "temperature")
    refused(c_verify(x, d.float(), u, q, o, a), "int32 or int64")
    refused(c_verify(x, d[:, :1], u, q, o, a), "drafts must be")
    refused(c_verify(x, d, None, q, o, a), "uniforms are needed")
    refused(c_verify(x, d, u.double(), q, o, a), "float32")
    refused(c_verify(x, d, u[:, :2], q, o, a), "uniforms must be")
    refused(c_verify(x, d, u, q[:, :1], o, a), "probs must be")
    refused(c_verify(x, d, u, q.double(), o, a), "probs must be")
    refused(c_verify(x, d, u, q, o.int(), a), "int64")
    refused(c_verify(x, d, u, q, o[:, :2], a), "tokens must be")
    refused(c_verify(x, d, u, q, o, a[:2]), "accepted")
    refused(c_verify(x, o[:, :2], u, q, o, a), "overlap")


def c_attend(q, k, v, ks, vs, pages, lengths, offsets, out, lse=None, longest=1, window=0, scale=1.0, flags=1, work=None):
    return C.lib().gpuos_attend(ref(q), arr([k, v]), arr([ks, vs]), ref(pages), ref(lengths), ref(offsets), ref(out), ref(lse),
                                None if work is None else work.data_ptr(), 0 if work is None else work.numel(), longest, window, scale, flags, None)


def test_attend_refuses():
    q, out = torch.zeros(3, 4, 32), torch.zeros(3, 4, 32)
    k, v = torch.zeros(5, 4, 2, 32, dtype=torch.int8), torch.zeros(5, 4, 2, 32, dtype=torch.int8)
    ks, vs = torch.zeros(5, 4, 2, 1), torch.zeros(5, 4, 2, 1)
    pages, lengths, off = torch.zeros(3, 2).int(), torch.zeros(3).int(), torch.zeros(4).int()

    def call(**new):
        a = dict(q=q, k=k, v=v, ks=ks, vs=vs, pages=pages, lengths=lengths, offsets=None, out=out)
        a.update(new)
        return c_attend(**a)

    refused(call(q=q.double()), "float32, float16 or bfloat16")
    refused(call(q=q[0]), "3 dims")
    refused(call(k=k.float(), v=v.float()), "int8 or float8")
    refused(call(k=k.view(torch.uint8), v=v.view(torch.uint8)), "4-bit")
    refused(call(v=v.view(E4)), "one format")
    refused(call(v=v[:4], vs=vs[:4]), "same sizes")
    refused(call(ks=ks[:, :3], vs=vs), "same pages")
    refused(call(ks=ks.half()), "float32")
    refused(call(k=k[..., :24], v=v[..., :24], q=q[..., :24], out=out[..., :24]), "multiple of 16")
    big = torch.zeros(5, 4, 2, 272, dtype=torch.int8)
    refused(call(k=big, v=big, q=torch.zeros(3, 4, 272), out=torch.zeros(3, 4, 272)), "at most 256")
    refused(call(q=torch.zeros(3, 4, 48)), "one head size")
    refused(call(ks=torch.zeros(5, 4, 2, 2), vs=torch.zeros(5, 4, 2, 2)), "multiple of 32")
    refused(call(q=q[:, :3], out=out[:, :3]), "multiple of the cache's")
    refused(call(pages=pages.float()), "int32 or int64")
    refused(call(lengths=lengths[:2]), "lengths")
    refused(call(q=q[:2], out=out[:2]), "one query")
    refused(call(offsets=off[:3]), "one element more")
    refused(call(offsets=off.float()), "int32 or int64")
    refused(call(longest=0), "longest")
    refused(call(window=-1), "window")
    refused(call(window=3, flags=0), "causal")
    refused(call(flags=2), "unknown flag")
    refused(call(scale=float("nan")), "scale")
    refused(call(out=out.half()), "one dtype")
    refused(call(out=out[:, :2]), "sizes of q")
    refused(call(out=q), "overlap")
    refused(call(out=torch.zeros(3, 1, 32).expand(3, 4, 32)), "overlap itself")
    refused(call(lse=torch.zeros(3, 3)), "lse must be")
    refused(call(lse=torch.zeros(3, 4).half()), "lse must be")
    refused(call(lse=out.view(3, 4, 32)[:, :, 0]), "overlap")
    refused(call(k=k[:, :0], v=v[:, :0], ks=ks[:, :0], vs=vs[:, :0]), "rows")
    refused(call(pages=torch.zeros(3, 1).int().expand(3, 1 << 30)), "2^31")
    n = ctypes.c_int64()
    refused(C.lib().gpuos_attend_workspace(ref(q), ref(k), ref(ks), ref(pages), 0, n), "longest")
    refused(C.lib().gpuos_attend_workspace(ref(q), ref(k), ref(ks), None, 1, n), "NULL")
    refused(C.lib().gpuos_attend_workspace(ref(q[0]), ref(k), ref(ks), ref(pages), 1, n), "dims")
    refused(C.lib().gpuos_attend_workspace(ref(q[:, :3]), ref(k), ref(ks), ref(pages), 1, n), "multiple of the cache's")


def test_python_refusals():
    x = torch.zeros(2, 4)
    o = R.Order(torch.zeros(2, 1).int(), torch.zeros(2).int(), torch.zeros(3).int(), torch.zeros(2).int())
    for f in (lambda: R.order(torch.zeros(2, 1).long(), 2), lambda: R.dispatch(x, o), lambda: R.combine(x, o), lambda: R.combine_grad(x, x, o, x),
              lambda: R.verify(torch.zeros(1, 1, 4), torch.zeros(1, 0).long(), torch.zeros(1, 1)),
              lambda: R.attend(x[None], (x, x), (x, x), x, x)):
        with pytest.raises(RuntimeError, match="must be CUDA"):
            f()
    with pytest.raises(TypeError, match="torch.Tensor"):
        R.order([1, 2], 2)


# ---------------------------------------------------------------------------
# Rows sorted by expert
# ---------------------------------------------------------------------------
def plain_order(experts, count, align):
    t, k = experts.shape
    rows = rows_of(t * k, count, align)
    places, sources = torch.full((t * k,), -1), torch.full((rows,), -1)
    offsets, counts, at = [], [], 0
    for e in range(count):
        mine = (experts.flatten() == e).nonzero()[:, 0]
        offsets.append(at)
        counts.append(len(mine))
        places[mine] = torch.arange(at, at + len(mine))
        sources[at: at + len(mine)] = mine
        at += -(-len(mine) // align) * align
    return places.view(t, k), sources, torch.tensor(offsets + [at]), torch.tensor(counts)


def check_order(experts, count, align, given=None):
    got = R.order(experts.to(DEV) if given is None else given, count, align=align)
    for x, y in zip(got, plain_order(experts.long(), count, align)):
        assert x.dtype == torch.int32 and torch.equal(x.cpu().long(), y)
    return got


@gpu
@pytest.mark.parametrize("tokens,k,count,align", [(0, 2, 4, 1), (0, 2, 4, 8), (1, 1, 1, 1), (1, 1, 1, 64), (8, 8, 64, 1), (33, 3, 7, 4), (100, 6, 1024, 16),
                                                  (1000, 8, 257, 1), (4099, 2, 8, 128), (16001, 8, 60, 1), (70001, 4, 1000, 5), (5, 64, 3, 1)])
@pytest.mark.parametrize("elsewhere", [0.0, 0.4, 1.0])
def test_order(tokens, k, count, align, elsewhere):
    g = gen(tokens + k)
    e = torch.randint(0, count, (tokens, k), generator=g)
    out = torch.rand(tokens, k, generator=g) < elsewhere
    e[out] = torch.tensor([-1, count, -(1 << 40), 1 << 40])[torch.randint(0, 4, (int(out.sum()),), generator=g)]
    check_order(e, count, align)


@gpu
def test_order_of_one_expert_and_of_other_layouts():
    g = gen(1)
    check_order(torch.full((9000, 4), 5), 8, 1)
    check_order(torch.full((900, 4), 5, dtype=torch.int32), 8, 32)
    e = torch.randint(-1, 12, (4, 300), generator=g)
    check_order(e.t(), 12, 1, e.to(DEV).t())
    e = torch.randint(-1, 12, (50, 9), generator=g, dtype=torch.int32)
    check_order(e[::3, 1:8:2], 12, 3, e.to(DEV)[::3, 1:8:2])
    check_order(e[:1].expand(40, 9), 12, 1, e.to(DEV)[:1].expand(40, 9))
    _, experts = R.route(randn(g, 40, 16).to(DEV), 4)
    check_order(experts.cpu(), 16, 1, experts)


def some_order(g, tokens, k, count, align, elsewhere=0.2):
    e = torch.randint(0, count, (tokens, k), generator=g)
    e[torch.rand(tokens, k, generator=g) < elsewhere] = -1
    return R.order(e.to(DEV), count, align=align), plain_order(e, count, align)


SHAPES = [(1, 1, 1, 1, 1), (1, 3, 7, 4, 1), (8, 8, 2048, 64, 1), (33, 2, 1000, 5, 4), (70, 6, 2050, 60, 1), (40, 1, 65, 3, 16), (9, 64, 24, 12, 1), (300, 4, 8200, 16, 8), (2, 2, 12345, 2, 1)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k,hidden,count,align", SHAPES)
def test_dispatch_combine_and_gradient(dtype, tokens, k, hidden, count, align):
    g = gen(tokens * 7 + hidden)
    order, (places, sources, _, _) = some_order(g, tokens, k, count, align)
    x, rows = randn(g, tokens, hidden, dtype=dtype), len(sources)
    at = (sources.clamp(min=0) // k)
    want = torch.where((sources >= 0)[:, None], x[at], torch.zeros((), dtype=dtype))
    assert torch.equal(R.dispatch(x.to(DEV), order).cpu(), want)

    y, w, dout = randn(g, rows, hidden, dtype=dtype), randn(g, tokens, k), randn(g, tokens, hidden, dtype=dtype)
    has = (places >= 0)[..., None].double()
    by = y.double()[places.clamp(min=0)] * has if rows else torch.zeros(tokens, k, hidden, dtype=torch.float64)
    for weights in (None, w):
        ww = torch.ones(tokens, k) if weights is None else w
        exact = (by * ww.double()[..., None]).sum(1)
        size = (by * ww.double()[..., None]).abs().sum(1)
        got = R.combine(y.to(DEV), order, None if weights is None else w.to(DEV)).cpu()
        # one fused product and sum a choice, in 32 bits, then the result's rounding
        assert ((got.double() - exact).abs() <= rounding(dtype, exact) + 1.01 * k * 2.0 ** -24 * size).all()
    gy, gw = R.combine_grad(dout.to(DEV), y.to(DEV), order, w.to(DEV))
    per_row = torch.where(sources >= 0, w.flatten()[sources.clamp(min=0)], torch.zeros(()))
    exact = dout.double()[at] * per_row.double()[:, None] if rows else torch.zeros(0, hidden, dtype=torch.float64)
    # the product in 32 bits, and the result's rounding
    assert ((gy.cpu().double() - exact).abs() <= rounding(dtype, exact) * 1.001 + 1.01 * 2.0 ** -24 * exact.abs()).all()
    exact, size = (by * dout.double()[:, None]).sum(-1), (by * dout.double()[:, None]).abs().sum(-1)
    # a thread's sum of hidden / 256 packs of up to 8, the warp's 5 steps and the 8 warps'
    assert ((gw.cpu().double() - exact).abs() <= 1.01 * (hidden / 256 + 8 + 13) * 2.0 ** -24 * size).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad", [0, 1, 2, 8])
def test_rows_of_other_strides(dtype, pad):
    """Rows as slices of wider ones (16-byte, 4-byte and single-element alignment), weights in other layouts."""
    g = gen(pad)
    t, k, h = 21, 3, 72
    order, plain = some_order(g, t, k, 6, 2)
    wide = randn(g, t, h + 2 * pad, dtype=dtype).to(DEV)
    x = wide[:, pad: pad + h]
    assert torch.equal(R.dispatch(x, order), R.dispatch(x.contiguous(), order))
    rows = len(plain[1])
    y = randn(g, rows, h + 2 * pad, dtype=dtype).to(DEV)[:, pad: pad + h]
    w = randn(g, k, 2 * t).to(DEV)[:, ::2].t()
    assert torch.equal(R.combine(y, order, w), R.combine(y.contiguous(), order, w.contiguous()))
    a, b = R.combine_grad(x, y, order, w), R.combine_grad(x.contiguous(), y.contiguous(), order, w.contiguous())
    assert torch.equal(a[0], b[0]) and torch.allclose(a[1], b[1], rtol=0, atol=1e-5 * h)  # (other packs, another order of sums)
    one = wide[:1, pad: pad + h].expand(t, h)
    assert torch.equal(R.dispatch(one, order), R.dispatch(one.contiguous(), order))


@gpu
def test_empty_rows():
    order = R.order(torch.zeros(0, 4, device=DEV).long(), 8)
    assert R.dispatch(torch.zeros(0, 16, device=DEV), order).shape == (0, 16)
    assert R.combine(torch.zeros(0, 16, device=DEV), order).shape == (0, 16)
    order = R.order(torch.full((5, 2), -1, device=DEV), 8, align=4)
    assert not R.dispatch(torch.ones(5, 16, device=DEV), order).any()
    y = torch.full((32, 16), float("nan"), device=DEV)  # rows of no choice are not read
    assert not R.combine(y, order).any()
    gy, gw = R.combine_grad(torch.ones(5, 16, device=DEV), y, order, torch.ones(5, 2, device=DEV))
    assert not gy.any() and not gw.any()
    assert R.dispatch(torch.ones(5, 0, device=DEV), order).shape == (len(order.sources), 0)


@gpu
def test_rows_named_by_a_wrong_order_stay_inside():
    """Places and sources outside the rows are skipped; nothing else is touched."""
    places = torch.tensor([[0, 7], [-5, 2 ** 31 - 1], [1, 3]], dtype=torch.int32, device=DEV)
    sources = torch.tensor([0, 4, -1, 5, 2 ** 31 - 1, -7], dtype=torch.int32, device=DEV)
    order = R.Order(places, sources, torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV))
    x = torch.arange(24, device=DEV).float().view(3, 8) + 1
    rows = R.dispatch(x, order)
    assert torch.equal(rows[[0, 1, 3]], x[[0, 2, 2]]) and not rows[[2, 5]].any()
    y = torch.arange(48, device=DEV).float().view(6, 8)
    out = R.combine(y, order)
    assert torch.equal(out[0], y[0]) and not out[1].any() and torch.equal(out[2], y[1] + y[3])
    R.combine_grad(x, y, order, torch.ones(3, 2, device=DEV))
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF])
def test_rows_gradients(dtype):
    g = gen(3)
    t, k, h, n = 12, 3, 40, 5
    order, (places, sources, _, _) = some_order(g, t, k, n, 4)
    x, w = randn(g, t, h, dtype=dtype), randn(g, t, k)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    scale = randn(g, len(sources), 1).to(DEV)
    out = R.combine(R.dispatch(xd, order) * scale.to(dtype), order, wd)
    dout = randn(g, t, h, dtype=dtype)
    gx, gw = torch.autograd.grad(out, (xd, wd), dout.to(DEV))
    has = (places >= 0).double()
    sc = scale.to(dtype).cpu().double()[places.clamp(min=0), 0] * has
    xr, wr = x.double().requires_grad_(), w.double().requires_grad_()
    (xr[:, None] * (sc * wr)[..., None]).sum(1).backward(dout.double())
    # every stage rounds to dtype: rows, scaled rows, their gradients (twice), and the result
    size = (dout.double().abs()[:, None] * (sc * w.double()).abs()[..., None]).sum(1)
    assert ((gx.cpu().double() - xr.grad).abs() <= 5 * half_step(dtype) * size + 1e-6 * size).all()
    size = (dout.double() * x.double()).abs().sum(-1, keepdim=True) * sc.abs()
    assert ((gw.cpu().double() - wr.grad).abs() <= 2 * half_step(dtype) * size + 64 * 2.0 ** -24 * size).all()
    if dtype is F32:  # linear in x and in w: a difference is exact but for the sums' rounding
        with torch.no_grad():
            dx, dw = randn(g, t, h).to(DEV), randn(g, t, k).to(DEV)

            def f(a, b):
                return (R.combine(R.dispatch(a, order) * scale, order, b).double() * dout.to(DEV).double()).sum()

            for p, at, grad in (((dx, 0), (xd + dx, wd), gx), ((dw, 1), (xd, wd + dw), gw)):
                change, along = f(*at) - f(xd, wd), (grad.double() * p[0].double()).sum()
                total = (dout.double().abs().sum() * 40).item()
                assert abs(change - along) <= 1e-6 * total
    # only one of the two is needed
    (only,) = torch.autograd.grad(R.combine(R.dispatch(x.to(DEV), order), order, wd).float().sum(), wd)
    assert only.shape == (t, k)
    y = randn(g, len(sources), h, dtype=dtype).to(DEV).requires_grad_()
    (only,) = torch.autograd.grad(R.combine(y, order, w.to(DEV)), y, dout.to(DEV))
    assert torch.equal(only, R.combine_grad(dout.to(DEV), y.detach(), order, w.to(DEV))[0])
    (only,) = torch.autograd.grad(R.combine(y, order), y, dout.to(DEV))
    assert torch.equal(only, R.dispatch(dout.to(DEV), order))
    # gradients of any strides
    (a,) = torch.autograd.grad(R.combine(y, order, w.to(DEV)).sum(), y)
    (b,) = torch.autograd.grad(R.dispatch(xd, order).float().sum(), xd)
    assert torch.equal(a, R.combine_grad(torch.ones(t, h, dtype=dtype, device=DEV), y.detach(), order, w.to(DEV))[0])
    assert torch.equal(b, R.combine(torch.ones(len(sources), h, dtype=dtype, device=DEV), order))


# ---------------------------------------------------------------------------
# Verification of drafted tokens
# ---------------------------------------------------------------------------
def plain_verify(x, drafts, u, probs, temperature):
    """The definition, draft by draft, in 64 bits."""
    b, rows, v = x.shape
    n = rows - 1
    tokens, accepted = torch.full((b, rows), -1), torch.zeros(b).long()
    for s in range(b):
        i, weight = 0, None
        while True:
            z = x[s, i].double()
            top = z[~z.isnan()].max() if (~z.isnan()).any() else torch.tensor(float("nan"))
            ok = not z.isnan().any() and math.isfinite(top)
            d = int(drafts[s, i]) if i < n else -1
            drafted = 0 <= d < v
            if not ok:
                break
            if temperature == 0:
                best = int((z == top).nonzero()[0, 0])
                if drafted and d == best:
                    tokens[s, i] = d
                    i += 1
                    continue
                tokens[s, i] = best
                break
            w = torch.exp((z - top) / temperature)
            total = w.sum()
            if drafted:
                q = probs[s, i].double() if probs is not None else None
                if float(u[s, i]) * (1.0 if q is None else float(q[d])) * total < w[d]:
                    tokens[s, i] = d
                    i += 1
                    continue
                weight = w - q * total if q is not None else w.clone()
                weight = torch.where(weight > 0, weight, 0.0)
                if q is None:
                    weight[d] = 0
            if weight is None or not weight.sum() > 0:
                weight = w
            sums = weight.cumsum(0)
            r = float(u[s, n])
            r = r if r > 0 else 0.0
            over = (sums > r * sums[-1]).nonzero()
            tokens[s, i] = int(over[0, 0]) if r < 1 and len(over) else int((weight > 0).nonzero()[-1, 0])
            break
        accepted[s] = i
    return tokens, accepted


def check_verify(x, drafts, u, probs=None, temperature=1.0, given=None):
    got = R.verify(x.to(DEV) if given is None else given, drafts.to(DEV), None if u is None else u.to(DEV),
                   probs=None if probs is None else probs.to(DEV), temperature=temperature)
    want = plain_verify(x, drafts, u, probs, temperature)
    assert torch.equal(got.accepted.cpu(), want[1]), (got.accepted.cpu(), want[1])
    assert torch.equal(got.tokens.cpu(), want[0])
    return want


def some_drafts(g, b, n, v, dtype, temperature, kind, by=2.0):
    x = randn(g, b, n + 1, v, dtype=dtype, by=by)
    z = x[:, :n].double() + 0.5 * torch.randn(b, n, v, generator=g).double()
    p = (z / (temperature or 1.0)).softmax(-1)
    drafts = torch.multinomial(p.view(b * n, v).float(), 1, generator=g).view(b, n) if n else torch.zeros(b, 0).long()
    if kind is None or temperature == 0:
        drafts = torch.where(torch.rand(b, n, generator=g) < 0.7, x[:, :n].argmax(-1), drafts)
    return x, drafts, torch.rand(b, n + 1, generator=g), None if kind is None or n == 0 else p.to(kind)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [None, F32, BF, FP])
@pytest.mark.parametrize("b,n,v", [(1, 0, 1), (3, 1, 1), (2, 2, 7), (5, 4, 33), (4, 3, 1000), (3, 7, 4097), (2, 63, 300), (2, 1, 50257), (1, 2, 140001)])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 0.0])
def test_verify(dtype, kind, b, n, v, temperature):
    g = gen(b + n + v)
    check_verify(*some_drafts(g, b, n, v, dtype, temperature, kind), temperature)


@gpu
@pytest.mark.parametrize("b,n,v", [(1400, 0, 9000), (300, 2, 5001), (0, 2, 10)])
def test_verify_many_sequences(b, n, v):
    g = gen(b)
    x, d, u, p = some_drafts(g, b, n, v, BF, 0.9, BF)
    check_verify(x, d.int(), u, p, 0.9)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_verify_masks_and_ties(dtype):
    g = gen(5)
    inf, low = float("inf"), torch.finfo(dtype).min
    b, n, v = 6, 2, 4096
    x = randn(g, b, n + 1, v, dtype=dtype)
    x[0, :, 100:] = -inf       # few tokens left
    x[1, 1] = -inf             # a row of nothing
    x[2] = low                 # masks of the lowest value: all alike
    x[3] = 0                   # equal logits: the sums are whole numbers, and the shares fall on their borders
    x[4, 0, :-1] = -inf
    x[5, :, ::2] = low
    drafts = torch.randint(0, 100, (b, n), generator=g)
    drafts[4, 0] = v - 1
    drafts[5] = torch.tensor([3, 2])
    for k in range(8):
        u = torch.rand(b, n + 1, generator=g)
        u[3, n] = k / 8
        u[2, n] = k / 8
        u[3, 0] = 1 / v if k < 4 else 0.0
        check_verify(x, drafts, u, None, 1.0)
        check_verify(x, drafts, u, None, 0.5)
        check_verify(x, drafts, u, None, 0.0)
        q = torch.full((b, n, v), 1 / v)
        check_verify(x, drafts, u, q, 1.0)
        check_verify(x, drafts, u, q.to(BF), 2.0)


@gpu
def test_verify_odd_numbers():
    g = gen(6)
    inf, nan = float("inf"), float("nan")
    b, n, v = 12, 3, 1500
    x, drafts, u, q = some_drafts(g, b, n, v, F32, 1.0, F32)
    x[0, 0, 77] = nan
    x[1, 1, 3] = inf
    x[2, 3, 1499] = nan         # the row behind the drafts
    u[3] = 0.0
    u[4, n] = 1.0
    u[5, n] = nan
    u[6, n] = -3.0
    u[7] = 1 - 2.0 ** -24
    drafts[8] = torch.tensor([-1, 5, 5])
    drafts[9, 1] = v            # outside: the drafts end
    q[10, 0] = 0                # a draft that could not have been drawn: accepted
    q[11, 0, 5:] = nan
    drafts[11, 0] = 700
    for t in (1.0, 0.0):
        check_verify(x, drafts, u, q, t)
        check_verify(x, drafts, u, None, t)
    q[:] = 2.0                  # nothing is left of any row: drawn from the target itself
    u[:, :n] = 0.999
    check_verify(x, drafts, u, q, 1.0)


@gpu
def test_verify_next_to_the_border():
    """Random numbers just below and above p / q, where 32-bit sums would not do."""
    g = gen(7)
    b, n, v = 40, 1, 3000
    x = randn(g, b, 2, v, by=2.0)
    p = x[:, 0].double().softmax(-1)
    drafts = p.argmax(-1)[:, None]
    border = p.gather(1, drafts)[:, 0]
    u = torch.rand(b, 2, generator=g)
    near = border.float()
    for step in (-3, -2, -1, 0, 1, 2, 3):
        at = near.clone()
        for _ in range(abs(step)):
            at = torch.nextafter(at, torch.full_like(at, 2.0 if step > 0 else -1.0))
        u[:, 0] = at
        want = check_verify(x, drafts, u)
        assert bool((want[1] == (at.double() < border)).all())
    # the drawn token, next to where one ends
    x = randn(g, 64, 1, v, by=2.0)
    w = (x[:, 0].double() - x[:, 0].double().amax(-1, keepdim=True)).exp()
    edge = w.cumsum(-1)[:, 1500] / w.sum(-1)
    near = edge.float()
    for at in (near, torch.nextafter(near, torch.zeros(())), torch.nextafter(near, torch.ones(()))):
        check_verify(x, torch.zeros(64, 0).long(), at[:, None].contiguous())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_verify_strides(dtype, shift):
    g = gen(shift)
    b, n, v = 5, 3, 2003
    x, drafts, u, q = some_drafts(g, b, n, v, dtype, 1.0, dtype)
    wide = torch.zeros(n + 1, b, v + 9, dtype=dtype)
    wide[:, :, shift: shift + v] = x.transpose(0, 1)
    given = wide.to(DEV)[:, :, shift: shift + v].transpose(0, 1)
    dd = torch.stack((drafts, drafts), -1).to(DEV)[..., 1]
    uu = torch.stack((u, u), -1).to(DEV)[..., 0]
    qq = torch.zeros(b, n, v + 7, dtype=dtype, device=DEV)
    qq[..., shift: shift + v] = q.to(DEV)
    got = R.verify(given, dd, uu, probs=qq[..., shift: shift + v])
    want = plain_verify(x, drafts, u, q, 1.0)
    assert torch.equal(got.tokens.cpu(), want[0]) and torch.equal(got.accepted.cpu(), want[1])
    one = R.verify(given[:1].expand(b, n + 1, v), dd, uu, probs=qq[..., shift: shift + v])
    want = plain_verify(x[:1].expand(b, n + 1, v), drafts, u, q, 1.0)
    assert torch.equal(one.tokens.cpu(), want[0])


@gpu
def test_verify_draws_as_the_target_alone():
    """First tokens over many random numbers: their shares are the target's, whatever the draft's are."""
    g = gen(9)
    v, b = 6, 60000
    x = torch.randn(1, 2, v, generator=g)
    q = torch.rand(1, 1, v, generator=g).softmax(-1)
    drafts = torch.multinomial(q[0, 0], b, replacement=True, generator=g)[:, None]
    got = R.verify(x.to(DEV).expand(b, 2, v), drafts.to(DEV), torch.rand(b, 2, generator=g).to(DEV), probs=q.to(DEV).expand(b, 1, v))
    share = torch.bincount(got.tokens[:, 0].cpu(), minlength=v).double() / b
    # six standard deviations of a share of b draws
    assert ((share - x[0, 0].double().softmax(-1)).abs() <= 6 * 0.5 / math.sqrt(b)).all()


# ---------------------------------------------------------------------------
# Attention over the cache
# ---------------------------------------------------------------------------
class Cache:
    """A paged cache of random codes; pages that belong to nobody, and rows behind a sequence's
    last one, hold NaN (scales) and the largest codes (e4m3: its NaN)."""

    def __init__(self, g, lengths, heads, d, page, fmt, groups=1, holes=False, wide=False):
        self.lengths, self.page, self.d, self.heads = lengths, page, d, heads
        used = [-(-n // page) for n in lengths]
        width = max(max(used), 1) + (2 if wide else 0)
        pool = sum(used) + 3
        perm = torch.randperm(pool, generator=g)
        self.pages = torch.full((len(lengths), width), -1)
        at = 0
        for s, n in enumerate(used):
            self.pages[s, :n] = perm[at: at + n]
            at += n
        if wide:
            self.pages[self.pages < 0] = torch.tensor([-1, pool, perm[-1].item()])[torch.randint(0, 3, (int((self.pages < 0).sum()),), generator=g)]
        if holes:  # pages that have been let go
            self.pages[torch.rand(self.pages.shape, generator=g) < 0.3] = -1
        self.codes, self.scales, self.values = [], [], []
        live = torch.zeros(pool, page, dtype=torch.bool)
        for s, n in enumerate(lengths):
            for p in range(-(-n // page)):
                if 0 <= self.pages[s, p] < pool:
                    live[self.pages[s, p], : min(page, n - p * page)] = True
        for most in (0.05, 0.02):
            if fmt == "int8":
                codes = torch.randint(-127, 128, (pool, page, heads, d), generator=g).to(torch.int8)
                codes[~live] = -128
            else:
                codes = (torch.randn(pool, page, heads, d, generator=g) * 100).clamp(-448, 448).to(E4)
                codes.view(torch.uint8)[~live] = 0x7F
            scales = torch.rand(pool, page, heads, groups, generator=g) * most + 1e-4
            scales[~live] = float("nan")
            self.codes.append(codes)
            self.scales.append(scales)
            self.values.append((codes.double().unflatten(-1, (groups, -1)) * scales.double()[..., None]).flatten(-2))

    def held(self, i, s, head):
        """(position, element) of sequence s, and which positions have a page."""
        n = self.lengths[s]
        j = torch.arange(n)
        p = self.pages[s, j // self.page] if n else torch.zeros(0).long()
        has = (p >= 0) & (p < len(self.codes[0]))
        return self.values[i][p.clamp(0, len(self.codes[0]) - 1), j % self.page, head], has

    def on(self, dev=DEV):
        return tuple(c.to(dev) for c in self.codes), tuple(s.to(dev) for s in self.scales)


def plain_attend(q, cache, queries, causal=True, window=None, scale=None, first=0):
    """(out, lse, size of what is summed, size of a score's terms), 64 bits."""
    t, hq, d = q.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, lse = torch.zeros(t, hq, d, dtype=torch.float64), torch.full((t, hq), -math.inf, dtype=torch.float64)
    size, terms, at = torch.zeros(t, hq, d, dtype=torch.float64), torch.zeros(t, hq, dtype=torch.float64), first
    for s, n in enumerate(queries):
        for h in range(hq):
            k, has = cache.held(0, s, h // (hq // cache.heads))
            v, _ = cache.held(1, s, h // (hq // cache.heads))
            length = len(k)
            if length == 0 or n == 0:
                continue
            j, last = torch.arange(length)[None], (length - n + torch.arange(n)) if causal else torch.full((n,), length - 1)
            seen = has[None] & (j <= last[:, None])
            if window:
                seen &= j > last[:, None] - window
            k, v = torch.where(has[:, None], k, 0.0), torch.where(has[:, None], v, 0.0)
            z = (q[at: at + n, h].double() @ k.T * scale).masked_fill(~seen, -math.inf)
            norm = torch.logsumexp(z, -1)
            p = torch.where(seen, (z - torch.where(norm > -math.inf, norm, 0.0)[:, None]).exp(), 0.0)
            out[at: at + n, h], lse[at: at + n, h] = p @ v, norm
            size[at: at + n, h] = p @ v.abs() + 2.0 ** -12 * v.abs().amax(0) * seen.any(-1)[:, None]
            terms[at: at + n, h] = (q[at: at + n, h].double().abs() @ k.abs().T * abs(scale)).masked_fill(~seen, 0).amax(-1)
        at += n
    return out, lse, size, terms


def check_attend(got, q, cache, queries, lse=None, first=0, **how):
    want, norm, size, terms = plain_attend(q, cache, queries, first=first, **how)
    d, longest = q.shape[-1], max(cache.lengths) + 1
    # a score: d products summed by tensor cores, 2^-23 a step of 16 and of what they add, and 6 roundings of its scales
    # and of the exponential's argument, the exponential 2^-22; it moves a weight and the sum of weights by as much
    score = 2 * ((d / 16 + 8) * 2.0 ** -23 * terms + 2.0 ** -22)
    # bf16: a weight, a value's scale and their product are 16-bit floats, half a step (2^-11) each; else weights of two
    # parts, 2^-22; the sums over the positions
    weight = 3 * 2.0 ** -11 if q.dtype is BF else 2.0 ** -21
    tol = rounding(q.dtype, want) + size * (weight + score[..., None] + (longest / 16 + 64) * 2.0 ** -23)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol + 1e-30).all()), (err / (tol + 1e-30)).max()
    if lse is not None:
        lse = lse.cpu().double()
        assert torch.equal(lse == -math.inf, norm == -math.inf)
        some = norm > -math.inf
        assert bool(((lse - norm).abs() <= score + (longest / 64 + 64) * 2.0 ** -23 + 2.0 ** -22 * norm.abs())[some].all())


def attend(q, cache, queries, longest=None, pages=torch.int32, **how):
    codes, scales = cache.on()
    off = torch.tensor([0] + queries).cumsum(0).to(DEV)
    return R.attend(q.to(DEV), codes, scales, cache.pages.to(pages).to(DEV), torch.tensor(cache.lengths).to(DEV), offsets=off,
                    longest=longest, lse=True, **how)


RAGGED = [0, 1, 2, 31, 33, 127, 128, 129, 300, 1025]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("d,hq,hk,page", [(128, 4, 1, 16), (64, 8, 8, 7), (256, 6, 2, 64), (80, 3, 3, 1), (16, 16, 2, 100), (192, 5, 1, 256)])
def test_attend_decode(dtype, fmt, d, hq, hk, page):
    g = gen(d + hq)
    cache = Cache(g, RAGGED, hk, d, page, fmt, wide=True)
    q = randn(g, len(RAGGED), hq, d, dtype=dtype, by=2.0)
    codes, scales = cache.on()
    out, lse = R.attend(q.to(DEV), codes, scales, cache.pages.to(DEV), torch.tensor(cache.lengths).to(DEV), lse=True)
    check_attend(out, q, cache, [1] * len(RAGGED), lse)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("d,groups,hq,hk", [(128, 1, 8, 2), (64, 2, 4, 4), (128, 4, 10, 1), (256, 2, 4, 2), (96, 3, 6, 3), (96, 1, 4, 4)])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 1), (True, 50), (False, None)])
def test_attend_queries(dtype, fmt, d, groups, hq, hk, causal, window):
    """Drafts and prompts of ragged lengths: none, more than there are positions, blocks that end inside a query's heads."""
    g = gen(d + groups + hq)
    lengths, queries = [5, 0, 200, 64, 1, 700, 130], [7, 3, 5, 64, 1, 0, 33]
    cache = Cache(g, lengths, hk, d, 16, fmt, groups)
    q = randn(g, sum(queries), hq, d, dtype=dtype, by=2.0)
    for longest in (None, 1, 64):
        out, lse = attend(q, cache, queries, longest, causal=causal, window=window)
        check_attend(out, q, cache, queries, lse, causal=causal, window=window)


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("d,hq,hk,page", [(64, 4, 1, 16), (16, 8, 2, 5), (48, 3, 3, 64), (80, 8, 1, 16), (128, 2, 2, 100), (112, 6, 2, 256)])
@pytest.mark.parametrize("window,causal,holes", [(None, True, False), (70, True, True), (None, False, False)])
def test_attend_prompts(dtype, fmt, d, hq, hk, page, window, causal, holes):
    """Blocks of 256 rows: heads that do not fill them, lengths and blocks that end anywhere, pages that are not there."""
    g = gen(d + hq + page)
    lengths, queries = [400, 1, 300, 131, 700], [400, 1, 129, 140, 65]
    cache = Cache(g, lengths, hk, d, page, fmt, holes=holes)
    q = randn(g, sum(queries), hq, d, dtype=dtype, by=2.0)
    out, lse = attend(q, cache, queries, max(queries), causal=causal, window=window)
    check_attend(out, q, cache, queries, lse, causal=causal, window=window)
    few, _ = attend(q, cache, queries, 1, causal=causal, window=window)  # the other kernel
    check_attend(few, q, cache, queries, causal=causal, window=window)
    # rows that do not lie on 16 bytes, and results between others
    wide = torch.zeros(sum(queries), hq, d + 3, dtype=dtype, device=DEV)
    wide[..., 1: d + 1] = q.to(DEV)
    codes, scales = cache.on()
    room = torch.full((sum(queries), hq, d + 5), 7.0, dtype=dtype, device=DEV)
    off = torch.tensor([0] + queries).cumsum(0).to(DEV)
    R.attend(wide[..., 1: d + 1], codes, scales, cache.pages.to(DEV), torch.tensor(lengths).to(DEV), offsets=off, causal=causal,
             window=window, out=room[..., 2: d + 2])
    assert torch.equal(room[..., 2: d + 2], out) and bool((room[..., :2] == 7).all()) and bool((room[..., d + 2:] == 7).all())


@gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_prompts_odd_numbers(dtype, d):
    """Scores that rise along the positions, queries far apart, scales that are not finite where some do not look."""
    g = gen(d)
    cache = Cache(g, [900], 1, d, 16, "int8")
    queries = [400]
    q = randn(g, 400, 2, d, dtype=dtype)
    # keys like one query, more and more so, and scales of values that rise: maxima are raised again and again
    j = torch.arange(900)
    at = (cache.pages[0, j // 16], j % 16)
    base = torch.randint(-100, 101, (d,), generator=g).to(torch.int8)
    cache.codes[0][at[0], at[1], 0] = base
    cache.scales[0][at[0], at[1], 0, 0] = (j.float() + 1) / 900 * 0.08
    cache.scales[1][at[0], at[1], 0, 0] = torch.exp2(j.float() / 60 - 10)
    q[::3] = (base.float() / 60).to(dtype)
    q[1::3] = (-base.float() / 60).to(dtype)

    def again():
        cache.values = [torch.where(s.isnan(), 0.0, c.double() * s.double()) for c, s in zip(cache.codes, cache.scales)]

    again()
    out, lse = attend(q, cache, queries)
    check_attend(out, q, cache, queries, lse)
    assert float((lse[399, 0] - lse[0, 0]).abs()) > 1  # (it does rise)
    # queries of other sizes, zeros among them, and one with NaN
    q2 = q.clone()
    q2[5] = 0
    q2[6] = (q2[6].float() * 2.0 ** -12).to(dtype)
    q2[7, 0] = (q2[7, 0].float() * 8).to(dtype)
    out, lse = attend(q2, cache, queries)
    check_attend(out, q2, cache, queries, lse)
    q3 = q2.clone()
    q3[9, 1, 3] = float("nan")
    q3[11, 0, 0] = float("inf")
    odd, _ = attend(q3, cache, queries)
    keep = torch.ones(400, 2, dtype=torch.bool)
    keep[9, 1] = keep[11, 0] = False
    assert not odd[~keep.to(DEV)].isfinite().all(-1).any()
    check_attend(torch.where(keep[..., None].to(DEV), odd, out), q2, cache, queries)
    # the last positions' scales are not finite: earlier queries do not see them
    for i, bad in ((1, float("nan")), (1, float("inf")), (0, float("nan"))):
        before = cache.scales[i].clone()
        cache.scales[i][at[0][880:], at[1][880:]] = bad
        for longest in (None, 1):
            odd, _ = attend(q2, cache, queries, longest)
            odd = odd.clone()
            assert not odd[399].isfinite().all()
            odd[380:] = out[380:]  # (query 380 is position 880)
            check_attend(odd, q2, cache, queries)
        cache.scales[i] = before


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("lengths,queries,hq,hk,d", [([20000], [1], 4, 1, 128), ([9000, 3, 15001], [1, 1, 1], 8, 2, 64), ([5000, 7000], [5, 3], 8, 2, 128), ([6000], [4], 2, 2, 256), ([3000, 4000, 1200], [40, 200, 1], 4, 2, 128)])
def test_attend_long(fmt, lengths, queries, hq, hk, d):
    """Lengths that are split over CTAs and joined."""
    g = gen(len(lengths) + d)
    cache = Cache(g, lengths, hk, d, 32, fmt)
    q = randn(g, sum(queries), hq, d, dtype=BF, by=3.0)
    out, lse = attend(q, cache, queries, max(queries), pages=torch.int64)
    check_attend(out, q, cache, queries, lse)
    again = attend(q, cache, queries, max(queries))
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_attend_holes_and_tokens_of_nobody(fmt, dtype):
    g = gen(4)
    cache = Cache(g, [300, 64, 1000], 2, 64, 16, fmt, holes=True)
    queries, d = [3, 64, 40], 64
    q = randn(g, sum(queries) + 9, 4, d, dtype=dtype, by=2.0)
    codes, scales = cache.on()
    off = torch.tensor([4, 7, 71, 111])  # 4 tokens before the first sequence, 5 behind the last
    out, lse = R.attend(q.to(DEV), codes, scales, cache.pages.to(DEV), torch.tensor(cache.lengths).to(DEV), offsets=off.to(DEV), lse=True)
    check_attend(out, q, cache, queries, lse, first=4)
    assert not out[:4].any() and not out[111:].any()
    # offsets and lengths that make no sense stay inside
    for bad, length in (([4, 2, 200, 1 << 40], [300, -5, 1 << 40]), ([-7, 90, 3, 4], [1 << 31, 0, 5])):
        R.attend(q.to(DEV), codes, scales, cache.pages.to(DEV), torch.tensor(length).to(DEV), offsets=torch.tensor(bad).to(DEV))
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_attend_layouts(fmt):
    """Heads before rows, caches that share a buffer, codes of any alignment, one scale a page, queries and results that are slices."""
    g = gen(8)
    cache = Cache(g, [70, 300, 9], 2, 64, 16, fmt)
    codes, scales = cache.on()
    q = randn(g, 3, 4, 64, dtype=BF).to(DEV)
    pages, lengths = cache.pages.to(DEV), torch.tensor(cache.lengths).int().to(DEV)
    want = R.attend(q, codes, scales, pages, lengths)
    check_attend(want, q.cpu(), cache, [1, 1, 1])
    turned = tuple(c.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(c.dtype) for c in codes)
    ts = tuple(s.transpose(1, 2).contiguous().transpose(1, 2) for s in scales)
    assert torch.equal(R.attend(q, turned, ts, pages, lengths), want)
    for by in (1, 4, 8):  # codes that start on a byte, or on four
        moved = []
        for c in codes:
            room = torch.zeros(*c.shape[:3], 64 + 16, dtype=torch.uint8, device=DEV)
            room[..., by: by + 64] = c.view(torch.uint8)
            moved.append(room[..., by: by + 64].view(c.dtype))
        assert torch.equal(R.attend(q, tuple(moved), scales, pages, lengths), want)
    both = torch.stack([c.view(torch.uint8) for c in codes], 3).view(codes[0].dtype)  # keys and values of a head side by side
    assert torch.equal(R.attend(q, (both[:, :, :, 0], both[:, :, :, 1]), scales, pages, lengths), want)
    wide = torch.zeros(3, 12, 80, dtype=BF, device=DEV)
    wide[:, 4:8, 8:72] = q
    out = torch.full((3, 8, 64), 7.0, dtype=BF, device=DEV)
    got = R.attend(wide[:, 4:8, 8:72], codes, scales, pages.t().contiguous().t(), lengths, out=out[:, 2:6])
    assert torch.equal(got, want) and bool((out[:, :2] == 7).all()) and bool((out[:, 6:] == 7).all())
    # one scale for a page and head
    per_page = [torch.rand(len(c), 1, 2, 1, generator=g) * 0.02 for c in codes]
    cache.values = [c.double() * s.double() for c, s in zip(cache.codes, per_page)]
    cache.values = [torch.where(torch.isnan(v), 0.0, v) for v in cache.values]
    got = R.attend(q, codes, tuple(s.to(DEV).expand(-1, 16, -1, -1) for s in per_page), pages, lengths)
    check_attend(got, q.cpu(), cache, [1, 1, 1])


@gpu
def test_attend_odd_numbers():
    """A query with NaN has results of its own; huge, tiny and zero queries; scales far apart."""
    g = gen(10)
    for fmt in ("int8", "e4m3"):
        cache = Cache(g, [200, 100], 1, 64, 16, fmt)
        q = randn(g, 8, 2, 64, dtype=BF)
        q[1, 0, 5] = float("nan")
        q[2] = 0
        q[3] *= 2.0 ** -120
        q[5, 1] *= 30
        queries = [6, 2]
        out, lse = attend(q, cache, queries)
        assert bool(out[1, 0].isnan().all()) and bool(lse[1, 0].isnan())
        q2 = q.clone()
        q2[1, 0, 5] = 0
        out2, lse2 = attend(q2, cache, queries)
        keep = torch.ones(8, 2, dtype=torch.bool)
        keep[1, 0] = False
        assert torch.equal(out[keep.to(DEV)], out2[keep.to(DEV)]) and torch.equal(lse[keep.to(DEV)], lse2[keep.to(DEV)])
        check_attend(out2, q2, cache, queries, lse2)
        # scales of values over many powers of two: each position's share is still its own
        cache.scales[1] = cache.scales[1] * torch.exp2(torch.randint(-20, 20, cache.scales[1].shape, generator=g).float())
        cache.values[1] = cache.codes[1].double() * cache.scales[1].double()
        out, _ = attend(q2, cache, queries)
        check_attend(out, q2, cache, queries)
        # a NaN code is a zero
        if fmt == "e4m3":
            cache.codes[1].view(torch.uint8)[:, ::3, :, 7] = 0x7F
            cache.codes[0].view(torch.uint8)[:, 1::3, :, 9] = 0xFF
            cache.values = [torch.where(c.double().isnan(), 0.0, c.double()) * s.double() for c, s in zip(cache.codes, cache.scales)]
            out, _ = attend(q2, cache, queries)
            check_attend(out, q2, cache, queries)


@gpu
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_attend_scales_and_no_sequences(scale, dtype):
    g = gen(17)
    cache = Cache(g, [300, 40], 1, 64, 16, "int8")
    q = randn(g, 210, 4, 64, dtype=dtype)
    out, lse = attend(q, cache, [200, 10], scale=scale)
    check_attend(out, q, cache, [200, 10], lse, scale=scale)
    out, lse = attend(q[:2], cache, [1, 1], scale=scale)
    check_attend(out, q[:2], cache, [1, 1], lse, scale=scale)
    # no sequence at all, and sequences without a table
    codes, scales = cache.on()
    none = torch.zeros(0, device=DEV).long()
    out, lse = R.attend(q.to(DEV), codes, scales, cache.pages[:0].to(DEV), none, offsets=torch.zeros(1, device=DEV).int(), lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    out = R.attend(q[:2].to(DEV), codes, scales, cache.pages[:, :0].to(DEV), torch.tensor([5, 7], device=DEV))
    assert not out.any()
    assert R.attend(q[:0].to(DEV), codes, scales, cache.pages[:0].to(DEV), none).shape == (0, 4, 64)


@gpu
def test_attend_past_32_bit_offsets():
    pages, page, heads, d = 17000, 256, 8, 128  # 4.4 GB of codes each
    g = gen(11)
    small = Cache(g, [600], heads, d, page, "int8")
    codes = [torch.zeros(pages, page, heads, d, dtype=torch.int8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(pages, page, heads, 1, device=DEV) for _ in range(2)]
    at = torch.tensor([16999, 3, 16990])
    for i in range(2):
        codes[i][at] = small.codes[i][small.pages[0]].to(DEV)
        scales[i][at] = small.scales[i][small.pages[0]].to(DEV)
    q = randn(g, 1, 16, d, dtype=BF)
    out = R.attend(q.to(DEV), tuple(codes), tuple(scales), at[None].to(DEV), torch.tensor([600]).to(DEV))
    check_attend(out, q, small, [1])


@gpu
def test_attend_reads_what_cache_write_wrote():
    g = gen(12)
    for fmt in ("int8", "e4m3"):
        k, v = randn(g, 150, 2, 64, dtype=BF), randn(g, 150, 2, 64, dtype=BF)
        codes, scales = zip(*(R.cache_alloc(12, 16, 2, 64, format=fmt, device=DEV) for _ in range(2)))
        table = torch.randperm(12, generator=g)[:10][None]
        slots = table[0][torch.arange(150) // 16] * 16 + torch.arange(150) % 16
        R.cache_write((k.to(DEV), v.to(DEV)), slots.to(DEV), codes, scales)
        cache = Cache(g, [150], 2, 64, 16, fmt)
        cache.pages = table
        cache.codes, cache.scales = [c.cpu() for c in codes], [s.cpu() for s in scales]
        cache.values = [c.double() * s.double() for c, s in zip(cache.codes, cache.scales)]
        q = randn(g, 5, 4, 64, dtype=BF)
        out, lse = attend(q, cache, [5])
        check_attend(out, q, cache, [5], lse)


@gpu
def test_attend_refuses_gradients_and_counts_as_written():
    g = gen(13)
    cache = Cache(g, [10], 1, 64, 16, "int8")
    codes, scales = cache.on()
    args = (codes, scales, cache.pages.to(DEV), torch.tensor([10], device=DEV))
    q = torch.randn(1, 2, 64, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        R.attend(q, *args)
    with torch.no_grad():
        R.attend(q, *args)
    out = torch.zeros(1, 2, 64, device=DEV)
    before = out._version
    assert R.attend(q.detach(), *args, out=out) is not None and out._version > before
    with pytest.raises(ValueError, match="window"):
        R.attend(q.detach(), *args, window=0)
    with pytest.raises(ValueError, match="gradient"):
        R.attend(q.detach(), *args, out=torch.zeros(1, 2, 64, device=DEV, requires_grad=True))
    with pytest.raises(ValueError, match="a tensor each"):
        R.attend(q.detach(), codes[:1], scales[:1], *args[2:])


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
class Step:
    """A step of a small model with experts: drafted tokens of two sequences go through positions, the cache, attention, the
    router and the experts, and their logits are checked."""

    def __init__(self, seed, fmt="int8"):
        g = gen(seed)
        self.b, self.n, self.hq, self.hk, self.d, self.e, self.k, self.v = 2, 3, 4, 2, 64, 6, 2, 500
        t, h = self.b * (self.n + 1), self.hq * self.d
        self.x = randn(g, t, (self.hq + 2 * self.hk) * self.d, dtype=BF).to(DEV)
        self.gate, self.up, self.out = (randn(g, *s, dtype=BF, by=s[-2] ** -0.5).to(DEV) for s in ((h, self.e), (self.e, h, h), (h, self.v)))
        self.codes, self.scales = zip(*(R.cache_alloc(20, 16, self.hk, self.d, format=fmt, device=DEV) for _ in range(2)))
        self.pages = torch.randperm(20, generator=g)[:10].view(2, 5).int().to(DEV)
        self.past = torch.tensor([70, 33])
        for s in range(2):
            n = int(self.past[s])
            old = (randn(g, n, self.hk, self.d, dtype=BF).to(DEV), randn(g, n, self.hk, self.d, dtype=BF).to(DEV))
            j = torch.arange(n, device=DEV)
            R.cache_write(old, self.pages[s][j // 16].long() * 16 + j % 16, self.codes, self.scales)
        self.f = R.rotary_frequencies(self.d, device=DEV)
        self.drafts = torch.randint(0, self.v, (self.b, self.n), generator=g).to(DEV)
        self.u = torch.rand(self.b, self.n + 1, generator=g).to(DEV)
        self.positions = (self.past[:, None] + torch.arange(self.n + 1)).flatten().to(DEV)
        seq = torch.arange(self.b).repeat_interleave(self.n + 1).to(DEV)
        self.slots = self.pages[seq, self.positions // 16].long() * 16 + self.positions % 16
        self.lengths = (self.past + self.n + 1).to(DEV)
        self.offsets = (torch.arange(self.b + 1) * (self.n + 1)).to(DEV)

    def run(self):
        t = len(self.x)
        q, k, v = self.x.view(t, -1, self.d).split((self.hq, self.hk, self.hk), 1)
        q, k = R.rotary((q, k), self.positions, self.f)
        R.cache_write((k, v), self.slots, self.codes, self.scales)
        y = R.attend(q, self.codes, self.scales, self.pages, self.lengths, offsets=self.offsets, longest=self.n + 1).flatten(1)
        w, e = R.route((y @ self.gate).float(), self.k, renormalize=True)
        order = R.order(e, self.e, align=4)
        rows = R.dispatch(y, order)
        at = torch.arange(len(rows), device=DEV)
        expert = torch.searchsorted(order.offsets[1:].contiguous(), at.int(), right=True).clamp(max=self.e - 1)
        rows = torch.stack([rows @ self.up[i] for i in range(self.e)])[expert, at]
        z = R.combine(rows, order, w)
        logits = ((z + y) @ self.out).view(self.b, self.n + 1, self.v) * 3
        got = R.verify(logits, self.drafts, self.u, temperature=0.8)
        return y, w, e, order, z, logits, rows, got

    def check(self, got):
        y, w, e, order, z, logits, rows, verified = got
        for a, b in zip(order, plain_order(e.cpu(), self.e, 4)):
            assert torch.equal(a.cpu().long(), b)
        exact = (rows.cpu().double()[order.places.cpu().long()] * w.cpu().double()[..., None]).sum(1)
        size = (rows.cpu().double()[order.places.cpu().long()] * w.cpu().double()[..., None]).abs().sum(1)
        assert ((z.cpu().double() - exact).abs() <= rounding(BF, exact) + 2.1 * 2.0 ** -24 * size).all()
        want = plain_verify(logits.cpu(), self.drafts.cpu(), self.u.cpu(), None, 0.8)
        assert torch.equal(verified.tokens.cpu(), want[0]) and torch.equal(verified.accepted.cpu(), want[1])
        cache = Cache(gen(0), self.lengths.tolist(), self.hk, self.d, 16, "int8")
        cache.pages = self.pages.cpu().long()
        cache.codes, cache.scales = [c.cpu() for c in self.codes], [s.cpu() for s in self.scales]
        cache.values = [c.double() * s.double() for c, s in zip(cache.codes, cache.scales)]
        t = len(self.x)
        q, k, _ = self.x.view(t, -1, self.d).split((self.hq, self.hk, self.hk), 1)
        q = R.rotary(q.contiguous(), self.positions, self.f).cpu()
        check_attend(y.view(t, self.hq, self.d), q, cache, [self.n + 1] * self.b)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_step(fmt):
    s = Step(1, fmt)
    s.check(s.run())


@gpu
def test_steps_in_graphs():
    steps = [Step(2), Step(3, "e4m3")]
    graphs, outs = [], []
    for s in steps:
        s.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.run())
        graphs.append(g)
    for s, new in zip(steps, (Step(4), Step(5))):
        for name in ("x", "drafts", "u"):
            getattr(s, name).copy_(getattr(new, name))
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for s, o in zip(steps, outs):
        s.check(o)


@gpu
def test_long_attention_on_two_streams_and_in_two_graphs():
    """Calls with workspaces, overlapping."""
    g = gen(14)
    jobs = []
    for seed in range(2):
        cache = Cache(g, [4000 + seed, 3000], 2, 64, 16, "int8")
        codes, scales = cache.on()
        q = randn(g, 2, 8, 64, dtype=BF)
        args = (q.to(DEV), codes, scales, cache.pages.to(DEV), torch.tensor(cache.lengths).to(DEV))
        jobs.append((q, cache, args, R.attend(*args)))
    streams = [torch.cuda.Stream() for _ in jobs]
    graphs = []
    torch.cuda.synchronize()
    for _, _, args, _ in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = R.attend(*args)
        graphs.append((graph, out))
    got = [[] for _ in jobs]
    for _ in range(20):
        for i, (_, _, args, _) in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                graphs[i][0].replay()
                got[i].append(R.attend(*args))
    torch.cuda.synchronize()
    for i, (q, cache, _, want) in enumerate(jobs):
        check_attend(want, q, cache, [1, 1])
        assert torch.equal(graphs[i][1], want) and all(torch.equal(x, want) for x in got[i])


@gpu
def test_first_calls_inside_a_capture():
    """Nothing is looked up that a capture forbids: a fresh process captures its first calls, of every kernel for attention."""
    code = """
import sys
import torch
sys.path[:0] = [%r, %r]
import test_operators as T
from gpuos_b200 import rowops as R
g = T.gen(3)
cache = T.Cache(g, [1500, 300], 2, 64, 16, "int8")
codes, scales = cache.on()
queries = [200, 5]
q = T.randn(g, sum(queries), 4, 64, dtype=T.BF)
off = torch.tensor([0] + queries).cumsum(0).to(T.DEV)
args = (q.to(T.DEV), codes, scales, cache.pages.to(T.DEV), torch.tensor(cache.lengths).to(T.DEV))
x, u, d = torch.randn(3, 2, 5000, device=T.DEV), torch.rand(3, 2, device=T.DEV), torch.zeros(3, 1, device=T.DEV).long()
e = torch.randint(0, 700, (300, 4), device=T.DEV)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = R.attend(*args, offsets=off)
    v = R.verify(x, d, u)
    order = R.order(e, 700)
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
T.check_attend(out, q, cache, queries)
want = T.plain_verify(x.cpu(), d.cpu(), u.cpu(), None, 1.0)
assert torch.equal(v.tokens.cpu(), want[0])
assert all(torch.equal(a.cpu().long(), b) for a, b in zip(order, T.plain_order(e.cpu(), 700, 1)))
print("as eager")
""" % (str(ROOT), str(ROOT / "tests"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as eager" in r.stdout, r.stderr[-2000:]


@gpu
def test_training_rows_in_a_graph():
    g = gen(15)
    order, plain = some_order(g, 64, 2, 6, 8)
    x, w = randn(g, 64, 128, dtype=BF).to(DEV), randn(g, 64, 2).to(DEV)
    dout = randn(g, 64, 128, dtype=BF).to(DEV)

    def step(a, b):
        rows = R.dispatch(a, order)
        R.combine(rows, order, b)
        gy, gw = R.combine_grad(dout, rows, order, b)
        return R.combine(gy, order), gw

    want = step(x, w)
    torch.cuda.synchronize()
    # an eager graph of the same leaves is alive while the calls are captured
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    eager = R.combine(R.dispatch(xl, order), order, wl)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        got = step(xl, wl)
    graph.replay()
    torch.cuda.synchronize()
    gx, gw = torch.autograd.grad(eager, (xl, wl), dout)
    for a, b, c in zip(got, want, (gx, gw)):
        assert torch.equal(a, b) and torch.equal(a, c)


@gpu
@pytest.mark.parametrize("mode", ["persistent", "stream"])
def test_inside_a_scheduler_context(mode, monkeypatch):
    monkeypatch.setenv("GPUOS_MODE", mode)
    monkeypatch.setenv("GPUOS_SCHEDULER_DISABLE_JIT", "0")
    g = gen(16)
    order, _ = some_order(g, 8, 2, 4, 1)
    a, b = randn(g, 8, 32).to(DEV), randn(g, 8, 32).to(DEV)
    x = randn(g, 2, 1, 100).to(DEV)
    u, none = torch.rand(2, 1, generator=g).to(DEV), torch.zeros(2, 0, device=DEV).long()
    cache = Cache(g, [40], 1, 32, 16, "int8")
    codes, scales = cache.on()
    more = (codes, scales, cache.pages.to(DEV), torch.tensor([40], device=DEV))
    q = randn(g, 1, 2, 32).to(DEV)
    plain = (R.combine(R.dispatch(a * b, order), order) + a, R.verify(x + x, none, u).tokens, R.attend(q * q, *more) + q)
    with torch.no_grad(), S.scheduler_context(auto_flush_ms=None):
        got = (R.combine(R.dispatch(a * b, order), order) + a, R.verify(x + x, none, u).tokens, R.attend(q * q, *more) + q)
    torch.cuda.synchronize()
    for p, y in zip(plain, got):
        assert torch.equal(p, y)


@gpu
def test_errors_leave_the_device_usable():
    x = torch.randn(4, 8, device=DEV)
    order = R.order(torch.zeros(4, 2, device=DEV).long(), 2)
    with pytest.raises(ValueError, match="tokens of places"):
        R.dispatch(x[:3], order)
    with pytest.raises(ValueError, match="sizes of places"):
        R.combine(x.repeat(2, 1), order, x)
    with pytest.raises(ValueError, match="count"):
        R.order(torch.zeros(4, 2, device=DEV).long(), 0)
    with pytest.raises(ValueError, match="align"):
        R.order(torch.zeros(4, 2, device=DEV).long(), 4, align=0)
    with pytest.raises(ValueError, match="temperature"):
        R.verify(x[None], torch.zeros(1, 3, device=DEV).long(), torch.zeros(1, 4, device=DEV), temperature=-1)
    with pytest.raises(TypeError):
        R.verify(x[None], torch.zeros(1, 3, device=DEV).long(), torch.zeros(1, 4, device=DEV), probs=torch.zeros(1, 3, 8, device=DEV).to(torch.complex64))
    with pytest.raises(NotImplementedError):
        import torch.autograd.forward_ad as fwd
        with fwd.dual_level():
            R.dispatch(fwd.make_dual(x, x), order)
    assert torch.equal(R.dispatch(x, order)[:4].sum(), R.dispatch(x, order)[:4].sum())
