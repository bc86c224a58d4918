"""The row operators (gpuos_b200.rowops and the gpuos_rotary, gpuos_cache_*,
gpuos_route*, gpuos_logprobs* entry points behind it).

CPU tests: every refusal of the entry points comes back as a status before
anything is launched, and the host-side frequencies.  GPU tests compare each
operator with its definition in 64 bits (the cache with its own 32-bit
arithmetic, bit for bit), over dtypes, layouts, strides, odd sizes, masks and
padding, then the operators together as a decode step uses them.

Tolerances count roundings: half a step of the output's type (eps / 2 of the
value), and what 32-bit intermediates may add, as derived beside each check.
"""
import ctypes
import itertools
import math

import numpy as np
import pytest
import torch

import gpuos_b200.cabi as C
from gpuos_b200 import rowops as R
from gpuos_b200 import scheduler as S

DEV = "cuda:0"
gpu = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF, FP, F32]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=F32, by=1.0):
    return (torch.randn(*shape, generator=g) * by).to(dtype)


# ---------------------------------------------------------------------------
# Refusals (CPU): the C ABI, with CPU tensors standing for device memory; every
# one of these returns before the first CUDA call.
# ---------------------------------------------------------------------------
def ref(t):
    return None if t is None else ctypes.byref(C.tensor(t))


def arr(ts):
    return (C.Tensor * max(len(ts), 1))(*[C.tensor(t) for t in ts])


def refused(rc, text):
    assert rc == C.EINVAL
    assert text in C.lib().gpuos_last_error().decode(), C.lib().gpuos_last_error()


def c_rotary(xs, outs, pos, f, scale=1.0, flags=0, n=None):
    return C.lib().gpuos_rotary(len(xs) if n is None else n, arr(xs), arr(outs), ref(pos), ref(f), scale, flags, None)


def test_rotary_refuses():
    x, pos = torch.zeros(4, 2, 16), torch.arange(4)
    f = torch.ones(8, dtype=torch.float64)
    o = torch.zeros_like(x)
    refused(c_rotary([x], [o], pos, f, n=0), "one or two")
    refused(c_rotary([x], [o], pos, f, n=3), "one or two")
    refused(c_rotary([x], [o], pos, f, flags=4), "unknown flag")
    refused(c_rotary([x], [o], pos, f, scale=float("nan")), "scale")
    refused(c_rotary([x], [o], pos, f, scale=float("inf")), "scale")
    refused(c_rotary([x], [o], pos, f, scale=-1.0), "scale")
    refused(c_rotary([x], [o], pos.float(), f), "int32 or int64")
    refused(c_rotary([x], [o], torch.arange(5), f), "token sizes")
    refused(c_rotary([x], [o], pos, torch.ones(9, dtype=torch.float64)), "more pairs")
    refused(c_rotary([x], [o], pos, torch.ones(8, dtype=torch.int64)), "float64 or float32")
    refused(c_rotary([x], [o.to(BF)], pos, f), "one dtype")
    refused(c_rotary([x.long()], [o.long()], pos, f), "float32, float16 or bfloat16")
    refused(c_rotary([x], [torch.zeros(4, 2, 18)], pos, f), "sizes of x")
    refused(c_rotary([x], [torch.zeros(4, 1, 16).expand(4, 2, 16)], pos, f), "overlap itself")
    refused(c_rotary([x.transpose(1, 2)], [o.transpose(1, 2)], pos, torch.ones(1, dtype=torch.float64)), "contiguous")
    refused(c_rotary([x[0]], [o[0]], pos, f), "3 dims")
    refused(c_rotary([x, torch.zeros(5, 2, 16)], [o, torch.zeros(5, 2, 16)], pos, f), "same tokens")
    refused(c_rotary([x, torch.zeros(4, 2, 16)], [o, o], pos, f), "outputs overlap")
    big = torch.zeros(5, 2, 16)
    refused(c_rotary([big[:4]], [big[1:]], pos, f), "not overlap")
    refused(c_rotary([x, big[1:]], [big[:4], o], pos, f), "another input")
    refused(c_rotary([torch.zeros(4, 2, 17)], [torch.zeros(4, 2, 17)], pos, f, flags=1), "even head")
    refused(C.lib().gpuos_rotary(1, arr([x]), arr([o]), None, ref(f), 1.0, 0, None), "NULL")
    t = C.tensor(x)
    t.data = x.data_ptr() + 2
    refused(C.lib().gpuos_rotary(1, (C.Tensor * 1)(t), arr([o]), ref(pos), ref(f), 1.0, 0, None), "aligned")
    t = C.tensor(x)
    t.strides[0] = -32
    refused(C.lib().gpuos_rotary(1, (C.Tensor * 1)(t), arr([o]), ref(pos), ref(f), 1.0, 0, None), "negative stride")
    t.strides[0] = 1 << 61
    refused(C.lib().gpuos_rotary(1, (C.Tensor * 1)(t), arr([o]), ref(pos), ref(f), 1.0, 0, None), "too large")


def test_side_by_side_slices_do_not_overlap():
    """Queries and keys as slices of one row: their spans cross, their elements
    do not.  Nothing is launched: there are no pairs and nothing to copy (in place)."""
    for order in ("token", "head"):
        qkv = torch.zeros(6, 12, 16) if order == "token" else torch.zeros(12, 6, 16).transpose(0, 1)
        q, k = qkv[:, :8], qkv[:, 8:10]
        f = torch.ones(0, dtype=torch.float64)
        assert c_rotary([q, k], [q, k], torch.arange(6), f) == C.OK
        refused(c_rotary([q, qkv[:, 7:9]], [q, qkv[:, 7:9]], torch.arange(6), f), "overlap")


def c_write(xs, slots, codes, scales):
    return C.lib().gpuos_cache_write(len(xs), arr(xs), ref(slots), arr(codes), arr(scales), None)


def c_read(slots, codes, scales, outs):
    return C.lib().gpuos_cache_read(len(outs), ref(slots), arr(codes), arr(scales), arr(outs), None)


def test_cache_refuses():
    x, slots = torch.zeros(3, 2, 32), torch.arange(3)
    codes, scales = torch.zeros(2, 4, 2, 32, dtype=torch.int8), torch.zeros(2, 4, 2, 1)
    for call in (lambda x=x, s=slots, c=codes, sc=scales: c_write([x], s, [c], [sc]),
                 lambda x=x, s=slots, c=codes, sc=scales: c_read(s, [c], [sc], [x])):
        refused(call(s=slots.float()), "int32 or int64")
        refused(call(s=torch.arange(4)), "one row for each token")
        refused(call(c=codes.to(torch.int32)), "codes must be int8")
        refused(call(c=codes[0]), "4 dims")
        refused(call(c=torch.zeros(2, 4, 2, 30, dtype=torch.int8)), "codes must be (page")
        refused(call(sc=torch.zeros(2, 4, 2, 3)), "divide the head")
        refused(call(sc=torch.zeros(2, 4, 2, 0)), "divide the head")
        refused(call(sc=torch.zeros(2, 3, 2, 1)), "pages, rows and heads")
        refused(call(sc=scales.double()), "float32")
        refused(call(x=x.transpose(1, 2)[:, :, :2].transpose(1, 2)[:, :, ::2]), "")
        refused(call(x=torch.zeros(3, 2, 64)[:, :, ::2]), "contiguous")
        refused(call(c=torch.zeros(2, 4, 2, 64, dtype=torch.int8)[..., ::2]), "contiguous")
        refused(call(x=x.long()), "float32, float16 or bfloat16")
    odd = torch.zeros(3, 2, 31)
    refused(c_write([odd], slots, [torch.zeros(2, 4, 2, 15, dtype=torch.uint8)], [scales]), "even head")
    refused(c_write([torch.zeros(3, 2, 6)], slots, [torch.zeros(2, 4, 2, 3, dtype=torch.uint8)], [torch.zeros(2, 4, 2, 2)]),
            "whole bytes")
    refused(c_write([torch.zeros(3, 2, 2048)], slots, [torch.zeros(2, 4, 2, 2048, dtype=torch.int8)], [scales]), "1024")
    refused(c_write([x, x], slots, [codes, codes], [scales, scales.clone()]), "overlap")
    refused(c_write([x, x], slots, [codes, codes.clone()], [scales, scales]), "overlap")
    refused(c_write([x, x], slots, [codes, torch.zeros(3, 4, 2, 32, dtype=torch.int8)], [scales, torch.zeros(3, 4, 2, 1)]),
            "same pages")
    refused(c_write([x, x], slots, [codes, codes.view(torch.float8_e4m3fn)], [scales, scales.clone()]), "one format")
    refused(c_write([x], slots, [codes[:1].expand(2, 4, 2, 32)], [scales]), "overlap itself")
    refused(c_read(slots, [codes], [scales], [x[:1].expand(3, 2, 32)]), "overlap itself")
    assert c_write([torch.zeros(0, 2, 32)], torch.arange(0), [codes], [scales]) == C.OK
    assert c_write([x], slots, [codes[:0]], [scales[:0]]) == C.OK  # no pages: nothing to write


def c_route(x, bias, w, e, score=0, groups=1, top_groups=1, group_score=0, renorm=0, scale=1.0):
    return C.lib().gpuos_route(ref(x), ref(bias), ref(w), ref(e), score, groups, top_groups, group_score, renorm, scale, None)


def test_route_refuses():
    x, w, e = torch.zeros(5, 16), torch.zeros(5, 4), torch.zeros(5, 4, dtype=torch.int64)
    refused(c_route(x[0], None, w, e), "2 dims")
    refused(c_route(x.double(), None, w, e), "float32, float16 or bfloat16")
    refused(c_route(x, None, w.half(), e), "weights must be float32")
    refused(c_route(x, None, w, e.float()), "int32 or int64")
    refused(c_route(x, None, w[:4], e), "row for each token")
    refused(c_route(x, None, w, e[:, :3]), "same columns")
    refused(c_route(torch.zeros(5, 3), None, w, e), "top_k")
    refused(c_route(torch.zeros(5, 1025), None, w, e), "[1, 1024]")
    refused(c_route(torch.zeros(5, 100), None, torch.zeros(5, 65), torch.zeros(5, 65, dtype=torch.int32)), "top_k")
    refused(c_route(torch.zeros(16, 5).t(), None, w, e), "contiguous")
    refused(c_route(x, torch.zeros(15), w, e), "bias")
    refused(c_route(x, torch.zeros(16, dtype=torch.float64), w, e), "bias")
    refused(c_route(x, None, w, e, score=2), "unknown score")
    refused(c_route(x, None, w, e, group_score=2, groups=2), "unknown group score")
    refused(c_route(x, None, w, e, groups=3), "groups")
    refused(c_route(x, None, w, e, groups=0), "groups")
    refused(c_route(x, None, w, e, groups=4, top_groups=5), "top_groups")
    refused(c_route(x, None, w, e, groups=8, top_groups=1), "open groups")
    refused(c_route(x, None, w, e, scale=float("nan")), "scale")
    refused(c_route(x, None, w[:1].expand(5, 4), e), "overlap itself")
    refused(c_route(x, None, x[:, :4], e), "overlap logits")
    L = C.lib()
    g = torch.zeros(5, 16)
    refused(L.gpuos_route_grad(ref(x), ref(e), ref(w), ref(x), 0, 0, 1.0, None), "overlap logits")
    refused(L.gpuos_route_grad(ref(x), ref(e), ref(w), ref(g.half()), 0, 0, 1.0, None), "dtype")
    refused(L.gpuos_route_grad(ref(x), ref(e), ref(w), ref(g[:4]), 0, 0, 1.0, None), "sizes of logits")
    refused(L.gpuos_route_grad(ref(x), None, ref(w), ref(g), 0, 0, 1.0, None), "NULL")
    assert c_route(x[:0], None, w[:0], e[:0]) == C.OK


def test_logprobs_refuses():
    L = C.lib()
    x, y, lp = torch.zeros(5, 16), torch.zeros(5, dtype=torch.int64), torch.zeros(5)
    ent, st, gx = torch.zeros(5), torch.zeros(5, 2), torch.zeros(5, 16)
    top, tok = torch.zeros(5, 3), torch.zeros(5, 3, dtype=torch.int64)

    def call(x=x, y=y, lp=lp, ent=None, top=None, tok=None, st=None, t=1.0):
        return L.gpuos_logprobs(ref(x), ref(y), ref(lp), ref(ent), ref(top), ref(tok), ref(st), t, None)

    refused(call(x=x[0]), "2 dims")
    refused(call(x=x.double()), "float32, float16 or bfloat16")
    refused(call(y=y.float()), "int32 or int64")
    refused(call(y=y[:4]), "one token for each row")
    refused(call(lp=None), "NULL")
    refused(call(lp=lp[:4]), "logprob must be")
    refused(call(ent=ent.double()), "entropy must be")
    refused(call(top=top), "together")
    refused(call(top=top, tok=tok[:, :2]), "row for each row")
    refused(call(top=torch.zeros(5, 17), tok=torch.zeros(5, 17, dtype=torch.int32)), "[1, min(64")
    refused(call(top=torch.zeros(5, 0), tok=tok[:, :0]), "[1, min(64")
    refused(call(st=torch.zeros(5, 3)), "stats")
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-38):
        refused(call(t=t), "temperature")
    refused(call(x=torch.zeros(16, 5).t()), "contiguous")
    refused(call(x=torch.zeros(5, 0)), "[1, 2^30)")
    refused(call(lp=lp[:1].expand(5)), "overlap itself")
    refused(call(ent=lp), "two outputs overlap")
    refused(call(lp=x[:, 0]), "overlaps logits")

    def grad(x=x, y=y, st=st, ent=None, gl=lp, ge=None, gx=gx, t=1.0):
        return L.gpuos_logprobs_grad(ref(x), ref(y), ref(st), ref(ent), ref(gl), ref(ge), ref(gx), t, None)

    refused(grad(gl=None), "must be given")
    refused(grad(ge=lp), "needs entropy")
    refused(grad(st=None), "NULL")
    refused(grad(gx=gx.half()), "dtype")
    refused(grad(gx=gx[:, :8]), "sizes of logits")
    refused(grad(gl=lp[:4]), "grad_logprob must be")
    refused(grad(gx=x.view(-1)[0:].view(5, 16)[:, :16].flip(0)[:0]), "sizes of logits")
    big = torch.zeros(6, 16)
    refused(grad(x=big[:5], gx=big[1:]), "not overlap")
    assert call(x=x[:0], y=y[:0], lp=lp[:0]) == C.OK


def test_python_refusals_without_a_gpu():
    x = torch.zeros(4, 2, 16)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        R.rotary(x, torch.arange(4), torch.ones(8))
    with pytest.raises(ValueError, match="score must be one of"):
        R.route(torch.zeros(2, 8), 2, score="tanh")
    with pytest.raises(ValueError, match="group_score must be one of"):
        R.route(torch.zeros(2, 8), 2, group_score="min")
    with pytest.raises(ValueError, match="format must be one of"):
        R.cache_alloc(1, 1, 1, 8, format="int2", device="cpu")
    with pytest.raises(ValueError, match="group must divide"):
        R.cache_alloc(1, 1, 1, 8, group=3, device="cpu")
    with pytest.raises(TypeError, match="dtype must be"):
        R.cache_read(torch.arange(1), torch.zeros(1, 1, 1, 8, dtype=torch.int8), torch.zeros(1, 1, 1, 1), dtype=torch.int32)
    with pytest.raises(ValueError, match="no stats"):
        R.logprobs_grad(torch.zeros(1, 4), torch.zeros(1), R.LogProbs(torch.zeros(1), None, None, None, None), torch.ones(1))
    with pytest.raises(TypeError, match="tuple of one or two"):
        R.rotary((x, x, x), torch.arange(4), torch.ones(8))
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        R.cache_write((1,), torch.arange(1), torch.zeros(1), torch.zeros(1))


def test_existing_requests_refuse_the_new_dtype_codes():
    a = C.tensor(torch.zeros(4))
    for code in (C.I32, C.F64, C.I64, C.U8, C.I8, C.E4M3):
        b = C.tensor(torch.zeros(4))
        b.dtype = code
        p = C.Plan()
        rc = C.lib().gpuos_plan_elementwise(C.variant("add"), 0.0, 0.0, ctypes.byref(a), ctypes.byref(b), ctypes.byref(a),
                                            ctypes.byref(p))
        refused(rc, "float32, float16 or bfloat16")


def test_rotary_frequencies():
    f = R.rotary_frequencies(8)
    assert torch.allclose(f, 10000.0 ** (-torch.tensor([0, 2, 4, 6], dtype=torch.float64) / 8), rtol=1e-15)
    assert torch.equal(R.rotary_frequencies(8, scaling="linear", factor=4.0), f / 4)
    n = R.rotary_frequencies(8, scaling="ntk", factor=4.0)
    assert n[0] == 1 and abs(n[-1] / (f[-1] / 4) - 1) < 1e-14  # the slowest pair is divided by the factor
    length = 1000
    r = R.rotary_frequencies(64, scaling="ramp", factor=4.0, low=1.0, high=8.0, length=length)
    f = R.rotary_frequencies(64)
    turns = length * f / (2 * math.pi)
    assert torch.equal(r[turns >= 8], f[turns >= 8]) and torch.equal(r[turns <= 1], f[turns <= 1] / 4)
    mid = (turns > 1) & (turns < 8)
    keep = (turns - 1) / 7
    assert mid.any() and torch.allclose(r[mid], (keep * f + (1 - keep) * f / 4)[mid], rtol=1e-14)
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, base=1.0), dict(rot_dim=8, factor=0.0),
                dict(rot_dim=8, scaling="other"), dict(rot_dim=8, scaling="ramp")):
        with pytest.raises(ValueError):
            R.rotary_frequencies(**bad)


# ---------------------------------------------------------------------------
# Rotary (GPU)
# ---------------------------------------------------------------------------
def rotary_oracle(x, pos, f, scale=1.0, interleaved=False, inverse=False):
    """(value, bound) in 64 bits on the CPU."""
    x, n = x.cpu().double(), 2 * f.numel()
    a = pos.cpu().double()[..., None] * f.cpu().double()
    c, s = (scale * a.cos())[..., None, :], (scale * a.sin())[..., None, :] * (-1 if inverse else 1)
    y, b = x.clone(), torch.zeros_like(x)
    if interleaved:
        i1, i2 = slice(0, n, 2), slice(1, n, 2)
    else:
        i1, i2 = slice(0, n // 2), slice(n // 2, n)
    p, q = x[..., i1], x[..., i2]
    y[..., i1], y[..., i2] = p * c - q * s, q * c + p * s
    # c and s: half a step of the reduced angle in turns (2 pi 2^-26), the sine's
    # documented 2 ulp (2^-23), the product with scale (2^-24), the 64-bit
    # product's error (below 2^-27 for positions to 2^24); then two 32-bit
    # roundings of the sum: 6 * 2^-24 of |p| + |q| in all, with scale
    b[..., i1] = b[..., i2] = (p.abs() + q.abs()) * scale * 7 * 2.0 ** -24
    return y, b


def check_rotary(got, x, pos, f, **how):
    want, bound = rotary_oracle(x, pos, f, **how)
    err = (got.cpu().double() - want).abs()
    bound = bound + want.abs() * half_step(got.dtype) + (2.0 ** -25 if got.dtype == FP else 1e-40)
    n = 2 * f.numel()
    assert bool((err <= bound).all()), float((err / bound).max())
    assert torch.equal(got[..., n:].cpu(), x[..., n:].cpu())  # copied


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,d,rot", [
    (1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (7, 4, 1, 64, 32), (33, 3, 2, 80, 20), (5, 2, 2, 18, 6),
    (130, 8, 8, 96, 96), (1025, 2, 1, 256, 64), (3, 5, 1, 40, 0), (300, 40, 8, 128, 128)])
def test_rotary(dtype, interleaved, tokens, hq, hk, d, rot):
    g = gen(tokens + rot)
    q, k = randn(g, tokens, hq, d, dtype=dtype).to(DEV), randn(g, tokens, hk, d, dtype=dtype).to(DEV)
    pos = torch.randint(-100, 1 << 24, (tokens,), generator=g).to(DEV)
    f = (R.rotary_frequencies(rot) if rot else torch.zeros(0, dtype=torch.float64)).to(DEV)
    for how in (dict(), dict(inverse=True, scale=1.25)):
        a, b = R.rotary((q, k), pos, f, interleaved=interleaved, **how)
        check_rotary(a, q, pos, f, interleaved=interleaved, **how)
        check_rotary(b, k, pos, f, interleaved=interleaved, **how)
        one = R.rotary(q, pos, f, interleaved=interleaved, **how)
        assert torch.equal(one, a)
        q2, k2 = q.clone(), k.clone()
        got = R.rotary((q2, k2), pos, f, interleaved=interleaved, out=(q2, k2), **how)
        assert got[0].data_ptr() == q2.data_ptr()
        assert torch.equal(q2, a) and torch.equal(k2, b)


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_rotary_layouts(dtype, interleaved):
    """Slices of one projection in place, heads before tokens, rows off 16-byte
    alignment, odd heads, expanded inputs and positions, 32-bit positions and frequencies."""
    g = gen(3)
    f = R.rotary_frequencies(32).to(DEV)
    how = dict(interleaved=interleaved)
    # queries, keys and values side by side, rotated in place; the values stay
    qkv = randn(g, 50, 12, 64, dtype=dtype).to(DEV)
    before = qkv.clone()
    pos = torch.arange(50, device=DEV, dtype=torch.int32)
    R.rotary((qkv[:, :8], qkv[:, 8:10]), pos, f, out=(qkv[:, :8], qkv[:, 8:10]), **how)
    check_rotary(qkv[:, :8], before[:, :8], pos, f, **how)
    check_rotary(qkv[:, 8:10], before[:, 8:10], pos, f, **how)
    assert torch.equal(qkv[:, 10:], before[:, 10:])
    # (batch, head, token, element) seen as (batch, token, head, element)
    x = randn(g, 3, 4, 17, 64, dtype=dtype).to(DEV).transpose(1, 2)
    pos = torch.randint(0, 10000, (3, 17), generator=g).to(DEV)
    y = R.rotary(x, pos, f, **how)
    assert y.stride() == x.stride()
    check_rotary(y, x, pos, f, **how)
    row = torch.arange(17, device=DEV).expand(3, 17)
    check_rotary(R.rotary(x, row, f.float(), **how), x, row, f.float(), **how)
    # rows that start one element off alignment, and an odd number of elements
    flat = randn(g, 20 * 3 * 65 + 1, dtype=dtype).to(DEV)
    x = flat[1:].view(20, 3, 65)
    if not interleaved:
        check_rotary(R.rotary(x, pos.view(-1)[:20], f), x, pos.view(-1)[:20], f)
    x = x[..., :64]
    check_rotary(R.rotary(x, pos.view(-1)[:20], f, **how), x, pos.view(-1)[:20], f, **how)
    # one head for all
    x = randn(g, 20, 1, 64, dtype=dtype).to(DEV).expand(20, 5, 64)
    check_rotary(R.rotary(x, pos.view(-1)[:20], f, **how), x, pos.view(-1)[:20], f, **how)
    # nothing
    assert R.rotary(x[:0], pos.view(-1)[:0], f, **how).shape == (0, 5, 64)


@gpu
def test_rotary_far_positions():
    """Angles of positions to 2^40: what a 32-bit angle would lose.  f is a
    power of two, so that the oracle's 64-bit product is exact."""
    pos = torch.tensor([0, 1, (1 << 31) + 5, (1 << 40) + 3, -(1 << 33) - 1], device=DEV)
    f = torch.tensor([2.0 ** -3, 2.0 ** -20], dtype=torch.float64, device=DEV)
    x = torch.ones(5, 1, 4, device=DEV)
    got = R.rotary(x, pos, f).cpu().double()
    # 64 bits: turns = p f / 2 pi carries a relative 3 * 2^-53, up to 2^38 turns: 2^-13 of one... so
    # the bound grows with the angle: 3 * 2^-53 |angle|, in the oracle's own cosine's argument too
    a = pos.cpu().double()[:, None] * f.cpu()
    want = torch.cat((a.cos() - a.sin(), a.cos() + a.sin()), -1)[:, None]
    bound = 2 * (7 * 2.0 ** -24 + 4 * 2.0 ** -53 * a.abs()) + 2.0 ** -23
    assert bool(((got - want).abs() <= torch.cat((bound, bound), -1)[:, None]).all())


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(interleaved):
    g = gen(5)
    q, k = randn(g, 2, 9, 4, 32).to(DEV), randn(g, 2, 9, 1, 32).to(DEV)
    pos, f = torch.arange(9, device=DEV).expand(2, 9), R.rotary_frequencies(16).to(DEV)
    q.requires_grad_(), k.requires_grad_()
    how = dict(scale=1.5, interleaved=interleaved)
    a, b = R.rotary((q, k), pos, f, **how)
    ga, gb = randn(g, *a.shape).to(DEV), randn(g, *b.shape).to(DEV)
    dq, dk = torch.autograd.grad((a, b), (q, k), (ga, gb), retain_graph=True)
    check_rotary(dq[..., :16], ga[..., :16], pos, f, inverse=True, **how)
    check_rotary(dk, gb, pos, f, inverse=True, **how)
    # against differences: the map is linear, so <g, R(x + e) - R(x)> = <dx, e> up to rounding
    e = randn(g, *q.shape).to(DEV)
    with torch.no_grad():
        lhs = ((R.rotary(q + e, pos, f, **how).double() - R.rotary(q, pos, f, **how).double()) * ga).sum()
    size = (ga.double().abs() * (q.double().abs() + e.double().abs() + 1)).sum()
    assert abs(float(lhs - (dq.double() * e).sum())) <= float(size) * 16 * 2.0 ** -24 * 1.5
    # only one of the two, a gradient of a broadcast input, an expanded incoming gradient
    (dk2,) = torch.autograd.grad(b, k, gb, retain_graph=True)
    assert torch.equal(dk2, dk)
    (dk3,) = torch.autograd.grad(b.sum(), k)
    check_rotary(dk3, torch.ones_like(b), pos, f, inverse=True, **how)
    w = randn(g, 1, 1, 1, 32).to(DEV).requires_grad_()
    y = R.rotary(w.expand(2, 9, 4, 32), pos, f, **how)
    (dw,) = torch.autograd.grad(y, w, ga)
    want = rotary_oracle(ga, pos, f, inverse=True, **how)[0].sum((0, 1, 2), keepdim=True)
    assert bool(((dw.cpu().double() - want).abs() <= 72 * 4 * 2.0 ** -20).all())
    with pytest.raises(ValueError, match="out cannot"):
        R.rotary(q, pos, f, out=torch.empty_like(q))
    # the gradient's own gradient: the rotation again
    x = q.detach().clone().requires_grad_()
    u = ga.clone().requires_grad_()
    (dx,) = torch.autograd.grad(R.rotary(x, pos, f, **how), x, u, create_graph=True)
    (du,) = torch.autograd.grad(dx, u, gb.expand_as(dx))
    check_rotary(du, gb.expand_as(dx), pos, f, **how)


# ---------------------------------------------------------------------------
# Cache (GPU): bit for bit against the definition's 32-bit arithmetic
# ---------------------------------------------------------------------------
QMAX = {"int8": 127.0, "e4m3": 448.0, "int4": 7.0}


def encode(x, group, fmt):
    """(codes as the cache holds them, scales) of float32 rows (numpy, CPU)."""
    full = np.float32(QMAX[fmt])
    with np.errstate(all="ignore"):
        v = x.float().numpy().reshape(*x.shape[:-1], -1, group)
        finite = np.isfinite(v)
        a = np.where(finite, np.abs(v), np.float32(0)).max(-1, keepdims=True)
        fits = a >= np.float32(2.0 ** -100)
        inv = np.where(fits, np.float32(1) / a * full, np.float32(0)).astype(np.float32)
        y = (v * inv).astype(np.float32)
        y = np.where(np.isinf(v), np.copysign(full, v), y)
        y = np.where(np.isnan(v), np.float32("nan") if fmt == "e4m3" else np.float32(0), y)
        scale = np.where(fits, a * (np.float32(1) / full), np.float32(0)).astype(np.float32)[..., 0]
    y = torch.from_numpy(y.reshape(x.shape).astype(np.float32))
    if fmt == "e4m3":
        codes = y.clamp(-448, 448).to(torch.float8_e4m3fn)
    else:
        codes = y.round().to(torch.int8)
        if fmt == "int4":
            n = (codes + 8).to(torch.uint8)
            codes = n[..., 0::2] | (n[..., 1::2] << 4)
    return codes, torch.from_numpy(scale)


def decode(codes, scales, fmt, dtype):
    if fmt == "int4":
        v = torch.stack(((codes & 15).float() - 8, (codes >> 4).float() - 8), -1).flatten(-2)
    else:
        v = codes.float()
    v = v.unflatten(-1, (scales.shape[-1], -1)) * scales[..., None]
    return v.flatten(-2).to(dtype)


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8).cpu(), b.contiguous().view(torch.uint8).cpu())


def special(x, g):
    """Rows of zeros, tiny values, infinities and NaN among ordinary ones."""
    if x.numel() >= 64:
        f = x.view(-1)
        n = f.numel()
        f[:: max(n // 7, 1)] = float("inf")
        f[3:: max(n // 5, 1)] = float("nan")
        f[5:: max(n // 5, 1)] = float("-inf")
        x[0] = 0
        if x.dtype != FP and x.shape[0] > 2:
            x[1] = 1e-33
        if x.shape[0] > 3:
            x[2] = float("inf")
    return x


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,d,group,page", [
    (1, 1, 2, 2, 1), (1, 8, 128, 128, 16), (5, 2, 80, 80, 16), (9, 3, 96, 32, 7), (33, 1, 20, 20, 4), (64, 2, 576, 576, 8),
    (17, 1, 1024, 1024, 3), (700, 4, 64, 16, 64), (3, 2, 22, 22, 5), (2500, 8, 128, 128, 100), (4, 1, 264, 264, 2)])
def test_cache_write_and_read(fmt, dtype, tokens, heads, d, group, page):
    g = gen(tokens * d)
    pages = -(-tokens * 2 // page)
    rows = pages * page
    slots = torch.randperm(rows, generator=g)[:tokens]
    if tokens > 2:
        slots[1] = -1
        slots[2] = rows + (5 if tokens % 2 else 1 << 40)
    k = special(randn(g, tokens, heads, d, dtype=dtype, by=3.0), g)
    v = randn(g, tokens, heads, d, dtype=dtype)
    kc, ks = R.cache_alloc(pages, page, heads, d, format=fmt, group=group, device=DEV)
    vc, vs = R.cache_alloc(pages, page, heads, d, format=fmt, group=group, device=DEV)
    for t in (kc.view(torch.uint8), vc.view(torch.uint8)):
        t.fill_(0x55)
    ks.fill_(7.0), vs.fill_(9.0)
    want = [kc.cpu().flatten(0, 1), ks.cpu().flatten(0, 1), vc.cpu().flatten(0, 1), vs.cpu().flatten(0, 1)]
    R.cache_write((k.to(DEV), v.to(DEV)), slots.to(DEV), (kc, vc), (ks, vs))
    inside = (slots >= 0) & (slots < rows)
    for i, x in ((0, k), (2, v)):
        codes, scales = encode(x[inside], group, fmt)
        want[i].view(torch.uint8)[slots[inside]] = codes.view(torch.uint8)
        want[i + 1][slots[inside]] = scales
    for got, w in zip((kc, ks, vc, vs), want):  # rows no slot names are as they were
        if got.dtype == torch.float8_e4m3fn:
            nan = torch.isnan(w.float())
            assert torch.equal(torch.isnan(got.cpu().flatten(0, 1).float()), nan)
            got, w = got.cpu().flatten(0, 1).float()[~nan], w.float()[~nan]
            assert same_bits(got, w)
        else:
            assert same_bits(got.flatten(0, 1), w)
    for out_dtype in TYPES:
        a, b = R.cache_read(slots.to(DEV), (kc, vc), (ks, vs), dtype=out_dtype)
        for got, c, s in ((a, want[0], want[1]), (b, want[2], want[3])):
            exp = torch.zeros(tokens, heads, d, dtype=out_dtype)
            exp[inside] = decode(c[slots[inside]], s[slots[inside]], fmt, out_dtype)
            nan = torch.isnan(exp)
            assert torch.equal(torch.isnan(got.cpu()), nan)
            assert torch.equal(got.cpu()[~nan], exp[~nan])


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
def test_cache_layouts(fmt):
    """Heads before rows in a page, codes and scales in one padded buffer,
    strided and expanded rows, different heads for keys and values, one tensor, 32-bit slots,
    repeated slots in a read, given outputs."""
    g = gen(11)
    pages, page, tokens = 6, 16, 40
    width = 32 if fmt == "int4" else 64
    raw = torch.zeros(pages, 2, page, width + 16, dtype=torch.uint8, device=DEV)
    codes = raw[..., :width].transpose(1, 2).view(R.CACHE_FORMATS[fmt])
    scales = raw.view(torch.float32)[..., width // 4:width // 4 + 2].transpose(1, 2)
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    qkv = randn(g, tokens, 6, 64, dtype=BF)
    x = qkv[:, 2:4]
    assert R.cache_write(x.to(DEV), slots.to(DEV), codes, scales) is None
    c, s = encode(x.contiguous(), 32, fmt)
    at = slots.long()
    got_c, got_s = codes.contiguous().flatten(0, 1)[at.to(DEV)], scales.contiguous().flatten(0, 1)[at.to(DEV)]
    assert same_bits(got_c, c) and same_bits(got_s, s)
    assert int(raw[..., width + 8:].sum()) == 0
    again = torch.cat((slots, slots.flip(0)))
    out = torch.zeros(2 * tokens, 2, 70, device=DEV)
    y = R.cache_read(again.to(DEV), codes, scales, out=out[..., :64], dtype=F32)
    assert y.data_ptr() == out.data_ptr() and int(out[..., 64:].abs().sum()) == 0
    w = decode(c, s, fmt, F32)
    assert torch.equal(y.cpu(), torch.cat((w, w.flip(0))))
    # keys of 3 heads x 48, values of 1 head x 32, the values' row expanded from one
    kc, ks = R.cache_alloc(4, 16, 3, 48, format=fmt, group=16, device=DEV)
    vc, vs = R.cache_alloc(4, 16, 1, 32, format=fmt, device=DEV)
    k, v = randn(g, 9, 3, 48, dtype=FP), randn(g, 1, 1, 32, dtype=FP).expand(9, 1, 32)
    sl = torch.arange(20, 29)
    R.cache_write((k.to(DEV), v.to(DEV)), sl.to(DEV), (kc, vc), (ks, vs))
    a, b = R.cache_read(sl.to(DEV), (kc, vc), (ks, vs), dtype=FP)
    assert torch.equal(a.cpu(), decode(*encode(k, 16, fmt), fmt, FP))
    assert torch.equal(b.cpu(), decode(*encode(v.contiguous(), 32, fmt), fmt, FP))
    # rows off 16-byte alignment
    flat = randn(g, 9 * 3 * 48 + 1, dtype=FP)
    x = flat[1:].view(9, 3, 48)
    R.cache_write(flat.to(DEV)[1:].view(9, 3, 48), sl.to(DEV), kc, ks)
    buf = torch.zeros(9 * 3 * 48 + 1, dtype=FP, device=DEV)
    R.cache_read(sl.to(DEV), kc, ks, dtype=FP, out=buf[1:].view(9, 3, 48))
    assert torch.equal(buf[1:].cpu(), decode(*encode(x, 16, fmt), fmt, FP).view(-1)) and buf[0] == 0
    # no tokens
    assert R.cache_read(sl[:0].to(DEV), kc, ks).shape == (0, 3, 48)
    R.cache_write(k[:0].to(DEV), sl[:0].to(DEV), kc, ks)


@gpu
def test_cache_past_32_bit_offsets():
    """The last rows of a cache of more than 2^32 bytes."""
    page, heads, d = 64, 8, 128
    pages = (1 << 32) // (page * heads * d) + 3
    codes = torch.empty(pages, page, heads, d, dtype=torch.int8, device=DEV)
    scales = torch.empty(pages, page, heads, 1, device=DEV)
    rows = pages * page
    slots = torch.tensor([rows - 1, 0, rows - 65, rows // 2])
    g = gen(12)
    x = randn(g, 4, heads, d, dtype=BF)
    R.cache_write(x.to(DEV), slots.to(DEV), codes, scales)
    got = R.cache_read(slots.to(DEV), codes, scales)
    assert torch.equal(got.cpu(), decode(*encode(x, d, "int8"), "int8", BF))


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
def test_cache_same_slot_twice_stays_inside(fmt):
    """A row named twice is left unspecified; the others must be right."""
    g = gen(13)
    x = randn(g, 6, 2, 64, dtype=BF)
    c, s = R.cache_alloc(2, 8, 2, 64, format=fmt, device=DEV)
    R.cache_write(x.to(DEV), torch.tensor([3, 5, 3, 9, 10, 3]).to(DEV), c, s)
    got = R.cache_read(torch.arange(16).to(DEV), c, s).cpu()
    want = torch.zeros(16, 2, 64, dtype=BF)
    want[[5, 9, 10]] = decode(*encode(x[[1, 3, 4]], 64, fmt), fmt, BF)
    keep = torch.arange(16) != 3
    assert torch.equal(got[keep], want[keep])


# ---------------------------------------------------------------------------
# Routing (GPU)
# ---------------------------------------------------------------------------
def route_oracle(x, top_k, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", renormalize=False,
                 scale=1.0):
    """Weights and experts in 64 bits; stable sorts put the lowest index first."""
    x = x.double()
    if score == "softmax":
        m = x.amax(-1, keepdim=True)
        e = torch.where((m == -math.inf), torch.zeros(()).double(), (x - m).exp())
        total = e.sum(-1, keepdim=True)
        s = torch.where(total == 0, torch.zeros(()).double(), e / total)
    else:
        s = 1 / (1 + (-x).exp())
    keys = x if bias is None else s + bias.double()
    if groups > 1:
        worth_of = s if bias is None and group_score == "top2" else keys
        by = worth_of.unflatten(-1, (groups, -1))
        worth = by.amax(-1) if group_score == "max" else by.sort(-1, descending=True)[0][..., :2].sum(-1)
        kept = worth.sort(dim=-1, descending=True, stable=True)[1][:, :top_groups]
        closed = torch.ones_like(worth, dtype=torch.bool).scatter(-1, kept, False)
        closed = closed[..., None].expand_as(by).flatten(-2)
        keys = torch.where(closed, torch.full((), -math.inf).double(), keys)
        # an open expert at -inf still comes before a closed one
        order = torch.where(closed, 1, 0).sort(dim=-1, stable=True)[1]
        experts = order.gather(-1, keys.gather(-1, order).sort(dim=-1, descending=True, stable=True)[1])[:, :top_k]
    else:
        experts = keys.sort(dim=-1, descending=True, stable=True)[1][:, :top_k]
    w = s.gather(-1, experts)
    if renormalize:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total == 0, torch.zeros(()).double(), w / total)
    return w * scale, experts


# a softmax or sigmoid score: expf 2 ulp, its argument's rounding (below a tenth of the score), sums of up to
# 1024 terms in 37 steps, a division, products: under 48 * 2^-24 of the value
ROUTE_REL = 48 * 2.0 ** -24


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts,top_k,groups,top_groups", [
    (1, 1, 1, 1, 1), (1, 8, 2, 1, 1), (3, 7, 7, 1, 1), (65, 60, 6, 1, 1), (257, 64, 8, 8, 3), (100, 160, 6, 8, 3),
    (33, 256, 8, 8, 4), (40, 100, 10, 4, 2), (9, 300, 64, 1, 1), (12, 384, 8, 12, 2), (5, 1024, 32, 64, 5), (700, 24, 4, 8, 4),
    (2100, 128, 8, 1, 1), (11, 6, 3, 6, 4)])
def test_route(dtype, score, tokens, experts, top_k, groups, top_groups):
    g = gen(tokens + experts)
    x = randn(g, tokens, experts, dtype=dtype, by=1.5)
    for bias, rule, renorm in itertools.product((None, randn(g, experts, by=0.05), torch.zeros(experts)),
                                                ("max", "top2") if groups > 1 else ("max",), (False, True)):
        how = dict(score=score, groups=groups, top_groups=top_groups, group_score=rule, renormalize=renorm, scale=2.5)
        w, e = R.route(x.to(DEV), top_k, bias=None if bias is None else bias.to(DEV), **how)
        ww, we = route_oracle(x, top_k, bias=bias, **how)
        assert e.dtype == torch.int64 and w.dtype == torch.float32
        assert torch.equal(e.cpu(), we)
        assert bool(((w.cpu().double() - ww).abs() <= ROUTE_REL * ww.abs() + 1e-37).all())


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_masks_and_near_ties(score):
    inf = math.inf
    base = torch.zeros(12, 32)
    base[1, 5:] = -inf                     # five left, eight wanted
    base[2] = -inf                         # nothing left
    base[3] = torch.finfo(F32).min         # the type's lowest value everywhere
    base[4, ::2] = torch.finfo(F32).min
    base[5] = torch.arange(32).float()
    base[6] = -torch.arange(32).float()
    base[7] = 1.0                          # all equal
    base[8, 20], base[8, 4] = 3.0, 3.0
    base[9, :] = torch.tensor([0.0, -0.0] * 16)
    base[10] = 80.0
    base[11, 7] = 100.0
    for bias, groups in itertools.product((None, torch.zeros(32), torch.linspace(0, 1e-7, 32)), (1, 4)):
        how = dict(score=score, groups=groups, top_groups=min(groups, 2), renormalize=True)
        w, e = R.route(base.to(DEV), 8, bias=None if bias is None else bias.to(DEV), **how)
        ww, we = route_oracle(base, 8, bias=bias, **how)
        assert torch.equal(e.cpu(), we)
        assert bool(((w.cpu().double() - ww).abs() <= ROUTE_REL * ww.abs() + 1e-37).all())
    # keys closer than 32-bit scores resolve: s + b of different logits that all but cancel
    g = gen(17)
    x = randn(g, 400, 64)
    s = x.double().softmax(-1) if score == "softmax" else torch.sigmoid(x.double())
    bias = (0.7 - s[0]).float()            # row 0: every key within half a 32-bit step of 0.7
    w, e = R.route(x.to(DEV), 8, score=score, bias=bias.to(DEV))
    ww, we = route_oracle(x, 8, score=score, bias=bias)
    assert torch.equal(e.cpu(), we)


@gpu
def test_route_nan_and_infinity_stay_in_range():
    x = torch.randn(6, 40, generator=gen(1))
    x[0, 3], x[1], x[2, 4], x[3, :38] = math.nan, math.nan, math.inf, math.nan
    for score, bias, groups in itertools.product(("softmax", "sigmoid"), (None, torch.zeros(40)), (1, 4)):
        w, e = R.route(x.to(DEV), 4, score=score, bias=None if bias is None else bias.to(DEV), groups=groups,
                       top_groups=min(groups, 2), group_score="top2")
        e = e.cpu()
        assert bool(((e >= 0) & (e < 40)).all())
        assert all(len(set(r.tolist())) == 4 for r in e)
        ww, we = route_oracle(x[4:], 4, score=score, bias=bias, groups=groups, top_groups=min(groups, 2), group_score="top2")
        assert torch.equal(e[4:], we)  # the other rows are as alone
    w, e = R.route(x[:1].to(DEV), 4, score="sigmoid")
    want = torch.where(torch.isnan(x[0]), torch.full((), -math.inf), x[0]).sort(descending=True, stable=True)[1][:4]
    assert torch.equal(e[0].cpu(), want)


@gpu
def test_route_strides():
    g = gen(19)
    big = randn(g, 50, 130, dtype=BF).to(DEV)
    for x in (big[:, :64], big[:, 1:65], big[::2, 3:63], big[:1, :64].expand(50, 64)):
        w, e = R.route(x, 5, renormalize=True)
        ww, we = route_oracle(x.cpu(), 5, renormalize=True)
        assert torch.equal(e.cpu(), we)
        gw = torch.randn(x.shape[0], 5, device=DEV)
        gx = R.route_grad(x, e, gw, renormalize=True)
        assert torch.equal(gx, R.route_grad(x.contiguous(), e.to(torch.int32), gw.t().contiguous().t(), renormalize=True))


def route_grad_oracle(x, experts, g, score, renormalize, scale):
    x = x.double()
    if score == "softmax":
        m = x.amax(-1, keepdim=True)
        e = torch.where(m == -math.inf, torch.zeros(()).double(), (x - m).exp())
        t = e.sum(-1, keepdim=True)
        s = torch.where(t == 0, torch.zeros(()).double(), e / t)
    else:
        s = 1 / (1 + (-x).exp())
    chosen = s.gather(-1, experts)
    total = chosen.sum(-1, keepdim=True) if renormalize else torch.ones(1).double()
    safe = torch.where(total == 0, torch.ones(()).double(), total)
    d = g.double() - ((g.double() * chosen).sum(-1, keepdim=True) / safe if renormalize else 0)
    d = torch.where(total == 0, torch.zeros(()).double(), d * scale / safe)
    ds = torch.zeros_like(s).scatter_add(-1, experts, d)
    size = torch.zeros_like(s).scatter_add(-1, experts, ((g.double().abs() + (
        (g.double().abs() * chosen).sum(-1, keepdim=True) / safe if renormalize else 0)) * scale / safe))
    if score == "sigmoid":
        return ds * s * (1 - s), size * s
    dot = (ds * s).sum(-1, keepdim=True)
    return s * (ds - dot), s * (size + (size * s).sum(-1, keepdim=True))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (3, 8, 2), (70, 60, 6), (33, 256, 8), (5, 1000, 40), (600, 64, 8)])
def test_route_gradient(dtype, score, renormalize, tokens, experts, top_k):
    g = gen(tokens)
    x = randn(g, tokens, experts, dtype=dtype, by=1.5)
    if tokens > 2:
        x[1] = -math.inf
        x[2, experts // 2:] = -math.inf
    xd = x.to(DEV).requires_grad_()
    how = dict(score=score, renormalize=renormalize, scale=1.5)
    w, e = R.route(xd, top_k, **how)
    gw = randn(g, tokens, top_k)
    (dx,) = torch.autograd.grad(w, xd, gw.to(DEV))
    assert dx.dtype == dtype
    want, size = route_grad_oracle(x, e.cpu(), gw, score, renormalize, 1.5)
    # the two differences' terms carry the scores' relative error each
    bound = size * 2 * ROUTE_REL + want.abs() * half_step(dtype) + (2.0 ** -25 if dtype == FP else 1e-37)
    err = (dx.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    assert torch.equal(dx, R.route_grad(xd.detach(), e, gw.to(DEV), **how))
    if dtype == F32 and experts <= 60 and tokens == 3:
        # against differences of the weights of the same experts, in 64 bits
        h = 1e-5
        for i, j in itertools.product((0,), range(experts)):
            up, dn = x.double().clone(), x.double().clone()
            up[i, j] += h
            dn[i, j] -= h
            f = lambda z: (route_oracle(z, top_k, **how)[0] * gw.double())[i].sum()  # noqa: E731
            if torch.equal(route_oracle(up, top_k, **how)[1][i], route_oracle(dn, top_k, **how)[1][i]):
                assert abs(float((f(up) - f(dn)) / (2 * h) - dx[i, j].cpu().double())) < 1e-6


@gpu
def test_route_gradient_of_given_experts():
    """Experts named twice add up in order; those outside the row count as not chosen."""
    x = randn(gen(2), 2, 8).to(DEV)
    e = torch.tensor([[1, 1, 3], [-1, 8, 2]], device=DEV)
    gw = torch.tensor([[1.0, 2.0, 0.5], [4.0, 5.0, 3.0]], device=DEV)
    got = R.route_grad(x, e, gw, score="sigmoid").cpu().double()
    s = torch.sigmoid(x.cpu().double())
    d = torch.zeros(2, 8).double()
    d[0, 1], d[0, 3], d[1, 2] = 3.0, 0.5, 3.0
    want = d * s * (1 - s)
    assert bool(((got - want).abs() <= 2 * ROUTE_REL * d).all())


# ---------------------------------------------------------------------------
# Log probabilities (GPU)
# ---------------------------------------------------------------------------
def logprobs_oracle(x, temperature):
    x = x.double()
    m = x.amax(-1, keepdim=True)
    none = m == -math.inf
    z = torch.where(none, torch.zeros(()).double(), x - m) / temperature
    s = z.exp().sum(-1, keepdim=True)
    lp = torch.where(none, torch.full((), -math.inf).double(), z - s.log())
    p = torch.where(none, torch.zeros(()).double(), lp.exp())
    ent = -(p * torch.where(p == 0, torch.zeros(()).double(), lp)).sum(-1)
    return lp, p, ent, z


def sum_error(cols):
    """Relative error of a 32-bit sum of 2^y: each term's exponential (2 ulp, 2^-22) and argument (two
    roundings of |y| below 30, weighted by the term: 2^-20 at most), and one rounding an
    addition: a thread adds cols / 128 of a short row, cols / 512 of a long one, then 15 joins
    of three roundings."""
    return 2.0 ** -22 + 2.0 ** -20 + (max(min(cols, 8192) / 128, cols / 512) + 60) * 2.0 ** -24


def check_logprobs(r, x, y, top, temperature, entropy):
    lp, p, ent, z = logprobs_oracle(x, temperature)
    rel = sum_error(x.shape[1])
    rows = torch.arange(len(y))
    inside = (y >= 0) & (y < x.shape[1])
    want = torch.where(inside, lp[rows, y.clamp(0, x.shape[1] - 1)], torch.zeros(()).double())
    got = r.logprob.cpu().double()
    assert torch.equal(torch.isnan(got), y >= x.shape[1])
    got = torch.where(y >= x.shape[1], torch.zeros(()).double(), got)
    # (x_y - m) / t is rounded twice, ln s once more on top of the sum's error, the difference once
    tol = rel + 2.0 ** -22 * (1 + want.abs() + math.log(x.shape[1]))
    same = torch.isinf(want) & (got == want)
    assert bool((same | ((got - want).abs() <= tol)).all()), float(((got - want).abs() - tol)[~same].max())
    if entropy:
        tol = (4 * rel + 2.0 ** -21) * (1 + ent + math.log(x.shape[1]))
        assert bool(((r.entropy.cpu().double() - ent).abs() <= tol).all())
    else:
        assert r.entropy is None
    if top:
        order = x.float().sort(dim=-1, descending=True, stable=True)[1][:, :top]
        assert torch.equal(r.top_tokens.cpu(), order)
        want = lp.gather(-1, order)
        got = r.top_logprobs.cpu().double()
        tol = rel + 2.0 ** -22 * (1 + want.abs() + math.log(x.shape[1]))
        assert bool((((got == want) & torch.isinf(want)) | ((got - want).abs() <= tol)).all())
    else:
        assert r.top_tokens is None and r.top_logprobs is None


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 3), (1, 7), (3, 9), (5, 64), (4, 1000), (40, 4097), (3, 8191), (2, 32000), (1, 50257),
                                       (70, 2050), (1, 262144), (300, 10007)])
@pytest.mark.parametrize("temperature", [1.0, 0.3])
def test_logprobs(dtype, rows, cols, temperature):
    g = gen(rows + cols)
    x = randn(g, rows, cols, dtype=dtype, by=4.0)
    y = torch.randint(0, cols, (rows,), generator=g)
    for top, entropy in ((0, False), (min(cols, 5), True), (min(cols, 64), False), (0, True)):
        r = R.logprobs(x.to(DEV), y.to(DEV), top=top, entropy=entropy, temperature=temperature)
        check_logprobs(r, x, y, top, temperature, entropy)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [50, 5000, 40000])
def test_logprobs_masks_ties_and_padding(dtype, cols):
    g = gen(cols)
    x = randn(g, 14, cols, dtype=dtype)
    low = torch.finfo(dtype).min
    x[0] = -math.inf                        # nothing left
    x[1, 3:] = -math.inf                    # three left, more alternatives wanted
    x[2] = low                              # the type's lowest value everywhere: uniform
    x[3, 1:] = low
    x[4] = 2.0                              # all equal
    x[5] = torch.linspace(-5, 5, cols).to(dtype)          # rising: each beats the ones before
    x[6] = torch.linspace(5, -5, cols).to(dtype)
    x[7, : cols // 2] = -math.inf
    x[8, -1] = 300.0                        # all the mass on the last
    x[9] = torch.tensor([0.0, -0.0]).repeat(cols)[:cols].to(dtype)
    x[10, ::2] = -math.inf
    y = torch.randint(0, cols, (14,), generator=g)
    y[0], y[1], y[3], y[11], y[12], y[13] = 2, 4, 5, -1, -100, cols
    for top, dev_y in ((0, y), (5, y.to(torch.int32)), (37, y)):
        r = R.logprobs(x.to(DEV), dev_y.to(DEV), top=top, entropy=True)
        check_logprobs(r, x, y, top, 1.0, True)


@gpu
@pytest.mark.parametrize("cols", [40, 30000])
def test_logprobs_nan_and_infinity(cols):
    x = randn(gen(4), 4, cols)
    x[0, 5], x[1, 7] = math.nan, math.inf
    x[2] = math.nan
    y = torch.tensor([5, 7, 0, 1])
    r = R.logprobs(x.to(DEV), y.to(DEV), top=20, entropy=True)
    for t in (r.logprob, r.entropy):
        assert bool(torch.isnan(t[:3]).all()) and not bool(torch.isnan(t[3]))
    assert bool(torch.isnan(r.top_logprobs[:3]).all())
    t = r.top_tokens.cpu()
    assert bool(((t >= 0) & (t < cols)).all()) and all(len(set(q.tolist())) == 20 for q in t)
    check_logprobs(R.LogProbs(r.logprob[3:], r.entropy[3:], r.top_logprobs[3:], r.top_tokens[3:], None), x[3:], y[3:], 20, 1.0,
                   True)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_strides(dtype):
    g = gen(6)
    big = randn(g, 12, 3001, dtype=dtype)
    dev = big.to(DEV)
    y = torch.randint(0, 2990, (12,), generator=g)
    for k in range(9):  # each alignment of a row's start
        r = R.logprobs(dev[:, k:k + 2990], y.to(DEV), top=7, entropy=True)
        check_logprobs(r, big[:, k:k + 2990], y, 7, 1.0, True)
    r = R.logprobs(dev[:1].expand(12, 3001), y.to(DEV), top=3)
    check_logprobs(r, big[:1].expand(12, 3001), y, 3, 1.0, False)
    yy = torch.stack((y, y), 1).to(DEV)[:, 0]
    r = R.logprobs(dev[::3], yy[::3], top=3)
    check_logprobs(r, big[::3], y[::3], 3, 1.0, False)
    assert R.logprobs(dev[:0], y[:0].to(DEV), top=3).top_tokens.shape == (0, 3)


def grad_oracle(x, y, g, h, t):
    lp, p, ent, z = logprobs_oracle(x, t)
    d = torch.zeros_like(p)
    size = torch.zeros_like(p)
    rows = torch.arange(len(y))
    lq = torch.where(p == 0, torch.zeros(()).double(), lp)
    if g is not None:
        gg = torch.where(y >= 0, g.double(), torch.zeros(()).double())
        hit = torch.zeros_like(p)
        hit[rows, y.clamp(min=0)] = 1
        none = (p.sum(-1) == 0)[:, None]
        d += gg[:, None] * torch.where(none, torch.zeros(()).double(), hit - p)
        size += gg.abs()[:, None] * (hit + p)
    if h is not None:
        d -= h.double()[:, None] * p * (lq + ent[:, None])
        size += h.double().abs()[:, None] * p * (lq.abs() + ent[:, None] + 2 * math.log(x.shape[1] + 1))
    return d / t, size / t


def check_grad(got, x, y, g, h, t):
    want, size = grad_oracle(x, y, g, h, t)
    # p: the sum's error and 2^-22 (1 + |y|) of its own exponential (|y| below 45 where p counts in
    # 32 bits: 2^-16 at most where p is below 2^-20; 2^-20 elsewhere), the sum A + B y four roundings
    lp, p, _, _ = logprobs_oracle(x, t)
    own = torch.where(p < 2.0 ** -20, 2.0 ** -16, 2.0 ** -18)
    bound = size * (2 * sum_error(x.shape[1]) + own) + want.abs() * half_step(got.dtype) + (
        2.0 ** -25 if got.dtype == FP else 2.0 ** -120)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 9), (4, 1000), (7, 4097), (2, 50257)])
@pytest.mark.parametrize("t", [1.0, 0.5])
def test_logprobs_gradient(dtype, rows, cols, t):
    gr = gen(rows * cols)
    x = randn(gr, rows, cols, dtype=dtype, by=2.0)
    y = torch.randint(0, cols, (rows,), generator=gr)
    if rows > 3:
        x[0] = -math.inf
        x[1, cols // 2:] = -math.inf
        y[1], y[2] = cols - 1, -1
    g, h = randn(gr, rows), randn(gr, rows, by=0.3)
    for gg, hh in ((g, None), (None, h), (g, h)):
        xd = x.to(DEV).requires_grad_()
        r = R.logprobs(xd, y.to(DEV), top=min(cols, 3), entropy=hh is not None or rows == 3, temperature=t)
        outs, gs = [], []
        if gg is not None:
            outs.append(r.logprob), gs.append(gg.to(DEV))
        if hh is not None:
            outs.append(r.entropy), gs.append(hh.to(DEV))
        (dx,) = torch.autograd.grad(outs, xd, gs)
        check_grad(dx, x, y, gg, hh, t)
        got = R.logprobs_grad(xd.detach(), y.to(DEV), r, None if gg is None else gg.to(DEV), None if hh is None else hh.to(DEV),
                              temperature=t)
        assert torch.equal(got, dx)
        inplace = xd.detach().clone()
        assert R.logprobs_grad(inplace, y.to(DEV), r, *(None if q is None else q.to(DEV) for q in (gg, hh)), temperature=t,
                               out=inplace).data_ptr() == inplace.data_ptr()
        assert torch.equal(inplace, dx)
    # rows whose starts differ in alignment from the output's
    buf = torch.zeros(rows * (cols + 1) + 3, dtype=dtype, device=DEV)
    view = buf[1:1 + rows * (cols + 1)].view(rows, cols + 1)[:, :cols]
    R.logprobs_grad(xd.detach(), y.to(DEV), r, g.to(DEV), h.to(DEV), temperature=t, out=view)
    assert torch.equal(view, dx)
    assert float(buf[0]) == 0 and float(buf[1:1 + rows * (cols + 1)].view(rows, cols + 1)[:, cols:].abs().sum()) == 0


@gpu
def test_logprobs_gradient_against_differences():
    gr = gen(9)
    x = randn(gr, 3, 11).double()
    y = torch.tensor([4, 0, 10])
    g, h = randn(gr, 3), randn(gr, 3)
    xd = x.float().to(DEV).requires_grad_()
    r = R.logprobs(xd, y.to(DEV), entropy=True, temperature=0.8)
    (dx,) = torch.autograd.grad((r.logprob * g.to(DEV)).sum() + (r.entropy * h.to(DEV)).sum(), xd)

    def value(z):
        lp, _, ent, _ = logprobs_oracle(z, 0.8)
        return (lp[torch.arange(3), y] * g.double() + ent * h.double())

    base = x.float().double()
    for i, j in itertools.product(range(3), range(11)):
        e = torch.zeros_like(base)
        e[i, j] = 1e-5
        d = float(((value(base + e) - value(base - e)) / 2e-5)[i])
        assert abs(d - float(dx[i, j])) < 2e-6 * (1 + abs(d))


# ---------------------------------------------------------------------------
# Together, and around the calls
# ---------------------------------------------------------------------------
class Step:
    """What one decode step of 4 sequences does with the operators: positions on
    queries and keys, the cache written and read, experts chosen, the sampled tokens scored."""

    def __init__(self, seed, fmt="int8"):
        g = gen(seed)
        self.fmt = fmt
        self.qkv = randn(g, 4, 12, 64, dtype=BF).to(DEV)
        self.pos = torch.tensor([5, 900, 31, 70000], device=DEV)
        self.f = R.rotary_frequencies(64, device=DEV)
        self.kc, self.ks = R.cache_alloc(8, 16, 2, 64, format=fmt, device=DEV)
        self.vc, self.vs = R.cache_alloc(8, 16, 2, 64, format=fmt, device=DEV)
        self.slots = torch.tensor([3, 100, -1, 64], device=DEV)
        self.gate = randn(g, 4, 32, dtype=BF).to(DEV)
        self.bias = randn(g, 32, by=0.1).to(DEV)
        self.logits = randn(g, 4, 5003, dtype=BF, by=3.0).to(DEV)
        self.tokens = torch.tensor([1, 5002, -1, 77], device=DEV)

    def run(self):
        q, k, v = self.qkv[:, :8], self.qkv[:, 8:10], self.qkv[:, 10:]
        q, k = R.rotary((q, k), self.pos, self.f)
        R.cache_write((k, v), self.slots, (self.kc, self.vc), (self.ks, self.vs))
        ko, vo = R.cache_read(self.slots, (self.kc, self.vc), (self.ks, self.vs))
        w, e = R.route(self.gate, 4, score="sigmoid", bias=self.bias, groups=4, top_groups=2, group_score="top2",
                       renormalize=True)
        r = R.logprobs(self.logits, self.tokens, top=5, entropy=True, temperature=0.9)
        return dict(q=q, k=k, ko=ko, vo=vo, w=w, e=e, lp=r.logprob, ent=r.entropy, tl=r.top_logprobs, tt=r.top_tokens)

    def check(self, o):
        check_rotary(o["q"], self.qkv[:, :8], self.pos, self.f)
        check_rotary(o["k"], self.qkv[:, 8:10], self.pos, self.f)
        for got, x in ((o["ko"], o["k"].cpu()), (o["vo"], self.qkv[:, 10:].cpu())):
            want = decode(*encode(x.contiguous(), 64, self.fmt), self.fmt, BF)
            want[2] = 0
            assert torch.equal(got.cpu(), want)
        w, e = route_oracle(self.gate.cpu(), 4, score="sigmoid", bias=self.bias.cpu(), groups=4, top_groups=2, group_score="top2",
                            renormalize=True)
        assert torch.equal(o["e"].cpu(), e) and bool(((o["w"].cpu().double() - w).abs() <= ROUTE_REL * w).all())
        check_logprobs(R.LogProbs(o["lp"], o["ent"], o["tl"], o["tt"], None), self.logits.cpu(), self.tokens.cpu(), 5, 0.9, True)


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3", "int4"])
def test_decode_step(fmt):
    s = Step(1, fmt)
    s.check(s.run())


@gpu
def test_decode_step_in_a_graph():
    """Captured once, replayed on new inputs in the same buffers; two graphs of
    the same kernels do not disturb one another."""
    steps = [Step(2), Step(3, "e4m3")]
    graphs, outs = [], []
    for s in steps:
        s.run()  # warm-up outside the capture
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.run())
        graphs.append(g)
    for s, new in zip(steps, (Step(4), Step(5))):
        for name in ("qkv", "gate", "logits"):
            getattr(s, name).copy_(getattr(new, name))
        s.pos.add_(17)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for s, o in zip(steps, outs):
        s.check(o)


@gpu
def test_two_streams_at_once():
    steps = [Step(6), Step(7, "int4")]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        outs = []
        for s, st in zip(steps, streams):
            with torch.cuda.stream(st):
                outs.append(s.run())
    torch.cuda.synchronize()
    for s, o in zip(steps, outs):
        s.check(o)


@gpu
def test_training_calls_in_a_graph():
    g = gen(8)
    x, y = randn(g, 64, 1003, dtype=BF).to(DEV), torch.randint(0, 1003, (64,), generator=g).to(DEV)
    gl, gw = randn(g, 64).to(DEV), randn(g, 64, 4).to(DEV)
    gate = randn(g, 64, 16, dtype=BF).to(DEV)

    def step():
        r = R.logprobs(x, y, entropy=True, stats=True)
        w, e = R.route(gate, 4)
        return R.logprobs_grad(x, y, r, gl, gl), R.route_grad(gate, e, gw)

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
@pytest.mark.parametrize("mode", ["persistent", "stream"])
def test_inside_a_scheduler_context(mode, monkeypatch):
    """Row operators read the results of requests the scheduler has not
    submitted yet, and requests read theirs."""
    monkeypatch.setenv("GPUOS_MODE", mode)
    monkeypatch.setenv("GPUOS_SCHEDULER_DISABLE_JIT", "0")
    g = gen(21)
    a, b = randn(g, 6, 2, 32).to(DEV), randn(g, 6, 2, 32).to(DEV)
    pos, f = torch.arange(6, device=DEV), R.rotary_frequencies(32, device=DEV)
    plain = R.rotary(a * b, pos, f) + b
    gate = randn(g, 6, 16).to(DEV)
    pw, pe = R.route(gate + gate, 3)
    with torch.no_grad(), S.scheduler_context(auto_flush_ms=None):
        y = R.rotary(a * b, pos, f) + b
        w, e = R.route(gate + gate, 3)
        z = a * b
        t = R.rotary(b, pos, f, out=z)  # a given output that a pending request writes
    assert not S.entered
    torch.cuda.synchronize()
    assert torch.equal(y, plain) and torch.equal(w, pw) and torch.equal(e, pe)
    assert torch.equal(t, R.rotary(b, pos, f)) and t.data_ptr() == z.data_ptr()


@gpu
def test_errors_leave_the_device_usable():
    x = torch.zeros(4, 8, device=DEV)
    with pytest.raises(ValueError, match="top_k"):
        R.route(x, 9)
    with pytest.raises(ValueError, match="2 dims"):
        R.route(x[0], 2)
    with pytest.raises(TypeError, match="not supported"):
        R.logprobs(x.to(torch.complex64), torch.zeros(4, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="temperature"):
        R.logprobs(x, torch.zeros(4, dtype=torch.int64, device=DEV), temperature=0.0)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        R.logprobs(x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="must be CUDA"):
        R.rotary(torch.zeros(4, 1, 8, device=DEV), torch.arange(4), torch.ones(4, device=DEV))
    w, e = R.route(x, 2)
    assert torch.equal(e.cpu(), torch.tensor([[0, 1]]).expand(4, 2))


@gpu
def test_backward_inside_a_scheduler_context(monkeypatch):
    """A backward pass schedules its small ops from a thread of autograd's; the
    row operators' gradients read what those have pending."""
    monkeypatch.setenv("GPUOS_MODE", "stream")
    monkeypatch.setenv("GPUOS_SCHEDULER_DISABLE_JIT", "0")
    g = gen(22)
    x, gw, lg = randn(g, 6, 16).to(DEV), randn(g, 6, 3).to(DEV), randn(g, 6).to(DEV)
    q, pos, f = randn(g, 6, 2, 32).to(DEV), torch.arange(6, device=DEV), R.rotary_frequencies(32, device=DEV)
    y = torch.arange(6, device=DEV)

    def grads():
        a, b, c = (t.clone().requires_grad_() for t in (x, x, q))
        w, _ = R.route(a * 1.5, 3)
        r = R.logprobs(b * 2.0, y, entropy=True)
        z = R.rotary(c * 0.5, pos, f)
        # the products' backward makes gradients that the operators' backward reads
        return torch.autograd.grad([w * gw, r.logprob * lg, r.entropy * lg, z * z], [a, b, c],
                                   [torch.ones_like(gw), lg, lg, torch.ones_like(z)])

    want = grads()
    with S.scheduler_context(auto_flush_ms=None):
        got = grads()
    torch.cuda.synchronize()
    for u, v in zip(got, want):
        assert torch.equal(u, v)


# ---------------------------------------------------------------------------
# Sizes that choose other kernels
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cols", [300, 1000, 4999, 13001])
@pytest.mark.parametrize("top", [0, 5, 16, 17, 33, 64])
def test_logprobs_many_rows(dtype, cols, top):
    """Rows enough for a warp each, with rows that make many candidates among
    them, and alternatives on both sides of every limit."""
    g = torch.Generator(device=DEV).manual_seed(cols + top)
    x = (torch.randn(1301, cols, generator=g, device=DEV) * 3).to(dtype)
    low = torch.finfo(dtype).min
    x[3] = 1.5
    x[10] = -math.inf
    x[17, 2:] = -math.inf
    x[24] = low
    x[31] = torch.linspace(-4, 4, cols, device=DEV).to(dtype)
    x[38] = torch.linspace(4, -4, cols, device=DEV).to(dtype)
    x[45, ::3] = -math.inf
    x[1300, : cols - 1] = low
    y = torch.randint(0, cols, (1301,), generator=g, device=DEV)
    y[1] = -1
    r = R.logprobs(x, y, top=min(top, cols), entropy=True)
    rows = torch.cat((torch.arange(60), torch.arange(1200, 1301)))
    keep = R.LogProbs(*(None if t is None else t[rows.to(DEV)] for t in r))
    check_logprobs(keep, x.cpu()[rows], y.cpu()[rows], min(top, cols), 1.0, True)
    if top:  # every row's tokens
        assert torch.equal(r.top_tokens, x.float().sort(dim=-1, descending=True, stable=True)[1][:, :min(top, cols)])


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cols,rows", [(50000, 3), (140001, 40), (262144, 1)])
@pytest.mark.parametrize("top", [1, 20, 40, 64])
def test_logprobs_long_rows_of_candidates(dtype, cols, rows, top):
    """Rows split over CTAs, and rows whose ties overflow the candidates."""
    g = torch.Generator(device=DEV).manual_seed(cols)
    x = (torch.randn(rows, cols, generator=g, device=DEV) * 3).to(dtype)
    x[rows - 1, cols // 3:] = 9.0                       # most are equal, and the largest
    x[0, : cols - 7] = -math.inf                        # seven left
    y = torch.zeros(rows, dtype=torch.int64, device=DEV)
    r = R.logprobs(x, y, top=top, entropy=True)
    assert torch.equal(r.top_tokens, x.float().sort(dim=-1, descending=True, stable=True)[1][:, :top])
    check_logprobs(r, x.cpu(), y.cpu(), top, 1.0, True)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(256, 8, 4, 8), (64, 1, 1, 6), (128, 4, 2, 31), (384, 6, 3, 8)])
def test_route_many_tokens_with_ties(dtype, score, experts, groups, top_groups, top_k):
    """Tokens enough for every CTA to take several, logits and biases of few
    distinct values, so that keys tie or nearly tie in every row."""
    g = torch.Generator(device=DEV).manual_seed(experts)
    x = (torch.randn(20011, experts, generator=g, device=DEV) * 4).round().div(4).to(dtype)
    x[::2] += torch.randn(10006, experts, generator=g, device=DEV).mul(1e-3).to(dtype)
    bias = torch.randn(experts, generator=g, device=DEV).mul(8).round().div(64)
    for b, rule in ((None, "max"), (bias, "max"), (bias, "top2"), (None, "top2")):
        how = dict(score=score, groups=groups, top_groups=top_groups, group_score=rule, renormalize=True)
        w, e = R.route(x, top_k, bias=b, **how)
        torch.set_default_device(DEV)
        try:
            ww, we = route_oracle(x, top_k, bias=b, **how)
        finally:
            torch.set_default_device("cpu")
        # The oracle's 64-bit keys carry 2^-50 of error: rows whose order two such keys leave open say nothing
        s = (x.double().softmax(-1) if score == "softmax" else torch.sigmoid(x.double()))
        k = x.double() if b is None else s + b.double()
        diff = (e != we).any(-1)
        near = torch.zeros_like(diff)
        if bool(diff.any()):
            a, c = k[diff].gather(-1, e[diff]), k[diff].gather(-1, we[diff])
            near[diff] = ((a - c).abs() <= 2.0 ** -50).all(-1)
            if groups > 1:
                # Nor do groups: with biases that are multiples of 1/64, (s1 + b1) + (s2 + b2) and
                # (s1 + b2) + (s2 + b1) are equal, but three additions of values below 4 leave up to
                # 3 * 2^-52 between their 64-bit sums (the rows that differed had 2^-52 or 2^-53 there).
                by = (s if b is None and rule == "top2" else k)[diff].unflatten(-1, (groups, -1))
                by = by.amax(-1) if rule == "max" else by.sort(-1, descending=True)[0][..., :2].sum(-1)
                by = by.sort(-1, descending=True)[0]
                near[diff] |= by[:, top_groups - 1] - by[:, top_groups] <= 2.0 ** -50
        assert not bool((diff & ~near).any())
        assert bool(((w.double() - ww).abs() <= ROUTE_REL * ww.abs() + 1e-37)[~diff].all())


@gpu
def test_more_pairs_than_threads_and_no_heads():
    g = gen(30)
    x = randn(g, 3, 2, 4200).to(DEV)
    pos, f = torch.tensor([0, 7, 900], device=DEV), R.rotary_frequencies(4096, device=DEV)
    for inter in (False, True):
        check_rotary(R.rotary(x, pos, f, interleaved=inter), x, pos, f, interleaved=inter)
    assert R.rotary(x[:, :0], pos, f).shape == (3, 0, 4200)
    c, s = R.cache_alloc(2, 4, 0, 16, device=DEV)
    R.cache_write(x[:, :0, :16], pos, c, s)
    assert R.cache_read(pos, c, s).shape == (3, 0, 16)


@gpu
def test_first_calls_inside_a_capture():
    """A process whose first call of each operator is captured."""
    import subprocess
    import sys
    code = """
import torch
from gpuos_b200 import rowops as R
x = torch.randn(9, 64, device="cuda"); y = torch.arange(9, device="cuda"); q = torch.randn(9, 2, 32, device="cuda")
f = R.rotary_frequencies(32, device="cuda"); c, s = R.cache_alloc(2, 8, 2, 32)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a = R.rotary(q, y, f); R.cache_write(a, y, c, s); b = R.cache_read(y, c, s, dtype=torch.float32)
    w, e = R.route(x, 4); r = R.logprobs(x, y, top=3, entropy=True, stats=True)
    d = R.logprobs_grad(x, y, r, r.logprob, r.entropy); h = R.route_grad(x, e, w)
g.replay(); torch.cuda.synchronize()
assert torch.equal(a, R.rotary(q, y, f)) and torch.equal(e, R.route(x, 4)[1])
assert torch.equal(r.logprob, R.logprobs(x, y).logprob) and float((a - b).abs().max()) < 0.05
print("captured")
"""
    from pathlib import Path
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240,
                         cwd=Path(__file__).resolve().parents[1])
    assert "captured" in out.stdout, out.stderr[-2000:]


@gpu
@pytest.mark.parametrize("by", [-80.0, -88.5])
def test_route_gradient_of_scores_near_the_smallest(by):
    """Renormalised sigmoid scores whose sum has no 32-bit inverse still have shares."""
    x = torch.tensor([[0.0, -0.125, -0.0625, 0.0]]) + by
    e, g = torch.tensor([[0, 1]]), torch.tensor([[1.0, -0.5]])
    got = R.route_grad(x.to(DEV), e.to(DEV), g.to(DEV), score="sigmoid", renormalize=True, scale=2.5)
    want, _ = route_grad_oracle(x, e, g, "sigmoid", True, 2.5)
    # Near 2^-128 the spacing of 2^-149 makes a rounding up to 2^-22 of a score.  A share takes three
    # (its score, the sum, the quotient), the mean of g five more; exp adds 2^-22 each: below 16 of
    # 2^-22, of terms up to 2.5 * 1.5.
    assert bool(((got.cpu().double() - want).abs() <= 16 * 2.0 ** -22 * 2.5 * 1.5).all()), got
    assert bool((got[0, 2:] == 0).all())


@gpu
def test_written_tensors_count_as_changed_in_place():
    """A backward pass that saved a tensor which an operator wrote over raises; what autograd
    follows is not written to behind its back."""
    g = gen(31)
    pos, f = torch.arange(4, device=DEV), R.rotary_frequencies(16, device=DEV)
    rows = randn(g, 4, 2, 16).to(DEV)

    def saved(shape):
        w = torch.ones(shape, device=DEV, requires_grad=True)
        t = torch.ones(shape, device=DEV)
        return t, (w * t).sum()

    q, loss = saved((4, 2, 16))
    R.rotary(q, pos, f, out=q)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    c, s = R.cache_alloc(1, 8, 2, 16, device=DEV)
    out, loss = saved((4, 2, 16))
    before = c._version, s._version
    R.cache_write(rows, pos, c, s)
    assert c._version > before[0] and s._version > before[1]
    R.cache_read(pos, c, s, out=out, dtype=F32)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    x, loss = saved((4, 16))
    r = R.logprobs(x, pos, stats=True)
    R.logprobs_grad(x, pos, r, torch.ones(4, device=DEV), out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    # calls with new outputs leave their inputs as they are
    before = rows._version
    R.rotary(rows, pos, f)
    assert rows._version == before
    followed = torch.zeros(4, 2, 16, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="requires a gradient"):
        R.rotary(rows, pos, f, out=followed)
    with pytest.raises(ValueError, match="requires a gradient"):
        R.cache_read(pos, c, s, out=followed, dtype=F32)
    with pytest.raises(ValueError, match="inv_freq takes no gradient"):
        R.rotary(rows, pos, f.clone().requires_grad_())
    assert not bool(followed.any())
    with torch.inference_mode():
        z = torch.zeros(4, 2, 16, device=DEV)
        assert torch.equal(R.rotary(rows, pos, f, out=z), R.rotary(rows, pos, f))
    assert torch.equal(R.rotary(rows, pos, f, out=z), R.rotary(rows, pos, f))


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,cols,top", [(3011, 24001, 5), (3011, 11999, 5), (1403, 7999, 16), (1301, 1990, 24), (1301, 1990, 25), (9, 901, 24)])
def test_logprobs_rows_of_a_warp_and_just_past_them(dtype, rows, cols, top):
    """Long rows by a warp each: several packs under a mark, more marks than are read at once, ties that overflow."""
    g = torch.Generator(device=DEV).manual_seed(cols + top)
    x = (torch.randn(rows, cols, generator=g, device=DEV) * 2).to(dtype)
    x[0] = 0.5
    x[1] = -math.inf
    x[2, 1:] = -math.inf
    x[3] = torch.linspace(-8, 8, cols, device=DEV).to(dtype)          # the largest all in the last mark
    x[4] = x[3].flip(0)
    x[5, cols // 2:] = 20.0
    x[6] = 0
    x[6, ::max(cols // 40, 1)] = 1.0                                  # forty of them, over all marks
    x[7, 7::97] = math.nan
    x[8, :] = torch.finfo(dtype).min
    y = torch.randint(0, cols, (rows,), generator=g, device=DEV)
    r = R.logprobs(x, y, top=top, entropy=True)
    order = torch.where(x != x, torch.tensor(-math.inf, device=DEV), x.float()).sort(dim=-1, descending=True, stable=True)[1]
    assert torch.equal(r.top_tokens, order[:, :top])
    assert bool(r.logprob[7].isnan())
    some = [i for i in range(min(rows, 40)) if i != 7] + list(range(rows - 3, rows))
    some = torch.tensor([i for i in some if i != 7])
    keep = R.LogProbs(*(None if t is None else t[some.to(DEV)] for t in r))
    check_logprobs(keep, x.cpu()[some], y.cpu()[some], top, 1.0, True)


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rot,dq,dk", [(32, 128, 32), (16, 128, 64), (96, 192, 104), (8, 264, 8), (64, 64, 64), (2, 50, 6)])
def test_rotary_shares_of_a_head(dtype, interleaved, rot, dq, dk):
    """More copied than rotated elements, heads of two sizes, one tensor in place beside one that is not, odd numbers of heads."""
    g = gen(rot + dq)
    f = R.rotary_frequencies(rot).to(DEV)
    how = dict(interleaved=interleaved, scale=1.25)
    for tokens, hq, hk in ((1, 7, 1), (37, 9, 3), (700, 5, 2)):
        q, k = randn(g, tokens, hq, dq, dtype=dtype).to(DEV), randn(g, tokens, hk, dk, dtype=dtype).to(DEV)
        pos = torch.randint(0, 5000, (tokens,), generator=g).to(DEV)
        room = torch.full((tokens, hq + 1, dq), 7.0, dtype=dtype, device=DEV)
        was = k.clone()
        a, b = R.rotary((q, k), pos, f, out=(room[:, :hq], k), **how)
        check_rotary(a, q, pos, f, **how)
        check_rotary(b, was, pos, f, **how)
        assert b.data_ptr() == k.data_ptr() and bool((room[:, hq] == 7).all())
