"""The row operators where 32-bit scores leave their range, where keys tie, where
autograd looks at a call in other ways than by a gradient, and where several threads meet.

Tolerances count roundings as in test_rowops.py, whose oracles these tests use.
"""
import itertools
import math
import threading
import time
import weakref

import pytest
import torch
import torch.autograd.forward_ad as fwd

from gpuos_b200 import load
from gpuos_b200 import rowops as R
from gpuos_b200 import scheduler as S
from test_rowops import BF, DEV, F32, FP, ROUTE_REL, TYPES, gen, gpu, randn, route_oracle


# ---------------------------------------------------------------------------
# Routing
# ---------------------------------------------------------------------------
def check_weights(got, want, rel=ROUTE_REL):
    got = got.cpu().double()
    assert bool(torch.isfinite(got).all()), got
    assert bool(((got - want).abs() <= rel * want.abs()).all()), (got, want)


@gpu
@pytest.mark.parametrize("scale", [1.0, 10.0, 1e30])
def test_renormalised_sigmoids_near_the_smallest_normal_number(scale):
    """scale / sum would leave 32 bits; the shares are ordinary numbers."""
    x = torch.tensor([[-86.5, -89.0, -95.0, -96.0], [-85.0, -85.5, -86.0, -100.0], [-86.25, -86.25, -87.0, -100.0]])
    for top_k in (1, 2):
        w, e = R.route(x.to(DEV), top_k, score="sigmoid", renormalize=True, scale=scale)
        ww, we = route_oracle(x, top_k, score="sigmoid", renormalize=True, scale=scale)
        assert torch.equal(e.cpu(), we)
        keep = [1, 2] if top_k == 2 else [0, 1, 2]
        check_weights(w[keep], ww[keep])
    # more ranks than a warp has lanes: the other selection
    x = -85.0 - torch.arange(40.0)[None] / 32
    w, e = R.route(x.to(DEV), 36, score="sigmoid", renormalize=True, scale=scale)
    ww, we = route_oracle(x, 36, score="sigmoid", renormalize=True, scale=scale)
    assert torch.equal(e.cpu(), we)
    check_weights(w, ww)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("below", [10.0, 80.0, 88.0, 96.0, 104.0, 200.0])
@pytest.mark.parametrize("experts,top_k,groups", [(3, 2, 1), (32, 4, 4), (256, 8, 8), (64, 36, 1), (48, 33, 2)])
def test_renormalised_softmax_of_experts_far_below_the_largest(dtype, below, experts, top_k, groups):
    """The bias picks experts whose scores leave 32 bits: their shares are those of their logits alone."""
    g = gen(experts + int(below))
    x = torch.zeros(5, experts)
    x[:, 1:] = -below - torch.rand(5, experts - 1, generator=g) * 4
    x = x.to(dtype)
    bias = 4.0 - torch.arange(experts).float() / 64  # falling by more than any picked score
    bias[0] = -4.0
    for rule in ("max", "top2"):
        how = dict(groups=groups, top_groups=max(1, groups // 2), group_score=rule, renormalize=True, scale=2.5)
        if top_k > experts // groups * how["top_groups"]:
            how["top_groups"] = groups
        w, e = R.route(x.to(DEV), top_k, bias=bias.to(DEV), **how)
        ww, we = route_oracle(x, top_k, bias=bias, **how)
        assert torch.equal(e.cpu(), we) and not bool((we == 0).any())
        check_weights(w, ww)


# Below 2^-126 a 32-bit score and its product with the scale are rounded to multiples of 2^-149: expf's
# 2 ulp, and half a step of each of two products.
SMALLEST = 3 * 2.0 ** -149


def sigmoid_weights_and_gradient(x, e, g, renormalize, scale):
    """In 64 bits from the logits: shares by e^(x - the largest), and their gradient on the chosen."""
    v = x.double().gather(-1, e)
    zero = v < -709.7827128933840
    top = v.amax(-1, keepdim=True).clamp(max=0) if renormalize else torch.zeros(len(x), 1).double()
    t = torch.where(v > 0, 1 / (1 + (-v).exp()), (v - top).exp() / (1 + v.exp()))
    t = torch.where(zero, torch.zeros(()).double(), t)
    d, size = g.double() * scale, g.double().abs() * scale
    if renormalize:
        total = t.sum(-1, keepdim=True)
        t = torch.where(total == 0, torch.zeros(()).double(), t / total)
        d, size = d - (d * t).sum(-1, keepdim=True), size + (size * t).sum(-1, keepdim=True)
    slope = t / (1 + v.exp())
    zeros = torch.zeros_like(x).double()
    return t * scale, zeros.scatter(-1, e, d * slope), zeros.scatter(-1, e, size * slope)


@gpu
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("by", [0.0, -60.0, -87.0, -87.5, -90.0, -100.0, -104.5, -300.0, -705.0, -712.0])
@pytest.mark.parametrize("experts,top_k", [(4, 2), (64, 8), (48, 40)])
def test_small_sigmoids_have_one_rule(renormalize, by, experts, top_k):
    """Weights by the lanes, by a warp (40 ranks) and their gradient keep scores that 32 bits flush."""
    g = gen(experts - int(by))
    x = torch.rand(6, experts, generator=g) * 4 + by
    x[1] = by                              # equal ones
    x[2, 1:] = -math.inf                   # one left
    x[3] = -math.inf
    gw = randn(g, 6, top_k)
    for scale in (1.5, 4096.0):
        how = dict(score="sigmoid", renormalize=renormalize, scale=scale)
        w, e = R.route(x.to(DEV), top_k, **how)
        assert torch.equal(e.cpu(), x.double().sort(dim=-1, descending=True, stable=True)[1][:, :top_k])
        ww, dd, size = sigmoid_weights_and_gradient(x, e.cpu(), gw, renormalize, scale)
        tiny = 0.0 if renormalize else SMALLEST * scale
        assert bool(((w.cpu().double() - ww).abs() <= ROUTE_REL * ww + tiny).all()), (w, ww)
        dx = R.route_grad(x.to(DEV), e, gw.to(DEV), **how).cpu().double()
        # a share of 2^-126 and less of the sum is rounded to multiples of 2^-149 too
        tiny = 4 * SMALLEST * scale * (1 + gw.abs().amax().double())
        assert bool(((dx - dd).abs() <= 2 * ROUTE_REL * size + tiny).all()), (dx - dd).abs().max()
        assert bool((dx[3] == 0).all())


@gpu
@pytest.mark.parametrize("dtype", [F32, FP, BF])
@pytest.mark.parametrize("experts,top_k", [(4, 2), (32, 8), (200, 8), (64, 34)])
def test_bias_of_experts_whose_scores_leave_the_series(dtype, experts, top_k):
    """Softmax scores hundreds below the largest logit differ in 64 bits until e^-745, in every path."""
    if experts == 4 and dtype == F32:
        x, bias = torch.tensor([[0.0, -700.0, -695.0, -800.0]]), torch.tensor([0.5, 0.0, 0.0, 0.0])
        w, e = R.route(x.to(DEV), 2, bias=bias.to(DEV))
        assert e.cpu().tolist() == [[0, 2]]
    g = gen(experts)
    # (steps that scores near 2^-1074, multiples of it, still tell apart)
    step = 4.0 if dtype == BF else 0.5
    x = -680.0 - torch.randint(0, int(60 / step) + 1, (40, experts), generator=g) * step
    x[20:] -= 80 * (torch.rand(20, experts, generator=g) < 0.3)  # and some of them 0
    x[:, 0] = 0.0
    x[5:10, 1:] += 500.0
    x[10, 3:] = -math.inf
    x[11, 3:] = torch.finfo(dtype).min
    x = x.to(dtype)
    bias = torch.zeros(experts)
    bias[0] = 0.5
    for renormalize in (False, True):
        w, e = R.route(x.to(DEV), top_k, bias=bias.to(DEV), renormalize=renormalize)
        ww, we = route_oracle(x, top_k, bias=bias, renormalize=renormalize)
        assert torch.equal(e.cpu(), we)
        assert bool(((w.cpu().double() - ww).abs() <= ROUTE_REL * ww + 1e-37).all())


@gpu
@pytest.mark.parametrize("dtype", [F32, FP, BF])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(32, 4, 2, 4), (256, 8, 4, 8), (64, 8, 3, 10), (1024, 64, 5, 8),
                                                             (128, 2, 1, 40)])
def test_groups_of_scores_near_nothing(dtype, score, experts, groups, top_groups, top_k):
    """The sum of a group's two largest scores, where those are far below 32 bits' smallest."""
    g = gen(experts + groups)
    for low, high in ((-120, -86), (-708, -640), (-760, -690)):
        step = 4.0 if dtype == BF else 0.5
        x = low + torch.randint(0, int((high - low) / step), (24, experts), generator=g) * step
        x[3] = low                                     # all equal: the first groups
        x[4, : experts // 2] = -math.inf
        if score == "softmax":
            x[::2, 5] = 0.0
        x = x.to(dtype)
        how = dict(score=score, groups=groups, top_groups=top_groups, group_score="top2")
        for bias in (None, torch.arange(experts).remainder(3) * 0.0):
            w, e = R.route(x.to(DEV), top_k, bias=None if bias is None else bias.to(DEV), **how)
            ww, we = route_oracle(x, top_k, **how)
            assert torch.equal(e.cpu(), we)


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("top_k,groups", [(2, 1), (2, 2), (40, 1)])
def test_one_bias_for_all_is_no_bias(score, top_k, groups):
    """Scores that 64 bits cannot tell apart (1 - e^-40, or a small one beside 0.5) are ordered by their logits."""
    x = torch.full((3, 48), -50.0)
    x[0, :4] = torch.tensor([40.0, 41.0, 42.0, 41.0])
    x[1, 20:24] = torch.tensor([-49.0, -48.0, -47.0, 90.0])
    how = dict(score=score, groups=groups)
    w, e = R.route(x.to(DEV), top_k, **how)
    assert torch.equal(e.cpu(), route_oracle(x, top_k, score="softmax", groups=groups)[1])
    for b in (0.0, 0.5, -3.0):
        wb, eb = R.route(x.to(DEV), top_k, bias=torch.full((48,), b, device=DEV), **how)
        assert torch.equal(e, eb) and torch.equal(w, wb)


# ---------------------------------------------------------------------------
# Around the calls
# ---------------------------------------------------------------------------
class Recorder:
    """In place of the extension: what a mode submits and flushes, and on which thread."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a, **k: self.calls.append((name, threading.get_ident()))


def test_only_the_threads_own_contexts_are_flushed():
    """Another thread's tables may be changing, and the addresses in them may be of tensors long gone."""
    def mode():
        return S._GPUOSSchedulerMode(Recorder(), size_threshold=1 << 16, auto_flush_ms=None, pending=set(), jit=True, fuse=True)

    shared = torch.zeros(8)
    mine, theirs = mode(), mode()
    entered, done = threading.Event(), threading.Event()

    def other():
        with theirs:
            S.entered.append(theirs)
            theirs._done(shared)
            entered.set()
            done.wait(30)
            S.entered.remove(theirs)

    t = threading.Thread(target=other)
    t.start()
    try:
        assert entered.wait(30)
        S.order_after_pending([shared], [shared])
        assert theirs.ext.calls == [] and theirs.pending
        with mine:
            S.entered.append(mine)
            mine._done(shared[2:4])
            S.order_after_pending([shared[4:]], [])
            assert mine.ext.calls == []            # reads nothing that is pending
            S.order_after_pending([shared], [])
            S.entered.remove(mine)
        assert mine.ext.calls == [("flush", threading.get_ident())] and not mine.pending
        assert theirs.ext.calls == [] and theirs.pending
    finally:
        done.set()
        t.join(30)


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_mode(interleaved):
    """Rotary's tangent is the operator of the tangent; the others have none and say so."""
    g = gen(40)
    q, k, tq = randn(g, 5, 3, 32).to(DEV), randn(g, 5, 1, 32).to(DEV), randn(g, 5, 3, 32).to(DEV)
    pos, f = torch.arange(5, device=DEV) * 100, R.rotary_frequencies(16, device=DEV)
    how = dict(interleaved=interleaved, scale=1.5)
    want = R.rotary(tq, pos, f, **how)
    for inverse in (False, True):
        with fwd.dual_level():
            a, b = R.rotary((fwd.make_dual(q, tq), k), pos, f, inverse=inverse, **how)
            assert torch.equal(fwd.unpack_dual(a).tangent, R.rotary(tq, pos, f, inverse=inverse, **how))
            assert fwd.unpack_dual(b).tangent is None or not bool(fwd.unpack_dual(b).tangent.any())
            assert torch.equal(fwd.unpack_dual(a).primal, R.rotary(q, pos, f, inverse=inverse, **how))
    with torch.no_grad(), fwd.dual_level():  # which leaves forward mode on
        a = R.rotary(fwd.make_dual(q, tq), pos, f, **how)
        assert torch.equal(fwd.unpack_dual(a).tangent, want)
        wide = fwd.make_dual(q, tq.transpose(0, 2).contiguous().transpose(0, 2))  # elements of a tangent's row apart
        assert torch.equal(fwd.unpack_dual(R.rotary(wide, pos, f, **how)).tangent, want)
        with pytest.raises(ValueError, match="out cannot"):
            R.rotary(fwd.make_dual(q, tq), pos, f, out=torch.empty_like(q))
        with pytest.raises(ValueError, match="inv_freq takes no gradient"):
            R.rotary(q, pos, fwd.make_dual(f, torch.ones_like(f)))
        x = fwd.make_dual(q[:, 0], tq[:, 0])
        with pytest.raises(NotImplementedError):
            R.route(x, 2)
        with pytest.raises(NotImplementedError):
            R.logprobs(x, pos // 100, entropy=True)
    # a gradient through the tangent
    t = tq.clone().requires_grad_()
    with fwd.dual_level():
        a = fwd.unpack_dual(R.rotary(fwd.make_dual(q, t), pos, f, **how)).tangent
        (dt,) = torch.autograd.grad(a, t, tq)
    assert torch.equal(dt, R.rotary(tq, pos, f, inverse=True, **how))


@gpu
@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("how", [torch.enable_grad, torch.no_grad])
def test_a_trace_keeps_the_calls(how):
    g = gen(41)
    x, other = randn(g, 5, 32).to(DEV), randn(g, 5, 32).to(DEV)
    pos, f = torch.arange(5, device=DEV), R.rotary_frequencies(16, device=DEV)

    def step(x):
        y = R.rotary(x[:, None], pos, f)[:, 0]
        w, e = R.route(y, 4)
        return y, w, e, R.logprobs(y, pos, top=2).top_logprobs

    with how():
        traced = torch.jit.trace(step, x, check_trace=False)
        for got, want in zip(traced(other), step(other)):
            assert torch.equal(got, want)
        c, s = R.cache_alloc(1, 8, 1, 32, device=DEV)
        with pytest.raises(RuntimeError, match="cannot record"):
            torch.jit.trace(lambda x: R.cache_read(pos, c, s), x)
        with pytest.raises(RuntimeError, match="cannot record"):
            torch.jit.trace(lambda x: R.cache_write(x[:, None], pos, c, s), x)
        r = R.logprobs(x, pos, stats=True)
        with pytest.raises(RuntimeError, match="cannot record"):
            torch.jit.trace(lambda x: R.logprobs_grad(x, pos, r, r.logprob), x)
        w, e = R.route(x, 2)
        with pytest.raises(RuntimeError, match="cannot record"):
            torch.jit.trace(lambda x: R.route_grad(x, e, w), x)
    with torch.inference_mode():
        for call in (lambda x: R.rotary(x[:, None], pos, f), lambda x: R.route(x, 2), lambda x: R.logprobs(x, pos).logprob):
            with pytest.raises(RuntimeError, match="cannot record"):
                torch.jit.trace(call, x)


@gpu
def test_outputs_that_autograd_follows_are_refused():
    g = gen(42)
    x, y = randn(g, 4, 16).to(DEV), torch.arange(4, device=DEV)
    r = R.logprobs(x, y, stats=True)
    gl = torch.ones(4, device=DEV)
    want = R.logprobs_grad(x, y, r, gl)
    for followed in (x.clone().requires_grad_(), x.clone().requires_grad_() * 1):
        before = followed.detach().clone()
        with pytest.raises(ValueError, match="out cannot be a tensor that requires a gradient"):
            R.logprobs_grad(followed, y, r, gl, out=followed)
        with pytest.raises(ValueError, match="out cannot be a tensor that requires a gradient"):
            R.logprobs_grad(x, y, r, gl, out=followed)
        assert torch.equal(followed, before)
        assert torch.equal(R.logprobs_grad(followed, y, r, gl), want)   # read, not written
        with torch.no_grad():
            assert R.logprobs_grad(followed, y, r, gl, out=followed) is followed
        assert torch.equal(followed, want)
    c, s = R.cache_alloc(1, 8, 1, 16, device=DEV)
    rows = x[:, None].clone().requires_grad_()
    with pytest.raises(ValueError, match="scales cannot be a tensor that requires a gradient"):
        R.cache_write(rows, y, c, s.clone().requires_grad_())
    R.cache_write(rows, y, c, s)                                     # rows count as detached
    assert not s.requires_grad and bool(s.flatten()[:4].all())


@gpu
def test_results_of_a_call_have_storages_of_their_own():
    """One may be resized, saved or kept without the others."""
    g = gen(43)
    x, y = randn(g, 6, 32).to(DEV), torch.arange(6, device=DEV)
    q = randn(g, 6, 2, 32).to(DEV)
    f = R.rotary_frequencies(32, device=DEV)
    c, s = R.cache_alloc(1, 8, 2, 32, device=DEV)
    calls = [lambda: R.route(x, 4), lambda: R.rotary((q, q), y, f), lambda: R.cache_read(y, (c, c), (s, s)),
             lambda: R.logprobs(x, y, top=3, entropy=True, stats=True)]
    for call in calls:
        got = list(call())
        kept = [t.clone() for t in got]
        assert len({t.untyped_storage().data_ptr() for t in got}) == len(got)
        for t in got:
            assert t.storage_offset() == 0 and t.untyped_storage().nbytes() == t.numel() * t.element_size()
        got[0].resize_(4096).fill_(7)
        assert all(torch.equal(a, b) for a, b in zip(got[1:], kept[1:]))
    # as other tensors' memory: kept for another stream that uses it, and none for no rows
    w, e = R.route(x, 4)
    w.record_stream(torch.cuda.Stream())
    assert R.route(x[:0], 4)[0].shape == (0, 4)
    with torch.inference_mode():
        assert R.route(x, 4)[0].is_inference()


@gpu
def test_tensors_of_a_request_submitted_during_a_flush_stay():
    """A flush waits outside the interpreter's lock; a request that another thread submits meanwhile
    is not among those it waits for, nor are its tensors."""
    ext = load()
    ext.init(mode="stream")
    try:
        x = torch.arange(64.0, device=DEV)
        first, out = torch.empty_like(x), x * 0 + 5.0    # (which loads the kernels that the wait must not meet)
        torch.cuda.synchronize()
        ext.submit_add(x, x, first)
        torch.cuda._sleep(1 << 30)                      # half a second, for which the flush waits
        waiting = threading.Thread(target=lambda: ext.flush(sync=True))
        waiting.start()
        time.sleep(0.1)
        assert waiting.is_alive()
        y = x * 0 + 5.0
        ext.submit_add(x, y, out)
        alive = weakref.ref(y)
        del y
        assert waiting.is_alive()
        waiting.join(60)
        assert alive() is not None
        ext.flush(sync=True)
        ext.flush(sync=True)                             # what the one before left is released here at the latest
        assert alive() is None and torch.equal(out, x + 5)
    finally:
        ext.shutdown()


@gpu
def test_of_a_pair_only_what_needs_a_gradient_is_followed():
    g = gen(44)
    q, k = randn(g, 5, 3, 32).to(DEV), randn(g, 5, 1, 32).to(DEV)
    pos, f = torch.arange(5, device=DEV), R.rotary_frequencies(32, device=DEV)
    for needs in ((True, False), (False, True), (True, True)):
        a, b = q.clone().requires_grad_(needs[0]), k.clone().requires_grad_(needs[1])
        y, z = R.rotary((a, b), pos, f)
        assert (y.requires_grad, z.requires_grad) == needs
        assert torch.equal(y, R.rotary(q, pos, f)) and torch.equal(z, R.rotary(k, pos, f))
        grads = torch.autograd.grad([t for t in (y, z) if t.requires_grad], [t for t in (a, b) if t.requires_grad],
                                    [w for t, w in ((y, q), (z, k)) if t.requires_grad])
        for got, w in zip(grads, [w for n, w in zip(needs, (q, k)) if n]):
            assert torch.equal(got, R.rotary(w, pos, f, inverse=True))


@gpu
@pytest.mark.parametrize("top_k", [2, 33])
def test_renormalised_softmax_of_masked_experts(top_k):
    """A bias that closes all experts but masked ones: by -inf nothing is left of those, by a finite
    number they share alike, in the weights as in their gradient."""
    x = torch.zeros(2, 48)
    x[0, 8:], x[1, 8:] = -math.inf, -65504.0
    bias = torch.zeros(48)
    bias[:8] = -2.0
    gw = randn(gen(45), 2, top_k)
    w, e = R.route(x.to(DEV), top_k, bias=bias.to(DEV), renormalize=True)
    assert bool((e >= 8).all())
    want = torch.stack((torch.zeros(top_k), torch.full((top_k,), 1 / top_k))).double()
    assert bool(((w.cpu().double() - want).abs() <= ROUTE_REL * want).all())
    dx = R.route_grad(x.to(DEV), e, gw.to(DEV), renormalize=True).cpu().double()
    d = torch.zeros(2, 48).double().scatter(-1, e.cpu(), want * (gw.double() - (gw.double() * want).sum(-1, keepdim=True)))
    assert bool(((dx - d).abs() <= 2 * ROUTE_REL * (gw.abs().amax().double() + 1)).all()) and not bool(dx[0].any())


@gpu
@pytest.mark.parametrize("experts", [8, 24, 64, 200])
def test_small_sigmoids_leave_the_other_tokens_of_a_warp_as_they_are(experts):
    x = -0.3 - torch.rand(64, experts, generator=gen(46))
    w, e = R.route(x.to(DEV), 3, score="sigmoid", renormalize=True)
    x[1::2] -= 95.0
    x[6] = -math.inf
    w2, e2 = R.route(x.to(DEV), 3, score="sigmoid", renormalize=True)
    keep = [i for i in range(0, 64, 2) if i != 6]
    assert torch.equal(w[keep], w2[keep]) and torch.equal(e[keep], e2[keep])


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [8, 24, 64])
def test_doubt_about_one_token_leaves_the_others_of_a_warp_as_they_are(score, experts):
    """Ties in every other row send them to later passes; the rows between have a score that those passes
    would not settle, but which decides nothing there."""
    g = gen(47)
    x, tied = randn(g, 256, experts), torch.zeros(256, experts)
    x[:, 5] = -700.0
    bias = torch.rand(experts, generator=g)
    bias[2] = bias[3] = 3.0                # the tie of a row of equal logits
    bias[5] = -3.0
    tied[::2] = x[::2]
    w, e = R.route(x.to(DEV), 3, score=score, bias=bias.to(DEV))
    w2, e2 = R.route(tied.to(DEV), 3, score=score, bias=bias.to(DEV))
    assert torch.equal(e2.cpu(), route_oracle(tied, 3, score=score, bias=bias)[1])
    assert torch.equal(w[::2], w2[::2]) and torch.equal(e[::2], e2[::2])
