"""Row operators of a language model's step, beside the executor's elementwise
requests and reductions: rotary positions, a quantised cache, routing to
experts, and log probabilities of given tokens.

Each call runs one kernel at once on torch's current stream of its tensors'
device; it allocates its outputs (where `out` gives none) and nothing else, so it
may be captured into a CUDA graph.  As with an op of torch's own, requests
submitted to an executor are seen once they are flushed; inside a
``scheduler_context``, pending requests on the call's tensors are flushed first.
Tensors are CUDA tensors of one device.  A call that breaks a rule raises
``ValueError`` (``TypeError`` for a dtype, ``RuntimeError`` for a device) and
launches nothing.

``rotary``, ``route`` and ``logprobs`` take part in autograd; their gradients
are also there as calls of their own (``rotary(..., inverse=True)``,
``route_grad``, ``logprobs_grad``), for steps that are captured or keep no graph.
In forward mode ``rotary`` carries tangents; ``route`` and ``logprobs`` raise.
A given `out` and a written cache count as changed in place: a backward pass that saved
one of them raises, as after an in-place op of torch's.
include/gpuos_b200.h states each operator's formula and its edge cases.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch
import torch.autograd.forward_ad as _fwd

from . import load as _load
from . import scheduler as _scheduler

_ext = _load()
_entered = _scheduler.entered  # empty outside scheduler contexts

_SCORE = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORE = {"max": 0, "top2": 1}
_ROW_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
CACHE_FORMATS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "int4": torch.uint8}

Tensors = Union[torch.Tensor, Tuple[torch.Tensor, ...]]


def _tuple(x) -> tuple:
    return (x,) if isinstance(x, torch.Tensor) else tuple(x)


def _order(reads, writes=()):
    """Flush what a scheduler context has pending on a call's tensors."""
    _scheduler.order_after_pending([t for t in reads if isinstance(t, torch.Tensor)],
                                   [t for t in writes if isinstance(t, torch.Tensor)])


def _choice(table, value, name):
    try:
        return table[value]
    except (KeyError, TypeError):
        raise ValueError(f"{name} must be one of {', '.join(map(repr, table))}, not {value!r}") from None


def _row(g: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """A gradient as the kernels read it: elements of a row side by side."""
    if g is None or g.dim() == 0 or g.stride(-1) == 1 or g.size(-1) == 1:
        return g
    return g.contiguous()


def _followed(t: torch.Tensor) -> bool:
    return (t.requires_grad and torch.is_grad_enabled()) or _fwd.unpack_dual(t).tangent is not None


# ---- rotary positions ----------------------------------------------------------
def rotary_frequencies(rot_dim: int, *, base: float = 10000.0, scaling: str = "none",
                       factor: float = 1.0, low: float = 1.0, high: float = 32.0,
                       length: Optional[int] = None, device=None) -> torch.Tensor:
    """``inv_freq`` of ``rotary``: float64 [rot_dim / 2], radians a position turns
    each pair by, ``base ** (-2 i / rot_dim)`` scaled for contexts `factor` times
    the trained one:

    * ``"none"``; ``"linear"``: all divided by `factor` (positions interpolated);
    * ``"ntk"``: the base grows so that the slowest pair is divided by `factor`;
    * ``"ramp"``: pairs that turn more than `high` times within the trained
      `length` stay, those that turn less than `low` times are divided by `factor`, the others are
      mixed linearly in their number of turns.
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError("rot_dim must be even and at least 2")
    if not (base > 1 and math.isfinite(base) and factor > 0 and math.isfinite(factor)):
        raise ValueError("base must be above 1 and factor above 0, both finite")
    if scaling == "ntk":
        if rot_dim > 2:
            base = base * factor ** (rot_dim / (rot_dim - 2))
    elif scaling not in ("none", "linear", "ramp"):
        raise ValueError(f"scaling must be 'none', 'linear', 'ntk' or 'ramp', not {scaling!r}")
    f = base ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    if scaling == "linear":
        f = f / factor
    if scaling == "ramp":
        if length is None or not high > low:
            raise ValueError("ramp needs length, and low below high")
        keep = ((length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
    return f if device is None else f.to(device)


def rotary(x: Tensors, positions: torch.Tensor, inv_freq: torch.Tensor, *, scale: float = 1.0,
           interleaved: bool = False, inverse: bool = False, out: Optional[Tensors] = None) -> Tensors:
    """Rotary positions on `x`, a tensor or a pair of tensors (queries and keys) of
    the same tokens: (token, head, element) or (batch, token, head, element), any
    strides but the last, which is 1.  `positions` (int32 or int64) has the token
    dims.  The first ``2 * len(inv_freq)`` elements of each head are rotated by
    ``position * inv_freq`` (in 64 bits) and multiplied by `scale`, in pairs (i, i + half),
    or (2i, 2i + 1) if `interleaved` (of an even head size); the others are copied.  `inverse` rotates back
    (the transposed map, also the gradient).  `out` may be `x`.  Returns tensors as `x` is given."""
    if _entered:
        _order((*_tuple(x), positions, inv_freq), () if out is None else _tuple(out))
    got = _ext.rotary(x, out, positions, inv_freq, scale, interleaved, inverse)
    if got is NotImplemented:  # autograd has to record it
        if out is not None:
            raise ValueError("out cannot be given where a gradient is needed, nor in a trace")
        xs = _tuple(x)
        got = _Rotary.apply(positions, inv_freq, scale, interleaved, inverse, *xs)
        # (of a pair, one whose input needs none follows no gradient)
        got = tuple(y if _followed(t) else y.detach() for t, y in zip(xs, got))
        return got[0] if isinstance(x, torch.Tensor) else got
    return got


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, positions, inv_freq, scale, interleaved, inverse, *xs):
        ctx.save_for_backward(positions, inv_freq)
        ctx.save_for_forward(positions, inv_freq)
        ctx.how = dict(scale=scale, interleaved=interleaved)
        ctx.inverse = inverse
        ctx.like = [(x.shape, x.dtype, x.device) for x in xs]
        ctx.set_materialize_grads(False)
        return _ext.rotary(xs, None, positions, inv_freq, scale, interleaved, inverse)

    @staticmethod
    def _turn(ctx, vectors, inverse):
        """The map, or its transpose, of those vectors that there are."""
        positions, inv_freq = ctx.saved_tensors
        need = [i for i, v in enumerate(vectors) if v is not None]
        got = [None] * len(vectors)
        if need:
            turned = rotary(tuple(_row(vectors[i]) for i in need), positions, inv_freq, inverse=inverse, **ctx.how)
            for i, v in zip(need, turned):
                got[i] = v
        return tuple(got)

    @staticmethod
    def backward(ctx, *grads):
        grads = [g if need else None for g, need in zip(grads, ctx.needs_input_grad[5:])]
        return (None,) * 5 + _Rotary._turn(ctx, grads, not ctx.inverse)

    @staticmethod
    def jvp(ctx, *tangents):  # linear: the map itself
        got = _Rotary._turn(ctx, tangents[5:], ctx.inverse)
        return tuple(torch.zeros(size, dtype=dtype, device=device) if t is None else t
                     for t, (size, dtype, device) in zip(got, ctx.like))


# ---- quantised cache -------------------------------------------------------------
def cache_alloc(pages: int, page_size: int, heads: int, head_dim: int, *, format: str = "int8",
                group: Optional[int] = None, device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """An empty cache: (codes, scales), zeros.  codes is (page, row, head, code) in
    the format's dtype (int8; float8_e4m3fn; uint8 with two 4-bit codes a byte);
    scales is float32 (page, row, head, group) with a scale for each `group`
    elements (default: the whole head)."""
    dtype = _choice(CACHE_FORMATS, format, "format")
    group = head_dim if group is None else group
    if group < 1 or head_dim % group or (format == "int4" and group % 2):
        raise ValueError("group must divide head_dim (and be even for int4)")
    width = head_dim // 2 if format == "int4" else head_dim
    device = "cuda" if device is None else device
    codes = torch.zeros(pages, page_size, heads, width, dtype=torch.uint8, device=device)
    scales = torch.zeros(pages, page_size, heads, head_dim // group, device=device)
    return codes.view(dtype), scales


def cache_write(x: Tensors, slots: torch.Tensor, codes: Tensors, scales: Tensors) -> None:
    """Quantise rows into a paged cache: `x` is a tensor or a pair (keys and
    values), (token, head, element); token t goes to row ``slots[t]`` of the cache, counted
    through its pages.  A slot outside the cache (-1: padding) writes nothing; the
    slots inside it must differ.  `codes` and `scales` as from ``cache_alloc``, one of each
    for each of `x`; any strides but the last (a page may hold its heads before its rows).
    `x` counts as detached: no gradient goes through a cache."""
    if _entered:
        _order((*_tuple(x), slots), (*_tuple(codes), *_tuple(scales)))
    _ext.cache_write(x, slots, codes, scales)


def cache_read(slots: torch.Tensor, codes: Tensors, scales: Tensors, *, dtype: torch.dtype = torch.bfloat16,
               out: Optional[Tensors] = None) -> Tensors:
    """The rows of a cache at `slots` (token, head, element) in `dtype`, or written
    to `out`; zeros for a slot outside the cache.  Returns tensors as `codes` is given."""
    if _entered:
        _order((slots, *_tuple(codes), *_tuple(scales)), () if out is None else _tuple(out))
    code = _ROW_DTYPE.get(dtype)
    if code is None:
        raise TypeError("dtype must be float32, float16 or bfloat16")
    return _ext.cache_read(slots, codes, scales, out, code)


# ---- routing -----------------------------------------------------------------------
def route(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None,
          groups: int = 1, top_groups: int = 1, group_score: str = "max", renormalize: bool = False,
          scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(weights float32, experts int64), both (token, top_k), of logits (token,
    expert): the `top_k` experts with the largest score (+ `bias`, float32 [expert], for balance:
    it chooses and does not weigh; one number for all is no bias), in falling order, of equal
    ones the lowest index first.  With `groups`, only experts of the best `top_groups` groups are chosen from; a group is
    worth its largest key, or with ``group_score="top2"`` the sum of its two
    largest.  Weights are the scores, divided by their sum if `renormalize`, times `scale`.
    The choice is that of keys in 64 bits."""
    if _entered:
        _order((logits, bias))
    kind, rule = _choice(_SCORE, score, "score"), _choice(_GROUP_SCORE, group_score, "group_score")
    got = _ext.route(logits, bias, top_k, kind, groups, top_groups, rule, renormalize, scale)
    if got is NotImplemented:  # autograd has to record it
        return _Route.apply(logits, bias, top_k, (kind, groups, top_groups, rule, renormalize, scale))
    return got


def route_grad(logits: torch.Tensor, experts: torch.Tensor, grad_weights: torch.Tensor, *, score: str = "softmax",
               renormalize: bool = False, scale: float = 1.0) -> torch.Tensor:
    """The gradient of the logits from that of ``route``'s weights (float32)."""
    if _entered:
        _order((logits, experts, grad_weights))
    return _ext.route_grad(logits, experts, grad_weights, _choice(_SCORE, score, "score"), renormalize, scale)


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, top_k, how):
        weights, experts = _ext.route(logits, bias, top_k, *how)
        ctx.save_for_backward(logits, experts)
        ctx.how = (how[0], how[4], how[5])
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_weights, _):
        logits, experts = ctx.saved_tensors
        if _entered:
            _order((logits, experts, grad_weights))
        return _ext.route_grad(logits, experts, grad_weights, *ctx.how), None, None, None


# ---- log probabilities ---------------------------------------------------------------
class LogProbs(NamedTuple):
    logprob: torch.Tensor                  # float32 [row]
    entropy: Optional[torch.Tensor]        # float32 [row], nats
    top_logprobs: Optional[torch.Tensor]   # float32 (row, top)
    top_tokens: Optional[torch.Tensor]     # int64 (row, top)
    stats: Optional[torch.Tensor]          # float32 (row, 2), for logprobs_grad


def logprobs(logits: torch.Tensor, targets: torch.Tensor, *, top: int = 0, entropy: bool = False,
             temperature: float = 1.0, stats: bool = False) -> LogProbs:
    """Log probabilities of `targets` (int32 or int64 [row]) under
    ``softmax(logits / temperature)``, logits (row, token); with `entropy` the
    distribution's entropy, with `top` the likeliest tokens and their log probabilities (at
    most 64; of equal logits the lowest index first), with `stats` what
    ``logprobs_grad`` needs.  A negative target is padding (0).  Gradients flow to
    the logits from ``logprob`` and ``entropy``."""
    if _entered:
        _order((logits, targets))
    got = _ext.logprobs(logits, targets, top, entropy, temperature, stats)
    if got is NotImplemented:  # autograd has to record it
        got = _LogProbs.apply(logits, targets, top, entropy, temperature)
    return LogProbs._make(got)


def logprobs_grad(logits: torch.Tensor, targets: torch.Tensor, result: LogProbs,
                  grad_logprob: Optional[torch.Tensor], grad_entropy: Optional[torch.Tensor] = None, *,
                  temperature: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of the logits from those of ``logprobs``'s logprob and entropy
    (float32 [row]); `result` is what ``logprobs(..., stats=True)`` gave for the same
    arguments.  `out` may be `logits`, if autograd does not follow those (detach them)."""
    if result.stats is None:
        raise ValueError("result has no stats: call logprobs(..., stats=True)")
    if _entered:
        _order((logits, targets, result.stats, result.entropy, grad_logprob, grad_entropy), (out,))
    return _ext.logprobs_grad(logits, targets, result.stats, result.entropy, grad_logprob, grad_entropy, temperature, out)


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, entropy, temperature):
        got = _ext.logprobs(logits, targets, top, entropy, temperature, True)
        ctx.save_for_backward(logits, targets, got[1], got[4])
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in got[2:] if t is not None))
        return got

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logprob, grad_entropy, *_):
        if grad_logprob is None and grad_entropy is None:
            return (None,) * 5
        logits, targets, entropy, stats = ctx.saved_tensors
        if _entered:
            _order((logits, targets, stats, entropy, grad_logprob, grad_entropy))
        return (_ext.logprobs_grad(logits, targets, stats, entropy, grad_logprob, grad_entropy, ctx.temperature,
                                   None),) + (None,) * 4
