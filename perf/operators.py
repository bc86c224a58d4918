"""Cases of the row operators of a language model's step (gpuos_b200.rowops):

  rotary     rotary positions on queries and keys, and the inverse rotation (their gradient)
  cache      quantising keys and values as they are written to a paged cache, and reading them back
  route      routing tokens to experts, and its gradient
  logprobs   log probabilities of given tokens with entropy and top alternatives, and their gradient

`run` computes a case in elementary torch operations (32 bits; 64 for the angles of far positions and for the
selection keys of the router, whose ties a 32-bit rounding could turn), or, where `own` is set, through
gpuos_b200.rowops.  `exact` computes it in 64 bits from the operator's definition.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
QMAX = {"int8": 127.0, "e4m3": 448.0, "int4": 7.0}
CODE_BYTES = {"int8": 1.0, "e4m3": 1.0, "int4": 0.5}
TINY = 2.0 ** -100  # groups below it are stored as zeros


def listed():
    return [
        # one decode step of 8 sequences: 32 query and 8 key heads of 128 (4096 columns), far positions
        {"name": "rotary_decode_b8", "op": "rotary", "tokens": 8, "q_heads": 32, "k_heads": 8, "head_dim": 128, "rot_dim": 128,
         "interleaved": False, "inverse": False, "scaling": "none", "far": 131072, "dtype": "bf16"},
        # a packed prompt, half of each head rotated, interleaved pairs, frequencies scaled for a long context
        {"name": "rotary_prompt_partial", "op": "rotary", "tokens": 9001, "q_heads": 32, "k_heads": 8, "head_dim": 128,
         "rot_dim": 64, "interleaved": True, "inverse": False, "scaling": "ramp", "far": 1000000, "dtype": "fp16"},
        # the gradient of a training batch: the inverse rotation of the gradients of queries and keys
        {"name": "rotary_grad", "op": "rotary", "tokens": 16384, "q_heads": 32, "k_heads": 32, "head_dim": 128, "rot_dim": 128,
         "interleaved": False, "inverse": True, "scaling": "none", "far": 4096, "dtype": "bf16"},
        # one decode step of 64 sequences: a token each into an 8-bit cache, and those rows read back
        {"name": "cache_decode_b64_int8", "op": "cache", "tokens": 64, "rows": 16384, "page": 16, "heads": 8, "head_dim": 128,
         "group": 128, "format": "int8", "write": True, "dtype": "bf16"},
        # a prompt written to an fp8 cache and read back for its attention
        {"name": "cache_prompt_e4m3", "op": "cache", "tokens": 16000, "rows": 32768, "page": 64, "heads": 8, "head_dim": 128,
         "group": 128, "format": "e4m3", "write": True, "dtype": "bf16"},
        # a long context read back from a 4-bit cache with a scale for each 32 values
        {"name": "cache_long_read_int4", "op": "cache", "tokens": 100003, "rows": 131072, "page": 16, "heads": 8,
         "head_dim": 128, "group": 32, "format": "int4", "write": False, "dtype": "fp16"},
        # one decode step of 64 tokens over 64 experts
        {"name": "route_decode_b64", "op": "route", "tokens": 64, "experts": 64, "top_k": 6, "score": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "renormalize": True, "grad": False, "dtype": "bf16"},
        # a prompt over 256 experts in 8 groups, sigmoid scores with a bias for balance
        {"name": "route_prompt_groups", "op": "route", "tokens": 16384, "experts": 256, "top_k": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "renormalize": True, "grad": False, "dtype": "fp32"},
        # a training batch over 128 experts: weights and the gradient of the logits
        {"name": "route_train", "op": "route", "tokens": 32749, "experts": 128, "top_k": 8, "score": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "renormalize": False, "grad": True, "dtype": "bf16"},
        # the sampled tokens of one decode step of 8 sequences, with 20 alternatives
        {"name": "logprobs_decode_b8", "op": "logprobs", "tokens": 8, "vocab": 32000, "top": 20, "entropy": True,
         "temperature": 0.7, "grad": False, "dtype": "bf16"},
        # a prompt scored over a large vocabulary with an odd row length
        {"name": "logprobs_prompt", "op": "logprobs", "tokens": 2048, "vocab": 128257, "top": 5, "entropy": False,
         "temperature": 1.0, "grad": False, "dtype": "bf16"},
        # a policy-gradient step: log probabilities and entropy, then the gradient of the logits
        {"name": "logprobs_train", "op": "logprobs", "tokens": 1500, "vocab": 50257, "top": 0, "entropy": True,
         "temperature": 1.0, "grad": True, "dtype": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "cache", "route", "logprobs"])
    if op == "rotary":
        head = rng.choice([64, 80, 96, 128, 192, 256])
        rot = rng.choice([head, head // 2, head // 4])
        q = rng.choice([1, 4, 8, 16, 20, 32, 40])
        k = rng.choice([x for x in (1, 2, 4, 8, q) if x <= q])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = 16384 * 64 * 128 * 2 // ((q + k) * head * SIZE[dtype])
        return {"op": op, "tokens": _log_int(rng, 1, min(most, 40000)), "q_heads": q, "k_heads": k, "head_dim": head,
                "rot_dim": rot, "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.3,
                "scaling": rng.choice(["none", "linear", "ntk", "ramp"]), "far": _log_int(rng, 64, 2000000),
                "dtype": dtype}
    if op == "cache":
        head = rng.choice([64, 80, 96, 128, 256])
        group = rng.choice([head, 32 if head % 32 == 0 else head, 16])
        heads = rng.choice([1, 2, 4, 8, 16])
        most = 50000 * 8 * 128 // (heads * head)  # written and read back
        tokens = _log_int(rng, 1, min(most, 100003))
        page = rng.choice([1, 16, 32, 64, 100])
        return {"op": op, "tokens": tokens, "rows": -(-tokens * rng.choice([2, 3]) // page) * page, "page": page, "heads": heads,
                "head_dim": head, "group": group, "format": rng.choice(["int8", "e4m3", "int4"]),
                "write": rng.random() < 0.6, "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * rng.choice([8, 16, 20, 32, 48]) if groups > 1 else rng.choice([8, 16, 60, 64, 100, 128, 256, 384])
        top_groups = 1 if groups == 1 else rng.choice([2, 4])
        score = rng.choice(["softmax", "sigmoid"])
        bias = rng.random() < 0.5
        return {"op": op, "tokens": _log_int(rng, 1, 32749), "experts": experts, "top_k": rng.choice([1, 2, 4, 6, 8]),
                "score": score, "bias": bias, "groups": groups, "top_groups": top_groups,
                "renormalize": rng.random() < 0.6, "grad": rng.random() < 0.4, "dtype": rng.choice(["bf16", "fp32"])}
    vocab = _log_int(rng, 1000, 262144)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    grad = rng.random() < 0.4
    most = 2000 * 128257 // vocab // (SIZE[dtype] // 2 * (2 if grad else 1))
    return {"op": op, "tokens": _log_int(rng, 1, min(most, 20000)), "vocab": vocab,
            "top": 0 if grad else rng.choice([0, 1, 5, 20]), "entropy": rng.random() < 0.5,
            "temperature": rng.choice([1.0, 0.6, 1.3]), "grad": grad, "dtype": dtype}


def _inverse_frequencies(case):
    """Radians a position turns each pair by, in 64 bits."""
    n = case["rot_dim"]
    base, factor, length, low, high = 10000.0, 8.0, 8192.0, 1.0, 32.0
    if case["scaling"] == "ntk":
        base *= factor ** (n / (n - 2.0)) if n > 2 else 1.0
    f = base ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "ramp":  # pairs of many turns within the trained length stay, those of few are stretched
        keep = ((length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
    return f.cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t, dtype = case["tokens"], DTYPES[case["dtype"]]

    def randn(*shape, by=1.0, to=dtype):
        return torch.randn(*shape, generator=g, device="cuda").mul_(by).to(to)

    s = {"case": case}
    if case["op"] == "rotary":
        s["q"] = randn(t, case["q_heads"], case["head_dim"])
        s["k"] = randn(t, case["k_heads"], case["head_dim"])
        s["positions"] = torch.randint(0, case["far"], (t,), generator=g, device="cuda")
        s["inv_freq"] = _inverse_frequencies(case)
    elif case["op"] == "cache":
        page, rows, h, d = case["page"], case["rows"], case["heads"], case["head_dim"]
        # every token has a row of its own; one in sixteen is padding and has none
        s["slots"] = torch.randperm(rows, generator=g, device="cuda")[:t].contiguous()
        s["slots"][torch.rand(t, generator=g, device="cuda") < 1 / 16] = -1
        if case["write"]:  # keys have a few channels far larger than the rest
            wide = 1 + 7 * (torch.rand(d, generator=g, device="cuda") < 0.05)
            s["k"] = randn(t, h, d, to=torch.float32).mul_(wide).to(dtype)
            s["v"] = randn(t, h, d)
        for name in ("k", "v"):
            if case["format"] == "int8":
                codes = torch.randint(-127, 128, (rows // page, page, h, d), generator=g, device="cuda", dtype=torch.int8)
            elif case["format"] == "e4m3":
                codes = randn(rows // page, page, h, d, by=100.0, to=torch.float32).clamp_(-448, 448).to(torch.float8_e4m3fn)
            else:  # two codes of -7..7 to a byte, each with 8 added, the even one in the low half
                low, high = (torch.randint(1, 16, (rows // page, page, h, d // 2), generator=g, device="cuda", dtype=torch.uint8)
                             for _ in range(2))
                codes = low + high * 16
            s[name + "_codes"] = codes
            s[name + "_scale"] = torch.rand(rows // page, page, h, d // case["group"], generator=g, device="cuda") * 0.02 + 0.001
    elif case["op"] == "route":
        s["logits"] = randn(t, case["experts"], by=1.5)
        s["bias"] = randn(case["experts"], by=0.05, to=torch.float32) if case["bias"] else None
        s["grad"] = randn(t, case["top_k"], to=torch.float32) if case["grad"] else None
    else:
        s["logits"] = randn(t, case["vocab"], by=2.5)
        # half of the given tokens are the likeliest one, the others any
        first = s["logits"].argmax(-1)
        other = torch.randint(0, case["vocab"], (t,), generator=g, device="cuda")
        s["targets"] = torch.where(torch.rand(t, generator=g, device="cuda") < 0.5, first, other)
        if case["grad"]:
            s["grad_logprob"] = randn(t, to=torch.float32)
            s["grad_entropy"] = randn(t, by=0.01, to=torch.float32) if case["entropy"] else None
    return s


def run(s):
    return {"rotary": _rotary, "cache": _cache, "route": _route, "logprobs": _logprobs}[s["case"]["op"]](s)


def _rotary(s):
    c = s["case"]
    if own:
        from gpuos_b200 import rowops
        return rowops.rotary((s["q"], s["k"]), s["positions"], s["inv_freq"], interleaved=c["interleaved"], inverse=c["inverse"])
    angle = s["positions"].double()[:, None, None] * s["inv_freq"]
    cos, sin = angle.cos().float(), angle.sin().float()
    if c["inverse"]:
        sin = -sin
    return _turned(s["q"], cos, sin, c), _turned(s["k"], cos, sin, c)


def _turned(x, cos, sin, c):
    n, dtype = c["rot_dim"], x.dtype
    x, rest = x[..., :n].float(), x[..., n:]
    if c["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., : n // 2], x[..., n // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y.to(dtype), rest), -1)


def _cache(s):
    c = s["case"]
    dtype = DTYPES[c["dtype"]]
    codes, scales = (s["k_codes"], s["v_codes"]), (s["k_scale"], s["v_scale"])
    if own:
        from gpuos_b200 import rowops
        if c["write"]:
            rowops.cache_write((s["k"], s["v"]), s["slots"], codes, scales)
        k, v = rowops.cache_read(s["slots"], codes, scales, dtype=dtype)
    else:
        if c["write"]:
            _write(s["k"], s["slots"], s["k_codes"], s["k_scale"], c)
            _write(s["v"], s["slots"], s["v_codes"], s["v_scale"], c)
        k = _read(s["slots"], s["k_codes"], s["k_scale"], c, dtype)
        v = _read(s["slots"], s["v_codes"], s["v_scale"], c, dtype)
    return (k, v) + scales if c["write"] else (k, v)


def _write(x, slots, codes, scales, c):
    has = slots >= 0
    x, slots = x[has].float(), slots[has]
    x = x.unflatten(-1, (-1, c["group"]))
    most, full = x.abs().amax(-1, keepdim=True), QMAX[c["format"]]
    fits = most >= TINY
    y = (x * torch.where(fits, full / most, 0.0)).flatten(-2)
    if c["format"] == "int8":
        y = y.round().clamp(-127, 127).to(torch.int8)
    elif c["format"] == "e4m3":
        y = y.clamp(-448, 448).to(torch.float8_e4m3fn)
    else:
        y = (y.round().clamp(-7, 7) + 8).to(torch.uint8)
        y = y[..., 0::2] + y[..., 1::2] * 16
    codes.flatten(0, 1)[slots] = y
    scales.flatten(0, 1)[slots] = torch.where(fits, most / full, 0.0)[..., 0]


def _values(codes, form):
    if form != "int4":
        return codes.float()
    return torch.stack(((codes & 15).float() - 8, (codes >> 4).float() - 8), -1).flatten(-2)


def _read(slots, codes, scales, c, dtype):
    has, at = slots >= 0, slots.clamp(min=0)
    y = _values(codes.flatten(0, 1)[at], c["format"]).unflatten(-1, (-1, c["group"]))
    y = (y * scales.flatten(0, 1)[at][..., None]).flatten(-2)
    return torch.where(has[:, None, None], y, 0.0).to(dtype)


def _route(s):
    c = s["case"]
    rule = "top2" if c["score"] == "sigmoid" else "max"
    if own:
        from gpuos_b200 import rowops
        how = {"score": c["score"], "renormalize": c["renormalize"], "scale": 1.5}
        weights, experts = rowops.route(s["logits"], c["top_k"], bias=s["bias"], groups=c["groups"], top_groups=c["top_groups"],
                                        group_score=rule, **how)
        if not c["grad"]:
            return weights, experts
        return weights, experts, rowops.route_grad(s["logits"], experts, s["grad"], **how)
    x = s["logits"].double()  # next to the border of the chosen ones
    scores = x.softmax(-1) if c["score"] == "softmax" else x.sigmoid()
    keys = scores if s["bias"] is None else scores + s["bias"].double()
    if c["groups"] > 1:
        by = keys.unflatten(-1, (c["groups"], -1))
        best = by.amax(-1) if rule == "max" else by.topk(2, -1)[0].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True)[1][:, : c["top_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter(-1, kept, True)
        keys = torch.where(open_[..., None], by, -math.inf).flatten(-2)
    experts = keys.sort(dim=-1, descending=True, stable=True)[1][:, : c["top_k"]].contiguous()
    scores = scores.float()
    chosen = scores.gather(-1, experts)
    total = chosen.sum(-1, keepdim=True) if c["renormalize"] else torch.ones_like(chosen[:, :1])
    weights = chosen / total * 1.5
    if not c["grad"]:
        return weights, experts
    d = s["grad"] * 1.5
    if c["renormalize"]:
        d = (d - (d * chosen / total).sum(-1, keepdim=True)) / total
    dense = torch.zeros_like(scores).scatter(-1, experts, d)
    if c["score"] == "softmax":
        dense = scores * (dense - (d * chosen).sum(-1, keepdim=True))
    else:
        dense = dense * scores * (1 - scores)
    return weights, experts, dense.to(s["logits"].dtype)


def _logprobs(s):
    c = s["case"]
    if own:
        from gpuos_b200 import rowops
        r = rowops.logprobs(s["logits"], s["targets"], top=c["top"], entropy=c["entropy"], temperature=c["temperature"],
                            stats=c["grad"])
        got = [r.logprob] + ([r.entropy] if c["entropy"] else []) + ([r.top_logprobs, r.top_tokens] if c["top"] else [])
        if c["grad"]:
            got.append(rowops.logprobs_grad(s["logits"], s["targets"], r, s["grad_logprob"], s["grad_entropy"],
                                            temperature=c["temperature"]))
        return got
    x, at = s["logits"].float(), s["targets"][:, None]
    z = (x - x.amax(-1, keepdim=True)) / c["temperature"]
    e = z.exp()
    total = e.sum(-1, keepdim=True)
    logs = total.log()
    got = [(z.gather(-1, at) - logs)[:, 0]]
    if c["entropy"]:
        entropy = logs - (z * e).sum(-1, keepdim=True) / total
        got.append(entropy[:, 0])
    if c["top"]:  # the value in the upper half of the key, and the lowest index first in the lower one
        bits = (x + 0.0).view(torch.int32).long()
        index = torch.arange(c["vocab"], device=x.device)
        keys = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * 2 ** 32 + (2 ** 32 - 1 - index)
        tokens = 2 ** 32 - 1 - (keys.topk(c["top"], -1)[0] & 0xFFFFFFFF)
        got += [z.gather(-1, tokens) - logs, tokens]
    if c["grad"]:
        p, g = e / total, s["grad_logprob"][:, None]
        d = -g * p
        d.scatter_add_(-1, at, g)
        if c["entropy"]:
            d -= s["grad_entropy"][:, None] * p * (z - logs + entropy)
        got.append((d / c["temperature"]).to(s["logits"].dtype))
    return got


def work(case):
    t, size = case["tokens"], SIZE[case["dtype"]]
    if case["op"] == "rotary":
        n = t * (case["q_heads"] + case["k_heads"])
        return {"bytes": 2 * n * case["head_dim"] * size + 8 * t + 4 * case["rot_dim"], "flops": 3 * n * case["rot_dim"]}
    if case["op"] == "cache":
        n = 2 * t * case["heads"] * case["head_dim"]
        held = n * CODE_BYTES[case["format"]] + n // case["group"] * 4
        passes = 2 if case["write"] else 1
        return {"bytes": passes * (n * size + held + 8 * t), "flops": (3 * (passes - 1) + 1) * n}
    if case["op"] == "route":
        n = t * case["experts"]
        back = n * size + 4 * t * case["top_k"] if case["grad"] else 0
        return {"bytes": n * size + 12 * t * case["top_k"] + back, "flops": 4 * n}
    n = t * case["vocab"]
    return {"bytes": n * size * (2 if case["grad"] else 1) + t * (16 + 12 * case["top"]), "flops": n * (10 if case["grad"] else 5)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "cache": _exact_cache, "route": _exact_route, "logprobs": _exact_logprobs}[case["op"]](s)


def _exact_rotary(s):
    """Each pair as a complex number, times e^(i position frequency)."""
    c = s["case"]
    n = c["rot_dim"]
    angle = torch.outer(s["positions"].double(), s["inv_freq"])
    turn = torch.polar(torch.ones_like(angle), -angle if c["inverse"] else angle)
    got = []
    for x in (s["q"], s["k"]):
        y = x.double().clone()
        for h in range(y.shape[1]):
            part = y[:, h, :n]
            pairs = part.reshape(-1, n // 2, 2) if c["interleaved"] else part.reshape(-1, 2, n // 2).transpose(1, 2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            y[:, h, :n] = z.reshape(-1, n) if c["interleaved"] else z.transpose(1, 2).reshape(-1, n)
        got.append(y)
    return tuple(got)


def _exact_cache(s):
    """What the codes and scales stand for; rows of this call by the definition of the format."""
    c = s["case"]
    page, group, full = c["page"], c["group"], QMAX[c["format"]]
    rows = (s["slots"] >= 0).nonzero()[:, 0]
    at = s["slots"][rows]
    got, scales = [], []
    for name in ("k", "v"):
        codes, scale = s[name + "_codes"], s[name + "_scale"].double()
        t, h, d = c["tokens"], c["heads"], c["head_dim"]
        out = torch.zeros(t, h, d, dtype=torch.float64, device="cuda")
        if c["write"]:
            x = s[name][rows].double().reshape(-1, h, d // group, group)
            a = x.abs().max(-1).values
            step = a / full
            q = x / step.clamp(min=1e-300)[..., None]
            if c["format"] == "e4m3":  # 4 bits of mantissa from 2^-6 on, steps of 2^-9 below
                unit = torch.exp2(q.abs().clamp(min=2.0 ** -6).log2().floor() - 3)
                q = torch.round(q / unit) * unit
            else:
                q = torch.round(q)
            out[rows] = (q * step[..., None]).reshape(-1, h, d)
            scale.view(-1, h, d // group)[at] = step
        else:
            held = codes.reshape(-1, h, codes.shape[-1])[at]
            if c["format"] == "int4":
                q = torch.empty(len(at), h, d, dtype=torch.float64, device="cuda")
                q[..., 0::2] = (held % 16).double() - 8
                q[..., 1::2] = torch.div(held, 16, rounding_mode="floor").double() - 8
            else:
                q = held.double()
            q = q.reshape(-1, h, d // group, group)
            out[rows] = (q * scale.reshape(-1, h, d // group)[at][..., None]).reshape(-1, h, d)
        got.append(out)
        scales.append(scale)
    return tuple(got + scales) if c["write"] else tuple(got)


def _exact_route(s):
    c = s["case"]
    x = s["logits"].double()
    if c["score"] == "softmax":
        e = torch.exp(x - x.max(-1, keepdim=True).values)
        p = e / e.sum(-1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-x))
    key = p.clone() if s["bias"] is None else p + s["bias"].double()
    t, n = x.shape
    if c["groups"] > 1:
        per = key.reshape(t, c["groups"], -1)
        top = per.sort(dim=-1, descending=True).values
        worth = top[..., 0] + top[..., 1] if c["score"] == "sigmoid" else top[..., 0]
        # a group is out where `top_groups` others are better, or as good and before it
        better = worth[:, None, :] > worth[:, :, None]
        before = (worth[:, None, :] == worth[:, :, None]) & (torch.arange(c["groups"], device="cuda")[None, :]
                                                             < torch.arange(c["groups"], device="cuda")[:, None])
        out = (better | before).sum(-1) >= c["top_groups"]
        key[out.repeat_interleave(n // c["groups"], -1)] = -math.inf
    picked = []
    for _ in range(c["top_k"]):
        best = key.max(-1, keepdim=True).values
        picked.append((key == best).int().argmax(-1))  # the first of the largest
        key[torch.arange(t, device="cuda"), picked[-1]] = -math.inf
    index = torch.stack(picked, -1)
    w = p.gather(-1, index)
    norm = w.sum(-1, keepdim=True) if c["renormalize"] else 1.0
    weights = 1.5 * w / norm
    if not c["grad"]:
        return weights, index
    g = 1.5 * s["grad"].double()
    if c["renormalize"]:
        g = g / norm - (g * w).sum(-1, keepdim=True) / norm ** 2
    dx = torch.zeros_like(p).scatter_(-1, index, g)
    if c["score"] == "softmax":
        dx = p * dx - p * (p * dx).sum(-1, keepdim=True)
    else:
        dx = dx * (p - p * p)
    return weights, index, dx


def _exact_logprobs(s):
    c = s["case"]
    parts = []
    for lo in range(0, c["tokens"], 256):
        hi = min(lo + 256, c["tokens"])
        x = s["logits"][lo:hi].double() / c["temperature"]
        y = s["targets"][lo:hi]
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        p = lp.exp()
        entropy = -(p * lp).sum(-1, keepdim=True)
        row = [lp.gather(-1, y[:, None])[:, 0]]
        if c["entropy"]:
            row.append(entropy[:, 0])
        if c["top"]:
            # the values alone: which of equal ones are meant is said by the whole numbers of the other forms
            row.append(lp.topk(c["top"], -1).values)
        if c["grad"]:
            d = -p * s["grad_logprob"][lo:hi, None].double()
            d[torch.arange(hi - lo, device="cuda"), y] += s["grad_logprob"][lo:hi].double()
            if c["entropy"]:
                d -= s["grad_entropy"][lo:hi, None].double() * p * (lp + entropy)
            row.append(d / c["temperature"])
        parts.append(row)
    got = [torch.cat(column) for column in zip(*parts)]
    if c["top"]:
        got.insert(2 + c["entropy"], None)
    return got
