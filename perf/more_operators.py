"""Cases of the operators of a serving and training step that stand beside the row operators (gpuos_b200.rowops):

  attend    attention of queries over a paged cache held in 8 bits (what cache_write left there)
  verify    drafted tokens checked against the target's probabilities from given random numbers, and the next token
  experts   token rows sorted by the experts that route chose, the experts' results brought back with their weights,
            and the gradient of both

`run` computes a case in elementary torch operations (32 bits; 64 for verify, whose accepted counts and tokens a
32-bit sum could turn), or, where `own` is set, through gpuos_b200.rowops.  `exact` computes it in 64 bits from the
operator's definition.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one decode step of one conversation: a token over 700 cached ones, 32 query and 8 key heads of 128 (4096 columns)
        {"name": "attend_decode_b1", "op": "attend", "sequences": 1, "longest": 700, "queries": 1, "q_heads": 32, "k_heads": 8,
         "head_dim": 128, "group": 128, "page": 16, "format": "int8", "causal": True, "window": 0, "lse": False, "dtype": "bf16"},
        # one decode step of 64 sequences of ragged lengths
        {"name": "attend_decode_b64", "op": "attend", "sequences": 64, "longest": 8000, "queries": 1, "q_heads": 32, "k_heads": 8,
         "head_dim": 128, "group": 128, "page": 64, "format": "e4m3", "causal": True, "window": 0, "lse": False, "dtype": "bf16"},
        # two long documents, one token each: the work of a head has to be split along its length
        {"name": "attend_long", "op": "attend", "sequences": 2, "longest": 200001, "queries": 1, "q_heads": 32, "k_heads": 8,
         "head_dim": 128, "group": 128, "page": 16, "format": "int8", "causal": True, "window": 0, "lse": True, "dtype": "bf16"},
        # five drafted tokens of each of 24 sequences, a scale for each 32 values, only the last 1000 positions seen
        {"name": "attend_drafts_window", "op": "attend", "sequences": 24, "longest": 4000, "queries": 5, "q_heads": 16, "k_heads": 4,
         "head_dim": 64, "group": 32, "page": 100, "format": "int8", "causal": True, "window": 1000, "lse": False, "dtype": "fp16"},
        # the next chunk of two prompts, behind what is cached of them
        {"name": "attend_prompt", "op": "attend", "sequences": 2, "longest": 8192, "queries": 4096, "q_heads": 32, "k_heads": 8,
         "head_dim": 128, "group": 128, "page": 64, "format": "int8", "causal": True, "window": 0, "lse": False, "dtype": "bf16"},
        # four drafted tokens of one conversation; the drafts come from a lookup, so they have no probabilities
        {"name": "verify_b1", "op": "verify", "sequences": 1, "drafts": 4, "vocab": 32000, "probs": "", "temperature": 0.7,
         "dtype": "bf16"},
        # seven drafted tokens of 32 sequences by a draft model, over a large vocabulary with an odd row length
        {"name": "verify_b32", "op": "verify", "sequences": 32, "drafts": 7, "vocab": 128257, "probs": "fp32", "temperature": 1.0,
         "dtype": "bf16"},
        # tokens of 64 sequences drawn from given random numbers, nothing drafted
        {"name": "verify_draw_b64", "op": "verify", "sequences": 64, "drafts": 0, "vocab": 50257, "probs": "", "temperature": 0.8,
         "dtype": "fp32"},
        # one decode step of 8 tokens, each to 8 of 64 experts
        {"name": "experts_decode", "op": "experts", "tokens": 8, "top_k": 8, "experts": 64, "hidden": 2048, "align": 1,
         "elsewhere": 0.0, "grad": False, "dtype": "bf16"},
        # a packed prompt, half of whose 256 experts are on another device, rows of an expert padded to whole tiles of 16
        {"name": "experts_prompt_half", "op": "experts", "tokens": 9001, "top_k": 8, "experts": 256, "hidden": 2048, "align": 16,
         "elsewhere": 0.5, "grad": False, "dtype": "bf16"},
        # a training batch, each token to 2 of 8 experts
        {"name": "experts_train", "op": "experts", "tokens": 16384, "top_k": 2, "experts": 8, "hidden": 4096, "align": 1,
         "elsewhere": 0.0, "grad": False, "dtype": "bf16"},
        # the gradients of the same batch
        {"name": "experts_train_grad", "op": "experts", "tokens": 16384, "top_k": 2, "experts": 8, "hidden": 4096, "align": 1,
         "elsewhere": 0.0, "grad": True, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["attend", "verify", "experts"])
    if op == "attend":
        kind = rng.choice(["decode", "decode", "drafts", "prompt"])
        head = rng.choice([64, 80, 96, 128, 128, 256])
        k = rng.choice([1, 2, 4, 8])
        each = rng.choice([1, 2, 4, 5, 8, 16])
        window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if kind == "decode":
            queries, sequences = 1, _log_int(rng, 1, 128)
        elif kind == "drafts":
            queries, sequences = rng.randint(2, 8), _log_int(rng, 1, 48)
        else:
            queries, sequences = _log_int(rng, 16, 4096), rng.randint(1, 4)
        # as many positions as the listed cases have bytes of cache, and scores
        most = min(2 * 200001 * 8 * 128 // (sequences * k * head), 2 * 32 * 4096 * 8192 // (sequences * queries * k * each))
        if kind == "prompt":  # no more products than the listed prompts
            most = min(most, 2 * 4096 * 8192 * 32 * 128 // (sequences * queries * k * each * head) // (4 if dtype == "fp32" else 1))
        queries = min(queries, max(most, 1))
        return {"op": op, "sequences": sequences, "longest": _log_int(rng, queries, min(most, 100000)), "queries": queries,
                "q_heads": k * each, "k_heads": k, "head_dim": head,
                "group": rng.choice([head, head, 32 if head % 32 == 0 else head]), "page": rng.choice([1, 16, 32, 64, 100, 256]),
                "format": rng.choice(["int8", "e4m3"]), "causal": window > 0 or rng.random() < 0.8, "window": window,
                "lse": rng.random() < 0.3, "dtype": dtype}
    if op == "verify":
        vocab, drafts = _log_int(rng, 1000, 262144), rng.randint(0, 8)
        most = 32 * 8 * 128257 // (vocab * (drafts + 1))
        probs = rng.choice(["", "fp32", "bf16"]) if drafts else ""
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return {"op": op, "sequences": _log_int(rng, 1, min(most // (2 if dtype == "fp32" else 1), 256)), "drafts": drafts,
                "vocab": vocab, "probs": probs, "temperature": rng.choice([1.0, 0.6, 1.3, 0.0]), "dtype": dtype}
    hidden = rng.choice([256, 1000, 1536, 2050, 2880, 4096, 5120, 7168])
    top_k, experts = rng.choice([1, 2, 4, 6, 8]), rng.choice([8, 16, 60, 64, 100, 128, 256, 384])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    # as many bytes as the listed gradients
    most = 16384 * (3 * 2 + 2) * 4096 * 2 // (hidden * (3 * top_k + 2) * SIZE[dtype])
    tokens = _log_int(rng, 1, min(most, 32749))
    align = rng.choice([1, 1, 16, 64])
    if min(experts, tokens * top_k) * align > max(tokens * top_k, 1024):
        align = 1  # padding would be most of it
    return {"op": op, "tokens": tokens, "top_k": top_k, "experts": experts, "hidden": hidden, "align": align,
            "elsewhere": rng.choice([0.0, 0.0, 0.5]), "grad": rng.random() < 0.4, "dtype": dtype}


def _ragged(case):
    """Lengths from half the longest to the longest, and each sequence's new tokens (at most its length)."""
    n, longest, queries = case["sequences"], case["longest"], case["queries"]
    lengths = [max(1, longest - i * longest // (2 * n)) for i in range(n)]
    if queries <= 8:
        return lengths, [min(queries, length) for length in lengths]
    return lengths, [min(max(1, queries - i * queries // (2 * n)), length) for i, length in enumerate(lengths)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    {"attend": _prepare_attend, "verify": _prepare_verify, "experts": _prepare_experts}[case["op"]](case, s, g)
    return s


def _prepare_attend(c, s, g):
    dtype, n, page, h, d = DTYPES[c["dtype"]], c["sequences"], c["page"], c["k_heads"], c["head_dim"]
    lengths, queries = (torch.tensor(x, device="cuda") for x in _ragged(c))
    order = torch.randperm(n, generator=g, device="cuda")
    lengths, queries = lengths[order], queries[order]
    total = sum(_ragged(c)[1])
    s["lengths"] = lengths.int()
    s["offsets"] = torch.cat((queries.new_zeros(1), queries.cumsum(0))).int()
    s["longest"] = c["queries"]
    # pages lie anywhere in the pool; places of the table behind a sequence's last page name none
    width = -(-c["longest"] // page)
    used = -(-lengths // page)
    pool = sum(-(-length // page) for length in _ragged(c)[0]) + 3
    some = torch.randperm(pool, generator=g, device="cuda").int()
    slot = torch.arange(width, device="cuda")
    first = used.cumsum(0) - used
    s["pages"] = torch.where(slot < used[:, None], some[(first[:, None] + slot).clamp(max=pool - 1)], -1)
    s["q"] = torch.randn(total, c["q_heads"], d, generator=g, device="cuda").to(dtype)
    for name, most in (("k", 0.06), ("v", 0.02)):
        if c["format"] == "int8":
            codes = torch.randint(-127, 128, (pool, page, h, d), generator=g, device="cuda", dtype=torch.int8)
        else:
            codes = torch.randn(pool, page, h, d, generator=g, device="cuda").mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn)
        s[name + "_codes"] = codes
        s[name + "_scales"] = torch.rand(pool, page, h, d // c["group"], generator=g, device="cuda") * most + 0.001


def _prepare_verify(c, s, g):
    n, k, v = c["sequences"], c["drafts"], c["vocab"]
    dtype = DTYPES[c["dtype"]]
    s["logits"] = torch.randn(n, k + 1, v, generator=g, device="cuda").mul_(2.5).to(dtype)
    s["uniforms"] = torch.rand(n, k + 1, generator=g, device="cuda")
    s["probs"] = None
    if k == 0:
        s["drafts"] = torch.zeros(n, 0, dtype=torch.int64, device="cuda")
        return
    # a draft model that is somewhat off the target, and tokens drawn from it
    z = s["logits"][:, :k].float() + torch.randn(n, k, v, generator=g, device="cuda").mul_(0.5)
    p = (z / (c["temperature"] or 1.0)).softmax(-1)
    s["drafts"] = torch.multinomial(p.view(n * k, v), 1, generator=g).view(n, k)
    if not c["probs"] or c["temperature"] == 0:  # a lookup, or greedy choice: half of the drafts are the likeliest token
        likely = torch.rand(n, k, generator=g, device="cuda") < 0.75
        s["drafts"] = torch.where(likely, s["logits"][:, :k].argmax(-1), s["drafts"])
    if c["probs"]:
        s["probs"] = p.to(DTYPES[c["probs"]])


def _prepare_experts(c, s, g):
    t, k, e, hidden = c["tokens"], c["top_k"], c["experts"], c["hidden"]
    dtype = DTYPES[c["dtype"]]
    score = torch.randn(t, e, generator=g, device="cuda") + torch.randn(e, generator=g, device="cuda") * 0.5
    weights, experts = score.softmax(-1).topk(k, -1)
    s["weights"] = weights.contiguous()
    s["experts"] = torch.where(experts < e * (1 - c["elsewhere"]), experts, -1)

    def randn(n):
        return torch.randn(n, hidden, generator=g, device="cuda").to(dtype)

    rows = _rows(c)
    s["y"] = randn(rows)  # what the experts make of the rows
    if c["grad"]:
        s["order"] = _order(s["experts"], e, c["align"], rows)  # kept from the forward pass
        s["grad_rows"], s["grad_out"] = randn(rows), randn(t)
    else:
        s["x"] = randn(t)


def _rows(c):
    """Rows that any choice of experts fits in."""
    n = c["tokens"] * c["top_k"]
    return (n + min(c["experts"], n) * (c["align"] - 1)) // c["align"] * c["align"]


def run(s):
    return {"attend": _attend, "verify": _verify, "experts": _experts}[s["case"]["op"]](s)


def _attend(s):
    c = s["case"]
    if own:
        from gpuos_b200 import rowops
        return rowops.attend(s["q"], (s["k_codes"], s["v_codes"]), (s["k_scales"], s["v_scales"]), s["pages"], s["lengths"],
                             offsets=s["offsets"], longest=s["longest"], causal=c["causal"], window=c["window"] or None,
                             lse=c["lse"])
    q, lengths, offsets, h, d = s["q"], s["lengths"].long(), s["offsets"].long(), c["k_heads"], c["head_dim"]
    count = offsets[1:] - offsets[:-1]
    row = torch.arange(s["longest"], device=q.device)
    at = (offsets[:-1, None] + row).clamp(max=len(q) - 1)
    # (sequence, key head, query head of it and query, element), the shorter sequences filled up
    x = q[at].float().unflatten(2, (h, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3) * d ** -0.5
    k = _held(s["pages"], s["k_codes"], s["k_scales"])
    score = x @ k.permute(0, 2, 3, 1)
    del k
    position = torch.arange(score.shape[-1], device=q.device)
    last = (lengths - count)[:, None] + row if c["causal"] else (lengths - 1)[:, None].expand(-1, len(row))
    seen = (position <= last[..., None]) & (position < lengths[:, None, None])
    if c["window"]:
        seen &= position > last[..., None] - c["window"]
    score = score.unflatten(2, (-1, len(row)))
    score.masked_fill_(~seen[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    score.sub_(torch.where(most > -math.inf, most, 0.0)).exp_()
    total = score.sum(-1, keepdim=True)
    v = _held(s["pages"], s["v_codes"], s["v_scales"]).transpose(1, 2)
    out = (score.flatten(2, 3) @ v).unflatten(2, (-1, len(row))) / torch.where(total > 0, total, 1.0)
    # back to the packed tokens
    token = torch.arange(len(q), device=q.device)
    seq = torch.searchsorted(offsets[1:].contiguous(), token, right=True)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, token - offsets[seq]].to(q.dtype)
    if not c["lse"]:
        return out
    lse = (most + total.log()).squeeze(-1).permute(0, 3, 1, 2).flatten(2)
    return out, lse[seq, token - offsets[seq]]


def _held(pages, codes, scales):
    """(sequence, position, head, element) in 32 bits; positions of no page hold anything finite."""
    at = pages.clamp(min=0)
    x = codes.view(torch.uint8)[at].view(codes.dtype).float().flatten(1, 2)
    x.unflatten(-1, (scales.shape[-1], -1)).mul_(scales[at].flatten(1, 2)[..., None])
    return x


def _verify(s):
    c = s["case"]
    if own:
        from gpuos_b200 import rowops
        return tuple(rowops.verify(s["logits"], s["drafts"], s["uniforms"], probs=s["probs"], temperature=c["temperature"]))
    x, drafts, n = s["logits"], s["drafts"], c["drafts"]
    u = s["uniforms"].double()
    likeliest = x.argmax(-1)
    if c["temperature"] == 0:
        taken = drafts == likeliest[:, :n]
        accepted = taken.long().cumprod(-1).sum(-1)
        final = likeliest.gather(1, accepted[:, None])
    else:
        w = ((x.double() - x.amax(-1, keepdim=True).double()) / c["temperature"]).exp()
        total = w.sum(-1, keepdim=True)
        mine = w[:, :n].gather(-1, drafts[..., None])[..., 0]
        theirs = 1.0 if s["probs"] is None else s["probs"].gather(-1, drafts[..., None])[..., 0].double()
        taken = u[:, :n] * theirs * total[:, :n, 0] < mine
        accepted = taken.long().cumprod(-1).sum(-1)
        here = accepted[:, None, None]
        w = w.gather(1, here.expand(-1, 1, c["vocab"]))[:, 0]
        if n:  # what the draft has too much of is not drawn where it was refused
            refused, place = accepted < n, accepted.clamp(max=n - 1)[:, None]
            if s["probs"] is None:
                less = w.scatter(1, drafts.gather(1, place), 0.0)
            else:
                less = s["probs"].gather(1, place[..., None].expand(-1, 1, c["vocab"]))[:, 0].double()
                less = (w - less * total.gather(1, here)[:, 0]).clamp(min=0)
            w = torch.where((refused & (less.sum(-1) > 0))[:, None], less, w)
        sums = w.cumsum(-1)
        # the first place whose sum exceeds the share
        final = (sums <= u[:, n:] * sums[:, -1:]).sum(-1, keepdim=True)
    place = torch.arange(n + 1, device=x.device)
    tokens = torch.cat((drafts, final), -1)
    tokens = torch.where(place < accepted[:, None], tokens, torch.where(place == accepted[:, None], final, -1))
    return tokens, accepted


def _order(experts, count, align, rows):
    """Where each choice's row is (-1: nowhere), which choice a row is of (-1: none), where each expert's rows begin, how many they are."""
    flat = experts.flatten()
    key = torch.where((flat >= 0) & (flat < count), flat, count)
    sizes = torch.zeros(count + 1, dtype=torch.int64, device=key.device).scatter_add_(0, key, torch.ones_like(key))
    by = key.argsort(stable=True)
    padded = (sizes + align - 1) // align * align
    padded[count] = 0
    begin = padded.cumsum(0) - padded
    sorted_key = key[by]
    place = begin[sorted_key] + torch.arange(len(key), device=key.device) - (sizes.cumsum(0) - sizes)[sorted_key]
    place = torch.where(sorted_key < count, place, -1)
    places = torch.empty_like(key).scatter_(0, by, place)
    sources = torch.full((rows + 1,), -1, dtype=torch.int64, device=key.device)
    sources.scatter_(0, torch.where(place >= 0, place, rows), by)
    return places.view(experts.shape).int(), sources[:rows].int(), begin.int(), sizes[:count].int()


def _gathered(x, at):
    """Rows of x in 32 bits, zeros where `at` is negative."""
    return torch.where((at >= 0)[..., None], x[at.clamp(min=0).long()].float(), 0.0)


def _experts(s):
    c = s["case"]
    if own:
        from gpuos_b200 import rowops
        if c["grad"]:
            order = rowops.Order(*s["order"])
            return (rowops.combine(s["grad_rows"], order),) + tuple(rowops.combine_grad(s["grad_out"], s["y"], order, s["weights"]))
        order = rowops.order(s["experts"], c["experts"], align=c["align"])
        return (rowops.dispatch(s["x"], order), rowops.combine(s["y"], order, s["weights"])) + tuple(order)
    k, dtype = c["top_k"], s["y"].dtype
    if c["grad"]:
        places, sources = s["order"][:2]
        grad_x = _gathered(s["grad_rows"], places).sum(1).to(dtype)
        weight = torch.where(sources >= 0, s["weights"].flatten()[sources.clamp(min=0).long()], 0.0)
        grad_y = (_gathered(s["grad_out"], sources.div(k, rounding_mode="floor")) * weight[:, None]).to(dtype)
        grad_weights = (_gathered(s["y"], places) * s["grad_out"].float()[:, None]).sum(-1)
        return grad_x, grad_y, grad_weights
    order = _order(s["experts"], c["experts"], c["align"], len(s["y"]))
    rows = _gathered(s["x"], order[1].div(k, rounding_mode="floor")).to(dtype)
    out = (_gathered(s["y"], order[0]) * s["weights"][..., None]).sum(1).to(dtype)
    return (rows, out) + order


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "attend":
        lengths, queries = _ragged(case)
        h, d, groups = case["k_heads"], case["head_dim"], case["head_dim"] // case["group"]
        held = products = 0
        for length, n in zip(lengths, queries):
            seen = [min(length if not case["causal"] else length - n + i + 1, case["window"] or length) for i in range(n)]
            first = length - n + 1 - seen[0] if case["causal"] else length - seen[0]
            held += length - first
            products += sum(seen)
        q = sum(queries) * case["q_heads"]
        return {"bytes": 2 * held * h * (d + 4 * groups) + 2 * q * d * size + (4 * q if case["lse"] else 0)
                + 4 * (2 * len(lengths) + 1 + held // case["page"]), "flops": 4 * products * case["q_heads"] * d}
    if case["op"] == "verify":  # the drafts' rows, and one row of the draft's probabilities where the first is refused
        rows, v = case["sequences"] * (case["drafts"] + 1), case["vocab"]
        probs = case["sequences"] * v * SIZE[case["probs"]] if case["probs"] and case["temperature"] else 0
        return {"bytes": rows * (v * size + 20) + probs, "flops": 4 * rows * v}
    t, k, hidden = case["tokens"], case["top_k"], case["hidden"]
    here = int(t * k * (1 - case["elsewhere"]))
    if case["grad"]:  # rows and results of the experts read, gradients of the results written, those of the tokens in and out
        return {"bytes": (3 * here + 2 * t) * hidden * size + 16 * t * k, "flops": 4 * here * hidden}
    return {"bytes": (here + _rows(case) + 2 * t) * hidden * size + 20 * t * k, "flops": 2 * here * hidden}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "verify": _exact_verify, "experts": _exact_experts}[case["op"]](s)


def _exact_attend(s):
    """Sequence by sequence and head by head, queries in slices."""
    c = s["case"]
    each, page = c["q_heads"] // c["k_heads"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    lengths, offsets = s["lengths"].tolist(), s["offsets"].tolist()
    for b, length in enumerate(lengths):
        lo, hi = offsets[b], offsets[b + 1]
        own_pages = s["pages"][b, : -(-length // page)].long()
        for h in range(c["k_heads"]):
            k, v = ((s[name + "_codes"][:, :, h].view(torch.uint8)[own_pages].view(s[name + "_codes"].dtype).double()
                     .reshape(-1, c["head_dim"] // c["group"], c["group"])
                     * s[name + "_scales"][own_pages, :, h].double().reshape(-1, c["head_dim"] // c["group"], 1)).flatten(1)[:length]
                    for name in ("k", "v"))
            for at in range(lo, hi, 1024):
                end = min(at + 1024, hi)
                x = s["q"][at:end, h * each: (h + 1) * each].double().transpose(0, 1)
                z = torch.einsum("gnd,ld->gnl", x, k) / math.sqrt(c["head_dim"])
                j = torch.arange(length, device="cuda")[None]
                i = torch.arange(at - lo, end - lo, device="cuda")[:, None] + length - (hi - lo)
                hidden = torch.zeros(len(i), length, dtype=torch.bool, device="cuda")
                if c["causal"]:
                    hidden |= j > i
                if c["window"]:
                    hidden |= i - j >= c["window"]
                z.masked_fill_(hidden, -math.inf)
                norm = torch.logsumexp(z, -1, keepdim=True)
                out[at:end, h * each: (h + 1) * each] = (torch.exp(z - norm) @ v).transpose(0, 1)
                lse[at:end, h * each: (h + 1) * each] = norm[..., 0].transpose(0, 1)
    return (out, lse) if c["lse"] else out


def _exact_verify(s):
    """Draft by draft, as it is told: accept with chance p / q, else draw from what p has more than q."""
    c = s["case"]
    n, v = c["drafts"], c["vocab"]
    tokens = torch.full((c["sequences"], n + 1), -1, dtype=torch.int64, device="cuda")
    accepted = torch.zeros(c["sequences"], dtype=torch.int64, device="cuda")
    drafts, uniforms = s["drafts"].tolist(), s["uniforms"].tolist()
    for b in range(c["sequences"]):
        i, weight = 0, None
        while True:
            x = s["logits"][b, i].double()
            if c["temperature"] == 0:
                best = (x == x.max()).nonzero()[0, 0].item()
                if i < n and drafts[b][i] == best:
                    tokens[b, i] = best
                    i += 1
                    continue
                final = best
                break
            p = torch.exp((x - x.max()) / c["temperature"])
            if i < n:
                d = drafts[b][i]
                q = torch.zeros(v, dtype=torch.float64, device="cuda")
                q[d] = 1.0
                if s["probs"] is not None:
                    q = s["probs"][b, i].double()
                if uniforms[b][i] * q[d] < p[d] / p.sum():
                    tokens[b, i] = d
                    i += 1
                    continue
                weight = torch.relu(p - q * p.sum())
            if weight is None or weight.sum() == 0:
                weight = p
            share = weight.cumsum(0)
            final = torch.searchsorted(share, share[-1:] * uniforms[b][n], right=True).item()
            break
        tokens[b, i] = final
        accepted[b] = i
    return tokens, accepted


def _exact_experts(s):
    c = s["case"]
    t, k, hidden, dev = c["tokens"], c["top_k"], c["hidden"], "cuda"
    rows = len(s["y"])
    weights = s["weights"].double()
    if c["grad"]:
        places = s["order"][0].long()
        grad_x = torch.zeros(t, hidden, dtype=torch.float64, device=dev)
        grad_y = torch.zeros(rows, hidden, dtype=torch.float64, device=dev)
        grad_weights = torch.zeros(t, k, dtype=torch.float64, device=dev)
        for j in range(k):
            has = (places[:, j] >= 0).nonzero()[:, 0]
            at = places[has, j]
            g = s["grad_out"][has].double()
            grad_x[has] += s["grad_rows"][at].double()
            grad_y[at] = g * weights[has, j, None]
            grad_weights[has, j] = torch.einsum("nh,nh->n", g, s["y"][at].double())
        return grad_x, grad_y, grad_weights
    experts = s["experts"]
    places = torch.full((t, k), -1, dtype=torch.int64, device=dev)
    sources = torch.full((rows,), -1, dtype=torch.int64, device=dev)
    begin, sizes, at = [], [], 0
    for e in range(c["experts"]):
        mine = (experts == e).flatten().nonzero()[:, 0]  # in the order of the tokens
        begin.append(at)
        sizes.append(len(mine))
        spot = torch.arange(at, at + len(mine), device=dev)
        places.view(-1)[mine] = spot
        sources[spot] = mine
        at += -(-len(mine) // c["align"]) * c["align"]
    begin.append(at)
    out = torch.zeros(t, hidden, dtype=torch.float64, device=dev)
    moved = torch.zeros(rows, hidden, dtype=torch.float64, device=dev)
    for j in range(k):
        has = (places[:, j] >= 0).nonzero()[:, 0]
        spot = places[has, j]
        moved[spot] = s["x"][has].double()
        out[has] += s["y"][spot].double() * weights[has, j, None]
    return moved, out, places.int(), sources.int(), torch.tensor(begin, device=dev).int(), torch.tensor(sizes, device=dev).int()
