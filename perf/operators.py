"""The serving and position operators as they are measured: rotary positions, the append to a paged
key/value cache, attention over that cache for a batch that shares a prefix, and the verification of
drafted tokens.

With ``own`` false every operator runs in its plain form (elementary torch operations in 32 bits, 64 where
32 lose what matters); with ``own`` true it is the call a user makes of this package.  ``listed`` gives the
cases, ``draw`` more of the same ranges, ``exact`` the results in 64 bits.
"""
import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"


# --- cases ------------------------------------------------------------------------------------------------


def listed():
    return [
        # Positions of a small decode batch: a few tokens far into their contexts; latency.
        {"name": "rotary-decode", "op": "rotary", "tokens": 7, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "interleaved": False, "dtype": "bf16", "scaling": "log_ramp", "factor": 16.0, "context": 8192,
         "far": 1000000, "backward": False},
        # Queries and keys of a training batch on their way into the attention.
        {"name": "rotary-train", "op": "rotary", "tokens": 16384, "hq": 32, "hkv": 8, "d": 128, "rot": 128,
         "interleaved": False, "dtype": "bf16", "scaling": "none", "factor": 1.0, "context": 8192,
         "far": 8192, "backward": False},
        # The same in the backward pass, f32, neighbours as pairs, half of each head rotated, an odd token count.
        {"name": "rotary-gradient", "op": "rotary", "tokens": 6001, "hq": 16, "hkv": 16, "d": 64, "rot": 32,
         "interleaved": True, "dtype": "f32", "scaling": "ramp", "factor": 8.0, "context": 8192,
         "far": 65536, "backward": True},
        # One decode step's keys and values of a running batch.
        {"name": "append-decode", "op": "append", "batch": 61, "new": 1, "len": 900, "prefix": 2048, "hq": 32,
         "hkv": 8, "d": 128, "rot": 128, "interleaved": False, "dtype": "bf16", "page": 16, "head_major": False},
        # Prompts of several requests packed into one batch, each its own length.
        {"name": "append-prompts", "op": "append", "batch": 12, "new": 1500, "len": 2000, "prefix": 0, "hq": 28,
         "hkv": 4, "d": 128, "rot": 64, "interleaved": True, "dtype": "f16", "page": 64, "head_major": True},
        # One user's long conversation: few rows, a long axis.
        {"name": "attention-one-long", "op": "attention", "batch": 1, "new": 1, "len": 50001, "prefix": 0,
         "hq": 32, "hkv": 8, "d": 128, "dtype": "bf16", "page": 16, "head_major": False},
        # A decode batch behind one long system prompt, each with a conversation of its own.
        {"name": "attention-shared", "op": "attention", "batch": 128, "new": 1, "len": 1000, "prefix": 8192,
         "hq": 64, "hkv": 8, "d": 128, "dtype": "bf16", "page": 64, "head_major": False},
        # Drafted tokens of a batch under verification: several queries a sequence.
        {"name": "attention-drafts", "op": "attention", "batch": 33, "new": 5, "len": 2500, "prefix": 500,
         "hq": 16, "hkv": 4, "d": 64, "dtype": "f16", "page": 32, "head_major": True},
        # Prompt chunks behind what is cached already.
        {"name": "attention-prompts", "op": "attention", "batch": 5, "new": 1024, "len": 3500, "prefix": 1111,
         "hq": 32, "hkv": 8, "d": 128, "dtype": "bf16", "page": 16, "head_major": False},
        # A small batch in f32, as the package's dense attention takes its operands.
        {"name": "attention-f32", "op": "attention", "batch": 9, "new": 2, "len": 700, "prefix": 333,
         "hq": 12, "hkv": 4, "d": 64, "dtype": "f32", "page": 16, "head_major": False},
        # One sequence's drafts, the target's and the drafter's probabilities in hand.
        {"name": "verify-one", "op": "verify", "batch": 1, "drafts": 5, "vocab": 32000, "certain": False},
        # A batch of them over a large odd vocabulary.
        {"name": "verify-batch", "op": "verify", "batch": 64, "drafts": 4, "vocab": 131071, "certain": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = [work(c) for c in listed()]
    while True:
        case = _drawn(rng)
        w = work(case)
        if w["bytes"] <= max(m["bytes"] for m in most) and w["flops"] <= max(m["flops"] for m in most):
            return case


def _drawn(rng):
    op = rng.choice(["rotary", "append", "attention", "attention", "verify"])
    if op == "verify":
        return {"op": op, "batch": _log(rng, 1, 64), "drafts": rng.randint(1, 8) if rng.random() < 0.7 else 1,
                "vocab": _log(rng, 257, 65536), "certain": rng.random() < 0.3}
    d = rng.choice([64, 128, 128, 96, 256, 80])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    hkv = rng.choice([1, 2, 4, 8])
    case = {"op": op, "hq": hkv * rng.choice([1, 3, 4, 7, 8]), "hkv": hkv, "d": d, "dtype": dtype}
    if op == "rotary":
        case |= {"tokens": _log(rng, 1, 8192), "rot": rng.choice([d, d, d // 2, 32]),
                 "interleaved": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "base", "ramp", "log_ramp"]),
                 "factor": rng.choice([2.0, 5.0, 16.0]), "context": 8192, "far": _log(rng, 2048, 4000000),
                 "backward": rng.random() < 0.5}
        if case["scaling"] == "none":
            case["factor"] = 1.0
        return case
    case |= {"page": rng.choice([8, 16, 32, 64, 128, 20]), "head_major": rng.random() < 0.5,
             "prefix": _log(rng, 100, 4096) if rng.random() < 0.6 else 0}
    many = rng.random() < 0.3
    if op == "append":
        case |= {"batch": _log(rng, 1, 8) if many else _log(rng, 1, 128), "new": _log(rng, 64, 1024) if many else rng.choice([1, 1, 5])}
        case |= {"len": case["new"] + _log(rng, 1, 1000), "rot": rng.choice([d, d, d // 2]), "interleaved": rng.random() < 0.5}
        return case
    case |= {"batch": _log(rng, 1, 4) if many else _log(rng, 1, 64), "new": _log(rng, 16, 512) if many else rng.choice([1, 1, 2, 6])}
    return case | {"len": case["new"] + _log(rng, 1, 2048)}


def _spread(n, lo, hi, salt):
    """n whole numbers of [lo, hi], spread over it and in no order, by the case alone; the first is hi."""
    return [lo + int((hi - lo) * (1.0 - (i * (0.6180339887 + 0.1 * salt)) % 1.0) + 0.5) for i in range(n)]


def _tokens(case):
    """(new tokens, cached tokens with them) of each sequence."""
    new = _spread(case["batch"], min(case["new"], max(1, case["new"] // 4)), case["new"], 0)
    cached = _spread(case["batch"], max(1, case["len"] // 4), case["len"], 1)
    return new, [max(a, b) for a, b in zip(new, cached)]


def work(case):
    if case["op"] == "verify":
        # one row of p and, but for certain drafts, of q: what a rejected sequence needs
        rows = 1 if case["certain"] else 2
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        return {"bytes": 4 * b * (rows * v + rows * k + 3 * k + 3), "flops": 3 * b * v}
    size, d = DTYPES[case["dtype"]].itemsize, case["d"]
    if case["op"] == "rotary":
        n = case["tokens"] * (case["hq"] + case["hkv"])
        return {"bytes": 2 * n * d * size + 8 * case["tokens"], "flops": 3 * n * case["rot"]}
    new, cached = _tokens(case)
    if case["op"] == "append":
        n = sum(new)
        return {"bytes": 2 * n * (case["hq"] + 2 * case["hkv"]) * d * size + 8 * case["batch"] + 4 * n,
                "flops": 3 * n * (case["hq"] + case["hkv"]) * case["rot"]}
    keys = case["prefix"] + sum(cached)
    pairs = sum(n * (case["prefix"] + c - n) + n * (n + 1) // 2 for n, c in zip(new, cached))
    return {"bytes": 2 * keys * case["hkv"] * d * size + 2 * sum(new) * case["hq"] * d * size + 4 * keys // case["page"],
            "flops": 4 * pairs * case["hq"] * d}


# --- inputs -----------------------------------------------------------------------------------------------


def _frequencies(case):
    """Radians a position of each pair, in 64 bits, on the GPU."""
    r, s, theta = case["rot"], case.get("factor", 1.0), 10000.0
    kind = case.get("scaling", "none")
    if kind == "base":
        theta *= s ** (r / (r - 2))
    f = theta ** (-torch.arange(0, r, 2, dtype=torch.float64, device=DEVICE) / r)
    if kind == "linear":
        f = f / s
    if kind in ("ramp", "log_ramp"):
        t = case["context"] * f / (2 * math.pi)
        w = (t - 1) / (32 - 1) if kind == "ramp" else torch.log(t) / math.log(32)
        w = w.clamp(0, 1)
        f = f * (w + (1 - w) / s)
    return f


def _magnitude(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case.get("scaling") == "log_ramp" else 1.0


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "verify":
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        logits = 2.5 * torch.randn(b, k + 1, v, device=DEVICE, generator=g)
        s["target"] = torch.softmax(logits, -1)
        if case["certain"]:
            s["draft"] = None
            s["tokens"] = logits[:, :k].argmax(-1).to(torch.int32)
        else:
            s["draft"] = torch.softmax(logits[:, :k] + 0.7 * torch.randn(b, k, v, device=DEVICE, generator=g), -1)
            s["tokens"] = torch.multinomial(s["draft"].reshape(b * k, v), 1, generator=g).reshape(b, k).to(torch.int32)
        s["u_accept"] = torch.rand(b, k, device=DEVICE, generator=g)
        s["u_sample"] = torch.rand(b, device=DEVICE, generator=g)
        s["accepted"] = torch.empty(b, dtype=torch.int32, device=DEVICE)
        s["out"] = torch.empty(b, k + 1, dtype=torch.int32, device=DEVICE)
        return _handle(s) if own else s
    dt, hq, hkv, d = DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"]
    if case["op"] == "rotary":
        n = case["tokens"]
        # queries, keys and values as one projection writes them, or their gradients
        qkv = torch.randn(n, hq + 2 * hkv, d, device=DEVICE, generator=g).to(dt)
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hkv]
        s["positions"] = torch.randint(0, case["far"], (n,), device=DEVICE, generator=g)
        s["frequencies"] = _frequencies(case)
        s["q_out"], s["k_out"] = torch.empty_like(s["q"], memory_format=torch.contiguous_format), torch.empty_like(s["k"], memory_format=torch.contiguous_format)
        return _handle(s) if own else s
    new, cached = _tokens(case)
    n, page, prefix = sum(new), case["page"], case["prefix"]
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    s["cu"], s["lengths"], s["tokens"], s["max_new"], s["max_len"] = _ints(cu), _ints(cached), n, max(new), max(cached)
    # pages handed out in no order, the prefix's first; a few stay free
    width, head = -(-max(cached) // page), -(-prefix // page)
    need = [-(-x // page) for x in cached]
    pages = head + sum(need) + 3
    order = torch.randperm(pages, device=DEVICE, generator=g).to(torch.int32)
    at = torch.tensor([head + sum(need[:b]) for b in range(len(need))], device=DEVICE)
    col = torch.arange(width, device=DEVICE)
    inside = col[None] < torch.tensor(need, device=DEVICE)[:, None]
    s["prefix_table"] = order[:head].contiguous()
    s["table"] = torch.where(inside, order[(at[:, None] + col[None]).clamp(max=pages - 1)], 0).to(torch.int32)
    shape = (pages, hkv, page, d) if case["head_major"] else (pages, page, hkv, d)
    s["k_cache"] = torch.randn(shape, device=DEVICE, generator=g, dtype=dt)
    s["v_cache"] = torch.randn(shape, device=DEVICE, generator=g, dtype=dt)
    s["pages"] = pages
    if case["op"] == "append":
        qkv = torch.randn(n, hq + 2 * hkv, d, device=DEVICE, generator=g).to(dt)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["frequencies"] = _frequencies(case)
        s["q_out"] = torch.empty(n, hq, d, device=DEVICE, dtype=dt)
    else:
        s["q"] = (1.5 * torch.randn(n, hq, d, device=DEVICE, generator=g)).to(dt)
        s["o"] = torch.empty_like(s["q"])
    return _handle(s) if own else s


# --- the package's calls ------------------------------------------------------------------------------------

_context = None


def _runtime():
    """The package's runtime and one context of it, as a program keeps them."""
    global _context
    rt = importlib.import_module("emmy-hackathon-2026_b200.runtime")
    if _context is None:
        _context = rt.Context(torch.cuda.current_device())
    return rt, _context


def _heads(rt, x):
    return rt.heads(x.data_ptr(), x.shape[1], x.stride(0), x.stride(1))


def _handle(s):
    """The plans, the workspace and the bound call that a program's loop keeps."""
    rt, ctx = _runtime()
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    if case["op"] == "verify":
        s["call"] = ctx.verify_drafts_call(
            s["target"].data_ptr(), s["tokens"].data_ptr(), s["u_accept"].data_ptr(), s["u_sample"].data_ptr(),
            s["accepted"].data_ptr(), s["out"].data_ptr(), case["batch"], case["drafts"], case["vocab"],
            draft=0 if s["draft"] is None else s["draft"].data_ptr(), stream=stream)
        return s
    dt = {"f32": rt.F32, "f16": rt.F16, "bf16": rt.BF16}[case["dtype"]]
    rope = None
    if "rot" in case:
        rope = rt.rope_plan(case["rot"], theta=10000.0, interleaved=case["interleaved"], scaling=case.get("scaling", "none"),
                            factor=case.get("factor", 1.0), context=case.get("context", 0), low=1.0, high=32.0,
                            magnitude=_magnitude(case))
    if case["op"] == "rotary":
        s["call"] = ctx.rotary_call(rope, dt, [(_heads(rt, s["q"]), _heads(rt, s["q_out"])), (_heads(rt, s["k"]), _heads(rt, s["k_out"]))],
                                    s["positions"].data_ptr(), case["tokens"], case["d"], transpose=case["backward"], stream=stream)
        return s
    cache = rt.paged_cache(s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), dt, s["pages"], case["page"], case["hkv"],
                           case["d"], head_major=case["head_major"])
    batch = rt.paged_batch(case["batch"], s["tokens"], s["cu"].data_ptr(), s["lengths"].data_ptr(), s["table"].data_ptr(),
                           s["table"].shape[1], max_new=s["max_new"], max_len=s["max_len"], prefix_len=case["prefix"],
                           prefix_table=s["prefix_table"].data_ptr())
    if case["op"] == "append":
        s["call"] = ctx.paged_append_call(cache, batch, _heads(rt, s["k"]), _heads(rt, s["v"]), q=_heads(rt, s["q"]),
                                          q_out=_heads(rt, s["q_out"]), rope=rope, stream=stream)
        return s
    nbytes = ctx.paged_attention_workspace(cache, batch, case["hq"])
    s["workspace"] = torch.empty(max(16, nbytes), dtype=torch.uint8, device=DEVICE)
    s["call"] = ctx.paged_attention_call(cache, batch, _heads(rt, s["q"]), _heads(rt, s["o"]), s["workspace"].data_ptr(), nbytes, stream=stream)
    return s


def run(state):
    if own:
        state["call"]()
        op = state["case"]["op"]
        if op == "verify":
            return {"accepted": state["accepted"], "tokens": state["out"]}
        if op == "rotary":
            return {"q": state["q_out"], "k": state["k_out"]}
        if op == "append":
            return {"q": state["q_out"], "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
        return {"o": state["o"]}
    return {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention, "verify": _plain_verify}[state["case"]["op"]](state)


# --- plain forms --------------------------------------------------------------------------------------------


def _rotate(x, positions, frequencies, case, sign=1.0):
    """x [tokens, heads, d] rotated to its positions; angles in 64 bits, the rest in 32, rounded once."""
    angle = positions.double()[:, None] * frequencies
    c = (torch.cos(angle) * _magnitude(case)).float()[:, None]
    s = (torch.sin(angle) * (sign * _magnitude(case))).float()[:, None]
    r, y = case["rot"], x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if case["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
    ra, rb = a * c - b * s, b * c + a * s
    turned = torch.stack([ra, rb], -1).flatten(-2) if case["interleaved"] else torch.cat([ra, rb], -1)
    return torch.cat([turned, y[..., r:]], -1).to(x.dtype)


def _plain_rotary(s):
    sign = -1.0 if s["case"]["backward"] else 1.0
    return {n: _rotate(s[n], s["positions"], s["frequencies"], s["case"], sign) for n in ("q", "k")}


def _places(s):
    """(sequence, position among its own tokens) of each packed token."""
    token = torch.arange(s["tokens"], device=DEVICE, dtype=torch.int32)
    b = torch.searchsorted(s["cu"], token, right=True) - 1
    new = s["cu"][1:] - s["cu"][:-1]
    return b, (s["lengths"] - new)[b] + token - s["cu"][b]


def _plain_append(s):
    case, page = s["case"], s["case"]["page"]
    b, at = _places(s)
    q = _rotate(s["q"], case["prefix"] + at, s["frequencies"], case)
    k = _rotate(s["k"], case["prefix"] + at, s["frequencies"], case)
    pages, row = s["table"][b, at // page], at % page
    if case["head_major"]:
        s["k_cache"][pages, :, row] = k
        s["v_cache"][pages, :, row] = s["v"]
    else:
        s["k_cache"][pages, row] = k
        s["v_cache"][pages, row] = s["v"]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _keys(cache, table, case, n):
    """cache rows of the pages in `table` [..., pages] in 32 bits: [..., heads, n, d]."""
    x = cache[table].float()
    x = x.movedim(-3, -4) if case["head_major"] else x
    # [..., pages, page, heads, d] or, head major, [..., heads, pages, page, d]
    if case["head_major"]:
        return x.flatten(-3, -2)[..., :n, :]
    return x.flatten(-4, -3).movedim(-2, -3)[..., :n, :]


def _plain_attention(s):
    case = s["case"]
    hq, hkv, d, p = case["hq"], case["hkv"], case["d"], case["prefix"]
    b, at = _places(s)
    n, batch, longest = s["tokens"], case["batch"], s["max_len"]
    j = torch.arange(n, device=DEVICE) - s["cu"][b]
    scaled = s["q"].float() / math.sqrt(d)
    # [sequence, kv head, new token, its query heads, d], short sequences filled up with zeros
    q = torch.zeros(batch, s["max_new"], hkv, hq // hkv, d, device=DEVICE)
    q[b, j] = scaled.view(n, hkv, hq // hkv, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)
    k, v = _keys(s["k_cache"], s["table"], case, longest), _keys(s["v_cache"], s["table"], case, longest)
    own_keys = torch.full((batch, s["max_new"]), -1, device=DEVICE, dtype=at.dtype)
    own_keys[b, j] = at
    seen = torch.arange(longest, device=DEVICE) <= own_keys[:, :, None]
    seen = seen[:, None, :, None].expand(-1, hkv, -1, hq // hkv, -1).reshape(batch, hkv, -1, longest)
    score = (q @ k.transpose(-1, -2)).masked_fill(~seen, -math.inf)
    qp = q.transpose(0, 1).reshape(hkv, -1, d)
    kp, vp = _keys(s["k_cache"], s["prefix_table"], case, p), _keys(s["v_cache"], s["prefix_table"], case, p)
    before = qp @ kp.transpose(-1, -2)
    rows = q.shape[2]
    before = before.view(hkv, batch, rows, p).transpose(0, 1)
    top = score.amax(-1, keepdim=True)
    if p:
        top = torch.maximum(top, before.amax(-1, keepdim=True))
    top = top.clamp(min=torch.finfo(torch.float32).min)
    score, before = torch.exp(score - top), torch.exp(before - top)
    total = score.sum(-1, keepdim=True) + before.sum(-1, keepdim=True)
    o = score @ v + (before.transpose(0, 1).reshape(hkv, batch * rows, p) @ vp).view(hkv, batch, rows, d).transpose(0, 1)
    o = (o / total).view(batch, hkv, s["max_new"], hq // hkv, d)[b, :, j]
    return {"o": o.reshape(n, hq, d).to(s["q"].dtype)}


def _plain_verify(s):
    b, k = s["tokens"].shape
    x = s["tokens"].long()[..., None]
    p = s["target"][:, :k].gather(-1, x)[..., 0].double()
    q = torch.ones_like(p) if s["draft"] is None else s["draft"].gather(-1, x)[..., 0].double()
    taken = (s["u_accept"].double() * q < p).long().cumprod(-1)
    accepted = taken.sum(-1)
    rows = torch.arange(b, device=DEVICE)
    p = s["target"][rows, accepted].double()
    last = accepted.clamp(max=k - 1)
    if s["draft"] is None:
        q = torch.zeros_like(p).scatter_(-1, x[rows, last], math.inf)
    else:
        q = s["draft"][rows, last].double()
    rest = torch.where((accepted < k)[:, None], (p - q).clamp(min=0), p)
    rest = torch.where((rest.amax(-1) > 0)[:, None], rest, p)
    total = rest.cumsum(-1)
    over = (total > s["u_sample"].double()[:, None] * total[:, -1:]) & (rest > 0)
    token = over.long().argmax(-1)
    i = torch.arange(k + 1, device=DEVICE)
    drafted = torch.cat([s["tokens"].long(), torch.full((b, 1), -1, device=DEVICE)], -1)
    out = torch.where(i < accepted[:, None], drafted, torch.where(i == accepted[:, None], token[:, None], -1))
    return {"accepted": accepted.to(torch.int32), "tokens": out.to(torch.int32)}


# --- 64 bits ------------------------------------------------------------------------------------------------


def _turned(x, positions, case, back=False):
    """x [tokens, heads, d] in 64 bits as complex numbers times exp(i position frequency)."""
    r, s, kind = case["rot"], case.get("factor", 1.0), case.get("scaling", "none")
    f = []
    for i in range(r // 2):
        w = math.exp(-2 * i / r * (math.log(10000.0) + (r / (r - 2) * math.log(s) if kind == "base" else 0.0)))
        t = case.get("context", 1) * w / (2 * math.pi)
        part = {"ramp": (t - 1) / 31, "log_ramp": math.log(t) / math.log(32), "linear": 0.0}.get(kind, 1.0)
        part = min(1.0, max(0.0, part))
        f.append(w * part + w * (1 - part) / s)
    f = torch.tensor(f, dtype=torch.float64, device=DEVICE)
    y = x.double().clone()
    first, second = (torch.arange(0, r, 2), torch.arange(1, r, 2)) if case["interleaved"] else (torch.arange(r // 2), torch.arange(r // 2, r))
    z = torch.complex(y[..., first.to(DEVICE)], y[..., second.to(DEVICE)])
    angle = positions.double()[:, None, None] * f
    z = z * torch.polar(torch.full_like(angle, _magnitude(case)), -angle if back else angle)
    y[..., first.to(DEVICE)], y[..., second.to(DEVICE)] = z.real, z.imag
    return y


def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    if case["op"] == "rotary":
        return {n: _turned(s[n], s["positions"], case, case["backward"]) for n in ("q", "k")}
    new, cached = _tokens(case)
    page, p, group = case["page"], case["prefix"], case["hq"] // case["hkv"]
    start = s["cu"].tolist()
    if case["op"] == "append":
        at = torch.cat([torch.arange(c - n, c) for n, c in zip(new, cached)]).to(DEVICE)
        q, k = _turned(s["q"], p + at, case), _turned(s["k"], p + at, case)
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        for b, n in enumerate(new):
            rows = at[start[b]:start[b + 1]]
            pages = s["table"][b].long()[rows // page]
            for cache, x in ((kc, k), (vc, s["v"].double())):
                view = cache.transpose(1, 2) if case["head_major"] else cache
                view[pages, rows % page] = x[start[b]:start[b + 1]]
        return {"q": q, "k_cache": kc, "v_cache": vc}
    kc, vc = (c.transpose(1, 2) if case["head_major"] else c for c in (s["k_cache"], s["v_cache"]))
    o = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for b, (n, c) in enumerate(zip(new, cached)):
        where = torch.cat([s["prefix_table"].long().repeat_interleave(page)[:p] * page + torch.arange(p, device=DEVICE) % page,
                           s["table"][b].long().repeat_interleave(page)[:c] * page + torch.arange(c, device=DEVICE) % page])
        hidden = torch.arange(p + c, device=DEVICE)[None] > p + c - n + torch.arange(n, device=DEVICE)[:, None]
        for h in range(case["hkv"]):
            k, v = (x[where // page, where % page, h].double() for x in (kc, vc))
            for m in range(group):
                q = s["q"][start[b]:start[b + 1], h * group + m].double()
                a = (q @ k.T) * case["d"] ** -0.5
                o[start[b]:start[b + 1], h * group + m] = torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v
    return {"o": o}

