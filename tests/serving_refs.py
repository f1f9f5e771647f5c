"""Plain 64-bit forms of the serving operators, and the batches their tests share.

Tolerances are bounds, not fits: each adds up the roundings an operator is allowed (the output's, the
probabilities' where they enter the tensor cores, FP32 arithmetic in between)."""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype) -> float:
    """Largest relative error of a rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def frequencies(rot, theta=10000.0, scaling="none", factor=1.0, context=0.0, low=1.0, high=32.0):
    out = []
    for i in range(rot // 2):
        f = (theta * factor ** (rot / (rot - 2)) if scaling == "base" else theta) ** (-2 * i / rot)
        if scaling == "linear":
            f /= factor
        if scaling in ("ramp", "log_ramp"):
            g = math.log if scaling == "log_ramp" else float
            w = (g(context * f / (2 * math.pi)) - g(low)) / (g(high) - g(low))
            w = min(1.0, max(0.0, w))
            f = f * w + f * (1 - w) / factor
        out.append(f)
    return out


def rotary(x, positions, freqs, interleaved, magnitude=1.0, transpose=False):
    """(y, tolerance before the output's rounding) of x [tokens, heads, d] in 64 bits."""
    r, y = 2 * len(freqs), x.double().clone()
    first, second = ((slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r)))
    angle = positions.double()[:, None, None] * torch.tensor(freqs, dtype=torch.float64, device=x.device)
    c, s = magnitude * torch.cos(angle), magnitude * torch.sin(angle) * (-1 if transpose else 1)
    a, b = x.double()[..., first], x.double()[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    # a coefficient: the angle's rounding (pi 2^-25 and 2^-32 pi), sincospif's two units (2^-23), its product
    # with the magnitude (2^-24); then two FP32 products and a sum (2^-23): 4e-7 of |a| + |b| covers them
    tol = torch.zeros_like(y)
    each = 4e-7 * abs(magnitude) * (a.abs() + b.abs())
    tol[..., first], tol[..., second] = each, each
    return y, tol


def close(got, want, tol, dtype, what=""):
    """|got - want| within `tol` plus the rounding to `dtype` (its subnormal step for f16)."""
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    bound = tol * (1 + half_step(dtype)) + half_step(dtype) * want.abs() + tiny
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float(((got.double() - want).abs() - bound)[bad].max()):.3g} over its bound")


def batch(new, lengths, *, prefix=0, page=16, heads=2, d=64, dtype=torch.bfloat16, head_major=False, seed=0, extra_rows=0,
          spare=2, poison=True):
    """Paged sequences with random keys and values; every row of the cache that holds no token is NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, need = len(new), [-(-x // page) for x in lengths]
    head = -(-prefix // page)
    pages = head + sum(need) + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = max(1, max(need, default=1))
    table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
    at = head
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    shape = (pages, heads, page, d) if head_major else (pages, page, heads, d)
    bt = SimpleNamespace(new=list(new), lengths=list(lengths), prefix=prefix, page=page, heads=heads, d=d, dtype=dtype,
                         head_major=head_major, pages=pages, table=table, prefix_table=order[:max(1, head)].clone(),
                         width=width, tokens=sum(new) + extra_rows, generator=g)
    bt.first = torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32, device="cuda")
    bt.lens = torch.tensor(list(lengths) or [0], dtype=torch.int32, device="cuda")
    bt.k = torch.full(shape, float("nan") if poison else 0.0, device="cuda", dtype=dtype)
    bt.v = bt.k.clone()
    for b in [None] + list(range(n)):
        count = prefix if b is None else lengths[b]
        for cache in (bt.k, bt.v):
            write_rows(bt, cache, b, torch.randn(count, heads, d, generator=g, device="cuda").to(dtype))
    return bt


def places(bt, b, count):
    pos = torch.arange(count, device="cuda")
    row = bt.prefix_table if b is None else bt.table[b]
    return row.long()[pos // bt.page], pos % bt.page


def write_rows(bt, cache, b, x):
    pages, rows = places(bt, b, x.shape[0])
    view = cache.transpose(1, 2) if bt.head_major else cache
    view[pages, rows] = x


def read_rows(bt, cache, b, count):
    pages, rows = places(bt, b, count)
    view = cache.transpose(1, 2) if bt.head_major else cache
    return view[pages, rows]


def attention(bt, q, scale=None):
    """(o, tolerance before the output's rounding) [tokens, heads, d] in 64 bits; rows of no sequence are NaN."""
    scale = math.sqrt(bt.d) if scale is None else scale
    hq = q.shape[1]
    o = torch.full(q.shape, float("nan"), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(o)
    u = 0.0 if q.dtype == torch.float32 else half_step(q.dtype)  # the probabilities' rounding
    at = 0
    for b, (n, length) in enumerate(zip(bt.new, bt.lengths)):
        k = torch.cat([read_rows(bt, bt.k, None, bt.prefix), read_rows(bt, bt.k, b, length)]).double()
        v = torch.cat([read_rows(bt, bt.v, None, bt.prefix), read_rows(bt, bt.v, b, length)]).double()
        k, v = (x.repeat_interleave(hq // bt.heads, 1) for x in (k, v))
        x = q[at:at + n].double()
        limit = bt.prefix + (length - n + 1 + torch.arange(n, device="cuda")).clamp(min=0)
        hidden = (torch.arange(k.shape[0], device="cuda")[None] >= limit[:, None])[:, None]
        s = torch.einsum("jhd,khd->jhk", x, k) / scale
        s = s.masked_fill(hidden, -math.inf)
        p = torch.softmax(s, -1).nan_to_num(0.0)
        o[at:at + n] = torch.einsum("jhk,khd->jhd", p, v)
        # a score: an FP32 sum of d products; a probability: twice its score's error, the exponential's and
        # its own rounding; sums over the keys, each addition good to 2^-23 in the worst (truncating) case
        spread = torch.einsum("jhd,khd->jhk", x.abs(), k.abs()).masked_fill(hidden, 0.0)
        spread = spread.amax(-1, keepdim=True) if k.shape[0] else torch.zeros(n, hq, 1, device="cuda", dtype=torch.float64)
        rel = u + 2 * (bt.d + 4) * 2.0 ** -23 * spread / scale + 2.0 ** -21 + 2 * k.shape[0] * 2.0 ** -23
        tol[at:at + n] = rel * torch.einsum("jhk,khd->jhd", p, v.abs()) + rel * o[at:at + n].abs()
        at += n
    return o, tol


def verify(target, draft, drafted, counts, u_accept, u_sample):
    """(accepted, tokens) one sequence at a time in 64 bits on the host."""
    target, drafted = target.double().cpu(), drafted.cpu().tolist()
    draft = None if draft is None else draft.double().cpu()
    u_accept, u_sample = u_accept.double().cpu(), u_sample.double().cpu()
    vocab, most = target.shape[-1], target.shape[1] - 1
    accepted, tokens = [], []
    for b in range(target.shape[0]):
        n = most if counts is None else min(max(int(counts[b]), 0), most)
        taken = 0
        while taken < n:
            x = drafted[b][taken]
            if not 0 <= x < vocab:
                break
            q = 1.0 if draft is None else float(draft[b, taken, x])
            if not float(u_accept[b, taken]) * q < float(target[b, taken, x]):
                break
            taken += 1
        p = target[b, taken].clone()
        rest = p
        if taken < n:
            if draft is None:
                rest = p.clone()
                if 0 <= drafted[b][taken] < vocab:
                    rest[drafted[b][taken]] = 0.0
            else:
                rest = (p - draft[b, taken]).clamp(min=0.0)
            if not (rest > 0).any():
                rest = p
        held = (rest > 0).nonzero()[:, 0]
        token = -1
        if len(held):
            total = rest.cumsum(0)
            over = ((total > u_sample[b] * total[-1]) & (rest > 0)).nonzero()[:, 0]
            token = int(over[0] if len(over) else held[-1])
        accepted.append(taken)
        tokens.append(drafted[b][:taken] + [token] + [-1] * (most - taken))
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32).reshape(len(accepted), most + 1)
