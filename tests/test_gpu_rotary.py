"""Rotary positions and the append to a paged cache against their 64-bit forms."""
from __future__ import annotations

import importlib

import pytest

from conftest import PKG

torch = pytest.importorskip("torch")
import serving_refs as refs  # noqa: E402

pytestmark = pytest.mark.gpu
rt = importlib.import_module(f"{PKG}.runtime")
CODES = {"f32": rt.F32, "f16": rt.F16, "bf16": rt.BF16}


def heads(x):
    return rt.heads(x.data_ptr(), x.shape[1], x.stride(0), x.stride(1))


SCALINGS = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
            dict(scaling="ramp", factor=8.0, context=8192.0, low=1.0, high=4.0),
            dict(scaling="log_ramp", factor=16.0, context=4096.0, low=1.0, high=32.0)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hkv,d,rot", [(1, 1, 1, 2, 2), (1, 8, 2, 128, 128), (7, 5, 1, 64, 32), (13, 3, 3, 80, 40),
                                                 (33, 4, 4, 96, 96), (5, 2, 1, 256, 256), (3, 2, 2, 7, 4),
                                                 (700, 12, 4, 128, 64), (2500, 8, 8, 64, 64), (9, 1, 1, 40, 38)])
def test_rotary_matches(ctx, torch_cuda, dtype, interleaved, tokens, hq, hkv, d, rot):
    dt, g = refs.DTYPES[dtype], torch.Generator(device="cuda").manual_seed(tokens + d)
    kw = SCALINGS[(tokens + rot) % 5 if rot > 2 else 0]
    magnitude = 1.0 if tokens % 2 else 1.25
    qkv = torch.randn(tokens, hq + 2 * hkv, d, device="cuda", generator=g).to(dt)
    x = [qkv[:, :hq], qkv[:, hq:hq + hkv]]
    y = [torch.full((tokens, h, d), 7.0, device="cuda", dtype=dt) for h in (hq, hkv)]
    pos = torch.randint(0, 100000, (tokens,), device="cuda", generator=g)
    rope = rt.rope_plan(rot, interleaved=interleaved, magnitude=magnitude, **kw)
    freqs = refs.frequencies(rot, **kw)
    for transpose in (False, True):
        ctx.rotary(rope, CODES[dtype], [(heads(a), heads(b)) for a, b in zip(x, y)], pos.data_ptr(), tokens, d,
                   transpose=transpose)
        ctx.sync()
        for a, b in zip(x, y):
            want, tol = refs.rotary(a, pos, freqs, interleaved, magnitude, transpose)
            refs.close(b, want, tol, dt, f"rotary {transpose=}")


@pytest.mark.parametrize("dtype,tokens,hq,hkv,d,rot,interleaved", [
    ("f32", 9601, 9, 10, 256, 256, False), ("bf16", 9500, 37, 5, 128, 64, True), ("f16", 5000, 24, 12, 64, 64, False),
    ("f32", 20000, 1, 1, 24, 8, True)])
def test_rotary_many_tokens(ctx, torch_cuda, dtype, tokens, hq, hkv, d, rot, interleaved):
    """A warp or two to a token, more heads than one batch of loads, odd token counts."""
    dt, g = refs.DTYPES[dtype], torch.Generator(device="cuda").manual_seed(tokens)
    q, k = (torch.randn(tokens, h, d, device="cuda", generator=g).to(dt) for h in (hq, hkv))
    pos = torch.randint(0, 100000, (tokens,), device="cuda", generator=g)
    yq, yk = (torch.full((tokens + 1,) + x.shape[1:], 7.0, device="cuda", dtype=dt) for x in (q, k))
    ctx.rotary(rt.rope_plan(rot, interleaved=interleaved), CODES[dtype],
               [(heads(q), heads(yq)), (heads(k), heads(yk))], pos.data_ptr(), tokens, d)
    ctx.sync()
    for x, y in ((q, yq), (k, yk)):
        want, tol = refs.rotary(x, pos, refs.frequencies(rot), interleaved)
        refs.close(y[:-1], want, tol, dt, "many tokens")
        assert (y[-1] == 7.0).all()


def test_rotary_far_and_negative_positions(ctx, torch_cuda):
    """Angles stay exact where a 32-bit product of position and frequency holds no digit of them."""
    d, pos = 64, torch.tensor([0, 1, -1, -12345, 2 ** 24 + 1, 2 ** 31 + 7, 2 ** 40 + 3, -(2 ** 33)], device="cuda")
    x = torch.randn(len(pos), 2, d, device="cuda")
    y = torch.empty_like(x)
    rope = rt.rope_plan(d)
    ctx.rotary(rope, rt.F32, [(heads(x), heads(y))], pos.data_ptr(), len(pos), d)
    ctx.sync()
    # the 64-bit form's own angles are off by |position| 2^-53: compare by the plan's exact integers
    for t, p in enumerate(pos.tolist()):
        for i in range(d // 2):
            turns = (rope.turn[i] * p) % 2 ** 64 / 2.0 ** 64
            a, b = float(x[t, 0, i]), float(x[t, 0, i + d // 2])
            import math
            c, s = math.cos(2 * math.pi * turns), math.sin(2 * math.pi * turns)
            assert abs(float(y[t, 0, i]) - (a * c - b * s)) <= 5e-7 * (abs(a) + abs(b))
            assert abs(float(y[t, 0, i + d // 2]) - (b * c + a * s)) <= 5e-7 * (abs(a) + abs(b))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(ctx, torch_cuda, interleaved):
    """transpose is the gradient: <g, dR x> by differences, and <R x, g> = <x, R^T g>."""
    tokens, h, d, rot = 6, 2, 32, 24
    g = torch.Generator(device="cuda").manual_seed(1)
    x, grad = (torch.randn(tokens, h, d, device="cuda", generator=g) for _ in range(2))
    pos = torch.randint(0, 5000, (tokens,), device="cuda", generator=g)
    rope = rt.rope_plan(rot, interleaved=interleaved, magnitude=1.5)

    def apply(v, transpose):
        y = torch.empty_like(v)
        ctx.rotary(rope, rt.F32, [(heads(v), heads(y))], pos.data_ptr(), tokens, d, transpose=transpose)
        ctx.sync()
        return y.double()

    back = apply(grad, True)
    for t, k, e in [(0, 0, 0), (2, 1, 5), (3, 0, 23), (5, 1, 31), (4, 0, 12)]:
        step = torch.zeros_like(x)
        step[t, k, e] = 0.5
        slope = ((apply(x + step, False) - apply(x - step, False)) * grad.double()).sum()
        # a linear map: the difference is exact but for FP32 roundings of values below 2^4, two entries of it
        assert abs(float(slope) - float(back[t, k, e])) <= 4e-6 * float(grad.abs().max())
    assert abs(float((apply(x, False) * grad.double()).sum() - (x.double() * back).sum())) <= 1e-6 * float(
        (x.double().abs() * back.abs()).sum())


def test_rotary_in_place_strides_and_tail(ctx, torch_cuda):
    """In place on a strided view: only the rows and heads of the call change."""
    buf = torch.randn(10, 9, 72, device="cuda").to(torch.bfloat16)
    keep = buf.clone()
    view = buf[2:8, 1:7, 4:68]  # 8-byte aligned rows: no 16-byte accesses
    x = view.clone()
    pos = torch.arange(100, 106, device="cuda")
    ctx.rotary(rt.rope_plan(64), rt.BF16, [(heads(view), heads(view))], pos.data_ptr(), 6, 64)
    ctx.sync()
    want, tol = refs.rotary(x, pos, refs.frequencies(64), False)
    refs.close(view, want, tol, torch.bfloat16, "in place")
    keep[2:8, 1:7, 4:68] = view
    assert torch.equal(buf, keep)


def test_rotary_values_outside_pairs_are_copied(ctx, torch_cuda):
    x = torch.full((2, 1, 16), float("inf"), device="cuda")
    x[:, :, :8] = 1.0
    y = torch.empty_like(x)
    ctx.rotary(rt.rope_plan(8, magnitude=3.0), rt.F32, [(heads(x), heads(y))],
               torch.tensor([5, 9], device="cuda").data_ptr(), 2, 16)
    ctx.sync()
    assert torch.equal(y[:, :, 8:], x[:, :, 8:]) and torch.isfinite(y[:, :, :8]).all()


def test_rotary_refusals(ctx, torch_cuda):
    x = torch.zeros(4, 2, 32, device="cuda")
    pos = torch.zeros(4, dtype=torch.int64, device="cuda")
    rope, pair = rt.rope_plan(32), [(heads(x), heads(x))]
    ctx.rotary(rope, rt.F32, pair, 0, 0, 32)  # no tokens: nothing to read
    narrow = rt.heads(x.data_ptr(), 2, 64, 16)
    for args in [(rope, 9, pair, pos.data_ptr(), 4, 32), (rope, rt.F32, pair, 0, 4, 32),
                 (rope, rt.F32, pair, pos.data_ptr(), -1, 32), (rope, rt.F32, pair, pos.data_ptr(), 4, 16),
                 (rope, rt.F32, pair, pos.data_ptr(), 4, 257), (rope, rt.F32, pair * 4, pos.data_ptr(), 4, 32),
                 (rope, rt.F32, [(heads(x), rt.heads(x.data_ptr(), 1, 64, 32))], pos.data_ptr(), 4, 32),
                 (rope, rt.F32, [(heads(x), rt.heads(0, 2, 64, 32))], pos.data_ptr(), 4, 32),
                 (rope, rt.F32, [(heads(x), rt.heads(x.data_ptr(), 2, 128, 32))], pos.data_ptr(), 4, 32),
                 (rope, rt.F32, [(narrow, narrow)], pos.data_ptr(), 4, 32),
                 # tokens of an output in one place
                 (rope, rt.F32, [(heads(x), rt.heads(x.data_ptr() + 4096, 2, 0, 32))], pos.data_ptr(), 2, 32),
                 # off an element's boundary
                 (rope, rt.F32, pair, pos.data_ptr() + 4, 2, 32),
                 (rope, rt.F32, [(heads(x), rt.heads(x.data_ptr() + 2, 2, 64, 32))], pos.data_ptr(), 2, 32)]:
        with pytest.raises(rt.B2KError) as e:
            ctx.rotary(*args)
        assert e.value.status == rt.B2K_EINVAL
    ctx.sync()


# --- append ------------------------------------------------------------------------------------------------


def call_parts(bt):
    cache = rt.paged_cache(bt.k.data_ptr(), bt.v.data_ptr(), {v: CODES[k] for k, v in refs.DTYPES.items()}[bt.dtype],
                           bt.pages, bt.page, bt.heads, bt.d, head_major=bt.head_major)
    batch = rt.paged_batch(len(bt.new), bt.tokens, bt.first.data_ptr(), bt.lens.data_ptr(), bt.table.data_ptr(), bt.width,
                           max_new=max(bt.new, default=0), max_len=max(bt.lengths, default=0), prefix_len=bt.prefix,
                           prefix_table=bt.prefix_table.data_ptr())
    return cache, batch


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,lengths,prefix,page,hq,hkv,d,rot,interleaved,head_major", [
    ([1], [1], 0, 16, 4, 4, 64, 64, False, False),
    ([1, 1, 1], [5, 16, 17], 33, 16, 8, 2, 128, 128, False, False),
    ([3, 0, 7, 1], [3, 12, 40, 1], 100, 8, 6, 2, 80, 40, False, True),
    ([20, 5], [25, 5], 0, 20, 4, 1, 96, 96, True, True),
    ([600, 1, 333], [700, 64, 333], 5, 64, 3, 3, 64, 32, True, False),
    ([2, 2], [2, 3], 1, 1, 2, 1, 10, 6, False, False),
    ([1100, 900, 800], [1500, 900, 1000], 0, 128, 4, 2, 256, 128, False, True),
])
def test_append_matches(ctx, torch_cuda, dtype, new, lengths, prefix, page, hq, hkv, d, rot, interleaved, head_major):
    dt = refs.DTYPES[dtype]
    bt = refs.batch(new, lengths, prefix=prefix, page=page, heads=hkv, d=d, dtype=dt, head_major=head_major, extra_rows=3,
                    poison=False)
    n = sum(new)
    qkv = torch.randn(bt.tokens, hq + 2 * hkv, d, device="cuda", generator=bt.generator).to(dt)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    q_out = torch.full((bt.tokens, hq, d), 7.0, device="cuda", dtype=dt)
    cache, batch = call_parts(bt)
    was_k, was_v = bt.k.clone(), bt.v.clone()
    ctx.paged_append(cache, batch, heads(k), heads(v), q=heads(q), q_out=heads(q_out),
                     rope=rt.rope_plan(rot, interleaved=interleaved))
    ctx.sync()
    freqs, at = refs.frequencies(rot), 0
    for b, (m, length) in enumerate(zip(new, lengths)):
        pos = prefix + torch.arange(length - m, length, device="cuda")
        for x, out in ((q, q_out[at:at + m]), (k, refs.read_rows(bt, bt.k, b, length)[length - m:])):
            want, tol = refs.rotary(x[at:at + m], pos, freqs, interleaved)
            refs.close(out, want, tol, dt, f"sequence {b}")
        assert torch.equal(refs.read_rows(bt, bt.v, b, length)[length - m:], v[at:at + m])
        # what was there before: put back, the caches are as they were
        for cache_t, was in ((bt.k, was_k), (bt.v, was_v)):
            rows = refs.read_rows(bt, cache_t, b, length)
            rows[length - m:] = refs.read_rows(bt, was, b, length)[length - m:]
            refs.write_rows(bt, cache_t, b, rows)
        at += m
    assert torch.equal(bt.k, was_k) and torch.equal(bt.v, was_v)
    assert (q_out[n:] == 7.0).all()


def test_append_without_rope_copies(ctx, torch_cuda):
    bt = refs.batch([2, 3], [9, 3], heads=3, d=40, dtype=torch.float16, poison=False)
    k, v = (torch.randn(5, 3, 40, device="cuda").half() for _ in range(2))
    cache, batch = call_parts(bt)
    ctx.paged_append(cache, batch, heads(k), heads(v))
    ctx.paged_append_call(cache, batch, heads(k), heads(v))()
    ctx.sync()
    assert torch.equal(refs.read_rows(bt, bt.k, 0, 9)[7:], k[:2]) and torch.equal(refs.read_rows(bt, bt.v, 1, 3), v[2:])


@pytest.mark.parametrize("what", ["page", "negative page", "past the table", "too many new", "first falls", "before the start"])
def test_append_index_out_of_bounds(ctx, torch_cuda, what):
    """A bad index writes nothing for its token, leaves the others right and is reported at the next sync."""
    bt = refs.batch([2, 1], [20, 5], heads=1, d=16, dtype=torch.float32, poison=False)
    k, v = (torch.randn(3, 1, 16, device="cuda") for _ in range(2))
    cache, batch = call_parts(bt)
    was = bt.k.clone()
    if what == "page":
        bt.table[0, 1] = bt.pages
    elif what == "negative page":
        bt.table[0, 1] = -1
    elif what == "past the table":
        bt.lens[0] = 40
    elif what == "too many new":
        batch.max_new = 1
    elif what == "first falls":
        bt.first[0], bt.first[1] = 3, 2  # -1 new tokens
    else:
        bt.lens[0] = 1  # two new tokens, one cached: the first has position -1
    ctx.paged_append(cache, batch, heads(k), heads(v))
    with pytest.raises(rt.B2KError) as e:
        ctx.sync()
    assert e.value.status == rt.B2K_EINDEX
    assert torch.equal(refs.read_rows(bt, bt.k, 1, 5)[4:], k[2:])
    if what in ("page", "negative page", "past the table", "too many new", "first falls"):
        refs.write_rows(bt, bt.k, 1, refs.read_rows(bt, was, 1, 5))
        assert torch.equal(bt.k, was)
    ctx.sync()  # the context is usable, the report is given once


def test_append_refusals(ctx, torch_cuda):
    bt = refs.batch([1], [4], heads=2, d=32, dtype=torch.float32)
    x = torch.zeros(1, 2, 32, device="cuda")
    cache, batch = call_parts(bt)

    def refused(cache=cache, batch=batch, k=heads(x), v=heads(x), **kw):
        with pytest.raises(rt.B2KError) as e:
            ctx.paged_append(cache, batch, k, v, **kw)
        assert e.value.status == rt.B2K_EINVAL

    def changed(s, **kw):
        c = type(s).from_buffer_copy(s)
        for name, value in kw.items():
            setattr(c, name, value)
        return c

    for kw in (dict(k=None), dict(dtype=5), dict(page_size=0), dict(pages=0), dict(heads=0), dict(d=0), dict(d=257), dict(k_row=31)):
        refused(cache=changed(cache, **kw))
    for kw in (dict(sequences=-1), dict(tokens=-1), dict(max_new=-1), dict(max_len=17), dict(first=None), dict(lengths=None),
               dict(table=None), dict(table_stride=0), dict(prefix_len=-1), dict(prefix_len=3, prefix_table=None)):
        refused(batch=changed(batch, **kw))
    refused(k=rt.heads(x.data_ptr(), 1, 64, 32))
    refused(q=heads(x), q_out=heads(x))            # no rope
    refused(q=heads(x), rope=rt.rope_plan(32))     # nowhere to
    refused(rope=rt.rope_plan(64))                 # beyond the head
    ctx.paged_append(cache, changed(batch, sequences=0, first=None), heads(x), heads(x))
    ctx.sync()
