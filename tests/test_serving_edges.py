"""Host side of the serving operators' edges: which operands meet, what a session keeps and checks, plans, turns (no GPU)."""
from __future__ import annotations

import ctypes as C
import importlib
import random
from decimal import Decimal, localcontext

import pytest

from conftest import PKG

rt = importlib.import_module(f"{PKG}.runtime")


def rows(x, tokens, d, size):
    return [x.data + (t * x.stride_token + h * x.stride_head) * size for t in range(tokens) for h in range(x.heads)]


def met(x, y, tokens, d, size):
    """By looking at every pair of rows; None where a tensor meets itself only in name (one row)."""
    a = rows(x, tokens, d, size)
    if y is None:
        a = sorted(a)
        return any(q - p < d * size for p, q in zip(a, a[1:]))
    return any(abs(p - q) < d * size for p in a for q in rows(y, tokens, d, size))


@pytest.mark.parametrize("seed", range(4))
def test_heads_that_meet_themselves(seed):
    rng, seen = random.Random(seed), set()
    for _ in range(1500):
        d, tokens = rng.randint(1, 5), rng.randint(1, 6)
        x = rt.heads(4096, rng.randint(1, 6), rng.randint(0, 40), rng.randint(0, 40))
        want = met(x, None, tokens, d, 2)
        assert rt.heads_overlap(x, None, tokens, d, rt.BF16) == want, (x.heads, x.stride_token, x.stride_head, tokens, d)
        seen.add(want)
    assert seen == {False, True}
    # interleaved on purpose, and neither axis within the other's step
    assert not rt.heads_overlap(rt.heads(4096, 3, 5, 7), None, 3, 2, rt.F32) and rt.heads_overlap(rt.heads(4096, 3, 5, 7), None, 3, 3, rt.F32)
    assert rt.heads_overlap(rt.heads(4096, 32, 128, 128), None, 4, 128, rt.BF16)      # token 1 in head 1's place
    assert rt.heads_overlap(rt.heads(4096, 8, 128, 256), None, 3, 128, rt.BF16)
    assert not rt.heads_overlap(rt.heads(4096, 8, 128, 3 * 128), None, 3, 128, rt.BF16)  # head-major
    assert not rt.heads_overlap(rt.heads(4096, 2 ** 15, 2 ** 61, 2 ** 45), None, 2 ** 31, 128, rt.F32)


@pytest.mark.parametrize("kind", ["same steps", "same token step", "any"])
@pytest.mark.parametrize("seed", range(4))
def test_heads_that_meet_each_other(kind, seed):
    """Exact for tensors with the same strides or the same token step; never a missed meeting for the others."""
    rng, seen = random.Random(seed), set()
    for _ in range(1500):
        d, tokens, size = rng.randint(1, 4), rng.randint(1, 5), rng.choice([2, 4])
        dtype = rt.F32 if size == 4 else rt.F16
        x = rt.heads(2 ** 20, rng.randint(1, 5), rng.randint(0, 40), rng.randint(d, 30))
        y = rt.heads(2 ** 20 + size * rng.randint(-90, 90), rng.randint(1, 5), rng.randint(0, 40), rng.randint(d, 30))
        if kind == "same steps":
            y.stride_token, y.stride_head = x.stride_token, x.stride_head
        elif kind == "same token step":
            wide = max((t.heads - 1) * t.stride_head + d for t in (x, y))
            x.stride_token = y.stride_token = wide + rng.randint(0, 20)
        want, got = met(x, y, tokens, d, size), rt.heads_overlap(x, y, tokens, d, dtype)
        if kind == "any":
            assert got or not want
        else:
            assert got == want, [(t.data, t.heads, t.stride_token, t.stride_head) for t in (x, y)] + [tokens, d, size]
        seen.add(want)
    assert seen == {False, True}


def test_heads_of_a_fused_projection_lie_apart():
    n, hq, hkv, d = 16384, 32, 8, 128
    wide = (hq + 2 * hkv) * d
    q, k = rt.heads(4096, hq, wide, d), rt.heads(4096 + 2 * hq * d, hkv, wide, d)
    assert not rt.heads_overlap(q, k, n, d, rt.BF16) and not rt.heads_overlap(k, q, n, d, rt.BF16)
    k.data -= 2  # one element into the last query head
    assert rt.heads_overlap(q, k, n, d, rt.BF16) and rt.heads_overlap(k, q, n, d, rt.BF16)
    o = rt.heads(4096 + 256, hq, wide, d)
    assert rt.heads_overlap(q, o, n, d, rt.BF16) and not rt.heads_overlap(q, o, 0, d, rt.BF16)
    for bad in [(rt.heads(4096, 0, 8, 8), 1, 8, rt.F32), (q, -1, 8, rt.F32), (q, 1, 0, rt.F32), (q, 1, 8, 3), (rt.heads(1, 1, -1, 8), 1, 8, 0)]:
        with pytest.raises(rt.B2KError) as e:
            rt.heads_overlap(bad[0], None, *bad[1:])
        assert e.value.status == rt.B2K_EINVAL


def test_paged_plan_refuses_outputs_that_meet_themselves():
    cache = rt.paged_cache(4096, 8192, rt.BF16, 100, 16, 8, 128)
    batch = rt.paged_batch(4, 4, 256, 256, 256, 8, max_new=1, max_len=100)
    q = rt.heads(2 ** 20, 32, 32 * 128, 128)
    for strides, fine in (((32 * 128, 128), True), ((128, 4 * 128), True), ((128, 128), False), ((128, 2 * 128), False), ((16 * 128, 128), False)):
        o, out = rt.heads(2 ** 21, 32, *strides), rt.PagedAttentionPlan()
        status = rt.library().b2k_paged_attention_plan(148, C.byref(cache), C.byref(batch), C.byref(q), C.byref(o), C.byref(out))
        assert status == (rt.B2K_OK if fine else rt.B2K_EINVAL)


# --- api.Session's side, with a session that has no device --------------------------------------------------


class FakeSession:
    """Hands out addresses and keeps count of them."""

    def __init__(self):
        self.live, self.next, self.calls, self.stream = set(), 4096, [], 0
        self.ctx = self

    def empty(self, shape, dtype="f4"):
        return importlib.import_module(f"{PKG}.api").DeviceArray(self, tuple(shape), dtype)

    def malloc(self, nbytes):
        at, self.next = self.next, self.next + (nbytes + 4095) // 4096 * 4096
        self.live.add(at)
        return at

    def free(self, ptr):
        self.live.remove(ptr)

    def sync(self, stream=0):
        pass

    def __getattr__(self, name):  # the context's calls
        return lambda *args, **kw: self.calls.append(name) or 64


def test_workspace_outlives_larger_calls():
    """A captured call goes on using the workspace of its time: a larger one takes a new one beside it."""
    api = importlib.import_module(f"{PKG}.api")
    s = FakeSession()
    kv = api.PagedKV(s, 4, 16, 2, 64)
    small, large = kv.workspace(100), kv.workspace(5000)
    assert {small.ptr, large.ptr} <= s.live and small.ptr != large.ptr
    assert kv.workspace(200).nbytes >= 200 and kv.workspace(5000).ptr == large.ptr
    sizes = [kv.workspace(n).nbytes for n in range(5000, 300000, 1000)]
    held = s.next - 4096
    assert sizes == sorted(sizes) and held <= 4 * max(sizes)  # a growing call does not pile up one for each size
    kv.free()
    assert not s.live
    kv.free()


def session(fake):
    api = importlib.import_module(f"{PKG}.api")
    s = api.Session.__new__(api.Session)
    s.ctx, s.stream, s._pinned = fake, 0, []
    return s


def test_session_checks_its_arrays():
    import numpy as np
    api = importlib.import_module(f"{PKG}.api")
    fake = FakeSession()
    s = session(fake)
    kv = s.paged_kv(8, 16, 2, 32)
    ints = lambda *shape: s.empty(shape, np.int32)  # noqa: E731
    batch = s.paged_batch(ints(3), ints(2), ints(2, 4), 5, max_new=3, max_len=60, prefix_table=ints(2), prefix_len=33)
    q, o, flat, k = s.empty((5, 4, 32)), s.empty((5, 4, 32)), s.empty((5, 32)), s.empty((5, 2, 32))
    with pytest.raises(ValueError):
        s.paged_attention(kv, batch, q, o)  # 33 tokens in two pages of 16: the third page would be read behind the table
    batch.prefix_len = 32
    s.paged_attention(kv, batch, q, o)
    for call in (lambda: s.paged_attention(kv, batch, flat, o), lambda: s.paged_append(kv, batch, flat, k),
                 lambda: s.paged_append(kv, batch, k, k, q=flat, q_out=q, rope=rt.rope_plan(32)),
                 lambda: s.rotary(rt.rope_plan(32), [], s.empty((5,), np.int64)),
                 lambda: s.rotary(rt.rope_plan(32), [(s.empty((5, 4, 32), np.float64),) * 2], s.empty((5,), np.int64)),
                 lambda: s.rotary(rt.rope_plan(32), [(flat, flat)], s.empty((5,), np.int64)),
                 lambda: s.paged_kv(8, 16, 2, 32, np.float64),
                 lambda: s.paged_batch(ints(3), ints(2), ints(8), 5, max_new=3, max_len=60)):
        with pytest.raises(ValueError):
            call()
    assert fake.calls.count("paged_attention") == 1 and "rotary" not in fake.calls and "paged_append" not in fake.calls
    assert api.ELEMENTS[np.dtype(np.uint16)] == rt.BF16


def test_prefix_splits_by_lengths_spread_below_their_bound():
    """128 sequences behind 8192 tokens: two splits while the own keys, half of the bound each, end before one would."""
    def splits(max_len):
        cache = rt.paged_cache(4096, 8192, rt.BF16, 10 ** 6, 16, 8, 128)
        batch = rt.paged_batch(128, 128, 256, 256, 256, 10 ** 4, max_new=1, max_len=max_len, prefix_len=8192, prefix_table=256)
        plan = rt.paged_attention_plan(148, cache, batch, rt.heads(2 ** 20, 64, 64 * 128, 128), rt.heads(2 ** 30, 64, 64 * 128, 128))
        assert plan["own_kernel"] == 1 and plan["prefix_kernel"] == 2
        return plan["prefix_splits"]
    assert [splits(n) for n in (1000, 2000, 2500)] == [2, 2, 1]


def test_plan_tells_the_f32_kernels_apart():
    """Up to 64 rows a cache head in 16-byte pieces stream; more, odd head dims and bases off 16 bytes do not."""
    def plan(new=1, prefix=0, sequences=2, d=64, at=4096, dtype=rt.F32, kernel=0):
        cache = rt.paged_cache(at, at, dtype, 1000, 16, 2, d)
        batch = rt.paged_batch(sequences, sequences * new, 256, 256, 256, 100, max_new=new, max_len=1000, prefix_len=prefix,
                               prefix_table=256)
        assert rt.library().b2k_paged_attention_set_kernel(kernel) == rt.B2K_OK
        try:
            return rt.paged_attention_plan(148, cache, batch, rt.heads(2 ** 20, 4, 4 * d, d), rt.heads(2 ** 30, 4, 4 * d, d))["streaming"]
        finally:
            rt.library().b2k_paged_attention_set_kernel(0)
    assert [plan(new=n) for n in (1, 32, 33)] == [1, 1, 0]
    assert plan(prefix=100) == 3 and plan(prefix=100, sequences=32) == 3 and plan(prefix=100, sequences=33) == 1
    assert plan(new=32, prefix=100, sequences=1) == 3 and plan(new=33, prefix=100, sequences=1) == 0
    assert plan(d=66) == 0 and plan(at=4100) == 0 and plan(kernel=1) == 0 and plan(dtype=rt.BF16, prefix=100) == 0


PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def exact_turns(rot, theta, scaling="none", factor=1.0, context=0.0, low=1.0, high=32.0):
    """f_i / 2 pi with 60 digits."""
    theta, s, out = Decimal(theta), Decimal(factor), []
    if scaling == "base":
        theta *= (s.ln() * rot / (rot - 2)).exp()
    for i in range(rot // 2):
        f = (theta.ln() * -2 * i / rot).exp()
        if scaling == "linear":
            f /= s
        if scaling in ("ramp", "log_ramp"):
            g = (lambda x: x.ln()) if scaling == "log_ramp" else (lambda x: x)
            t, lo, hi = Decimal(context) * f / (2 * PI), Decimal(low), Decimal(high)
            w = min(Decimal(1), max(Decimal(0), (g(t) - g(lo)) / (g(hi) - g(lo))))
            f = f * w + f * (1 - w) / s
        out.append(f / (2 * PI))
    return out


@pytest.mark.parametrize("kw", [dict(), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
                                dict(scaling="ramp", factor=8.0, context=8192.0, low=1.0, high=4.0),
                                dict(scaling="log_ramp", factor=16.0, context=4096.0, low=1.0, high=32.0),
                                dict(scaling="log_ramp", factor=2.5, context=131072.0, low=3.0, high=6.0)])
@pytest.mark.parametrize("rot,theta", [(128, 10000.0), (64, 500000.0), (6, 10.0), (256, 1e6), (32, 1.0), (96, 1e7)])
def test_turns_are_good_to_their_bound(kw, rot, theta):
    """The plan's fractions of a turn against 60 digits: within 2^-62, as b2k_rope_plan's comment derives."""
    with localcontext() as c:
        c.prec = 60
        for i, exact in enumerate(exact_turns(rot, theta, **kw)):
            off = abs(Decimal(rt.rope_plan(rot, theta=theta, **kw).turn[i]) / 2 ** 64 - exact)
            assert min(off, 1 - off) * 2 ** 62 < 1, (i, off * 2 ** 64)
