"""Host side of the serving operators: rotary plans and the page lookup (no GPU)."""
from __future__ import annotations

import ctypes as C
import importlib
import math
from fractions import Fraction

import pytest

from conftest import PKG

rt = importlib.import_module(f"{PKG}.runtime")

SCALINGS = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
            dict(scaling="ramp", factor=8.0, context=8192.0, low=1.0, high=4.0),
            dict(scaling="log_ramp", factor=16.0, context=4096.0, low=1.0, high=32.0)]


@pytest.mark.parametrize("kw", SCALINGS)
@pytest.mark.parametrize("rot,theta", [(128, 10000.0), (64, 500000.0), (6, 10.0), (256, 1e6), (32, 0.5)])
def test_rope_plan_turns(kw, rot, theta):
    torch = pytest.importorskip("torch")  # noqa: F841  (serving_refs needs it)
    import serving_refs as refs
    plan = rt.rope_plan(rot, theta=theta, interleaved=True, magnitude=1.25, **kw)
    assert plan.rot == rot and plan.interleaved == 1 and plan.magnitude == 1.25
    for i, f in enumerate(refs.frequencies(rot, theta, **kw)):
        turns = f / (2 * math.pi)
        got = plan.turn[i] / 2.0 ** 64
        off = abs(got - turns % 1.0)
        assert min(off, 1 - off) <= 8 * 2.0 ** -53 * max(1.0, turns)  # the 64-bit form's own roundings


def test_rope_plan_first_pair_is_one_radian():
    plan = rt.rope_plan(128)
    assert abs(Fraction(plan.turn[0], 2 ** 64) * Fraction("6.28318530717958647692528676655900576839") - 1) < Fraction(1, 2 ** 62)
    assert all(plan.turn[i] > plan.turn[i + 1] for i in range(63)) and not any(plan.turn[64:])


@pytest.mark.parametrize("kw", [dict(rot=0), dict(rot=3), dict(rot=258), dict(theta=0.0), dict(theta=float("nan")),
                                dict(theta=float("inf")), dict(scaling="linear", factor=0.0),
                                dict(scaling="base", factor=2.0, rot=2), dict(scaling="ramp", context=0.0),
                                dict(scaling="ramp", context=10.0, low=4.0, high=4.0), dict(magnitude=float("inf")),
                                dict(scaling="log_ramp", context=10.0, low=0.0, high=4.0)])
def test_rope_plan_refuses(kw):
    kw = {"rot": 64, **kw}
    with pytest.raises(rt.B2KError) as e:
        rt.rope_plan(**kw)
    assert e.value.status == rt.B2K_EINVAL


def test_rope_plan_refuses_null_and_unknown_scaling():
    lib, p, out = rt.library(), rt.RopeParams(8, 0, 7, 10.0, 1.0, 0.0, 0.0, 0.0, 1.0), rt.Rope()
    assert lib.b2k_rope_plan(C.byref(p), C.byref(out)) == rt.B2K_EINVAL
    assert lib.b2k_rope_plan(None, C.byref(out)) == rt.B2K_EINVAL


@pytest.mark.parametrize("page_size", [1, 16, 20])
def test_paged_slot(page_size):
    row = [7, 0, 3]
    for pos in range(3 * page_size):
        assert rt.paged_slot(row, 8, page_size, pos) == row[pos // page_size] * page_size + pos % page_size
    for pos in (-1, 3 * page_size, 2 ** 31, 2 ** 40, -(2 ** 40)):
        assert rt.paged_slot(row, 8, page_size, pos) == -1


def test_paged_slot_refuses_bad_pages():
    assert rt.paged_slot([5, 8, -1, 2 ** 31 - 1], 8, 4, 0) == 20
    assert [rt.paged_slot([5, 8, -1, 2 ** 31 - 1], 8, 4, p) for p in (4, 8, 12)] == [-1, -1, -1]
    assert rt.paged_slot([], 8, 4, 0) == -1 and rt.paged_slot([0], 8, 0, 0) == -1
    assert rt.paged_slot([2 ** 31 - 1], 2 ** 33, 2 ** 20, 5) == (2 ** 31 - 1) * 2 ** 20 + 5  # beyond 32 bits


def test_contexts_calls_need_a_context():
    lib = rt.library()
    assert lib.b2k_rotary(None, None, 0, 1, None, None, None, 0, 1, 0, None) == rt.B2K_EINVAL
    assert lib.b2k_paged_append(None, None, None, None, None, None, None, None, None) == rt.B2K_EINVAL
    assert lib.b2k_paged_attention(None, None, None, None, None, 1.0, None, 0, None) == rt.B2K_EINVAL
    assert lib.b2k_verify_drafts(None, None, None, None, None) == rt.B2K_EINVAL


# --- the plan of a paged attention call: host arithmetic on made-up addresses ------------------------------------


def parts(sequences=4, new=1, length=1000, prefix=0, hq=32, hkv=8, d=128, dtype=rt.BF16, page=16, at=4096, **kw):
    cache = rt.paged_cache(at, at + 64, dtype, 1000, page, hkv, d)
    batch = rt.paged_batch(sequences, sequences * new, 256, 256, 256, -(-length // page), max_new=new, max_len=length,
                           prefix_len=prefix, prefix_table=256)
    x = rt.heads(kw.get("q", 4096), hq, hq * d, d)
    return cache, batch, x, rt.heads(kw.get("o", 8192), hq, hq * d, d)


def test_paged_plan_kernels():
    plain, warp, memory = 0, 1, 2
    plan = lambda **kw: rt.paged_attention_plan(148, *parts(**kw))  # noqa: E731
    assert plan()["own_kernel"] == warp                                   # decode
    assert plan(dtype=rt.F32)["own_kernel"] == plain
    assert plan(d=100)["own_kernel"] == plain                             # no 16-byte pieces
    assert plan(at=4098)["own_kernel"] == plain and plan(q=4098)["own_kernel"] == plain and plan(o=8194)["own_kernel"] == plain
    assert plan(new=512, length=4096)["own_kernel"] == memory             # prompts
    assert plan(new=512, length=4096, d=256)["own_kernel"] == memory
    assert plan(new=512, length=4096, d=256, page=20)["own_kernel"] == warp   # no boxes, which wide heads need there
    assert plan(new=8, length=64)["own_kernel"] == warp                   # 32 rows fit the warp kernel
    assert plan(new=9, length=40)["own_kernel"] == warp                   # more, but too little work to repay a block's start
    decode = plan(sequences=128, prefix=8192, hq=64)
    assert (decode["own_kernel"], decode["prefix_kernel"], decode["joined"]) == (warp, memory, 0)
    assert plan(prefix=64)["prefix_kernel"] == warp and plan()["prefix_kernel"] == -1
    chunk = plan(new=512, length=4096, prefix=1000)
    assert (chunk["joined"], chunk["prefix_kernel"], chunk["prefix_splits"]) == (1, -1, 0)


@pytest.mark.parametrize("kw", [dict(), dict(sequences=1, length=50001), dict(sequences=128, prefix=8192, hq=64),
                                dict(new=512, length=4096, prefix=1000), dict(dtype=rt.F32, prefix=77), dict(d=256, new=33),
                                dict(sequences=1, length=1), dict(length=2 ** 30, page=2 ** 20), dict(new=40, length=700, prefix=129)])
def test_paged_plan_covers_the_keys(kw):
    """Splits cover the keys without an empty one, whole tiles each, and the workspace holds every part."""
    p, (cache, batch, q, _) = rt.paged_attention_plan(148, *parts(**kw)), parts(**kw)
    step = 128 if p["own_kernel"] == 2 else 64
    start = 0 if not p["joined"] else -(-batch.prefix_len // 128) * 128 if p["own_kernel"] == 2 else batch.prefix_len
    assert p["own_chunk"] % step == 0
    assert (p["own_splits"] - 1) * p["own_chunk"] < batch.max_len + start <= p["own_splits"] * p["own_chunk"]
    if p["prefix_splits"]:
        assert (p["prefix_splits"] - 1) * p["prefix_chunk"] < batch.prefix_len <= p["prefix_splits"] * p["prefix_chunk"]
    slots = p["own_splits"] + p["prefix_splits"]
    need = slots * batch.tokens * q.heads * (cache.d + 2) * 4
    assert slots == 1 or need <= p["workspace_bytes"]


def changed(s, **kw):
    c = type(s).from_buffer_copy(s)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("which,kw", [
    (0, dict(k=None)), (0, dict(v=None)), (0, dict(dtype=3)), (0, dict(page_size=0)), (0, dict(pages=0)), (0, dict(heads=0)),
    (0, dict(d=0)), (0, dict(d=257)), (0, dict(k_row=1)), (0, dict(v_head=1)), (0, dict(k_page=1)),
    (1, dict(sequences=-1)), (1, dict(tokens=-1)), (1, dict(max_new=-1)), (1, dict(max_len=-1)), (1, dict(prefix_len=-1)),
    (1, dict(first=None)), (1, dict(lengths=None)), (1, dict(table=None)), (1, dict(table_stride=1)), (1, dict(max_len=10 ** 6)),
    (1, dict(prefix_len=5, prefix_table=None)), (1, dict(tokens=2 ** 31)),
    (2, dict(heads=12)), (2, dict(heads=0)), (2, dict(data=None)), (2, dict(stride_head=3)), (2, dict(stride_token=-1)),
    (3, dict(heads=8)), (3, dict(data=4096)), (3, dict(data=None)), (3, dict(stride_token=0)), (3, dict(stride_token=1)),
    # off an element's boundary: loads there would fault
    (0, dict(k=4097)), (0, dict(v=4099)), (1, dict(first=258)), (1, dict(lengths=257)), (1, dict(table=258)),
    (1, dict(prefix_table=258)), (2, dict(data=4097)), (3, dict(data=8193))])
def test_paged_plan_refuses(which, kw):
    args = list(parts())
    args[which] = changed(args[which], **kw)
    with pytest.raises(rt.B2KError) as e:
        rt.paged_attention_plan(148, *args)
    assert e.value.status == rt.B2K_EINVAL


@pytest.mark.parametrize("kw", [dict(sequences=65536), dict(tokens=2 ** 31 - 1), dict(max_new=2 ** 30)])
def test_paged_plan_too_large(kw):
    cache, batch, q, o = parts()
    with pytest.raises(rt.B2KError) as e:
        rt.paged_attention_plan(148, cache, changed(batch, **kw), q, o)
    assert e.value.status == rt.B2K_EUNSUPPORTED
    assert rt.library().b2k_paged_attention_set_kernel(4) == rt.B2K_EINVAL
    assert rt.library().b2k_paged_attention_plan(0, C.byref(cache), C.byref(batch), C.byref(q), C.byref(o),
                                                 C.byref(rt.PagedAttentionPlan())) == rt.B2K_EINVAL
