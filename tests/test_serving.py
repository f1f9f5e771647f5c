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
