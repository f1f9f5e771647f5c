"""Calls of the serving operators at the edges of what their documentation allows: bounds far above the lengths in use,
arrays that meet, steps that follow each other without a synchronisation."""
from __future__ import annotations

import importlib
from types import SimpleNamespace

import pytest

from conftest import PKG

torch = pytest.importorskip("torch")
import serving_refs as refs  # noqa: E402

pytestmark = pytest.mark.gpu
rt = importlib.import_module(f"{PKG}.runtime")
CODES = {torch.float32: rt.F32, torch.float16: rt.F16, torch.bfloat16: rt.BF16}


def heads(x):
    return rt.heads(x.data_ptr(), x.shape[1], x.stride(0), x.stride(1))


def attend(ctx, cache, batch, q, stream=0):
    o = torch.full(q.shape, 7.0, device="cuda", dtype=q.dtype)
    nbytes = ctx.paged_attention_workspace(cache, batch, q.shape[1])
    ws = torch.full((nbytes // 4 + 4,), float("nan"), device="cuda")
    ctx.paged_attention(cache, batch, heads(q), heads(o), ws.data_ptr(), nbytes, stream=stream)
    ctx.sync(stream)
    return o


# --- bounds -----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 70])
def test_max_len_near_its_limit(ctx, torch_cuda, dtype, new):
    """The bound alone is near 2^31: a split is as long, and numbers of keys rounded up to splits pass 32 bits."""
    dt, page, width, n, d = refs.DTYPES[dtype], 2 ** 20, 2048, 600 // new, 8
    lengths = [new + i % 20 for i in range(n)]
    lengths[3], lengths[-2] = 70001, 100000  # a length and the longest split are beyond 2^31 together
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(2, page, 1, d, device="cuda", generator=g).to(dt) for _ in range(2))
    bt = SimpleNamespace(new=[new] * n, lengths=lengths, prefix=64, page=page, heads=1, d=d, head_major=False, k=k, v=v,
                         table=torch.zeros(n, width, dtype=torch.int32, device="cuda"),
                         prefix_table=torch.ones(1, dtype=torch.int32, device="cuda"))
    first = torch.arange(n + 1, dtype=torch.int32, device="cuda") * new
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    cache = rt.paged_cache(k.data_ptr(), v.data_ptr(), CODES[dt], 2, page, 1, d)
    q = torch.randn(n * new, 1, d, device="cuda", generator=g).to(dt)
    want, tol = refs.attention(bt, q)
    for max_len in (2 ** 31 - 65665, 2 ** 30 + 12345):
        batch = rt.paged_batch(n, n * new, first.data_ptr(), lens.data_ptr(), bt.table.data_ptr(), width, max_new=new,
                               max_len=max_len, prefix_len=64, prefix_table=bt.prefix_table.data_ptr())
        refs.close(attend(ctx, cache, batch, q), want, tol, dt, f"{max_len=}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("length", [41, 48, -1])
def test_append_refuses_lengths_outside_max_len(ctx, torch_cuda, dtype, tokens, length):
    """Above max_len, and within the table all the same: nothing of the sequence is written, its neighbours are."""
    dt = refs.DTYPES[dtype]
    bt = refs.batch([tokens, 2], [40, 9], page=16, heads=2, d=16, dtype=dt, poison=False)
    bt.table[0] = torch.tensor([3, 4, 5])
    bt.table[1] = torch.tensor([1, 2, 0])
    k, v, q = (torch.randn(tokens + 2, 2, 16, device="cuda", generator=bt.generator).to(dt) for _ in range(3))
    q_out = torch.full_like(q, 7.0)
    cache = rt.paged_cache(bt.k.data_ptr(), bt.v.data_ptr(), CODES[dt], bt.pages, 16, 2, 16)
    batch = rt.paged_batch(2, tokens + 2, bt.first.data_ptr(), bt.lens.data_ptr(), bt.table.data_ptr(), bt.width,
                           max_new=tokens, max_len=40)
    batch.max_new = max(2, tokens)
    bt.lens[0] = length
    was = bt.v.clone()
    ctx.paged_append(cache, batch, heads(k), heads(v), q=heads(q), q_out=heads(q_out), rope=rt.rope_plan(16))
    with pytest.raises(rt.B2KError) as e:
        ctx.sync()
    assert e.value.status == rt.B2K_EINDEX
    assert torch.equal(refs.read_rows(bt, bt.v, 1, 9)[7:], v[tokens:]) and (q_out[:tokens] == 7.0).all()
    refs.write_rows(bt, bt.v, 1, refs.read_rows(bt, was, 1, 9))
    assert torch.equal(bt.v, was)
    ctx.sync()


def test_append_without_a_table(ctx, torch_cuda):
    """max_len = 0 needs no table, and then no length from the device makes the kernel read one."""
    lens, first = torch.tensor([5, 0], dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 2], dtype=torch.int32, device="cuda")
    k = torch.zeros(1, 16, 1, 16, device="cuda")
    x = torch.ones(2, 1, 16, device="cuda")
    cache = rt.paged_cache(k.data_ptr(), k.data_ptr(), rt.F32, 1, 16, 1, 16)
    batch = rt.paged_batch(2, 2, first.data_ptr(), lens.data_ptr(), 0, 4, max_new=2, max_len=0)
    ctx.paged_append(cache, batch, heads(x), heads(x))
    with pytest.raises(rt.B2KError) as e:
        ctx.sync()
    assert e.value.status == rt.B2K_EINDEX and not k.any()
    lens.zero_()
    ctx.paged_append(cache, batch, heads(x), heads(x))  # two new tokens of none: positions -2 and -1
    with pytest.raises(rt.B2KError):
        ctx.sync()
    assert not k.any()
