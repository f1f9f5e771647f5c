"""Attention over a paged cache behind a shared prefix against its 64-bit form."""
from __future__ import annotations

import importlib

import pytest

from conftest import PKG

torch = pytest.importorskip("torch")
import serving_refs as refs  # noqa: E402

pytestmark = pytest.mark.gpu
rt = importlib.import_module(f"{PKG}.runtime")
CODES = {torch.float32: rt.F32, torch.float16: rt.F16, torch.bfloat16: rt.BF16}


KERNELS = {"rule": 0, "plain": 1, "warp": 2, "memory": 3}


@pytest.fixture(params=list(KERNELS))
def kernel(request, ctx):
    """Each kernel in turn, wherever it applies, and the rule that chooses among them."""
    ctx.set_paged_attention_kernel(KERNELS[request.param])
    yield request.param
    ctx.set_paged_attention_kernel(0)


def heads(x):
    return rt.heads(x.data_ptr(), x.shape[1], x.stride(0), x.stride(1))


def call_parts(bt, **kw):
    cache = rt.paged_cache(bt.k.data_ptr(), bt.v.data_ptr(), CODES[bt.dtype], bt.pages, bt.page, bt.heads, bt.d,
                           head_major=bt.head_major)
    batch = rt.paged_batch(len(bt.new), bt.tokens, bt.first.data_ptr(), bt.lens.data_ptr(), bt.table.data_ptr(), bt.width,
                           **{**dict(max_new=max(bt.new, default=0), max_len=max(bt.lengths, default=0)), **kw},
                           prefix_len=bt.prefix, prefix_table=bt.prefix_table.data_ptr())
    return cache, batch


def run(ctx, bt, q, scale=None, parts=None, stream=0, o=None):
    cache, batch = parts or call_parts(bt)
    o = torch.full(q.shape, 7.0, device="cuda", dtype=q.dtype) if o is None else o
    nbytes = ctx.paged_attention_workspace(cache, batch, q.shape[1])
    # a workspace of exactly the stated size, NaN all over, with a guard behind it
    ws = torch.full((nbytes // 4 + 64,), float("nan"), device="cuda")
    ws[nbytes // 4:] = 5.0
    ctx.paged_attention(cache, batch, heads(q), heads(o), ws.data_ptr() if nbytes else 0, nbytes, scale=scale, stream=stream)
    ctx.sync(stream)
    assert (ws[nbytes // 4:] == 5.0).all()
    return o


def check(ctx, bt, q, **kw):
    o = run(ctx, bt, q, **kw)
    n = sum(bt.new)
    want, tol = refs.attention(bt, q[:n], kw.get("scale"))
    refs.close(o[:n], want, tol, q.dtype, "attention")
    assert (o[n:] == 7.0).all()  # rows behind the last sequence
    return o


CASES = [
    # new, lengths, prefix, page, hq, hkv, d, head_major
    ([1], [1], 0, 16, 1, 1, 64, False),
    ([1], [0], 0, 16, 2, 1, 64, False),                       # a token that sees nothing
    ([1, 1, 1], [15, 16, 17], 0, 16, 8, 2, 128, False),       # page ends
    ([1, 0, 1, 1], [300, 50, 1, 129], 0, 32, 8, 8, 64, True),  # a sequence without new tokens
    ([1, 1, 1, 1, 1], [31, 257, 64, 1, 700], 65, 16, 16, 2, 128, False),
    ([1] * 40, [1 + 13 * i for i in range(40)], 500, 64, 8, 1, 128, True),
    ([1], [5000], 0, 16, 4, 1, 128, False),                   # one long row: many splits
    ([1], [3], 4097, 128, 7, 1, 64, False),                   # all of it prefix
    ([5, 1, 3], [100, 33, 3], 77, 8, 4, 2, 80, True),
    ([8, 8], [8, 200], 1000, 20, 12, 4, 96, False),
    ([4, 2, 1], [40, 1, 0], 10, 16, 4, 1, 64, False),         # more new tokens than cached: the first see the prefix alone
    ([4, 3], [2, 3], 0, 16, 4, 1, 64, False),                 # and without a prefix nothing
    ([40, 17], [150, 17], 50, 32, 8, 2, 128, False),
    ([130, 1, 250], [130, 70, 600], 0, 64, 4, 2, 64, True),
    ([200, 64, 5], [333, 100, 5], 301, 16, 8, 2, 128, False),  # prefix joined to the own keys
    ([300], [1500], 128, 128, 4, 4, 256, False),
    ([1, 2], [900, 40], 333, 16, 8, 2, 256, True),
    ([3], [77], 13, 4, 3, 3, 24, False),
    ([700], [700], 0, 16, 2, 1, 128, False),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_matches(ctx, torch_cuda, kernel, dtype, case):
    if dtype == "f32" and kernel != "rule":
        pytest.skip("f32 has one kernel")
    new, lengths, prefix, page, hq, hkv, d, head_major = CASES[case]
    bt = refs.batch(new, lengths, prefix=prefix, page=page, heads=hkv, d=d, dtype=refs.DTYPES[dtype], head_major=head_major,
                    seed=case, extra_rows=2)
    q = (1.5 * torch.randn(bt.tokens, hq, d, device="cuda", generator=bt.generator)).to(bt.dtype)
    check(ctx, bt, q)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [1, 3, 8, 36, 100, 136])
def test_attention_odd_head_dims(ctx, torch_cuda, dtype, d):
    bt = refs.batch([1, 3], [50, 9], prefix=21, heads=2, d=d, dtype=refs.DTYPES[dtype], seed=d)
    q = torch.randn(bt.tokens, 4, d, device="cuda", generator=bt.generator).to(bt.dtype)
    check(ctx, bt, q, scale=0.7)


@pytest.mark.parametrize("page", [1, 4, 8, 16, 20, 24, 64, 128, 256, 384])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (3, 1, 128), (14, 2, 80), (16, 1, 128), (32, 2, 40), (12, 4, 256), (8, 4, 192)])
def test_attention_page_sizes_and_groups(ctx, torch_cuda, kernel, page, hq, hkv, d):
    """Boxes of pages, of tokens by heads, and what neither fits; tiles that end in a prefix, a page and a length."""
    dt = torch.bfloat16 if page % 16 else torch.float16
    bt = refs.batch([33, 1, 0, 150], [260, 129, 7, 150], prefix=157, page=page, heads=hkv, d=d, dtype=dt, seed=page + d,
                    head_major=bool(hq % 2), extra_rows=1)
    q = torch.randn(bt.tokens, hq, d, device="cuda", generator=bt.generator).to(dt)
    check(ctx, bt, q)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1])
def test_attention_strided_operands(ctx, torch_cuda, kernel, dtype, shift):
    """Keys and values side by side in one buffer, queries out of a fused projection, outputs with gaps; shift moves every
    base off its 16 bytes."""
    dt, d, h = refs.DTYPES[dtype], 64, 2
    bt = refs.batch([2, 1, 9], [70, 33, 40], prefix=40, heads=h, d=d, dtype=dt)
    both = torch.full((bt.pages * bt.page * h * 2 * d + 8,), float("nan"), device="cuda", dtype=dt)
    view = both[shift:shift + bt.pages * bt.page * h * 2 * d].view(bt.pages, bt.page, h, 2, d)
    view[:, :, :, 0], view[:, :, :, 1] = bt.k, bt.v
    strides = (bt.page * h * 2 * d, h * 2 * d, 2 * d)
    cache = rt.paged_cache(view.data_ptr(), view[:, :, :, 1].data_ptr(), CODES[dt], bt.pages, bt.page, h, d,
                           k_strides=strides, v_strides=strides)
    fused = torch.randn(bt.tokens * 9 * d + 8, device="cuda").to(dt)[shift:shift + bt.tokens * 9 * d].view(bt.tokens, 9, d)
    q = fused[:, 1:7]
    o = torch.full((bt.tokens, 13, d + 8), 7.0, device="cuda", dtype=dt)
    run(ctx, bt, q, parts=(cache, call_parts(bt)[1]), o=o[:, 3:9, :d])
    want, tol = refs.attention(bt, q)
    refs.close(o[:, 3:9, :d], want, tol, dt, "strided")
    o[:, 3:9, :d] = 7.0
    assert (o == 7.0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,lengths,prefix", [([1, 3], [200, 90], 64), ([70, 150], [170, 150], 100)])
def test_attention_large_scores_and_one_hot_rows(ctx, torch_cuda, kernel, dtype, new, lengths, prefix):
    """Scores of hundreds: the running maximum moves far, and a row may be one key alone."""
    dt = refs.DTYPES[dtype]
    bt = refs.batch(new, lengths, prefix=prefix, heads=2, d=64, dtype=dt, seed=9)
    q = (40.0 * torch.randn(bt.tokens, 8, 64, device="cuda", generator=bt.generator)).to(dt)
    check(ctx, bt, q)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_far_pages(ctx, torch_cuda, kernel, dtype):
    """Pages beyond 2^31 elements of the cache's start."""
    dt, page, h, d = refs.DTYPES[dtype], 64, 4, 128
    per = page * h * d
    pages = 2 ** 31 // per + 40
    if torch.cuda.mem_get_info()[0] < 3 * pages * per * dt.itemsize:
        pytest.skip("not enough device memory")
    bt = refs.batch([1, 2, 150], [100, 200, 170], prefix=70, page=page, heads=h, d=d, dtype=dt)
    far = torch.empty(pages, page, h, d, device="cuda", dtype=dt)
    lift = pages - bt.pages
    far[lift:] = bt.k
    k_far = far
    v_far = torch.empty_like(far)
    v_far[lift:] = bt.v
    bt.k, bt.v, bt.pages = k_far, v_far, pages
    bt.table += lift
    bt.prefix_table += lift
    q = torch.randn(bt.tokens, 8, d, device="cuda").to(dt)
    check(ctx, bt, q)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [[1, 1], [3, 90]])
def test_attention_in_graphs_and_streams(ctx, torch_cuda, kernel, dtype, new):
    """Two captured calls with workspaces of their own, replayed at once with lengths changed since the capture."""
    dt, runs = refs.DTYPES[dtype], []
    for seed in (1, 2):
        bt = refs.batch(new, [400, 333], prefix=150, heads=2, d=128, dtype=dt, seed=seed)
        q = torch.randn(bt.tokens, 8, 128, device="cuda", generator=bt.generator).to(dt)
        cache, batch = call_parts(bt)
        nbytes = ctx.paged_attention_workspace(cache, batch, 8)
        ws, o = torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda"), torch.zeros_like(q)
        call = ctx.paged_attention_call(cache, batch, heads(q), heads(o), ws.data_ptr(), nbytes)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            call.with_stream(torch.cuda.current_stream().cuda_stream)()
        bt.lengths = [211, 97]
        bt.lens.copy_(torch.tensor(bt.lengths, dtype=torch.int32))
        runs.append((bt, q, o, graph, stream, ws))
    torch.cuda.synchronize()
    for _ in range(3):
        for bt, q, o, graph, stream, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    ctx.sync()
    for bt, q, o, *_ in runs:
        want, tol = refs.attention(bt, q)
        refs.close(o, want, tol, dt, "replayed")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_same_bits_every_time(ctx, torch_cuda, kernel, dtype):
    bt = refs.batch([1, 4, 60], [900, 500, 300], prefix=800, heads=2, d=128, dtype=refs.DTYPES[dtype])
    q = torch.randn(bt.tokens, 8, 128, device="cuda").to(bt.dtype)
    one = run(ctx, bt, q)
    for _ in range(4):
        assert torch.equal(one, run(ctx, bt, q))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [[1, 1, 1], [2, 80, 1]])
@pytest.mark.parametrize("what", ["page", "negative page", "prefix page", "long", "too many new"])
def test_attention_index_out_of_bounds(ctx, torch_cuda, kernel, dtype, new, what):
    """A bad page hides its keys, a bad length or count leaves its rows alone; the next sync reports it."""
    bt = refs.batch(new, [90, 90, 45], prefix=40, heads=2, d=64, dtype=refs.DTYPES[dtype])
    q = torch.randn(bt.tokens, 4, 64, device="cuda", generator=bt.generator).to(bt.dtype)
    cache, batch = call_parts(bt)
    good, page = run(ctx, bt, q), int(bt.table[1, 2])
    if what in ("page", "negative page"):
        bt.table[1, 2] = bt.pages if what == "page" else -3
    elif what == "prefix page":
        bt.prefix_table[1] = 2 ** 31 - 1
    elif what == "long":
        bt.lens[1] = 91
    else:
        batch.max_new = max(new) - 1 if max(new) > 1 else 1
        if max(new) == 1:
            bt.first.copy_(torch.tensor([0, 1, 3, 3], dtype=torch.int32))
    o = torch.full(q.shape, 7.0, device="cuda", dtype=bt.dtype)
    nbytes = ctx.paged_attention_workspace(cache, batch, 4)
    ws = torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")
    ctx.paged_attention(cache, batch, heads(q), heads(o), ws.data_ptr(), nbytes)
    with pytest.raises(rt.B2KError) as e:
        ctx.sync()
    assert e.value.status == rt.B2K_EINDEX
    ctx.sync()
    at = [sum(new[:b]) for b in range(4)]
    if what in ("page", "negative page"):
        keep = torch.cat([torch.arange(32), torch.arange(48, 90)])
        some = refs.attention(bt_without(bt, 1, page, keep), q)
        got = o[at[1] + new[1] - 1].double()
        refs.close(got[None], some[0][at[1] + new[1] - 1][None], some[1][at[1] + new[1] - 1][None], bt.dtype, "rest")
    elif what != "prefix page":
        assert (o[at[1]:at[1] + 1] == 7.0).all()
    if what != "prefix page" and what != "too many new":
        for b in (0, 2):
            assert torch.equal(o[at[b]:at[b + 1]], good[at[b]:at[b + 1]])


def bt_without(bt, b, page, keep):
    """The batch with sequence b's keys `keep` alone, for its last row; `page` is the right third page of its table."""
    import copy
    c = copy.copy(bt)
    c.table = bt.table.clone()
    c.table[b, 2] = page
    rows_k, rows_v = refs.read_rows(c, bt.k, b, 90), refs.read_rows(c, bt.v, b, 90)
    c.k, c.v, c.lengths = bt.k.clone(), bt.v.clone(), list(bt.lengths)
    c.lengths[b] = len(keep)
    for cache, rows in ((c.k, rows_k), (c.v, rows_v)):
        refs.write_rows(c, cache, b, rows[keep.cuda()])
    return c


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_only_prefix(ctx, torch_cuda, kernel, dtype):
    """No own keys at all, and no table for them: every row sees the prefix alone."""
    bt = refs.batch([1, 2], [0, 0], prefix=333, heads=2, d=64, dtype=refs.DTYPES[dtype])
    q = torch.randn(3, 4, 64, device="cuda", generator=bt.generator).to(bt.dtype)
    cache, batch = call_parts(bt)
    batch.table, batch.table_width, batch.table_stride = None, 0, 0
    o = run(ctx, bt, q, parts=(cache, batch))
    want, tol = refs.attention(bt, q)
    refs.close(o, want, tol, q.dtype, "prefix alone")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_calls_side_by_side(ctx, torch_cuda, kernel, dtype):
    """Calls on several streams at once, each with its own workspace, and back to back in one with one workspace."""
    dt, jobs = refs.DTYPES[dtype], []
    for seed in range(4):
        bt = refs.batch([1 + seed, 40], [500, 200 + seed], prefix=200, heads=2, d=128, dtype=dt, seed=seed)
        q = torch.randn(bt.tokens, 8, 128, device="cuda", generator=bt.generator).to(dt)
        cache, batch = call_parts(bt)
        nbytes = ctx.paged_attention_workspace(cache, batch, 8)
        jobs.append((bt, q, torch.zeros_like(q), torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda"), nbytes,
                     cache, batch, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(3):
        for bt, q, o, ws, nbytes, cache, batch, s in jobs:
            ctx.paged_attention(cache, batch, heads(q), heads(o), ws.data_ptr(), nbytes, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for bt, q, o, *_ in jobs:
        want, tol = refs.attention(bt, q)
        refs.close(o, want, tol, dt, "streams")
        o.zero_()
    shared = torch.empty(max(16, *(j[4] for j in jobs)), dtype=torch.uint8, device="cuda")
    for bt, q, o, _, nbytes, cache, batch, _ in jobs:
        ctx.paged_attention(cache, batch, heads(q), heads(o), shared.data_ptr(), nbytes)
    ctx.sync()
    for bt, q, o, *_ in jobs:
        want, tol = refs.attention(bt, q)
        refs.close(o, want, tol, dt, "one after the other")


def test_attention_values_of_later_tokens(ctx, torch_cuda):
    """The plain kernel keeps what a row may not see out of it altogether."""
    bt = refs.batch([4], [20], heads=1, d=64, dtype=torch.float32)
    refs.write_rows(bt, bt.v, 0, torch.cat([refs.read_rows(bt, bt.v, 0, 20)[:19], torch.full((1, 1, 64), float("nan"), device="cuda")]))
    q = torch.randn(4, 2, 64, device="cuda")
    o = run(ctx, bt, q)
    assert torch.isfinite(o[:3]).all() and torch.isnan(o[3]).all()


def test_attention_refusals(ctx, torch_cuda):
    bt = refs.batch([1, 1], [300, 20], prefix=20, heads=2, d=32, dtype=torch.float32)
    q, o = torch.zeros(2, 4, 32, device="cuda"), torch.zeros(2, 4, 32, device="cuda")
    cache, batch = call_parts(bt)
    nbytes = ctx.paged_attention_workspace(cache, batch, 4)
    ws = torch.empty(nbytes + 16, dtype=torch.uint8, device="cuda")
    assert nbytes > 0

    def refused(status=rt.B2K_EINVAL, cache=cache, batch=batch, q=heads(q), o=heads(o), ws=ws.data_ptr(), nbytes=nbytes, **kw):
        with pytest.raises(rt.B2KError) as e:
            ctx.paged_attention(cache, batch, q, o, ws, nbytes, **kw)
        assert e.value.status == status

    def changed(s, **kw):
        c = type(s).from_buffer_copy(s)
        for name, value in kw.items():
            setattr(c, name, value)
        return c

    refused(ws=0)
    refused(nbytes=nbytes - 1)
    refused(ws=ws.data_ptr() + 4)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(scale=scale)
    refused(o=heads(q))
    refused(q=rt.heads(q.data_ptr(), 3, 96, 32), o=rt.heads(o.data_ptr(), 3, 96, 32))  # three heads over two
    refused(q=rt.heads(q.data_ptr(), 2, 64, 32))
    refused(o=rt.heads(0, 4, 128, 32))
    for kw in (dict(v=None), dict(dtype=-1), dict(page_size=0), dict(d=300), dict(v_head=8)):
        refused(cache=changed(cache, **kw))
    for kw in (dict(max_len=10 ** 6), dict(tokens=-1), dict(prefix_table=None), dict(table_stride=1)):
        refused(batch=changed(batch, **kw))
    refused(status=rt.B2K_EUNSUPPORTED, batch=changed(batch, sequences=70000))
    ctx.paged_attention(cache, changed(batch, sequences=0), heads(q), heads(o))
    ctx.sync()
