"""Calls of the serving operators at the edges of what their documentation allows: bounds far above the lengths in use,
arrays that meet, steps that follow each other without a synchronisation."""
from __future__ import annotations

import importlib
from types import SimpleNamespace

import pytest

from conftest import PKG

torch = pytest.importorskip("torch")
import serving_refs as refs  # noqa: E402
from test_gpu_paged import CASES, call_parts, check  # noqa: E402

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


# --- steps without a synchronisation -----------------------------------------------------------------------


# prefix part and own part in two kernels side by side: (dtype, prefix, kernels the plan names)
TWO_KERNELS = [("bf16", 6000, (1, 2)), ("bf16", 4000, (1, 1)), ("f16", 300, (1, 1)), ("f32", 300, (0, 0))]


class Steps:
    """A decode loop of 40 sequences behind a prefix; everything that a step reads is overwritten by the next."""

    def __init__(self, ctx, dtype, prefix, seed=0, steps=24):
        self.ctx, self.dt, self.n, self.hq, self.hkv, self.d = ctx, refs.DTYPES[dtype], 40, 8, 2, 64
        lengths = [1 + 17 * i % 500 for i in range(self.n)]
        self.bt = refs.batch([1] * self.n, [x + steps for x in lengths], prefix=prefix, heads=self.hkv, d=self.d, dtype=self.dt,
                             seed=seed, poison=False)
        g = torch.Generator(device="cuda").manual_seed(seed + 100)
        self.inputs = torch.randn(steps, self.n, self.hq + 2 * self.hkv, self.d, device="cuda", generator=g).to(self.dt)
        self.start, self.k0, self.v0 = torch.tensor(lengths, dtype=torch.int32, device="cuda"), self.bt.k.clone(), self.bt.v.clone()
        self.lens, self.qkv = self.start.clone(), torch.zeros_like(self.inputs[0])
        self.turned, self.o = (torch.zeros(self.n, self.hq, self.d, device="cuda", dtype=self.dt) for _ in range(2))
        bt = self.bt
        self.cache = rt.paged_cache(bt.k.data_ptr(), bt.v.data_ptr(), CODES[self.dt], bt.pages, bt.page, self.hkv, self.d)
        self.batch = rt.paged_batch(self.n, self.n, bt.first.data_ptr(), self.lens.data_ptr(), bt.table.data_ptr(), bt.width,
                                    max_new=1, max_len=max(bt.lengths), prefix_len=prefix, prefix_table=bt.prefix_table.data_ptr())
        self.nbytes = ctx.paged_attention_workspace(self.cache, self.batch, self.hq)
        self.ws = torch.empty(self.nbytes, dtype=torch.uint8, device="cuda")
        self.rope = rt.rope_plan(self.d)
        self.outs = torch.zeros(steps, *self.o.shape, device="cuda", dtype=self.dt)

    def rewind(self):
        self.lens.copy_(self.start)
        self.bt.k.copy_(self.k0)
        self.bt.v.copy_(self.v0)
        self.outs.zero_()
        self.ws.fill_(255)
        torch.cuda.synchronize()

    def calls(self, after=lambda: None):
        stream = torch.cuda.current_stream().cuda_stream
        q, k, v = self.qkv[:, :self.hq], self.qkv[:, self.hq:self.hq + self.hkv], self.qkv[:, self.hq + self.hkv:]
        self.lens.add_(1)
        after()
        self.ctx.paged_append(self.cache, self.batch, heads(k), heads(v), q=heads(q), q_out=heads(self.turned), rope=self.rope,
                              stream=stream)
        after()
        self.ctx.paged_attention(self.cache, self.batch, heads(self.turned), heads(self.o), self.ws.data_ptr(), self.nbytes,
                                 stream=stream)
        after()

    def run(self, one, after=lambda: None):
        for i, x in enumerate(self.inputs):
            self.qkv.copy_(x)
            one()
            self.outs[i].copy_(self.o)
            after()

    def state(self):
        torch.cuda.synchronize()
        self.ctx.sync()
        return [x.clone() for x in (self.outs, self.bt.k, self.bt.v)]


@pytest.mark.parametrize("dtype,prefix,kernels", TWO_KERNELS)
def test_steps_back_to_back(ctx, torch_cuda, dtype, prefix, kernels):
    """Append, attention in two kernels, append ... on the same buffers, eager and captured: the bits of steps that are
    waited for one by one."""
    s = Steps(ctx, dtype, prefix)
    plan = rt.paged_attention_plan(torch.cuda.get_device_properties(0).multi_processor_count, s.cache, s.batch, heads(s.turned),
                                   heads(s.o))
    assert (plan["own_kernel"], plan["prefix_kernel"], plan["joined"]) == (*kernels, 0)
    s.run(lambda: s.calls(after=torch.cuda.synchronize), torch.cuda.synchronize)
    want = s.state()
    s.bt.lengths = s.lens.tolist()
    exact, tol = refs.attention(s.bt, s.turned)
    refs.close(want[0][-1], exact, tol, s.dt, "last step")
    for _ in range(3):
        s.rewind()
        s.run(s.calls)
        assert all(torch.equal(a, b) for a, b in zip(want, s.state()))
    graph = torch.cuda.CUDAGraph()
    s.rewind()
    with torch.cuda.graph(graph):
        s.calls()
    for _ in range(3):
        s.rewind()
        s.run(graph.replay)
        assert all(torch.equal(a, b) for a, b in zip(want, s.state()))


@pytest.mark.parametrize("dtype,prefix,kernels", TWO_KERNELS)
def test_steps_on_two_streams(ctx, torch_cuda, dtype, prefix, kernels):
    """Two loops at once, of one context: eager in both, then captured in one and eager in the other."""
    loops, want = [Steps(ctx, dtype, prefix, seed) for seed in (1, 2)], []
    for s in loops:
        s.run(s.calls)
        want.append(s.state())
        s.rewind()
    streams = [torch.cuda.Stream() for _ in loops]

    def both(*ones):
        for s in loops:
            s.rewind()
        for i in range(len(loops[0].inputs)):
            for s, stream, one in zip(loops, streams, ones):
                with torch.cuda.stream(stream):
                    s.qkv.copy_(s.inputs[i])
                    one()
                    s.outs[i].copy_(s.o)
        for s, w in zip(loops, want):
            assert all(torch.equal(a, b) for a, b in zip(w, s.state()))

    both(loops[0].calls, loops[1].calls)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        loops[0].calls()
    both(graph.replay, loops[1].calls)


def test_capture_that_begins_with_attention(ctx, torch_cuda):
    """Nothing before the two kernels in the graph, and an eager call between its captures."""
    s = Steps(ctx, "bf16", 6000, steps=1)
    s.lens.add_(1)
    q = torch.randn(s.turned.shape, device="cuda").to(s.dt)
    s.bt.lengths = s.lens.tolist()
    want, tol = refs.attention(s.bt, q)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            ctx.paged_attention(s.cache, s.batch, heads(q), heads(s.o), s.ws.data_ptr(), s.nbytes,
                                stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
        refs.close(attend(ctx, s.cache, s.batch, q), want, tol, s.dt, "eager")
    for graph in graphs:
        s.o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        ctx.sync()
        refs.close(s.o, want, tol, s.dt, "replayed")


# --- operands that meet ------------------------------------------------------------------------------------


def test_outputs_that_meet_are_refused(ctx, torch_cuda):
    """Two rows of an output, an output and another operand: refused before anything is launched; places side by side
    are not."""
    n, h, d = 6, 4, 32
    buf = torch.randn(4 * n, 2 * h, d, device="cuda").bfloat16()
    at = lambda row, head=0, heads_=h, st=2 * h * d, sh=d: rt.heads(buf[row, head].data_ptr(), heads_, st, sh)  # noqa: E731
    pos, rope = torch.arange(n, device="cuda"), rt.rope_plan(d)
    keep = buf.clone()

    def refused(call, *args, **kw):
        with pytest.raises(rt.B2KError) as e:
            call(*args, **kw)
        assert e.value.status == rt.B2K_EINVAL

    rotate = lambda pairs: ctx.rotary(rope, rt.BF16, pairs, pos.data_ptr(), n, d)  # noqa: E731
    for pairs in ([(at(0), at(n, st=d))], [(at(0), at(n, st=d, sh=2 * d))],     # the output's tokens in its heads' places
                  [(at(0), at(1))], [(at(0), at(0, 1))],                          # a row, a head further
                  [(at(0), at(n)), (at(n), at(2 * n))],                           # an output over the other tensor's input
                  [(at(0), at(2 * n)), (at(n), at(2 * n, 3))]):                   # two outputs in one place
        refused(rotate, pairs)
    bt = refs.batch([1] * n, [20] * n, heads=h, d=d, poison=False)
    cache = rt.paged_cache(bt.k.data_ptr(), bt.v.data_ptr(), rt.BF16, bt.pages, bt.page, h, d)
    batch = rt.paged_batch(n, n, bt.first.data_ptr(), bt.lens.data_ptr(), bt.table.data_ptr(), bt.width, max_new=1, max_len=20)
    append = lambda q_out, **kw: ctx.paged_append(cache, batch, at(0), at(0, h), q=at(n), q_out=q_out, rope=rope)  # noqa: E731
    for q_out in (at(0), at(0, 1), at(n, 1), at(n + 1), at(2 * n, st=d)):
        refused(append, q_out)
    nbytes = ctx.paged_attention_workspace(cache, batch, h)
    ws = torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")
    for o in (at(0), at(0, 1), at(1), at(n, st=d)):
        refused(ctx.paged_attention, cache, batch, at(0), o, ws.data_ptr(), nbytes)
    cache.v = cache.k  # rotated keys and values in one place
    refused(append, at(n, h))
    cache.v = bt.v.data_ptr()
    ctx.sync()
    assert torch.equal(buf, keep)
    # side by side in one buffer
    rotate([(at(0), at(0, h)), (at(n), at(n, h)), (at(2 * n), at(2 * n))])
    append(at(n, h))
    ctx.paged_attention(cache, batch, at(0), at(0, h), ws.data_ptr(), nbytes)
    rotate([(at(0, heads_=1, sh=0), rt.heads(buf[3 * n].data_ptr(), 1, d, 0))])
    ctx.sync()


@pytest.mark.parametrize("kernel", [0, 1, 2, 3])
@pytest.mark.parametrize("d,new", [(64, [1, 3]), (128, [40, 90]), (256, [70, 1])])
def test_attention_of_head_major_queries(ctx, torch_cuda, kernel, d, new):
    """q and o as [heads][tokens][d]."""
    bt = refs.batch(new, [130, 200], prefix=70, heads=2, d=d, dtype=torch.bfloat16)
    q = torch.randn(8, bt.tokens, d, device="cuda").bfloat16().transpose(0, 1)
    o = torch.zeros(8, bt.tokens, d, device="cuda").bfloat16().transpose(0, 1)
    ctx.set_paged_attention_kernel(kernel)
    try:
        cache = rt.paged_cache(bt.k.data_ptr(), bt.v.data_ptr(), rt.BF16, bt.pages, bt.page, 2, d)
        batch = rt.paged_batch(2, bt.tokens, bt.first.data_ptr(), bt.lens.data_ptr(), bt.table.data_ptr(), bt.width,
                               max_new=max(new), max_len=200, prefix_len=70, prefix_table=bt.prefix_table.data_ptr())
        nbytes = ctx.paged_attention_workspace(cache, batch, 8)
        ws = torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")
        ctx.paged_attention(cache, batch, heads(q), heads(o), ws.data_ptr(), nbytes)
        ctx.sync()
    finally:
        ctx.set_paged_attention_kernel(0)
    want, tol = refs.attention(bt, q)
    refs.close(o, want, tol, torch.bfloat16, "head-major")


def test_verification_refuses_outputs_in_other_arrays(ctx, torch_cuda):
    batch, drafts, vocab = 3, 2, 8
    ints, floats = torch.zeros(256, dtype=torch.int32, device="cuda"), torch.full((256,), 0.125, device="cuda")
    i, f = (lambda n: ints.data_ptr() + 4 * n), (lambda n: floats.data_ptr() + 4 * n)  # noqa: E731
    # drafted 0..5, counts 6..8, accepted 16..18, tokens 32..40; target 0..71, u_accept 72..77, u_sample 78..80, draft 96..143
    good = dict(target=f(0), drafted=i(0), u_accept=f(72), u_sample=f(78), accepted=i(16), tokens=i(32), batch=batch,
                drafts=drafts, vocab=vocab, counts=i(6), draft=f(96))
    bad = [dict(tokens=i(5)), dict(tokens=i(8)), dict(tokens=i(8), accepted=i(40)), dict(tokens=i(18)), dict(accepted=i(5)),
           dict(accepted=i(31)), dict(accepted=i(40)), dict(accepted=i(8)), dict(tokens=f(71)), dict(tokens=f(77)), dict(accepted=f(80)),
           dict(tokens=f(143)), dict(accepted=f(95)), dict(drafted=i(27)), dict(target=i(0), tokens=i(32)),
           dict(ld_draft=16, accepted=f(96 + 5 * 16 + 7))]
    for kw in bad:
        with pytest.raises(rt.B2KError) as e:
            ctx.verify_drafts(**{**good, **kw})
        assert e.value.status == rt.B2K_EINVAL, kw
    ctx.sync()
    assert not ints.any()
    for kw in (dict(), dict(tokens=i(9), accepted=i(60)), dict(tokens=i(19)), dict(accepted=i(9)), dict(accepted=i(13)), dict(accepted=i(41)),
               dict(accepted=f(144)), dict(tokens=f(81)),
               dict(drafts=0, drafted=i(33), u_accept=i(33), draft=i(33), accepted=i(60))):  # arrays of no elements
        ctx.verify_drafts(**{**good, **kw})
    ctx.sync()


# --- what is copied ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [1, 3000])
@pytest.mark.parametrize("d,rot", [(40, 34), (48, 16), (37, 6)])
def test_elements_outside_pairs_keep_their_bits(ctx, torch_cuda, dtype, interleaved, tokens, d, rot):
    """NaNs with signs and payloads behind the rotated part, in vectors that are rotated in part."""
    dt = refs.DTYPES[dtype]
    bits = torch.int32 if dt == torch.float32 else torch.int16
    odd = {"f32": 0x7f800001, "f16": 0x7c01, "bf16": 0x7f81}[dtype]
    x = torch.randn(tokens, 3, d, device="cuda").to(dt)
    tail = torch.tensor([-1, -2, odd, -5] * d, device="cuda")[:d - rot]
    x.view(bits)[:, :, rot:] = tail.to(bits)
    y, pos = torch.zeros_like(x), torch.arange(tokens, device="cuda")
    ctx.rotary(rt.rope_plan(rot, interleaved=interleaved), CODES[dt], [(heads(x), heads(y))], pos.data_ptr(), tokens, d)
    ctx.sync()
    assert torch.equal(x.view(bits)[:, :, rot:], y.view(bits)[:, :, rot:])
    want, tol = refs.rotary(x[..., :rot], pos, refs.frequencies(rot), interleaved)
    refs.close(y[..., :rot], want, tol, dt, "rotated part")


# --- f32: the kernel that streams, and the blocks of 4, 8 and 32 rows ---------------------------------------


@pytest.mark.parametrize("case", range(len(CASES)))
def test_f32_blocks_of_rows(ctx, torch_cuda, case):
    """The plain kernel where the rule takes the streaming one."""
    new, lengths, prefix, page, hq, hkv, d, head_major = CASES[case]
    bt = refs.batch(new, lengths, prefix=prefix, page=page, heads=hkv, d=d, dtype=torch.float32, head_major=head_major,
                    seed=case, extra_rows=2)
    q = 1.5 * torch.randn(bt.tokens, hq, d, device="cuda", generator=bt.generator)
    ctx.set_paged_attention_kernel(1)
    try:
        check(ctx, bt, q)
    finally:
        ctx.set_paged_attention_kernel(0)


@pytest.mark.parametrize("kernel", [0, 1])
@pytest.mark.parametrize("page", [1, 4, 16, 20, 128, 384])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (6, 2, 80), (12, 2, 128), (4, 4, 256)])
def test_f32_page_sizes_and_groups(ctx, torch_cuda, kernel, page, hq, hkv, d):
    """Pages that end in, at and behind a tile; one to eight rows of a decode, and many."""
    for new, lengths in (([1, 1, 0, 2], [260, 129, 7, 2]), ([33, 1, 0, 150], [260, 129, 7, 150])):
        bt = refs.batch(new, lengths, prefix=157, page=page, heads=hkv, d=d, dtype=torch.float32, seed=page + d,
                        head_major=bool(page % 3), extra_rows=1)
        q = torch.randn(bt.tokens, hq, d, device="cuda", generator=bt.generator)
        ctx.set_paged_attention_kernel(kernel)
        try:
            check(ctx, bt, q)
        finally:
            ctx.set_paged_attention_kernel(0)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [4, 5, 8, 9, 32, 33, 63, 64, 65])
def test_f32_rows_around_the_rules(ctx, torch_cuda, rows, d):
    bt = refs.batch([rows, 1], [300, 77], prefix=50, heads=2, d=d, dtype=torch.float32, seed=rows)
    q = torch.randn(bt.tokens, 2, d, device="cuda", generator=bt.generator)
    cache, batch = call_parts(bt)
    plan = rt.paged_attention_plan(torch.cuda.get_device_properties(0).multi_processor_count, cache, batch, heads(q), heads(torch.empty_like(q)))
    assert plan["streaming"] & 1 == (rows <= 64)
    for kernel in (0, 1):
        ctx.set_paged_attention_kernel(kernel)
        try:
            check(ctx, bt, q)
        finally:
            ctx.set_paged_attention_kernel(0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_at_the_ends_of_the_scales(ctx, torch_cuda, dtype):
    """A scale whose reciprocal FP32 does not hold is refused; the largest leaves the mean of the values."""
    bt = refs.batch([1, 2], [30, 20], heads=1, d=64, dtype=refs.DTYPES[dtype])
    q, (cache, batch) = torch.randn(3, 2, 64, device="cuda").to(bt.dtype), call_parts(bt)
    o = torch.zeros_like(q)
    ws = torch.empty(max(16, ctx.paged_attention_workspace(cache, batch, 2)), dtype=torch.uint8, device="cuda")
    for scale in (1e-39, 4e-39, 1e-45):
        with pytest.raises(rt.B2KError) as e:
            ctx.paged_attention(cache, batch, heads(q), heads(o), ws.data_ptr(), ws.numel(), scale=scale)
        assert e.value.status == rt.B2K_EINVAL
    for kernel in (0, 1, 2, 3):
        ctx.set_paged_attention_kernel(kernel)
        try:
            check(ctx, bt, q, scale=3e38)
        finally:
            ctx.set_paged_attention_kernel(0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("new", [[1, 1, 3], [700, 900, 800]])
def test_append_into_a_shared_buffer(ctx, torch_cuda, dtype, shift, new):
    """Keys and values side by side in one buffer, queries rotated in place in a fused projection; shift moves every base
    off its 16 bytes."""
    dt, d, h, page = refs.DTYPES[dtype], 64, 2, 16
    bt = refs.batch(new, [n + 5 for n in new], prefix=40, page=page, heads=h, d=d, dtype=dt, extra_rows=1, poison=False)
    both = torch.full((bt.pages * page * h * 3 * d + 8,), 7.0, device="cuda", dtype=dt)
    view = both[shift:shift + bt.pages * page * h * 3 * d].view(bt.pages, page, h, 3, d)
    strides = (page * h * 3 * d, h * 3 * d, 3 * d)
    cache = rt.paged_cache(view.data_ptr(), view[:, :, :, 2].data_ptr(), CODES[dt], bt.pages, page, h, d, k_strides=strides,
                           v_strides=strides)
    fused = torch.randn(bt.tokens * 9 * d + 8, device="cuda").to(dt)[shift:shift + bt.tokens * 9 * d].view(bt.tokens, 9, d)
    was = fused.clone()
    ctx.paged_append(cache, call_parts(bt)[1], heads(fused[:, 5:7]), heads(fused[:, 7:]), q=heads(fused[:, 1:5]),
                     q_out=heads(fused[:, 1:5]), rope=rt.rope_plan(d))
    ctx.sync()
    freqs, first = refs.frequencies(d), 0
    expect = torch.full_like(view, 7.0)
    for b, n in enumerate(new):
        pos = 40 + torch.arange(5, n + 5, device="cuda")
        for x, got in ((was[first:first + n, 1:5], fused[first:first + n, 1:5]),
                       (was[first:first + n, 5:7], refs.read_rows(bt, view[:, :, :, 0], b, n + 5)[5:])):
            want, tol = refs.rotary(x, pos, freqs, False)
            refs.close(got, want, tol, dt, f"sequence {b}")
        pages, rows = refs.places(bt, b, n + 5)
        expect[pages[5:], rows[5:], :, 0] = view[pages[5:], rows[5:], :, 0]
        expect[pages[5:], rows[5:], :, 2] = was[first:first + n, 7:]
        first += n
    assert torch.equal(view, expect) and (both[:shift] == 7.0).all()
    fused[:first, 1:5] = was[:first, 1:5]
    assert torch.equal(fused, was)


@pytest.mark.parametrize("dtype,prefix,kernels", TWO_KERNELS)
def test_steps_without_programmatic_launch(ctx, torch_cuda, dtype, prefix, kernels):
    s = Steps(ctx, dtype, prefix, steps=4)
    s.run(s.calls)
    want = s.state()
    ctx.lib.b2k_set_pdl(0)
    try:
        s.rewind()
        s.run(s.calls)
        assert all(torch.equal(a, b) for a, b in zip(want, s.state()))
    finally:
        ctx.lib.b2k_set_pdl(1)
