"""The serving operators together, as one step of a server uses them: a shared prompt goes into the cache, then
sequences append drafted tokens, attend to everything, and have the drafts verified against probabilities that the
package's GEMM and row softmax make of the attention's output."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from conftest import PKG

torch = pytest.importorskip("torch")
import serving_refs as refs  # noqa: E402

pytestmark = pytest.mark.gpu
rt = importlib.import_module(f"{PKG}.runtime")
CODES = {torch.float32: rt.F32, torch.float16: rt.F16, torch.bfloat16: rt.BF16}


def heads(x):
    return rt.heads(x.data_ptr(), x.shape[1], x.stride(0), x.stride(1))


class Server:
    """A cache of pages and the sequences in it; every call goes through the package."""

    def __init__(self, ctx, sequences, dtype, hq=4, hkv=2, d=64, page=16, width=8, prefix_len=0, prefix_pages=8):
        self.ctx, self.dtype, self.hq, self.hkv, self.d, self.page, self.width = ctx, dtype, hq, hkv, d, page, width
        pages = prefix_pages + sequences * width
        self.k = torch.full((pages, page, hkv, d), float("nan"), device="cuda", dtype=dtype)
        self.v = self.k.clone()
        order = torch.randperm(pages).to(torch.int32).cuda()
        self.prefix_table, self.table = order[:prefix_pages].clone(), order[prefix_pages:].view(sequences, width).clone()
        self.lengths, self.prefix_len = torch.zeros(sequences, dtype=torch.int32, device="cuda"), prefix_len
        self.cache = rt.paged_cache(self.k.data_ptr(), self.v.data_ptr(), CODES[dtype], pages, page, hkv, d)
        self.rope = rt.rope_plan(d, scaling="log_ramp", factor=4.0, context=64.0, magnitude=1.125)

    def step(self, qkv, new, table=None, lengths=None, prefix_len=None):
        """Append `new` tokens to each sequence and attend; qkv [tokens, hq + 2 hkv, d]."""
        table = self.table if table is None else table
        lengths = self.lengths if lengths is None else lengths
        new_t = torch.tensor(new, dtype=torch.int32, device="cuda")
        lengths += new_t
        first = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), new_t.cumsum(0).to(torch.int32)])
        n = sum(new)
        batch = rt.paged_batch(len(new), n, first.data_ptr(), lengths.data_ptr(), table.data_ptr(), table.shape[1],
                               max_new=max(new), max_len=table.shape[1] * self.page,
                               prefix_len=self.prefix_len if prefix_len is None else prefix_len,
                               prefix_table=self.prefix_table.data_ptr())
        q, k, v = qkv[:, :self.hq], qkv[:, self.hq:self.hq + self.hkv], qkv[:, self.hq + self.hkv:]
        turned, o = (torch.empty(n, self.hq, self.d, device="cuda", dtype=self.dtype) for _ in range(2))
        nbytes = self.ctx.paged_attention_workspace(self.cache, batch, self.hq)
        ws = torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")
        self.ctx.paged_append(self.cache, batch, heads(k), heads(v), q=heads(q), q_out=heads(turned), rope=self.rope)
        self.ctx.paged_attention(self.cache, batch, heads(turned), heads(o), ws.data_ptr(), nbytes)
        self.ctx.sync()
        return o


def dense(histories, new, d, hq, hkv, freqs):
    """Attention of the last `new` tokens of each sequence's whole history in 64 bits, causal, rotated."""
    outs = []
    for qkv, n in zip(histories, new):
        pos = torch.arange(qkv.shape[0], device="cuda")
        q, _ = refs.rotary(qkv[:, :hq], pos, freqs, False, 1.125)
        k, _ = refs.rotary(qkv[:, hq:hq + hkv], pos, freqs, False, 1.125)
        v = qkv[:, hq + hkv:].double()
        k, v = (x.repeat_interleave(hq // hkv, 1) for x in (k, v))
        s = torch.einsum("jhd,khd->hjk", q[-n:], k) / d ** 0.5
        hidden = pos[None] > pos[-n:, None]
        outs.append(torch.einsum("hjk,khd->jhd", torch.softmax(s.masked_fill(hidden, -float("inf")), -1), v))
    return torch.cat(outs)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_steps_of_a_server(ctx, torch_cuda, dtype):
    dt, hq, hkv, d, vocab, drafts = refs.DTYPES[dtype], 4, 2, 64, 500, 3
    g = torch.Generator(device="cuda").manual_seed(3)
    draw = lambda n: torch.randn(n, hq + 2 * hkv, d, device="cuda", generator=g).to(dt)  # noqa: E731
    server = Server(ctx, 3, dt, prefix_len=0)
    freqs = refs.frequencies(d, scaling="log_ramp", factor=4.0, context=64.0)
    # u: what the operands' roundings leave of an output of unit size: those of the rotated queries and keys (each a
    # score's relative error, scores up to about 8), of the probabilities and of the output
    u = 2 * 8 * refs.half_step(dt) + 4 * refs.half_step(dt) + 2e-5

    def same(o, histories, new):
        want = dense(histories, new, d, hq, hkv, freqs)
        assert float((o.double() - want).abs().max()) <= u * float(want.abs().max())
        return want

    # the shared prompt, as the one sequence of its own pages, in two chunks; then it is everybody's prefix
    prompt = draw(101)
    table, length = server.prefix_table.view(1, -1), torch.zeros(1, dtype=torch.int32, device="cuda")
    o = torch.cat([server.step(prompt[:70], [70], table, length, 0), server.step(prompt[70:], [31], table, length, 0)])
    same(o, [prompt], [101])
    server.prefix_len = 101
    histories = [prompt] * 3
    weights = (torch.randn(hq * d, vocab, device="cuda", generator=g) / 4).contiguous()
    rng = np.random.default_rng(0)
    for new in ([5, 1, 17], [1, 1, 1], [drafts + 1] * 3, [drafts + 1] * 3):
        qkv = draw(sum(new))
        histories = [torch.cat([h, x]) for h, x in zip(histories, qkv.split(new))]
        o = server.step(qkv, new)
        same(o, histories, new)
    # the last step's rows are the places of three drafted tokens and one more: probabilities, then the verdict
    rows = 3 * (drafts + 1)
    x, logits = o.float().reshape(rows, hq * d).contiguous(), torch.empty(rows, vocab, device="cuda")
    target = torch.empty_like(logits)
    ctx.gemm(x.data_ptr(), weights.data_ptr(), logits.data_ptr(), rows, vocab, hq * d)
    ctx.row_softmax(logits.data_ptr(), target.data_ptr(), rows, vocab)
    ctx.sync()
    exact = torch.softmax(x.double() @ weights.double(), -1)
    assert float((target.double() - exact).abs().max()) <= 1e-5 * float(exact.max()) * 10
    target = target.view(3, drafts + 1, vocab)
    draft = torch.softmax(target[:, :drafts].log() + torch.randn(3, drafts, vocab, device="cuda", generator=g), -1).contiguous()
    tokens = torch.tensor(rng.integers(0, vocab, (3, drafts)), dtype=torch.int32, device="cuda")
    tokens[:, 0] = draft[:, 0].argmax(-1)
    u_accept, u_sample = torch.rand(3, drafts, device="cuda", generator=g) / 8, torch.rand(3, device="cuda", generator=g)
    accepted, out = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, drafts + 1, dtype=torch.int32, device="cuda")
    ctx.verify_drafts(target.data_ptr(), tokens.data_ptr(), u_accept.data_ptr(), u_sample.data_ptr(), accepted.data_ptr(),
                      out.data_ptr(), 3, drafts, vocab, draft=draft.data_ptr())
    ctx.sync()
    want = refs.verify(target, draft, tokens, None, u_accept, u_sample)
    assert torch.equal(accepted.cpu(), want[0]) and torch.equal(out.cpu(), want[1])
    # refused drafts leave the cache by the lengths alone: the next step overwrites them
    kept = accepted.tolist()
    server.lengths -= torch.tensor([drafts - a for a in kept], dtype=torch.int32, device="cuda")
    histories = [h[:h.shape[0] - (drafts - a)] for h, a in zip(histories, kept)]
    qkv = draw(3)
    histories = [torch.cat([h, x]) for h, x in zip(histories, qkv.split([1, 1, 1]))]
    same(server.step(qkv, [1, 1, 1]), histories, [1, 1, 1])


def test_rotary_before_dense_attention(ctx, torch_cuda):
    """Rotated queries and keys in the package's dense attention, and the same rows over a paged cache."""
    n, d = 200, 128
    bt = refs.batch([1], [n], heads=1, d=d, dtype=torch.float32, poison=False)
    qk = torch.randn(2, n, 1, d, device="cuda", generator=bt.generator)
    pos, rope = torch.arange(n, device="cuda"), rt.rope_plan(d, interleaved=True)
    ctx.rotary(rope, rt.F32, [(heads(qk[0]), heads(qk[0])), (heads(qk[1]), heads(qk[1]))], pos.data_ptr(), n, d)
    v = refs.read_rows(bt, bt.v, 0, n)
    o = torch.empty(1, n, d, device="cuda")
    q, k, flat = (x.reshape(1, n, d).contiguous() for x in (qk[0], qk[1], v))
    ctx.attention(q.data_ptr(), k.data_ptr(), flat.data_ptr(), o.data_ptr(), 1, n, n, d, d)
    ctx.sync()
    refs.write_rows(bt, bt.k, 0, qk[1])
    cache = rt.paged_cache(bt.k.data_ptr(), bt.v.data_ptr(), rt.F32, bt.pages, bt.page, 1, d)
    batch = rt.paged_batch(1, 1, bt.first.data_ptr(), bt.lens.data_ptr(), bt.table.data_ptr(), bt.width, max_new=1, max_len=n)
    last, paged = qk[0][-1:].contiguous(), torch.empty(1, 1, d, device="cuda")
    nbytes = ctx.paged_attention_workspace(cache, batch, 1)
    ws = torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")
    ctx.paged_attention(cache, batch, heads(last), heads(paged), ws.data_ptr(), nbytes)
    ctx.sync()
    want, _ = refs.attention(bt, last)
    assert float((paged.double() - want).abs().max()) <= 1e-5 and float((o[0, -1].double() - want[0, 0]).abs().max()) <= 1e-5


def test_append_and_attention_in_one_graph(ctx, torch_cuda):
    """A captured decode step, replayed while the lengths move on."""
    server = Server(ctx, 2, torch.bfloat16)
    hq, hkv, d = 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    server.step(torch.randn(30, hq + 2 * hkv, d, device="cuda", generator=g).bfloat16(), [20, 10])
    qkv = torch.zeros(2, hq + 2 * hkv, d, device="cuda", dtype=torch.bfloat16)
    first = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    batch = rt.paged_batch(2, 2, first.data_ptr(), server.lengths.data_ptr(), server.table.data_ptr(), server.width, max_new=1,
                           max_len=server.width * server.page)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    turned, o = (torch.zeros(2, hq, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    nbytes = ctx.paged_attention_workspace(server.cache, batch, hq)
    ws = torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        s = torch.cuda.current_stream().cuda_stream
        ctx.paged_append(server.cache, batch, heads(k), heads(v), q=heads(q), q_out=heads(turned), rope=server.rope, stream=s)
        ctx.paged_attention(server.cache, batch, heads(turned), heads(o), ws.data_ptr(), nbytes, stream=s)
    for _ in range(20):
        x = torch.randn(2, hq + 2 * hkv, d, device="cuda", generator=g).bfloat16()
        mirror = Server(ctx, 2, torch.bfloat16)
        mirror.__dict__.update({n: getattr(server, n) for n in ("table", "prefix_table")})
        mirror.k, mirror.v, mirror.lengths = server.k.clone(), server.v.clone(), server.lengths.clone()
        mirror.cache = rt.paged_cache(mirror.k.data_ptr(), mirror.v.data_ptr(), rt.BF16, server.k.shape[0], 16, hkv, d)
        want = mirror.step(x, [1, 1])
        qkv.copy_(x)
        server.lengths += 1
        graph.replay()
        torch.cuda.synchronize()
        ctx.sync()
        assert torch.equal(o, want) and torch.equal(server.k.nan_to_num(9.0), mirror.k.nan_to_num(9.0))


def test_session_arrays(ctx, torch_cuda):
    """The same step from NumPy arrays, without PyTorch on the package's side."""
    api = importlib.import_module(f"{PKG}.api")
    rng = np.random.default_rng(4)
    with api.Session(0) as s:
        n, hq, hkv, d, page = 3, 4, 2, 32, 16
        kv = s.paged_kv(8, page, hkv, d)
        qkv = [rng.standard_normal((n, h, d)).astype(np.float32) for h in (hq, hkv, hkv)]
        q, k, v = (s.upload(x) for x in qkv)
        first, lengths = s.upload(np.array([0, 2, 3], np.int32)), s.upload(np.array([2, 1], np.int32))
        table = s.upload(np.array([[5, 1], [3, 0]], np.int32))
        batch = s.paged_batch(first, lengths, table, n, max_new=2, max_len=2)
        rope, turned, o = rt.rope_plan(d), s.empty((n, hq, d)), s.empty((n, hq, d))
        s.paged_append(kv, batch, k, v, q=q, q_out=turned, rope=rope)
        s.paged_attention(kv, batch, turned, o)
        pos, back = s.upload(np.array([0, 1, 0], np.int64)), s.empty((n, hq, d))
        s.rotary(rope, [(turned, back)], pos, transpose=True)
        s.sync()
        got, same, cache = s.download(o), s.download(back), s.download(kv.k)
        s.sync()
        # a rotation's transpose is its inverse: two passes of FP32 roundings
        assert np.abs(same - qkv[0]).max() <= 4e-6
        keys = torch.from_numpy(np.stack([cache[5, 0], cache[5, 1], cache[3, 0]]))
        want, tol = refs.rotary(torch.from_numpy(qkv[1]), torch.tensor([0, 1, 0]), refs.frequencies(d), False)
        refs.close(keys, want, tol, torch.float32, "keys")
        assert np.abs(got[0] - np.repeat(qkv[2][0], 2, 0)).max() <= 1e-6  # a first token sees itself alone
        assert np.abs(got[2] - np.repeat(qkv[2][2], 2, 0)).max() <= 1e-6
        target = rng.random((2, 3, 50)).astype(np.float32)
        drafted = rng.integers(0, 50, (2, 2)).astype(np.int32)
        u, us = rng.random((2, 2)).astype(np.float32), rng.random(2).astype(np.float32)
        accepted, tokens = s.empty((2,), np.int32), s.empty((2, 3), np.int32)
        s.verify_drafts(s.upload(target), s.upload(drafted), s.upload(u), s.upload(us), accepted, tokens)
        s.sync()
        a, out = s.download(accepted), s.download(tokens)
        s.sync()
        want = refs.verify(*(torch.from_numpy(target), None, torch.from_numpy(drafted), None, torch.from_numpy(u), torch.from_numpy(us)))
        assert np.array_equal(a, want[0].numpy()) and np.array_equal(out, want[1].numpy())
        with pytest.raises(ValueError):
            s.rotary(rope, [(turned, back)], lengths)
        with pytest.raises(ValueError):
            s.paged_attention(kv, batch, s.empty((n, hq, d), np.float16), o)
        with pytest.raises(ValueError):
            s.paged_batch(first, first, table, n, max_new=2, max_len=2)
        kv.free()
