"""Public Python API over the C ABI, for callers that bring host arrays.

:class:`Session` owns one library context, device buffers allocated through
the library (no PyTorch), page-locked host staging buffers, and the host <->
device copies around each kernel -- the work the reference's runner does per
launch request (tools/local_runner.py:246-342: allocate, copy in, reset
``zero_outputs``, launch, copy out).
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np

from . import runtime

F32 = np.dtype(np.float32)
#: Element types of the serving operators by NumPy type; uint16 holds bf16 bit patterns.
ELEMENTS = {np.dtype(np.float32): runtime.F32, np.dtype(np.float16): runtime.F16, np.dtype(np.uint16): runtime.BF16}


class DeviceArray:
    """A device allocation made by the library (freed on :meth:`free`)."""

    def __init__(self, session: "Session", shape: tuple[int, ...], dtype=F32):
        self.session, self.shape, self.dtype = session, tuple(int(s) for s in shape), np.dtype(dtype)
        self.nbytes = int(math.prod(self.shape)) * self.dtype.itemsize
        self.ptr = session.ctx.malloc(max(1, self.nbytes))

    @property
    def size(self) -> int:
        return int(math.prod(self.shape))

    def free(self) -> None:
        if self.ptr:
            self.session.ctx.free(self.ptr)
            self.ptr = 0


def _element(dtype) -> int:
    code = ELEMENTS.get(np.dtype(dtype))
    if code is None:
        raise ValueError(f"expected float32, float16 or uint16 (bf16 bits), got {np.dtype(dtype)}")
    return code


def _heads(x: DeviceArray) -> runtime.Heads:
    if len(x.shape) != 3:
        raise ValueError(f"expected [tokens, heads, d], got shape {x.shape}")
    return runtime.heads(x.ptr, x.shape[1], x.shape[1] * x.shape[2], x.shape[2])


class PagedKV:
    """Keys and values in pages [pages, page_size, heads, d], and the workspace of the attention over them.

    All calls on one PagedKV share its workspace, so they go one after the other: the session's stream sees to
    that, and captured ones are replayed on one stream at a time.  Calls that overlap need
    ``runtime.Context.paged_attention`` with a workspace each."""

    def __init__(self, session: "Session", pages: int, page_size: int, heads: int, d: int, dtype=F32):
        self.session, self.dtype = session, np.dtype(dtype)
        shape, code = (pages, page_size, heads, d), _element(dtype)
        self.k, self.v = session.empty(shape, dtype), session.empty(shape, dtype)
        self.cache = runtime.paged_cache(self.k.ptr, self.v.ptr, code, pages, page_size, heads, d)
        self._workspaces: list[DeviceArray] = []

    def workspace(self, nbytes: int) -> DeviceArray:
        """At least `nbytes` of device memory, kept from call to call.  A larger one does not replace those before
        it until :meth:`free`: calls captured into a graph go on using theirs.  (Each is twice the last at least, so
        all of them are no more than twice the largest.)"""
        if not self._workspaces or self._workspaces[-1].nbytes < nbytes:
            last = self._workspaces[-1].nbytes if self._workspaces else 8
            self._workspaces.append(self.session.empty((max(2 * last, nbytes),), np.uint8))
        return self._workspaces[-1]

    def free(self) -> None:
        """Free keys, values and workspaces; graphs with calls on them must not be replayed any more."""
        for array in (self.k, self.v, *self._workspaces):
            array.free()


class Session:
    """One device, one context, one stream (the legacy default stream unless given)."""

    def __init__(self, device: int = 0, stream: int = 0):
        self.ctx = runtime.Context(device)
        self.stream = stream
        self._pinned: list[int] = []

    def close(self) -> None:
        for ptr in self._pinned:
            self.ctx.host_free(ptr)
        self._pinned.clear()
        self.ctx.close()

    def __enter__(self) -> "Session":
        return self

    def __exit__(self, *exc) -> None:
        self.close()

    # --- memory --------------------------------------------------------------
    def empty(self, shape, dtype=F32) -> DeviceArray:
        return DeviceArray(self, tuple(shape), dtype)

    def pinned(self, shape, dtype=F32) -> np.ndarray:
        """A NumPy array backed by page-locked host memory (lives with the session)."""
        dtype = np.dtype(dtype)
        count = int(math.prod(shape))
        ptr = self.ctx.host_alloc(max(1, count * dtype.itemsize))
        self._pinned.append(ptr)
        raw = (C.c_uint8 * max(1, count * dtype.itemsize)).from_address(ptr)
        return np.frombuffer(raw, dtype=dtype, count=count).reshape(shape)

    def upload(self, host: np.ndarray, out: DeviceArray | None = None) -> DeviceArray:
        host = np.ascontiguousarray(host)
        out = out or self.empty(host.shape, host.dtype)
        if out.nbytes != host.nbytes:
            raise ValueError("upload: size mismatch")
        if host.nbytes:
            self.ctx.htod(out.ptr, host.ctypes.data, host.nbytes, self.stream)
        return out

    def download(self, dev: DeviceArray, out: np.ndarray | None = None) -> np.ndarray:
        out = np.empty(dev.shape, dev.dtype) if out is None else out
        if not out.flags.c_contiguous or out.nbytes != dev.nbytes:
            raise ValueError("download: destination must be contiguous and the same size")
        if dev.nbytes:
            self.ctx.dtoh(out.ctypes.data, dev.ptr, dev.nbytes, self.stream)
        return out

    def sync(self) -> None:
        self.ctx.sync(self.stream)

    # --- kernels on device arrays ---------------------------------------------
    def gemm(self, a: DeviceArray, b: DeviceArray, c: DeviceArray, *, b_layout: str = "kn",
             bias: DeviceArray | None = None, relu: bool = False) -> None:
        m, k = a.shape
        n = b.shape[1] if b_layout == "kn" else b.shape[0]
        if c.shape != (m, n):
            raise ValueError(f"gemm: output shape {c.shape} != {(m, n)}")
        self.ctx.gemm(a.ptr, b.ptr, c.ptr, m, n, k, b_layout=runtime.B_KN if b_layout == "kn" else runtime.B_NK,
                      bias=bias.ptr if bias is not None else 0, relu=relu, stream=self.stream)

    def row_softmax(self, x: DeviceArray, y: DeviceArray) -> None:
        rows, cols = x.shape
        self.ctx.row_softmax(x.ptr, y.ptr, rows, cols, stream=self.stream)

    def pointwise(self, program, inputs: list[DeviceArray], out: DeviceArray) -> None:
        self.ctx.pointwise(program, [t.ptr for t in inputs], out.ptr, out.size, stream=self.stream)

    # --- serving: rotary positions, paged cache, drafted tokens -------------------
    # Arrays are [tokens, heads, d] of float32, float16 or uint16 (bf16 bits);
    # first, lengths, table (int32) and positions (int64) are device arrays too.
    def rotary(self, rope: runtime.Rope, pairs: list[tuple[DeviceArray, DeviceArray]], positions: DeviceArray, *,
               transpose: bool = False) -> None:
        """y = rotary(x) for each (x, y); ``transpose`` gives the inputs' gradients from the outputs'."""
        if not pairs:
            raise ValueError("rotary: no tensors")
        tokens, _, d = pairs[0][0].shape
        if positions.shape != (tokens,) or positions.dtype != np.int64:
            raise ValueError("rotary: positions must be int64, one for each token")
        for x, y in pairs:
            if x.shape != y.shape or x.shape[0] != tokens or x.shape[2] != d or {x.dtype, y.dtype} != {pairs[0][0].dtype}:
                raise ValueError(f"rotary: {x.shape} {x.dtype} to {y.shape} {y.dtype}")
        self.ctx.rotary(rope, _element(pairs[0][0].dtype), [(_heads(x), _heads(y)) for x, y in pairs], positions.ptr, tokens,
                        d, transpose=transpose, stream=self.stream)

    def paged_kv(self, pages: int, page_size: int, heads: int, d: int, dtype=F32) -> PagedKV:
        return PagedKV(self, pages, page_size, heads, d, dtype)

    @staticmethod
    def paged_batch(first: DeviceArray, lengths: DeviceArray, table: DeviceArray, tokens: int, *, max_new: int,
                    max_len: int, prefix_table: DeviceArray | None = None, prefix_len: int = 0) -> runtime.PagedBatch:
        """The sequences of a call: first [n + 1], lengths [n], table [n, pages], all int32."""
        n, width = table.shape
        arrays = [first, lengths, table] + ([prefix_table] if prefix_table is not None else [])
        if first.shape != (n + 1,) or lengths.shape != (n,) or any(x.dtype != np.int32 for x in arrays):
            raise ValueError("paged_batch: first [n + 1], lengths [n] and table [n, pages] must be int32")
        batch = runtime.paged_batch(n, tokens, first.ptr, lengths.ptr, table.ptr, width, max_new=max_new, max_len=max_len,
                                    prefix_len=prefix_len, prefix_table=prefix_table.ptr if prefix_table is not None else 0)
        batch.prefix_pages = prefix_table.size if prefix_table is not None else 0
        return batch

    def paged_append(self, kv: PagedKV, batch: runtime.PagedBatch, k: DeviceArray, v: DeviceArray, *,
                     q: DeviceArray | None = None, q_out: DeviceArray | None = None,
                     rope: runtime.Rope | None = None) -> None:
        for x in (k, v, q, q_out):
            if x is not None and (x.dtype != kv.dtype or len(x.shape) != 3 or (x.shape[0], x.shape[2]) != (batch.tokens, kv.cache.d)):
                raise ValueError(f"paged_append: {x.shape} {x.dtype} for {batch.tokens} tokens of a {kv.dtype} cache")
        self.ctx.paged_append(kv.cache, batch, _heads(k), _heads(v), q=None if q is None else _heads(q),
                              q_out=None if q_out is None else _heads(q_out), rope=rope, stream=self.stream)

    def paged_attention(self, kv: PagedKV, batch: runtime.PagedBatch, q: DeviceArray, o: DeviceArray, *,
                        scale: float | None = None) -> None:
        for x in (q, o):
            if x.dtype != kv.dtype or len(x.shape) != 3 or (x.shape[0], x.shape[2]) != (batch.tokens, kv.cache.d):
                raise ValueError(f"paged_attention: {x.shape} {x.dtype} for {batch.tokens} tokens of a {kv.dtype} cache")
        # the kernels read the prefix's table up to its last token (a batch made by runtime.paged_batch says nothing of it)
        pages = getattr(batch, "prefix_pages", None)
        if pages is not None and batch.prefix_len > pages * kv.cache.page_size:
            raise ValueError(f"paged_attention: a prefix of {batch.prefix_len} tokens in {pages} pages of {kv.cache.page_size}")
        nbytes = self.ctx.paged_attention_workspace(kv.cache, batch, q.shape[1])
        self.ctx.paged_attention(kv.cache, batch, _heads(q), _heads(o), kv.workspace(nbytes).ptr if nbytes else 0, nbytes,
                                 scale=scale, stream=self.stream)

    def verify_drafts(self, target: DeviceArray, drafted: DeviceArray, u_accept: DeviceArray, u_sample: DeviceArray,
                      accepted: DeviceArray, tokens: DeviceArray, *, draft: DeviceArray | None = None,
                      counts: DeviceArray | None = None) -> None:
        """target [batch, drafts + 1, vocab], draft [batch, drafts, vocab] float32; drafted [batch, drafts], accepted
        [batch], tokens [batch, drafts + 1] int32; u_accept [batch, drafts], u_sample [batch] float32."""
        batch, rows, vocab = target.shape
        want = [(target, F32, (batch, rows, vocab)), (drafted, np.int32, (batch, rows - 1)), (u_accept, F32, (batch, rows - 1)),
                (u_sample, F32, (batch,)), (accepted, np.int32, (batch,)), (tokens, np.int32, (batch, rows)),
                (draft, F32, (batch, rows - 1, vocab)), (counts, np.int32, (batch,))]
        for x, dtype, shape in want:
            if x is not None and (x.dtype != dtype or x.shape != shape):
                raise ValueError(f"verify_drafts: {x.shape} {x.dtype} where {shape} {np.dtype(dtype)} is wanted")
        self.ctx.verify_drafts(target.ptr, drafted.ptr, u_accept.ptr, u_sample.ptr, accepted.ptr, tokens.ptr, batch, rows - 1,
                               vocab, draft=draft.ptr if draft is not None else 0,
                               counts=counts.ptr if counts is not None else 0, stream=self.stream)

    # --- end to end from host arrays --------------------------------------------
    # One library call per operation: the inputs are copied in slab by slab on
    # a copy stream, each slab computes as soon as it has landed, and finished
    # output slabs are copied out on a second copy stream (b2k_*_host).  The
    # calls are asynchronous: `out` is complete after :meth:`sync`.  Host
    # arrays from :meth:`pinned` give full copy/compute overlap.
    @staticmethod
    def _host_in(x: np.ndarray) -> np.ndarray:
        x = np.asarray(x)
        if x.dtype != F32 or not x.flags.c_contiguous:
            raise ValueError("host inputs must be C-contiguous float32 arrays")
        return x

    @staticmethod
    def _host_out(out: np.ndarray | None, shape: tuple) -> np.ndarray:
        if out is None:
            return np.empty(shape, F32)
        if out.dtype != F32 or not out.flags.c_contiguous or out.shape != tuple(shape):
            raise ValueError(f"output must be a C-contiguous float32 array of shape {tuple(shape)}")
        return out

    def gemm_host(self, a: np.ndarray, b: np.ndarray, out: np.ndarray | None = None, *, b_layout: str = "kn",
                  bias: np.ndarray | None = None, relu: bool = False) -> np.ndarray:
        a, b = self._host_in(a), self._host_in(b)
        m, k = a.shape
        n = b.shape[1] if b_layout == "kn" else b.shape[0]
        out = self._host_out(out, (m, n))
        bias = self._host_in(bias) if bias is not None else None
        self.ctx.gemm_host(a.ctypes.data, b.ctypes.data, out.ctypes.data, m, n, k,
                           b_layout=runtime.B_KN if b_layout == "kn" else runtime.B_NK,
                           bias=bias.ctypes.data if bias is not None else 0, relu=relu, stream=self.stream)
        return out

    def row_softmax_host(self, x: np.ndarray, out: np.ndarray | None = None) -> np.ndarray:
        x = self._host_in(x)
        rows, cols = x.shape
        out = self._host_out(out, x.shape)
        self.ctx.row_softmax_host(x.ctypes.data, out.ctypes.data, rows, cols, stream=self.stream)
        return out

    def pointwise_host(self, program, inputs: list[np.ndarray], out: np.ndarray) -> np.ndarray:
        inputs = [self._host_in(t) for t in inputs]
        out = self._host_out(out, out.shape)
        self.ctx.pointwise_host(program, [t.ctypes.data for t in inputs], out.ctypes.data, out.size,
                                stream=self.stream)
        return out

    def attention_host(self, q: np.ndarray, k: np.ndarray, v: np.ndarray, out: np.ndarray | None = None, *,
                       scale: float | None = None, k_layout: str = "sd") -> np.ndarray:
        """q [bh, s_q, d], k [bh, s_kv, d] (or [bh, d, s_kv] with k_layout "ds"), v [bh, s_kv, dv]."""
        q, k, v = self._host_in(q), self._host_in(k), self._host_in(v)
        bh, s_q, d = q.shape
        s_kv, dv = v.shape[1], v.shape[2]
        out = self._host_out(out, (bh, s_q, dv))
        self.ctx.attention_host(q.ctypes.data, k.ctypes.data, v.ctypes.data, out.ctypes.data, bh, s_q, s_kv, d, dv,
                                scale=scale, k_layout=runtime.K_SD if k_layout == "sd" else runtime.K_DS,
                                stream=self.stream)
        return out
