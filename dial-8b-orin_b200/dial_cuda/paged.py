"""Serving over a paged KV cache: the post-QKV step, the attention of a chunk of
new tokens, reading rows back, and the verification of drafted tokens.

A serving loop keeps one `PagedKVCache` per layer and, per step, one `PagedBatch`
(which chunk of tokens belongs to which sequence, and where its rows are):

    cache = PagedKVCache(n_pages=4096, n_kv_heads=8, page_size=64, dtype=torch.bfloat16, quantized=True)
    batch = PagedBatch(block_table, kv_len, q_start, max_q=5, max_kv=8192)
    q = cache.append(qkv, batch, cos, sin, positions, q_norm=qn, k_norm=kn, sections=(24, 20, 20))
    out = cache.attention(q, batch)
    ids, count, logprob = verify_drafts(logits, ids, batch.q_start, temperature, accept_u, sample_u)

Nothing here copies to the host or waits: lengths and page tables stay on the
device, and every call can be captured into a CUDA graph, whose replays read the
tensors' contents of that time.  Calls run on the current stream of the tensors'
device.  A page id, a length or a position outside its array is reported by
`dial_device_error` (see include/dial_cuda.h for what each call then does).
The kernels are in libdial_cuda.so; there is no CPU path.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Sequence, Tuple

from . import _torch, check, dtype_code, lib

KV_INT8 = 3
_byref = ctypes.byref


class _PagedKv(ctypes.Structure):
    _fields_ = [("k_pages", ctypes.c_void_p), ("v_pages", ctypes.c_void_p),
                ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("format", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("page_size", ctypes.c_int32),
                ("n_pages", ctypes.c_int64)]


class _PagedBatch(ctypes.Structure):
    _fields_ = [("block_table", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("q_start", ctypes.c_void_p), ("n_seqs", ctypes.c_int32),
                ("max_pages", ctypes.c_int64), ("max_q", ctypes.c_int64), ("max_kv", ctypes.c_int64)]


class _RopeAxes(ctypes.Structure):
    _fields_ = [("n_axes", ctypes.c_int32), ("section", ctypes.c_int32 * 4), ("interleaved", ctypes.c_int32)]


def _tensor(t, name: str, dtype, shape: tuple, index: int):
    """t: a contiguous `dtype` tensor of `shape` on CUDA device `index`."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous():
        return
    if not t.is_cuda:
        raise RuntimeError(f"{name}: dial_cuda ops take CUDA tensors; there is no CPU path")
    if not t.is_contiguous():
        raise RuntimeError(f"{name}: dial_cuda ops take contiguous tensors")
    if t.dtype is not dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {shape}, got {tuple(t.shape)}")
    raise RuntimeError(f"{name}: on {t.device}, the others on cuda:{index}")


_fns = {}
_cuda = None  # torch._C's current device and raw stream


def _bind_cuda():
    """(current device, raw current stream of a device), as bare functions where torch has
    them: a Stream object costs 3 us a call, as much as a launch."""
    global _cuda
    torch = _torch()
    dev = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
    torch.cuda.current_device()  # (initialises CUDA)
    _cuda = dev, raw
    return _cuda


def _call(name: str, index: int, *args):
    """A library call on the current stream of CUDA device `index` (made current for the call)."""
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(lib(), name)
    dev, raw = _cuda or _bind_cuda()
    if index == dev():
        status = fn(*args, raw(index))
    else:
        with _torch().cuda.device(index):
            status = fn(*args, raw(index))
    if status:
        check(status, name)


class PagedBatch:
    """Chunks of new tokens of several sequences over a paged cache.

    block_table int32 [n_seqs, max_pages], kv_len int32 [n_seqs] (cache rows, the new
    tokens' counted), q_start int32 [n_seqs + 1] (token rows of each chunk).  max_q and
    max_kv are host-side bounds of a chunk and of kv_len (the largest possible by
    default); a chunk must not pass max_q, max_kv only sizes the work split.  Give max_q
    where chunks are short: it picks the attention kernel, and without it a batch of
    single tokens runs as one of chunks (32 over 2049 int8 rows: 88 us instead of 33).
    The tensors may be rewritten in place between calls (the object keeps them alive);
    other tensors or bounds take a new object."""

    def __init__(self, block_table, kv_len, q_start, max_q: Optional[int] = None, max_kv: Optional[int] = None):
        torch = _torch()
        if block_table.dim() != 2 or 0 in block_table.shape:
            raise ValueError(f"block_table must be [n_seqs, max_pages], got {tuple(block_table.shape)}")
        n, pages = block_table.shape
        index = max(block_table.get_device(), 0)
        _tensor(block_table, "block_table", torch.int32, (n, pages), index)
        _tensor(kv_len, "kv_len", torch.int32, (n,), index)
        _tensor(q_start, "q_start", torch.int32, (n + 1,), index)
        for name, v in (("max_q", max_q), ("max_kv", max_kv)):
            if v is not None and v <= 0:
                raise ValueError(f"{name} must be positive (got {v})")
        self.block_table, self.kv_len, self.q_start, self._index = block_table, kv_len, q_start, index
        self.n_seqs, self.max_pages, self.max_q, self.max_kv = n, pages, max_q, max_kv
        self._c = {}

    def _struct(self, page_size: int):
        c = self._c.get(page_size)
        if c is None:
            cap = self.max_pages * page_size
            c = self._c[page_size] = _byref(_PagedBatch(
                self.block_table.data_ptr(), self.kv_len.data_ptr(), self.q_start.data_ptr(), self.n_seqs,
                self.max_pages, self.max_q or (1 << 31) - 1, min(self.max_kv or cap, cap)))
        return c


class PagedKVCache:
    """Keys and values of one layer in pages [n_pages, n_kv_heads, page_size, 128], in the
    activations' type or (`quantized`) as int8 codes with an f32 scale per row."""

    def __init__(self, n_pages: int, n_kv_heads: int, page_size: int = 64, dtype=None, quantized: bool = False,
                 device=None):
        torch = _torch()
        dtype = dtype or torch.float16
        device = torch.device(device if device is not None else "cuda")
        shape = (n_pages, n_kv_heads, page_size, 128)
        pages = [torch.zeros(shape, dtype=torch.int8 if quantized else dtype, device=device) for _ in range(2)]
        scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)] if quantized else [None] * 2
        self._init(*pages, *scales)

    @classmethod
    def from_tensors(cls, k_pages, v_pages, k_scale=None, v_scale=None) -> "PagedKVCache":
        """A cache over existing pages (16-bit, or int8 with their scales)."""
        self = cls.__new__(cls)
        self._init(k_pages, v_pages, k_scale, v_scale)
        return self

    def _init(self, k, v, ks, vs):
        torch = _torch()
        if k.dim() != 4 or k.shape[3] != 128:
            raise ValueError(f"pages must be [n_pages, n_kv_heads, page_size, 128], got {tuple(k.shape)}")
        if k.shape[2] not in (16, 32, 64, 128, 256):
            raise ValueError(f"page_size must be 16, 32, 64, 128 or 256, got {k.shape[2]}")
        if 0 in k.shape:
            raise ValueError(f"pages must not be empty, got {tuple(k.shape)}")
        if k.dtype not in (torch.float16, torch.bfloat16, torch.int8):
            raise TypeError(f"pages must be f16, bf16 or int8, got {k.dtype}")
        self.quantized = k.dtype == torch.int8
        if self.quantized != (ks is not None) or self.quantized != (vs is not None):
            raise ValueError("int8 pages, and only they, have k_scale and v_scale")
        index = max(k.get_device(), 0)
        _tensor(k, "k_pages", k.dtype, k.shape, index)
        _tensor(v, "v_pages", k.dtype, k.shape, index)
        for name, s in (("k_scale", ks), ("v_scale", vs)):
            if s is not None:
                _tensor(s, name, torch.float32, k.shape[:3], index)
        self.k_pages, self.v_pages, self.k_scale, self.v_scale = k, v, ks, vs
        self.n_pages, self.n_kv_heads, self.page_size, _ = k.shape
        self.device, self._index = k.device, index
        self._codes = {torch.float16: 1, torch.bfloat16: 2} if self.quantized else {k.dtype: dtype_code(k.dtype)}
        self._c = _byref(_PagedKv(k.data_ptr(), v.data_ptr(), ks.data_ptr() if ks is not None else None,
                                  vs.data_ptr() if vs is not None else None,
                                  KV_INT8 if self.quantized else dtype_code(k.dtype), self.n_kv_heads, 128,
                                  self.page_size, self.n_pages))

    @property
    def bytes(self) -> int:
        b = 2 * self.k_pages.numel() * self.k_pages.element_size()
        return b + (2 * self.k_scale.numel() * 4 if self.quantized else 0)

    def _act(self, t, name: str) -> int:
        """The code of an activation tensor's type."""
        code = self._codes.get(t.dtype)
        if code is None:
            raise TypeError(f"{name}: expected {' or '.join(map(str, self._codes))}, got {t.dtype}")
        return code

    def _batch(self, batch: PagedBatch):
        if batch._index != self._index:
            raise RuntimeError(f"batch: on cuda:{batch._index}, the cache on cuda:{self._index}")
        return batch._c.get(self.page_size) or batch._struct(self.page_size)

    def append(self, qkv, batch: PagedBatch, cos, sin, positions, q_norm=None, k_norm=None, eps: float = 1e-6,
               sections: Sequence[int] = (64,), interleaved: bool = True, out=None):
        """Norm, rotary positions and the cache write of a chunk's fused qkv
        [T, (Hq + 2 Hkv) * 128]; returns q [T, Hq, 128].

        cos, sin: f32 tables [rows, 64] (`rope_tables`); positions int32 [T] or [n_axes, T],
        one axis per entry of `sections` (pairs of each axis, summing to 64; interleaved as
        Qwen3-VL, or consecutive).  q_norm, k_norm: [128] weights, or neither."""
        torch = _torch()
        dt, index, n = self._act(qkv, "qkv"), self._index, len(sections)
        T, hq = qkv.shape[0], qkv.shape[1] // 128 - 2 * self.n_kv_heads if qkv.dim() == 2 else 0
        if hq <= 0 or qkv.shape[1] % 128:
            raise ValueError(f"qkv must be [T, (Hq + 2 * {self.n_kv_heads}) * 128], got {tuple(qkv.shape)}")
        _tensor(qkv, "qkv", qkv.dtype, (T, (hq + 2 * self.n_kv_heads) * 128), index)
        axes = _axes(tuple(sections), bool(interleaved))
        _tensor(positions, "positions", torch.int32, (T,) if n == 1 and positions.dim() == 1 else (n, T), index)
        rows = cos.shape[0]
        _tensor(cos, "cos", torch.float32, (rows, 64), index)
        _tensor(sin, "sin", torch.float32, (rows, 64), index)
        if (q_norm is None) != (k_norm is None):
            raise ValueError("q_norm and k_norm go together")
        if q_norm is not None:
            _tensor(q_norm, "q_norm", qkv.dtype, (128,), index)
            _tensor(k_norm, "k_norm", qkv.dtype, (128,), index)
        if out is None:
            out = torch.empty((T, hq, 128), dtype=qkv.dtype, device=self.device)
        else:
            _tensor(out, "out", qkv.dtype, (T, hq, 128), index)
        if T:
            _call("dial_paged_kv_append", index, qkv.data_ptr(), q_norm.data_ptr() if q_norm is not None else None,
                  k_norm.data_ptr() if k_norm is not None else None, cos.data_ptr(), sin.data_ptr(), rows,
                  positions.data_ptr(), axes, self._c, self._batch(batch), out.data_ptr(), dt, T, hq, eps)
        return out

    def attention(self, q, batch: PagedBatch, scale: Optional[float] = None, out=None):
        """Attention of the batch's tokens, q [T, Hq, 128] -> [T, Hq, 128]: each attends its
        sequence's rows up to its own.  scale: 1/sqrt(128) by default."""
        dt, shape, index = self._act(q, "q"), q.shape, self._index
        if len(shape) != 3 or shape[2] != 128:
            raise ValueError(f"q must be [T, Hq, 128], got {tuple(shape)}")
        _tensor(q, "q", q.dtype, shape, index)
        if out is None:
            out = _torch().empty_like(q)
        else:
            _tensor(out, "out", q.dtype, shape, index)
        if shape[0]:
            _call("dial_paged_attention", index, q.data_ptr(), self._c, self._batch(batch), out.data_ptr(), dt, shape[0],
                  shape[1], 0.08838834764831845 if scale is None else scale)
        return out

    def read(self, batch: PagedBatch, tokens: Optional[int] = None, dtype=None, out=None) -> Tuple:
        """The batch's rows back from their pages: (k, v), each [T, Hkv, 128], either new
        (`tokens` rows in `dtype`: the pages' own, or f16 for int8) or `out`."""
        torch = _torch()
        if out is None:
            if tokens is None:
                raise ValueError("give the number of token rows, or out")
            dtype = dtype or (torch.float16 if self.quantized else self.k_pages.dtype)
            out = tuple(torch.empty((tokens, self.n_kv_heads, 128), dtype=dtype, device=self.device) for _ in range(2))
        k, v = out
        dt, shape, index = self._act(k, "out[0]"), k.shape, self._index
        if len(shape) != 3 or shape[1:] != (self.n_kv_heads, 128):
            raise ValueError(f"out must be [T, {self.n_kv_heads}, 128], got {tuple(shape)}")
        _tensor(k, "out[0]", k.dtype, shape, index)
        _tensor(v, "out[1]", k.dtype, shape, index)
        if shape[0]:
            _call("dial_paged_kv_read", index, self._c, self._batch(batch), k.data_ptr(), v.data_ptr(), dt, shape[0])
        return k, v


_AXES = {}


def _axes(sections: tuple, interleaved: bool):
    """The dial_rope_axes of these sections, made once."""
    a = _AXES.get((sections, interleaved))
    if a is None:
        if not 1 <= len(sections) <= 4:
            raise ValueError(f"1 to 4 position axes, got {len(sections)}")
        a = _byref(_RopeAxes(len(sections), (ctypes.c_int32 * 4)(*sections), int(interleaved)))
        if len(_AXES) < 64:
            _AXES[sections, interleaved] = a
    return a


def rope_tables(rows: int, theta: float, device=None):
    """f32 rotary tables (cos, sin), each [rows, 64], for `PagedKVCache.append`."""
    torch = _torch()
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    cos = torch.empty((rows, 64), dtype=torch.float32, device=device)
    sin = torch.empty_like(cos)
    _call("dial_rope_tables", cos.get_device(), cos.data_ptr(), sin.data_ptr(), dtype_code(torch.float32), rows, 128, theta)
    return cos, sin


@functools.lru_cache(maxsize=256)
def _verify_bytes(rows: int, vocab: int) -> int:
    return lib().dial_verify_drafts_workspace_bytes(rows, vocab)


def verify_drafts(logits, ids, q_start, temperature, accept_u, sample_u, draft_probs=None,
                  max_q: Optional[int] = None):
    """Verifies drafted tokens against the target's probabilities; with one row a sequence
    it draws the next token.

    logits [R, V] (f32, f16 or bf16) of the chunk ids int32 [R] (per sequence its last
    accepted token, then the drafts), rows q_start int32 [n_seqs + 1]; temperature f32
    [n_seqs] (0: greedy); accept_u f32 [R] and sample_u f32 [n_seqs] uniform in [0, 1);
    draft_probs f32 [R, V], row r the distribution that ids[r + 1] was drawn from (None: the
    drafts were certain).  Returns (out_ids int32 [R], n_out int32 [n_seqs], logprob f32
    [R]): the accepted drafts and the drawn token of each sequence, -1 behind them.  Rows
    from q_start[n_seqs] on belong to no sequence and are not written."""
    torch = _torch()
    index = max(logits.get_device(), 0)
    if logits.dim() != 2 or 0 in logits.shape:
        raise ValueError(f"logits must be [R, V], got {tuple(logits.shape)}")
    R, V = logits.shape
    n = q_start.numel() - 1
    if n < 1:
        raise ValueError("q_start must hold n_seqs + 1 values")
    f32, i32 = torch.float32, torch.int32
    _tensor(logits, "logits", logits.dtype, (R, V), index)
    _tensor(ids, "ids", i32, (R,), index)
    _tensor(q_start, "q_start", i32, (n + 1,), index)
    _tensor(temperature, "temperature", f32, (n,), index)
    _tensor(accept_u, "accept_u", f32, (R,), index)
    _tensor(sample_u, "sample_u", f32, (n,), index)
    if draft_probs is not None:
        _tensor(draft_probs, "draft_probs", f32, (R, V), index)
    # one allocation: tokens, counts, log-probabilities, workspace
    need = _verify_bytes(R, V)
    at = (2 * R + n + 3) // 4 * 4
    buf = torch.empty(at + need // 4, dtype=i32, device=logits.device)
    out, count, logp, _ = buf.split_with_sizes((R, n, R, at + need // 4 - 2 * R - n))
    p = buf.data_ptr()
    _call("dial_verify_drafts", index, logits.data_ptr(), dtype_code(logits.dtype), ids.data_ptr(),
          draft_probs.data_ptr() if draft_probs is not None else None, q_start.data_ptr(), n,
          temperature.data_ptr(), accept_u.data_ptr(), sample_u.data_ptr(), p, p + 4 * R, p + 4 * (R + n),
          R, V, max_q or R, p + 4 * at, need)
    return out, count, logp.view(f32)
