"""Prompt attention, the 4-bit key/value cache with its step attention, and
eviction from it (include/rvq_b200.h: ``rvq_prompt_attention``,
``rvq_cache4_write`` / ``_read`` / ``_attention`` / ``_evict``).

As in ``rvq_b200.step``, each ``*Op`` resolves its pointers once and
``launch()`` queues its kernels on the current stream of its tensors' device,
so launches can be captured in a CUDA graph.  The tensors an op was built
from must outlive it and keep their storage; an op with a workspace of its own
(``PromptAttentionOp``, ``Cache4AttentionOp``) runs one launch at
a time and outlives its launches and graphs, or, launched on the stream it was
built on, may be dropped with the work still queued there (what the stream
allocates later comes after it).
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _native
from .step import RvqVec

_HALF = (torch.bfloat16, torch.float16)


class RvqPromptAttnArgs(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("lse", ctypes.c_void_p), ("cu_q", ctypes.c_void_p), ("cu_k", ctypes.c_void_p),
                ("tokens", ctypes.c_int64), ("keys", ctypes.c_int64),
                ("q_stride", ctypes.c_int64 * 2), ("k_stride", ctypes.c_int64 * 2),
                ("v_stride", ctypes.c_int64 * 2), ("out_stride", ctypes.c_int64 * 2),
                ("n_seq", ctypes.c_int32), ("n_heads", ctypes.c_int32), ("n_kv", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("scaling", ctypes.c_float), ("causal", ctypes.c_int32),
                ("kind", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class RvqCache4(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("n_seq", ctypes.c_int32), ("n_kv", ctypes.c_int32),
                ("max_len", ctypes.c_int32), ("head_dim", ctypes.c_int32)]


class RvqCache4RowsArgs(ctypes.Structure):
    _fields_ = [("cache", RvqCache4), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("cu", ctypes.c_void_p),
                ("start", ctypes.c_void_p), ("tokens", ctypes.c_int64), ("k_stride", ctypes.c_int64 * 2),
                ("v_stride", ctypes.c_int64 * 2), ("kind", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class RvqCache4AttnArgs(ctypes.Structure):
    _fields_ = [("q", RvqVec), ("k", RvqVec), ("v", RvqVec), ("q_norm", ctypes.c_void_p), ("k_norm", ctypes.c_void_p),
                ("cos", ctypes.c_void_p), ("sin", ctypes.c_void_p), ("pos", ctypes.c_void_p), ("cache", RvqCache4),
                ("rows", ctypes.c_void_p), ("out", ctypes.c_void_p), ("weights", ctypes.c_void_p),
                ("n_heads", ctypes.c_int32), ("table_len", ctypes.c_int32),
                ("eps", ctypes.c_float), ("scaling", ctypes.c_float)]


class RvqCache4EvictArgs(ctypes.Structure):
    _fields_ = [("cache", RvqCache4), ("out", RvqCache4), ("weights", ctypes.c_void_p),
                ("out_weights", ctypes.c_void_p), ("rows", ctypes.c_void_p), ("new_rows", ctypes.c_void_p),
                ("kept", ctypes.c_void_p), ("keep", ctypes.c_int32), ("recent", ctypes.c_int32)]


_bound = False


def _lib():
    global _bound
    lib = _native.load()
    if not _bound:
        vp, i32, P = ctypes.c_void_p, ctypes.c_int, ctypes.POINTER
        lib.rvq_prompt_attention_workspace_size.restype = ctypes.c_size_t
        lib.rvq_prompt_attention_workspace_size.argtypes = [P(RvqPromptAttnArgs)]
        lib.rvq_prompt_attention.restype = i32
        lib.rvq_prompt_attention.argtypes = [P(RvqPromptAttnArgs), vp, ctypes.c_size_t, vp]
        lib.rvq_take_attention_timeout.restype = i32
        lib.rvq_take_attention_timeout.argtypes = []
        lib.rvq_cache4_record_bytes.restype = i32
        lib.rvq_cache4_record_bytes.argtypes = [i32]
        for name in ("rvq_cache4_write", "rvq_cache4_read"):
            getattr(lib, name).restype = i32
            getattr(lib, name).argtypes = [P(RvqCache4RowsArgs), vp]
        lib.rvq_cache4_attention_workspace_size.restype = ctypes.c_size_t
        lib.rvq_cache4_attention_workspace_size.argtypes = [P(RvqCache4AttnArgs)]
        lib.rvq_cache4_attention.restype = i32
        lib.rvq_cache4_attention.argtypes = [P(RvqCache4AttnArgs), vp, ctypes.c_size_t, vp]
        lib.rvq_cache4_evict.restype = i32
        lib.rvq_cache4_evict.argtypes = [P(RvqCache4EvictArgs), vp]
        _bound = True
    return lib


def record_bytes(head_dim: int) -> int:
    """Bytes of one cached token of one kv head (K and V)."""
    n = _lib().rvq_cache4_record_bytes(int(head_dim))
    if n == 0:
        raise NotImplementedError(f"the 4-bit cache holds heads of 64 or 128, not {head_dim}")
    return n


def take_timeout() -> bool:
    """Reads and clears the flag of a bounded attention wait that gave up; synchronises the device."""
    r = _lib().rvq_take_attention_timeout()
    if r < 0:
        _native.check(-r, "rvq_take_attention_timeout")
    return bool(r)


# -- argument checks: shapes and types first, the device last -----------------------------------------------------------
def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _heads3(t: torch.Tensor, name: str, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """A [tokens, heads, head_dim] tensor whose heads are adjacent elements at 16-byte steps."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim]")
    if t.dtype not in _HALF:
        raise NotImplementedError(f"{name} must be bf16 or fp16, not {t.dtype}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must have the type of the others ({dtype})")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"the head_dim elements of {name} must be adjacent")
    if t.data_ptr() % 16 or any(t.shape[d] > 1 and t.stride(d) % 8 for d in (0, 1)):
        raise ValueError(f"the heads of {name} must start at 16-byte steps")
    if any(t.stride(d) < 0 or (t.stride(d) == 0 and t.shape[d] > 1) for d in (0, 1)):
        raise ValueError(f"{name} must not repeat its rows (expanded dimension)")
    return t


def _strides(t: torch.Tensor):
    """Token and head strides; those of dimensions of one element, which torch leaves open, as for a packed tensor."""
    head = t.stride(1) if t.shape[1] > 1 else t.shape[2]
    return (ctypes.c_int64 * 2)(t.stride(0) if t.shape[0] > 1 else head * t.shape[1], head)


def _ints(t: torch.Tensor, n: int, dtype: torch.dtype, name: str) -> torch.Tensor:
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be {n} contiguous {dtype} values")
    return t


def _plain(t: torch.Tensor, shape, dtype: torch.dtype, name: str) -> torch.Tensor:
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")
    return t


def _span(t: torch.Tensor):
    """First byte and the one behind the last of a tensor's elements."""
    n, first = t.numel(), t.data_ptr()
    if n and not t.is_contiguous():
        n = 1 + sum((m - 1) * s for m, s in zip(t.shape, t.stride()))
    return first, first + n * t.element_size()


def _distinct(t: torch.Tensor, name: str) -> None:
    """Refuses a written [tokens, heads, head_dim] view whose rows share elements."""
    dims = sorted((t.stride(d), t.shape[d]) for d in (0, 1) if t.shape[d] > 1)
    end = t.shape[2]
    for stride, n in dims:
        if stride < end:
            raise ValueError(f"the rows of {name} must not overlap")
        end = stride * (n - 1) + end


def _interleaved(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [tokens, heads, head_dim] views of one buffer with the same strides share no element (columns of one
    packed projection, say)."""
    if a.dim() != 3 or b.dim() != 3 or a.stride() != b.stride() or a.dtype != b.dtype or a.shape[2] != b.shape[2]:
        return False
    off = (b.data_ptr() - a.data_ptr()) // a.element_size()
    (s0, d0), (s1, d1) = sorted(((a.stride(d), d) for d in (0, 1)), reverse=True)
    if max(a.shape[d1], b.shape[d1]) * s1 > s0:
        return False
    near = lambda rest, s, d: [i for i in range(-rest // s - 1, -rest // s + 2) if -a.shape[d] < i < b.shape[d]]
    return all(abs(off + i * s0 + j * s1) >= a.shape[2] for i in near(off, s0, d0) for j in near(off + i * s0, s1, d1))


def _in_gaps(view: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether the contiguous tensor ``t`` lies in the gaps of a [tokens, heads, head_dim] view."""
    if view.dim() != 3 or not t.is_contiguous():
        return False
    size = view.element_size()
    lo, hi = t.data_ptr() - view.data_ptr(), t.data_ptr() - view.data_ptr() + t.numel() * t.element_size()
    (s0, n0), (s1, n1) = sorted(((view.stride(d) * size, view.shape[d]) for d in (0, 1)), reverse=True)
    # for every place along the shorter stride: the last row that starts before t's end ends before t starts
    return all(j * s1 + min(n0 - 1, (hi - 1 - j * s1) // max(s0, 1)) * s0 + view.shape[2] * size <= lo
               for j in range(n1) if j * s1 < hi)


def _all_apart(written, read=()) -> None:
    """Refuses written (tensor, name) pairs that share memory with one another or with a read one; None: not there."""
    written, read = ([(*_span(t), t, n) for t, n in pairs if t is not None] for pairs in (written, read))
    for i, (a0, a1, a, an) in enumerate(written):
        for b0, b1, b, bn in written[i + 1:] + read:
            if a0 < b1 and b0 < a1 and not (_interleaved(a, b) or _in_gaps(a, b) or _in_gaps(b, a)):
                raise ValueError(f"{an} and {bn} must not overlap")


class _Op:
    """Device and stream of an op's launches."""

    def _on(self, *tensors) -> None:
        self._keep = [t for t in tensors if t is not None]
        dev = self._keep[0].device
        if any(not t.is_cuda for t in self._keep):
            raise ValueError("every tensor must be on a CUDA device")
        if any(t.device != dev for t in self._keep):
            raise ValueError("every tensor must be on the same device")
        self.device = dev

    def _workspace(self, size) -> int:
        """Allocates what ``self.args`` needs; its bytes."""
        with torch.cuda.device(self.device):
            n = size(ctypes.byref(self.args))
        self._ws = torch.empty(n, dtype=torch.uint8, device=self.device) if n else None
        return n

    def _bind(self, where: str, *args) -> None:
        """The C entry point and its arguments but the stream, resolved once."""
        self._where, self._fn, self._args = where, getattr(_lib(), where), args

    def launch(self) -> None:
        if torch.cuda.current_device() == self.device.index:
            rc = self._fn(*self._args, torch._C._cuda_getCurrentRawStream(self.device.index))
        else:
            with torch.cuda.device(self.device):
                rc = self._fn(*self._args, torch.cuda.current_stream().cuda_stream)
        if rc:
            where = self._where
            if rc == _native.RVQ_ERR_UNSUPPORTED:
                raise NotImplementedError(f"{where}: {_native.status_string(rc)}")
            if rc == _native.RVQ_ERR_INVALID:
                raise ValueError(f"{where}: {_native.status_string(rc)}")
            _native.check(rc, where)


class PromptAttentionOp(_Op):
    """``out = softmax(scaling q k^T, masked) v`` of whole prompts.

    ``q`` and ``out``: [tokens, n_heads, head_dim]; ``k``, ``v``: [keys, n_kv, head_dim], bf16 or fp16, any strides whose
    heads start at 16-byte steps (a slice of a packed q/k/v projection will do); ``n_kv`` divides ``n_heads``.
    ``cu_q`` / ``cu_k``: int32 [sequences + 1] offsets of packed sequences on the device (``cu_k`` None: the keys are
    packed as the queries); without them all tokens and all keys are one sequence.  ``causal``: the last query of a
    sequence sees all its keys, each one before it one key less (with more keys than queries the first keys are
    a past that every query sees).  ``lse``: fp32 [n_heads, tokens], gets log(sum(exp(scores))).
    Scores, softmax statistics and sums are fp32; the probabilities are rounded to q's type for the product with v.
    A query that sees no key gets zeros (lse -inf); rows outside every sequence are left as they were."""

    def __init__(self, q, k, v, out, *, scaling: float, causal: bool = True, cu_q: Optional[torch.Tensor] = None,
                 cu_k: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None):
        _heads3(q, "q")
        for t, name in ((k, "k"), (v, "v"), (out, "out")):
            _heads3(t, name, q.dtype)
        tokens, nh, hd = q.shape
        keys, nkv = k.shape[:2]
        if out.shape != q.shape:
            raise ValueError("out must have q's shape")
        _distinct(out, "out")
        if v.shape != k.shape or k.shape[2] != hd:
            raise ValueError("k and v must be [keys, n_kv, head_dim] with q's head_dim")
        if nkv < 1 or nh < 1 or nh % nkv:
            raise ValueError("n_kv must divide n_heads")
        if hd < 8 or hd % 8 or hd > 128:
            raise NotImplementedError("head_dim must be a multiple of 8, at most 128")
        if nh // nkv > 64:
            raise NotImplementedError("at most 64 query heads a kv head")
        if max(tokens, keys) > 2 ** 30:
            raise ValueError("at most 2^30 tokens")
        if cu_q is None:
            if cu_k is not None:
                raise ValueError("cu_k needs cu_q")
            n_seq = 1
        else:
            n_seq = cu_q.numel() - 1
            if n_seq < 1:
                raise ValueError("cu_q must hold sequences + 1 offsets")
            _ints(cu_q, n_seq + 1, torch.int32, "cu_q")
            if cu_k is not None:
                _ints(cu_k, n_seq + 1, torch.int32, "cu_k")
        if lse is not None:
            _plain(lse, (nh, tokens), torch.float32, "lse")
        _all_apart([(out, "out"), (lse, "lse")], [(q, "q"), (k, "k"), (v, "v"), (cu_q, "cu_q"), (cu_k, "cu_k")])
        self._on(q, k, v, out, cu_q, cu_k, lse)
        self.args = RvqPromptAttnArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(cu_q), _ptr(cu_k), tokens,
                                      keys, _strides(q), _strides(k), _strides(v), _strides(out), n_seq, nh, nkv, hd,
                                      float(scaling), int(bool(causal)), _native.kind_of(q), 0)
        n = self._workspace(_lib().rvq_prompt_attention_workspace_size)
        self._fresh = n > 0
        self._bind("rvq_prompt_attention", ctypes.byref(self.args), _ptr(self._ws), n)

    def launch(self) -> None:
        if self._fresh:
            # the workspace is zero-filled in front of its first call, on that call's stream (this one may not be the one the
            # op was built on); a capture only records that, so the first call outside of one does it again
            with torch.cuda.device(self.device), torch.inference_mode():      # it may have been built in that mode
                self._ws.zero_()
                self._fresh = torch.cuda.is_current_stream_capturing()
        super().launch()


class Cache4:
    """Keys and values of ``n_seq`` sequences (or layers) in 4 bits: ``data`` [n_seq, n_kv, max_len, record] bytes, a zero
    and a step for each 32 values; 5 head_dim / 4 bytes a token and kv head, against 4 head_dim in bf16."""

    def __init__(self, n_seq: int, n_kv: int, max_len: int, head_dim: int, device=None,
                 data: Optional[torch.Tensor] = None):
        if min(n_seq, n_kv, max_len) < 1 or max(n_seq, n_kv, max_len) > 2 ** 30:
            raise ValueError("n_seq, n_kv and max_len must be 1 to 2^30")
        shape = (n_seq, n_kv, max_len, record_bytes(head_dim))
        if data is None:
            data = torch.zeros(shape, dtype=torch.uint8, device=device)
        _plain(data, shape, torch.uint8, "data")
        if data.data_ptr() % 16:
            raise ValueError("data must be 16-byte aligned")
        self.data, self.n_seq, self.n_kv, self.max_len, self.head_dim = data, n_seq, n_kv, max_len, head_dim

    def seq(self, i: int) -> "Cache4":
        """Sequence (layer) ``i`` alone, on the same storage."""
        return Cache4(1, self.n_kv, self.max_len, self.head_dim, data=self.data[i:i + 1])

    def struct(self) -> RvqCache4:
        return RvqCache4(self.data.data_ptr(), self.n_seq, self.n_kv, self.max_len, self.head_dim)


class _Cache4RowsOp(_Op):
    name = ""

    def __init__(self, cache: Cache4, k: torch.Tensor, v: torch.Tensor, *, cu: Optional[torch.Tensor] = None,
                 start: Optional[torch.Tensor] = None):
        _heads3(k, "k")
        _heads3(v, "v", k.dtype)
        if k.shape != v.shape or k.shape[1] != cache.n_kv or k.shape[2] != cache.head_dim:
            raise ValueError("k and v must be [tokens, n_kv, head_dim] of the cache")
        if k.shape[0] > 2 ** 30:
            raise ValueError("at most 2^30 tokens")
        if cu is None and cache.n_seq != 1:
            raise ValueError("a cache of several sequences needs cu")
        if cu is not None:
            _ints(cu, cache.n_seq + 1, torch.int32, "cu")
        if start is not None:
            _ints(start, cache.n_seq, torch.int64, "start")
        rows, store, at = [(k, "k"), (v, "v")], [(cache.data, "the cache")], [(cu, "cu"), (start, "start")]
        if self.name == "rvq_cache4_read":
            _all_apart(rows, store + at)
            _distinct(k, "k")
            _distinct(v, "v")
        else:
            _all_apart(store, rows + at)
        self._on(k, v, cache.data, cu, start)
        self.args = RvqCache4RowsArgs(cache.struct(), _ptr(k), _ptr(v), _ptr(cu), _ptr(start), k.shape[0], _strides(k),
                                      _strides(v), _native.kind_of(k), 0)
        self._bind(self.name, ctypes.byref(self.args))


class Cache4WriteOp(_Cache4RowsOp):
    """Quantise ``k``, ``v`` [tokens, n_kv, head_dim] into the cache: token ``cu[b] + i`` becomes row ``start[b] + i`` of
    sequence ``b`` (``cu`` None: one sequence; ``start`` None: from row 0).  Rows outside the cache are dropped."""
    name = "rvq_cache4_write"


class Cache4ReadOp(_Cache4RowsOp):
    """The held values back as ``k``, ``v`` (the reverse of ``Cache4WriteOp``); rows outside the cache read as zeros."""
    name = "rvq_cache4_read"


def _operand(t: Optional[torch.Tensor], tiles: int, shape, name: str) -> RvqVec:
    """A contiguous bf16 / fp16 tensor, or fp32 partials [tiles, elements]."""
    if t is None:
        return RvqVec(None, 0, 0, 0)
    n = shape[0] * shape[1] * shape[2]
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.dtype == torch.float32:
        if tiles < 1 or t.numel() != tiles * n:
            raise ValueError(f"{name} must hold {tiles} partials of {n} elements")
        return RvqVec(t.data_ptr(), n, tiles, _native.RVQ_F32)
    if t.dtype not in _HALF:
        raise NotImplementedError(f"{name} must be bf16, fp16 or fp32 partials, not {t.dtype}")
    if tiles != 1 or t.numel() != n:
        raise ValueError(f"{name} must hold {n} elements (one tile)")
    return RvqVec(t.data_ptr(), n, 1, _native.kind_of(t))


class Cache4AttentionOp(_Op):
    """Attention of one new token of every sequence over the 4-bit cache, the token appended.

    ``q`` [n_seq, n_heads, head_dim], ``k`` / ``v`` [n_seq, n_kv, head_dim] (or both None: attend only): bf16, fp16 or
    the fp32 tile partials of a projection (``q_tiles`` / ``kv_tiles``).  ``rows``: int64 [n_seq] on the device, live rows
    of each sequence before the call; the token goes to row ``rows[b]`` and ``rows`` is left as it is (a replayed
    launch does the same again).  A sequence with ``rows[b] < 0`` is skipped.  ``out`` [n_seq, n_heads, head_dim]
    (any shape of that many elements): bf16, or fp16 for fp16 operands.
    ``q_norm`` / ``k_norm`` (bf16 [head_dim]) and ``cos`` / ``sin`` (bf16 [positions, head_dim]) with ``pos`` (int64
    [n_seq]): per-head RMSNorm and rotary embedding of q and k first, as ``AttentionOp`` does them.
    ``weights``: fp32 [n_seq, n_kv, max_len], gets the softmax weight of every attended row, summed over the query
    heads of its kv head, added (the new row's: set).
    Scores, softmax statistics and sums are fp32; a weight times a record's step keeps 16 bits for the product with the codes."""

    def __init__(self, q, k, v, cache: Cache4, rows: torch.Tensor, out: torch.Tensor, *, scaling: float,
                 n_heads: Optional[int] = None, weights: Optional[torch.Tensor] = None, q_norm=None, k_norm=None,
                 cos=None, sin=None, pos: Optional[torch.Tensor] = None, eps: float = 1e-6, q_tiles: int = 1,
                 kv_tiles: int = 1):
        n, nkv, hd = cache.n_seq, cache.n_kv, cache.head_dim
        if n_heads is None:
            if q.dim() != 3:
                raise ValueError("q must be [n_seq, n_heads, head_dim], or n_heads given")
            n_heads = q.shape[1]
        if n_heads < 1 or n_heads % nkv:
            raise ValueError("n_kv must divide n_heads")
        if n_heads // nkv > 64:
            raise NotImplementedError("at most 64 query heads a kv head")
        if (k is None) != (v is None):
            raise ValueError("k and v are given together")
        qv = _operand(q, q_tiles, (n, n_heads, hd), "q")
        kv_, vv = (_operand(t, kv_tiles, (n, nkv, hd), name) for t, name in ((k, "k"), (v, "v")))
        if k is not None and not q.dtype == k.dtype == v.dtype:
            raise ValueError("q, k and v must have the same type")
        if (q_norm is None) != (k_norm is None) or len({t is None for t in (cos, sin, pos)}) != 1:
            raise ValueError("q_norm comes with k_norm, cos with sin and pos")
        if q.dtype == torch.float16 and (q_norm is not None or cos is not None):
            raise NotImplementedError("norm and rotation compute in bf16")
        table = 0
        for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
            if t is not None:
                _plain(t, (hd,), torch.bfloat16, name)
        if cos is not None:
            table = int(cos.shape[0])
            if table < 1:
                raise ValueError("cos and sin must hold positions")
            _plain(cos, (table, hd), torch.bfloat16, "cos")
            _plain(sin, (table, hd), torch.bfloat16, "sin")
            _ints(pos, n, torch.int64, "pos")
        _ints(rows, n, torch.int64, "rows")
        if out.numel() != n * n_heads * hd or not out.is_contiguous() or \
                out.dtype != (torch.float16 if q.dtype == torch.float16 else torch.bfloat16):
            raise ValueError("out must be contiguous, with q's elements and type (bf16 for partials)")
        if weights is not None:
            _plain(weights, (n, nkv, cache.max_len), torch.float32, "weights")
        _all_apart([(out, "out"), (cache.data, "the cache"), (weights, "weights")],
                   [(q, "q"), (k, "k"), (v, "v"), (rows, "rows"), (q_norm, "q_norm"), (k_norm, "k_norm"), (cos, "cos"), (sin, "sin"),
                    (pos, "pos")])
        self._on(q, k, v, cache.data, rows, out, weights, q_norm, k_norm, cos, sin, pos)
        self.args = RvqCache4AttnArgs(qv, kv_, vv, _ptr(q_norm), _ptr(k_norm), _ptr(cos), _ptr(sin), _ptr(pos),
                                      cache.struct(), _ptr(rows), _ptr(out), _ptr(weights), n_heads, table, float(eps),
                                      float(scaling))
        n = self._workspace(_lib().rvq_cache4_attention_workspace_size)
        self._bind("rvq_cache4_attention", ctypes.byref(self.args), _ptr(self._ws), n)


class Cache4EvictOp(_Op):
    """Keep ``keep`` rows of every (sequence, kv head): the last ``recent`` and, of the others, those with the largest
    ``weights`` [n_seq, n_kv, max_len] (ties: the lowest row).  ``rows``: int64 [n_seq] live rows.  The kept records and weights move,
    in order, to the first rows of ``out`` and ``out_weights`` (None: in place); ``kept`` (int32 [n_seq, n_kv, keep], made
    here if None) gets their old rows, -1 behind the last, ``new_rows`` (int64 [n_seq], a tensor apart from ``rows``)
    the new live rows."""

    def __init__(self, cache: Cache4, weights: torch.Tensor, rows: torch.Tensor, *, keep: int, recent: int = 0,
                 kept: Optional[torch.Tensor] = None, out: Optional[Cache4] = None,
                 out_weights: Optional[torch.Tensor] = None, new_rows: Optional[torch.Tensor] = None):
        n, nkv = cache.n_seq, cache.n_kv
        if not 1 <= keep <= cache.max_len or not 0 <= recent <= keep:
            raise ValueError("1 <= keep <= max_len and 0 <= recent <= keep")
        _plain(weights, (n, nkv, cache.max_len), torch.float32, "weights")
        _ints(rows, n, torch.int64, "rows")
        if (out is None) != (out_weights is None):
            raise ValueError("out and out_weights are given together")
        apart = out is not None
        if not apart:
            out, out_weights = cache, weights
        else:
            if (out.n_seq, out.n_kv, out.head_dim) != (n, nkv, cache.head_dim) or out.max_len < keep:
                raise ValueError("out must hold keep rows of the same sequences and heads")
            _plain(out_weights, (n, nkv, out.max_len), torch.float32, "out_weights")
        if kept is not None:
            _plain(kept, (n, nkv, keep), torch.int32, "kept")
        if new_rows is not None:
            _ints(new_rows, n, torch.int64, "new_rows")
        _all_apart([(out.data, "out"), (out_weights, "out_weights"), (kept, "kept"), (new_rows, "new_rows")],
                   [(rows, "rows")] + ([(cache.data, "the cache"), (weights, "weights")] if apart else []))
        self._on(cache.data, weights, rows, out.data, out_weights, kept, new_rows)
        self.kept = torch.empty(n, nkv, keep, dtype=torch.int32, device=self.device) if kept is None else kept
        self.args = RvqCache4EvictArgs(cache.struct(), out.struct(), _ptr(weights), _ptr(out_weights), _ptr(rows),
                                       _ptr(new_rows), _ptr(self.kept), int(keep), int(recent))
        self._bind("rvq_cache4_evict", ctypes.byref(self.args))
