"""Attention between the q|k|v and the o matmul of a decoder layer, over a paged key/value cache.

Mirrors what the reference's attention functions do to the projections (native_model.cc:788-897,
976-1129, 1131-1282): RMSNorm of every query and key head, the values norm without a weight (:844),
``fast::rope``, the cache update and ``fast::scaled_dot_product_attention`` with a causal or
sliding-window mask. A layer's step is two launches around the matmuls::

    qkv = quantized_matmul(x, w_qkv)
    q, k, v = (t.unflatten(1, (-1, head_dim)) for t in qkv.split(...))
    q = kv_append(q, k, v, cache, batch, rope, q_norm, k_norm)       # norms, rotation, store
    attn = attention(q, cache, batch, scale=scale, window=1024)      # PagedAttention
    o = quantized_matmul(attn.flatten(1), w_o)

All compute runs in libg4q.so on the current CUDA stream; tensors are torch CUDA tensors, bf16.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib

__all__ = ["Rope", "PagedKVCache", "PagedBatch", "PagedAttention", "qk_norm_rope", "kv_append"]


_BF16 = torch.bfloat16
_raw_stream = torch._C._cuda_getCurrentRawStream
_HeadRows = _lib.G4qHeadRows


def _head_rows(t: torch.Tensor, head_dim: int, device: int, name: str, out: bool = False) -> _lib.G4qHeadRows:
    """The C view of a [tokens, heads, head_dim] tensor (any strides that keep 16-byte chunks whole). These
    checks run on every call of a decode step, so they stay a few attribute reads per tensor."""
    if t.dtype is not _BF16 or t.get_device() != device:
        raise ValueError(f"{name} must be a bfloat16 CUDA tensor on cuda:{device} (got {t.dtype} on {t.device})")
    shape = t.shape
    if len(shape) != 3 or shape[2] != head_dim:
        raise ValueError(f"{name} must be [tokens, heads, {head_dim}] (got {tuple(shape)})")
    st, sh, sd = t.stride()
    data = t.data_ptr()
    if sd != 1 or (st | sh) & 7 or data & 15:
        raise ValueError(f"{name}: the last dimension must be contiguous, strides multiples of 8 and data 16-byte aligned")
    if shape[1] == 1:
        sh = max(sh, head_dim)
    if out and (sh < head_dim or (shape[0] > 1 and st < head_dim)):
        raise ValueError(f"{name}: its rows overlap")
    return _HeadRows(data, st, sh, shape[1])


def _norm_weight(w: Optional[torch.Tensor], head_dim: int, device: int, name: str) -> Optional[int]:
    if w is None:
        return None
    if w.dtype is not _BF16 or w.get_device() != device or w.shape != (head_dim,) or not w.is_contiguous():
        raise ValueError(f"{name} must be a contiguous bf16 tensor of shape ({head_dim},) on cuda:{device}")
    return w.data_ptr()


def _int32(t: torch.Tensor, dims: int, name: str) -> torch.Tensor:
    if t.dtype is not torch.int32 or not t.is_cuda or t.dim() != dims or (t.numel() and t.stride(-1) != 1):
        raise ValueError(f"{name} must be a {dims}-D int32 CUDA tensor with contiguous rows")
    return t


def _same_device(device: int, **what) -> None:
    for name, x in what.items():
        if x.device != device:
            raise ValueError(f"{name} is on cuda:{x.device}, not on cuda:{device}")


def _output(t: torch.Tensor, heads: int, head_dim: int, device: int, out: Optional[torch.Tensor], name: str):
    """The output tensor for t's shape (a new contiguous one for None) and its C view."""
    if out is None:
        out = torch.empty_like(t, memory_format=torch.contiguous_format)
        return out, _HeadRows(out.data_ptr(), heads * head_dim, head_dim, heads)
    if out.shape != t.shape:
        raise ValueError(f"{name} must be shaped {tuple(t.shape)}")
    return out, _head_rows(out, head_dim, device, name, True)


class Rope:
    """Rotary position frequencies of one head layout, on the current GPU.

    ``inv_freq`` defaults to ``base ** (-2 i / rotary_dim)`` (radians per position), as ``fast::rope(x,
    dims=rotary_dim, traditional=False, base, scale)`` with ``scale`` multiplying the positions; pass
    ``rotary_dim / 2`` values of your own for other schemes (a pair with frequency 0 is not rotated). Pairs
    are (i, i + rotary_dim / 2); elements from rotary_dim on are left as they are."""

    def __init__(self, head_dim: int, base: float = 10000.0, *, rotary_dim: Optional[int] = None, scale: float = 1.0,
                 inv_freq: Optional[Sequence[float]] = None):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if inv_freq is None:
            if not (base > 0 and math.isfinite(base)):
                raise ValueError("base must be finite and positive")
            freqs = [scale * base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
        else:
            freqs = [float(f) * scale for f in inv_freq]
            if len(freqs) * 2 != rotary_dim:
                raise ValueError(f"inv_freq must hold rotary_dim / 2 = {rotary_dim // 2} values (got {len(freqs)})")
        self._h = ctypes.c_void_p()
        arr = (ctypes.c_double * max(len(freqs), 1))(*freqs)
        _lib.call("g4q_rope_create", head_dim, rotary_dim, arr, ctypes.byref(self._h))
        self.head_dim, self.rotary_dim = head_dim, rotary_dim
        self.device = torch.cuda.current_device()

    @property
    def handle(self) -> ctypes.c_void_p:
        if not self._h:
            raise ValueError("Rope has been freed")
        return self._h

    def free(self) -> None:
        if self._h:
            _lib.call("g4q_rope_free", self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class PagedKVCache:
    """One layer's keys and values in pages: ``k`` and ``v`` bf16 [pages, kv_heads, page_size, head_dim]
    CUDA tensors of equal strides (page_size a power of two, 16 or more). Any stride order qualifies while
    head_dim is contiguous, so ``t.transpose(1, 2)`` of a [pages, page_size, kv_heads, head_dim] tensor does,
    and so does one layer's slice of a tensor that holds them all. The tensors stay the caller's."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        for t, name in ((k, "k"), (v, "v")):
            if t.dtype != torch.bfloat16 or not t.is_cuda or t.dim() != 4:
                raise ValueError(f"{name} must be a 4-D bfloat16 CUDA tensor [pages, kv_heads, page_size, head_dim]")
            if t.stride(3) != 1:
                raise ValueError(f"{name}: head_dim must be contiguous")
        if k.shape != v.shape or k.stride() != v.stride() or k.device != v.device:
            raise ValueError("k and v must have the same shape, strides and device")
        self.k, self.v, self.device = k, v, k.get_device()
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        sp, sh, ss, _ = k.stride()
        # the stride of a dimension of one is never used, but has to be a legal one
        d = self.head_dim
        self.c = _lib.G4qPagedCache(k.data_ptr(), v.data_ptr(), self.n_pages, self.page_size, self.n_kv_heads, d,
                                    max(sp, d) if self.n_pages == 1 else sp, max(sh, d) if self.n_kv_heads == 1 else sh, ss)

    @classmethod
    def allocate(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int) -> "PagedKVCache":
        """A zeroed cache on the current GPU."""
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        dev = torch.device("cuda", torch.cuda.current_device())
        return cls(torch.zeros(shape, dtype=torch.bfloat16, device=dev), torch.zeros(shape, dtype=torch.bfloat16, device=dev))


class PagedBatch:
    """The sequences of one step. int32 CUDA tensors, read on the device when the kernels run (a captured
    graph replays with what they hold then; change them in place): ``q_offsets`` [n + 1], sequence b's new tokens are the rows
    q_offsets[b] .. q_offsets[b + 1]; ``kv_lens`` [n], its tokens in the cache with the new ones, which are
    the last; ``block_table`` [n, max_pages], position j is in page block_table[b, j // page_size]. ``max_q``:
    at least the longest sequence's new tokens. ``max_kv``: at least the longest kv_len where the caller
    knows it below the table's capacity; the table is then taken to end there.

    Contents that do not fit are refused on the device without touching other memory, and reported by
    ``_lib.device_error()`` as ERR_PAGE, ERR_TABLE or ERR_LENS."""

    def __init__(self, q_offsets: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, *, max_q: int,
                 max_kv: Optional[int] = None):
        self.q_offsets = _int32(q_offsets, 1, "q_offsets")
        self.kv_lens = _int32(kv_lens, 1, "kv_lens")
        self.block_table = _int32(block_table, 2, "block_table")
        n = kv_lens.shape[0]
        if n < 1 or q_offsets.shape[0] != n + 1 or block_table.shape[0] != n:
            raise ValueError(f"q_offsets must hold {n + 1} and block_table {n} rows for {n} sequences (at least one)")
        self.device = kv_lens.get_device()
        if q_offsets.get_device() != self.device or block_table.get_device() != self.device:
            raise ValueError("q_offsets, kv_lens and block_table must be on one device")
        if not 1 <= max_q < 2 ** 31 or (max_kv is not None and max_kv < 1):
            raise ValueError("max_q and max_kv must be >= 1 (and max_q below 2^31)")
        self.max_q, self.max_kv = max_q, max_kv
        self._views = {}

    def view(self, page_size: int) -> _lib.G4qPagedBatch:
        """The C view for a cache of this page size."""
        v = self._views.get(page_size)
        if v is None:
            v = self._views[page_size] = self._view(page_size)
        return v

    def _view(self, page_size: int) -> _lib.G4qPagedBatch:
        t = self.block_table
        pages = t.shape[1]
        if self.max_kv is not None:
            pages = min(pages, -(-self.max_kv // page_size))
        return _lib.G4qPagedBatch(self.q_offsets.data_ptr(), self.kv_lens.data_ptr(), t.data_ptr(),
                                  t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1]), t.shape[0], pages,
                                  self.max_q)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rope: Rope,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                 q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``rope(rms_norm(q) * q_weight)`` and the same for k, in one launch: q [tokens, q_heads, head_dim],
    k [tokens, kv_heads, head_dim] (views of the q|k|v matmul's output qualify), ``positions`` int32 [tokens].
    fp32 inside, one rounding at the end. The outputs may be the inputs (in place)."""
    d, dev = rope.head_dim, rope.device
    cq, ck = _head_rows(q, d, dev, "q"), _head_rows(k, d, dev, "k")
    n = q.shape[0]
    if k.shape[0] != n:
        raise ValueError("q and k must have the same number of tokens")
    if positions.dtype is not torch.int32 or positions.get_device() != dev or positions.shape != (n,) or (
            n > 1 and positions.stride(0) != 1):
        raise ValueError(f"positions must be a contiguous int32 tensor on cuda:{dev} with one entry per token")
    q_out, co = _output(q, cq.n_heads, d, dev, q_out, "q_out")
    k_out, cko = _output(k, ck.n_heads, d, dev, k_out, "k_out")
    _lib.call("g4q_qk_norm_rope", rope.handle, cq, ck, n, positions.data_ptr(),
              _norm_weight(q_weight, d, dev, "q_weight"), _norm_weight(k_weight, d, dev, "k_weight"), eps, co, cko,
              _raw_stream(dev))
    return q_out, k_out


def kv_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, cache: PagedKVCache, batch: PagedBatch,
              rope: Rope, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *,
              eps: float = 1e-6, norm_values: bool = True, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """The new tokens of a step, at their positions: keys normalized, weighted and rotated into the cache's
    pages, values normalized (without a weight; ``norm_values=False`` stores them as they are) beside them,
    and the queries, treated like the keys with ``q_weight``, returned (None for q None). One launch. ``v``
    may be ``k``. Sequences may share pages of a common prefix, but no two may append to one slot. Rows that belong to no sequence are left as they were (in ``q_out`` too)."""
    d, dev = rope.head_dim, rope.device
    _same_device(dev, cache=cache, batch=batch)
    ck = _head_rows(k, d, dev, "k")
    cv = ck if v is k else _head_rows(v, d, dev, "v")
    n = k.shape[0]
    if v.shape[0] != n or (q is not None and q.shape[0] != n):
        raise ValueError("q, k and v must have the same number of tokens")
    cq = co = None
    if q is not None:
        cq = _head_rows(q, d, dev, "q")
        q_out, co = _output(q, cq.n_heads, d, dev, q_out, "q_out")
    elif q_out is not None:
        raise ValueError("q_out without q")
    _lib.call("g4q_kv_append", rope.handle, cq, ck, cv, n, _norm_weight(q_weight, d, dev, "q_weight"),
              _norm_weight(k_weight, d, dev, "k_weight"), eps, 0 if norm_values else _lib.APPEND_RAW_VALUES, co,
              cache.c, batch.view(cache.page_size), _raw_stream(dev))
    return q_out


class PagedAttention:
    """Attention of a step's new tokens over a paged cache, for one head layout, on the current GPU.

    Owns the scratch of partial results: calls on one object must not overlap on the GPU (one stream, or
    events), replays of graphs that captured it included."""

    def __init__(self, n_q_heads: int, n_kv_heads: int, head_dim: int):
        self._h = ctypes.c_void_p()
        _lib.call("g4q_attn_create", n_q_heads, n_kv_heads, head_dim, ctypes.byref(self._h))
        self.n_q_heads, self.n_kv_heads, self.head_dim = n_q_heads, n_kv_heads, head_dim
        self.device = torch.cuda.current_device()

    @property
    def handle(self) -> ctypes.c_void_p:
        if not self._h:
            raise ValueError("PagedAttention has been freed")
        return self._h

    def __call__(self, q: torch.Tensor, cache: PagedKVCache, batch: PagedBatch, *, scale: Optional[float] = None,
                 window: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``softmax(scale * q k^T + mask) v``: q [tokens, q_heads, head_dim] as :func:`kv_append` returns it;
        the query at position t sees the keys j <= t, and j > t - window when window > 0. ``scale`` defaults
        to ``head_dim ** -0.5``. Single tokens, drafted blocks and prompt chunks may be mixed. A row that sees
        no key is zero; rows that belong to no sequence are left as they were (in ``out``, which must not overlap
        q)."""
        d, dev = self.head_dim, self.device
        _same_device(dev, cache=cache, batch=batch)
        cq = _head_rows(q, d, dev, "q")
        if not 0 <= window < 2 ** 31:
            raise ValueError("window must be >= 0 (0: none) and below 2^31")
        out, co = _output(q, cq.n_heads, d, dev, out, "out")
        _lib.call("g4q_paged_attention", self.handle, cq, q.shape[0], cache.c, batch.view(cache.page_size),
                  d ** -0.5 if scale is None else scale, window, co, _raw_stream(dev))
        return out

    def free(self) -> None:
        if self._h:
            _lib.call("g4q_attn_free", self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass
