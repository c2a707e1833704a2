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

All compute runs in libg4q.so on the current CUDA stream; tensors are torch CUDA tensors, bf16. The calls of a
step go through a small CPython module (csrc/g4q_torch.cpp), which checks the tensors and makes the outputs.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib

__all__ = ["Rope", "PagedKVCache", "PagedBatch", "PagedAttention", "qk_norm_rope", "kv_append"]


_raw_stream = torch._C._cuda_getCurrentRawStream


def _int32(t: torch.Tensor, dims: int, name: str) -> torch.Tensor:
    if t.dtype is not torch.int32 or not t.is_cuda or t.dim() != dims or (t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must be a {dims}-D int32 CUDA tensor with contiguous rows")
    return t


def _same_device(device: int, cache, batch) -> None:
    if cache.device != device or batch.device != device:
        raise ValueError(f"the cache (cuda:{cache.device}) and the batch (cuda:{batch.device}) must be on cuda:{device}")


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
        self._ops = _lib.torch_ops()

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
    CUDA tensors of equal strides (page_size a power of two, 16 or more). Any stride order qualifies while head_dim is
    contiguous, so ``t.transpose(1, 2)`` of a [pages, page_size, kv_heads, head_dim] tensor does, and so does one
    layer's slice of a tensor that holds them all. The tensors stay the caller's; other ones are another cache.
    Elements that ``k`` and ``v``, or two of a tensor's slots, share can be read; :func:`kv_append` refuses them."""

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
        self.c_addr = ctypes.addressof(self.c)

    def __setattr__(self, name, value):
        if "c_addr" in self.__dict__ and name in self.__dict__:    # the structure for the kernels would not follow
            raise AttributeError(f"a PagedKVCache stays as it was made ({name} assigned): make another one")
        super().__setattr__(name, value)

    @classmethod
    def allocate(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int) -> "PagedKVCache":
        """A zeroed cache on the current GPU."""
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        dev = torch.device("cuda", torch.cuda.current_device())
        return cls(torch.zeros(shape, dtype=torch.bfloat16, device=dev), torch.zeros(shape, dtype=torch.bfloat16, device=dev))


def _field(name: str) -> property:
    return property(lambda self: getattr(self, "_" + name), lambda self, value: self._set(**{name: value}))


class PagedBatch:
    """The sequences of one step. int32 CUDA tensors, read on the device when the kernels run (a captured
    graph replays with what they hold then; change them in place): ``q_offsets`` [n + 1], sequence b's new
    tokens are the rows q_offsets[b] .. q_offsets[b + 1]; ``kv_lens`` [n], its tokens in the cache with the new ones, which are
    the last; ``block_table`` [n, max_pages], position j is in page block_table[b, j // page_size]. ``max_q``:
    at least the longest sequence's new tokens. ``max_kv``: at least the longest kv_len where the caller
    knows it below the table's capacity; the table is then taken to end there.

    The five may be assigned later too (a wider table, a larger ``max_q``): from the next call on that holds; a
    captured graph stays with what it captured, tensors that have to live as long. Another number of sequences is
    another batch. Contents that do not fit are refused on the device without touching other memory, and reported by
    ``_lib.device_error()`` as ERR_PAGE, ERR_TABLE or ERR_LENS."""

    _FIELDS = ("q_offsets", "kv_lens", "block_table", "max_q", "max_kv")
    q_offsets, kv_lens, block_table, max_q, max_kv = map(_field, _FIELDS)

    def __init__(self, q_offsets: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, *, max_q: int,
                 max_kv: Optional[int] = None):
        self._set(q_offsets=q_offsets, kv_lens=kv_lens, block_table=block_table, max_q=max_q, max_kv=max_kv)

    def _set(self, **fields) -> None:
        """Take the fields if they fit together with the others; the views for the kernels are made anew."""
        f = {**{n: getattr(self, "_" + n, None) for n in self._FIELDS}, **fields}
        q_offsets, kv_lens = _int32(f["q_offsets"], 1, "q_offsets"), _int32(f["kv_lens"], 1, "kv_lens")
        block_table, max_q, max_kv = _int32(f["block_table"], 2, "block_table"), f["max_q"], f["max_kv"]
        n = kv_lens.shape[0]
        if n < 1 or q_offsets.shape[0] != n + 1 or block_table.shape[0] != n:
            raise ValueError(f"q_offsets must hold {n + 1} and block_table {n} rows for {n} sequences (at least one)")
        device = kv_lens.get_device()
        if q_offsets.get_device() != device or block_table.get_device() != device:
            raise ValueError("q_offsets, kv_lens and block_table must be on one device")
        if not 1 <= max_q < 2 ** 31 or (max_kv is not None and max_kv < 1):
            raise ValueError("max_q and max_kv must be >= 1 (and max_q below 2^31)")
        self.device = device
        for name in self._FIELDS:
            setattr(self, "_" + name, f[name])
        self._views = {}

    def view(self, page_size: int) -> int:
        """Address of the C view for a cache of this page size; valid until a field is assigned."""
        return self._held(page_size)[0]

    def _held(self, page_size: int) -> Tuple[int, _lib.G4qPagedBatch]:
        """The C view's address, and the view, which a call keeps while it runs."""
        v = self._views.get(page_size)
        if v is None:
            c = self._view(page_size)
            v = self._views[page_size] = (ctypes.addressof(c), c)
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
    fp32 inside, one rounding at the end. The outputs may be the inputs (in place), else they must not overlap
    any other rows of the call."""
    dev = rope.device
    return rope._ops.qk_norm_rope(rope.handle.value, rope.head_dim, dev, _raw_stream(dev), q, k, positions, q_weight, k_weight,
                                  eps, q_out, k_out)


def kv_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, cache: PagedKVCache, batch: PagedBatch,
              rope: Rope, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *,
              eps: float = 1e-6, norm_values: bool = True, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """The new tokens of a step, at their positions: keys normalized, weighted and rotated into the cache's
    pages, values normalized (without a weight; ``norm_values=False`` stores them as they are) beside them,
    and the queries, treated like the keys with ``q_weight``, returned (None for q None). One launch. ``v``
    may be ``k``. Sequences may share pages of a common prefix, but no two new tokens may go to one slot. Rows that
    belong to no sequence are left as they were (in ``q_out`` too). No tensor may overlap the cache."""
    dev = rope.device
    _same_device(dev, cache, batch)
    view = batch._held(cache.page_size)
    return rope._ops.kv_append(rope.handle.value, rope.head_dim, dev, _raw_stream(dev), q, k, v, cache.c_addr,
                               view[0], q_weight, k_weight, eps,
                               0 if norm_values else _lib.APPEND_RAW_VALUES, q_out)


class PagedAttention:
    """Attention of a step's new tokens over a paged cache, for one head layout, on the current GPU.

    Owns the scratch of partial results: calls on one object must not overlap on the GPU (one stream, or
    events), replays of graphs that captured it included."""

    def __init__(self, n_q_heads: int, n_kv_heads: int, head_dim: int):
        self._h = ctypes.c_void_p()
        _lib.call("g4q_attn_create", n_q_heads, n_kv_heads, head_dim, ctypes.byref(self._h))
        self.n_q_heads, self.n_kv_heads, self.head_dim = n_q_heads, n_kv_heads, head_dim
        self.device = torch.cuda.current_device()
        self._ops = _lib.torch_ops()

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
        q or the cache)."""
        dev = self.device
        _same_device(dev, cache, batch)
        view = batch._held(cache.page_size)
        return self._ops.paged_attention(self.handle.value, self.head_dim, dev, _raw_stream(dev), q, cache.c_addr,
                                         view[0], self.head_dim ** -0.5 if scale is None else scale, window,
                                         out)

    def free(self) -> None:
        if self._h:
            _lib.call("g4q_attn_free", self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass
