"""A paged key/value cache held in 4 bits and the attention over it, on an MI355X.

For serving: the decode path of ``flash_attn_forward_gqa`` reads dense 16-bit
keys and values; here they are pages of 17/32 byte an element that sequences
share a pool of.

    cache = PagedKVCache(num_pages, 64, num_kv_heads, head_dim, dtype=torch.bfloat16)
    # page_table (B, pages a sequence) int32, start (B,) int32: tokens held so far
    q = append_paged(cache, k, v, page_table, start, q=q, rotary=rotary)
    out = attend_paged(q, cache, page_table, start + q.shape[1])

``append_paged`` rotates the new keys (and queries) by their positions on the
way; ``attend_paged`` serves single tokens, speculated ones and whole prompt
chunks, causal with the mask aligned to the bottom right as everywhere in this
package; ``read_paged`` gives the held values back.  All run on the current
stream, synchronise nothing and can be captured into a graph; lengths, page
tables and counts are read on the device, so a replay serves what they hold
then.  None of them has a gradient.

The reference has no counterpart: its patch falls back to eager attention with
a cache (flash_attn_volta/patch_hf.py:145-162).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _capi, _runtime
from .autograd import _compiling, _cpp
from .forward import (NATIVE_HEAD_DIMS, _DTYPES, _kernel_ready, _on_device, _require, _stream_ptr,
                      kernel_strides)
from .rotary import RotaryPositions

__all__ = ["PagedKVCache", "append_paged", "attend_paged", "read_paged"]


def _shapes(N, P, H, D):
    return {"k_codes": (N, H, P, D // 2), "k_scales": (N, H, P, D // 32),
            "v_codes": (N, H, P // 4, 16, 4, D // 32), "v_scales": (N, H, P // 4, D // 32, 4)}


class PagedKVCache:
    """Pages of keys and values in 4 bits: e2m1 elements (0, 0.5, 1, 1.5, 2, 3,
    4, 6 and a sign), 32 along D to a power of two.

    PagedKVCache(num_pages, page_size, num_kv_heads, head_dim, dtype, device)
    allocates an empty cache; ``from_tensors`` wraps existing pages.  page_size
    is a power of two, at least 16; head_dim 32, 64 or 128; dtype (fp16 or
    bf16) is that of the keys, values and queries of its calls.

    Tensors (uint8, contiguous; token t of page n, head h):
      k_codes  (N, H, P, D/2)            byte d / 2, low half: even d
      k_scales (N, H, P, D/32)           power of two + 127
      v_codes  (N, H, P/4, 16, 4, D/32)  t = 4a + r, d = (D/16) m + j at
                                         [a, m, r, j / 2], low half: even j
      v_scales (N, H, P/4, D/32, 4)      t = 4a + r at [a, block, r]
    The value interleaving of 4 tokens is the order in which the attention's
    matrix instructions take them.  append_paged writes scales of 1 to 252 (140
    in an fp16 cache); larger ones must not be put there.
    """

    __slots__ = ("_tensors", "_dtype", "_sizes", "_structs", "_half", "_like", "_head_dim")

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        for name, n in (("num_pages", num_pages), ("num_kv_heads", num_kv_heads)):
            _require(isinstance(n, int) and n > 0, lambda: f"{name} must be positive, got {n!r}")
        _require(head_dim in NATIVE_HEAD_DIMS,
                 lambda: f"unsupported head_dim {head_dim} (allowed: {NATIVE_HEAD_DIMS})")
        _require(isinstance(page_size, int) and page_size >= 16
                 and page_size & (page_size - 1) == 0,
                 lambda: f"page_size must be a power of two, at least 16, got {page_size!r}")
        shapes = _shapes(num_pages, page_size, num_kv_heads, head_dim)
        self._adopt({n: torch.zeros(s, dtype=torch.uint8, device=device)
                     for n, s in shapes.items()}, dtype)

    @classmethod
    def from_tensors(cls, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                     v_scales: torch.Tensor, dtype: torch.dtype) -> "PagedKVCache":
        """A cache over existing page tensors (shared, not copied)."""
        self = cls.__new__(cls)
        self._adopt({"k_codes": k_codes, "k_scales": k_scales, "v_codes": v_codes,
                     "v_scales": v_scales}, dtype)
        return self

    def _adopt(self, tensors, dtype):
        _require(dtype in _DTYPES, lambda: f"dtype must be fp16 or bf16, got {dtype}")
        codes = tensors["k_codes"]
        _require(all(isinstance(t, torch.Tensor) and t.dtype == torch.uint8
                     for t in tensors.values()), "the cache's tensors must be uint8")
        _require(codes.dim() == 4, lambda: f"k_codes must be (N, H, P, D/2), got {tuple(codes.shape)}")
        N, H, P, D = *codes.shape[:3], codes.shape[3] * 2
        _require(N > 0 and H > 0, "the cache must have pages and heads")
        _require(D in NATIVE_HEAD_DIMS,
                 lambda: f"unsupported head_dim {D} (allowed: {NATIVE_HEAD_DIMS})")
        _require(P >= 16 and P & (P - 1) == 0,
                 lambda: f"page_size must be a power of two, at least 16, got {P}")
        for name, shape in _shapes(N, P, H, D).items():
            t = tensors[name]
            _require(tuple(t.shape) == shape,
                     lambda: f"{name} must be {shape}, got {tuple(t.shape)}")
            _require(t.device == codes.device, "the cache's tensors must be on one device")
            _require(t.is_contiguous() and t.data_ptr() % 16 == 0,
                     lambda: f"{name} must be contiguous and 16-byte aligned")
        # (fixed from here on: the calls' structs hold addresses and sizes)
        self._tensors, self._like, self._dtype = dict(tensors), codes, dtype
        self._sizes, self._head_dim = (N, H, P), D
        self._structs, self._half = {}, dtype == torch.float16

    k_codes = property(lambda self: self._tensors["k_codes"])
    k_scales = property(lambda self: self._tensors["k_scales"])
    v_codes = property(lambda self: self._tensors["v_codes"])
    v_scales = property(lambda self: self._tensors["v_scales"])
    num_pages = property(lambda self: self._sizes[0])
    num_kv_heads = property(lambda self: self._sizes[1])
    page_size = property(lambda self: self._sizes[2])
    head_dim = property(lambda self: self._head_dim)
    dtype = property(lambda self: self._dtype)
    device = property(lambda self: self._like.device)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() for t in self._tensors.values())

    def __reduce__(self):               # copies and pickles: their own addresses
        return PagedKVCache.from_tensors, (self.k_codes, self.k_scales, self.v_codes,
                                           self.v_scales, self.dtype)

    def _struct(self, width: int):
        """(fa_paged_cache for a table of `width` pages a sequence, its address)."""
        s = self._structs.get(width)
        if s is None:
            c = _capi.PagedCacheStruct(
                self.k_codes.data_ptr(), self.k_scales.data_ptr(), self.v_codes.data_ptr(),
                self.v_scales.data_ptr(), self.num_pages, self.page_size, self.num_kv_heads, width)
            s = self._structs[width] = (c, ctypes.addressof(c))
        return s

    def __repr__(self):
        return (f"PagedKVCache({self.num_pages} pages of {self.page_size} tokens, "
                f"{self.num_kv_heads} heads of {self.head_dim}, {self.dtype}, {self.device})")


def _cache(cache, device):
    _require(isinstance(cache, PagedKVCache),
             lambda: f"cache must be a PagedKVCache, got {type(cache).__name__}")
    _require(cache.device == device and device.type == "cuda",
             lambda: f"the cache is on {cache.device}, the tensors on {device}: one GPU is needed")


def _table(t, B: int, device):
    _require(isinstance(t, torch.Tensor) and t.dtype == torch.int32,
             "page_table must be an int32 tensor")
    _require(t.dim() == 2 and t.shape[0] == B and t.shape[1] > 0,
             lambda: f"page_table must be (B, pages) = ({B}, 1 or more), got {tuple(t.shape)}")
    _require(t.device == device, lambda: f"page_table must be on {device}")
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _counts(t, name: str, B: int, device):
    if t is None:
        return None
    _require(isinstance(t, torch.Tensor) and t.dtype == torch.int32,
             lambda: f"{name} must be an int32 tensor")
    _require(t.shape == (B,), lambda: f"{name} must be ({B},), got {tuple(t.shape)}")
    _require(t.device == device, lambda: f"{name} must be on {device}")
    return t if B == 1 or t.stride(0) == 1 else t.contiguous()


def _rows(t, name: str, cache, heads=None, like=None):
    _require(isinstance(t, torch.Tensor) and t.dim() == 4 and t.shape[3] == cache.head_dim,
             lambda: f"{name} must be (B, S, heads, {cache.head_dim}), got "
                     f"{tuple(getattr(t, 'shape', ()))}")
    _require(t.dtype == cache.dtype, lambda: f"{name} must be {cache.dtype}, got {t.dtype}")
    _require(t.device == cache.device, lambda: f"{name} must be on {cache.device}")
    if heads is not None:
        _require(t.shape[2] == heads, lambda: f"{name} must have {heads} heads, got {t.shape[2]}")
    if like is not None:
        _require(t.shape[:2] == like.shape[:2],
                 lambda: f"{name} {tuple(t.shape)} and k {tuple(like.shape)} differ in B or S")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _fast(cache, page_table, *tensors) -> int:
    """The address that the C++ calls of _fa_torch take for this cache and table,
    0 where a call goes the general way: the C++ module is not there, the call is
    being traced, or the arguments are not what they should be (the general
    way names what is wrong).  The C++ calls also leave to it whatever needs a
    copy or is empty."""
    if _cpp is None or type(cache) is not PagedKVCache or _compiling():
        return 0
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            return 0
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2 or page_table.shape[1] == 0:
        return 0
    return cache._struct(page_table.shape[1])[1]


def append_paged(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
                 start: torch.Tensor, counts: torch.Tensor | None = None, *,
                 q: torch.Tensor | None = None,
                 rotary: RotaryPositions | None = None) -> torch.Tensor | None:
    """Store the keys and values of new tokens in a paged 4-bit cache.

    Args:
        k, v: (B, S, Hk, D) in the cache's dtype, any strides with unit D stride.
        page_table: (B, pages) int32: position p of sequence b is slot
            p % page_size of page page_table[b, p // page_size].  Positions past
            the table, and ids that are no page of the cache (-1, say), store
            nothing.
        start: (B,) int32, the position of each sequence's first new token
            (the tokens it held before).
        counts: (B,) int32, how many of the S rows are tokens (a padded batch;
            clamped to 0 .. S), None: all.  Rows behind are not stored.
        q: (B, S, H, D), the same tokens' queries, rotated beside the keys.
        rotary: keys (and queries) are rotated by their positions; None: stored
            as they are.

    Returns q rotated, (B, S, H, D) contiguous (every row, those behind
    ``counts`` too), or None without q.  Each block of 32 columns is rounded
    to the nearest codes of its power of two, rotated keys directly from
    their 64-bit values; NaN is stored as 0 and an infinity as the dtype's
    largest value.  Pages that sequences share must not be appended to by
    more than one of them at the same slot: either's values may stay.
    """
    addr = _fast(cache, page_table, k, v, start)
    if addr and (q is None or isinstance(q, torch.Tensor)) \
            and (counts is None or isinstance(counts, torch.Tensor)) \
            and (rotary is None or isinstance(rotary, RotaryPositions)):
        done, out = _cpp.paged_append(
            addr, cache._like, cache._half, cache._head_dim, page_table, k, v, q, start, counts,
            *((None, 1.0, 0, 0) if rotary is None else rotary._args))
        if done:
            return out
    _require(isinstance(k, torch.Tensor), "k must be a tensor")
    _cache(cache, k.device)
    _rows(k, "k", cache, cache.num_kv_heads)
    _rows(v, "v", cache, cache.num_kv_heads, k)
    B, S, Hk, D = k.shape
    q_out, H = None, 0
    if q is not None:
        _rows(q, "q", cache, None, k)
        H = q.shape[2]
        q_out = torch.empty((B, S, H, D), dtype=q.dtype, device=q.device)
    page_table = _table(page_table, B, k.device)
    _require(start is not None, "start must be an int32 tensor")
    start, counts = _counts(start, "start", B, k.device), _counts(counts, "counts", B, k.device)
    steps, factor, R, flags = None, 1.0, 0, 0
    if rotary is not None:
        _require(isinstance(rotary, RotaryPositions),
                 lambda: f"rotary must be a RotaryPositions, got {type(rotary).__name__}")
        _require(rotary.steps.device == k.device,
                 lambda: f"rotary is on {rotary.steps.device}, k on {k.device}")
        _require(rotary.rotary_dim <= D,
                 lambda: f"rotary_dim {rotary.rotary_dim} is over the head_dim {D}")
        steps, factor = rotary.steps.data_ptr(), rotary.attention_factor
        R, flags = rotary.rotary_dim, rotary._flags
    if B == 0 or S == 0:
        return q_out
    k, v = _kernel_ready(k), _kernel_ready(v)
    rows = H > 0
    if rows:
        q = _kernel_ready(q)
    lib = _capi.load()
    with _on_device(k.device):
        rc = lib.fa_paged_append(
            cache._struct(page_table.shape[1])[0], page_table.data_ptr(), page_table.stride(0),
            k.data_ptr(), v.data_ptr(), q.data_ptr() if rows else None, _ptr(q_out) if rows else None,
            start.data_ptr(), _ptr(counts), steps, factor, R, flags, B, S, H, D,
            kernel_strides(k), kernel_strides(v), kernel_strides(q) if rows else None,
            kernel_strides(q_out) if rows else None, _DTYPES[cache.dtype], _stream_ptr(k.device))
    _capi.check(rc, "fa_paged_append")
    return q_out


def read_paged(cache: PagedKVCache, page_table: torch.Tensor, start: torch.Tensor, length: int,
               counts: torch.Tensor | None = None):
    """(k, v): the values held at positions start[b] .. start[b] + length - 1,
    each (B, length, Hk, D) contiguous in the cache's dtype, exactly what the
    attention sees; 0 behind counts[b] tokens and where the table names no page.
    For moving a sequence, a dense prefill over its prefix, or inspection."""
    addr = _fast(cache, page_table, start)
    if addr and isinstance(length, int) and (counts is None or isinstance(counts, torch.Tensor)):
        out = _cpp.paged_read(addr, cache._like, cache._half, cache._head_dim, page_table, start,
                              length, counts)
        if out is not None:
            return out
    _require(isinstance(page_table, torch.Tensor) and page_table.dim() == 2,
             "page_table must be a (B, pages) int32 tensor")
    _cache(cache, page_table.device)
    _require(isinstance(length, int) and length >= 0,
             lambda: f"length must be a non-negative int, got {length!r}")
    B, Hk, D = page_table.shape[0], cache.num_kv_heads, cache.head_dim
    page_table = _table(page_table, B, cache.device)
    _require(start is not None, "start must be an int32 tensor")
    start, counts = _counts(start, "start", B, cache.device), _counts(counts, "counts", B,
                                                                      cache.device)
    k, v = (torch.empty((B, length, Hk, D), dtype=cache.dtype, device=cache.device)
            for _ in range(2))
    if k.numel() == 0:
        return k, v
    lib = _capi.load()
    with _on_device(cache.device):
        rc = lib.fa_paged_read(
            cache._struct(page_table.shape[1])[0], page_table.data_ptr(), page_table.stride(0),
            k.data_ptr(), v.data_ptr(), start.data_ptr(), _ptr(counts), B, length, D,
            _DTYPES[cache.dtype], _stream_ptr(cache.device))
    _capi.check(rc, "fa_paged_read")
    return k, v


# Workspace bytes by sizes and device (the device's compute units decide).
_WS_BYTES: dict = {}


def _ws_bytes(lib, B, Sq, H, Hk, D) -> int:
    key = (B, Sq, H, Hk, D, _runtime.current_device())
    n = _WS_BYTES.get(key)
    if n is None:
        n = _WS_BYTES[key] = int(lib.fa_paged_attn_workspace_bytes(B, Sq, H, Hk, D))
    return n


def attend_paged(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor,
                 lengths: torch.Tensor, counts: torch.Tensor | None = None, *,
                 sm_scale: float | None = None, return_softmax_lse: bool = False):
    """Attention of each sequence's newest queries over a paged 4-bit cache.

    Args:
        q: (B, Sq, H, D) in the cache's dtype, H a multiple of the cache's
            heads (query head h reads head h // (H // Hk)), rotated like the
            keys were; any strides with unit D stride.
        page_table: (B, pages) int32 as for append_paged; keys of ids that are
            no page are not seen.
        lengths: (B,) int32, the tokens each sequence holds, those of the
            queries among them (append first).
        counts: (B,) int32, how many of the Sq rows are queries (a padded
            batch; clamped to 0 .. Sq), None: all.
        sm_scale: softmax scale (default 1/sqrt(D)).
        return_softmax_lse: also return the per-row natural-log LSE.

    Query i sees positions <= lengths[b] - counts[b] + i.  Returns out (B, Sq,
    H, D) contiguous in q's dtype and, if asked, lse (B, H, Sq) fp32; a query
    that sees no key, and every one behind ``counts``, gets 0 and +inf.
    """
    addr = _fast(cache, page_table, q, lengths)
    if addr and (counts is None or isinstance(counts, torch.Tensor)):
        out = _cpp.paged_attend(
            addr, cache._like, cache._half, cache._head_dim, q, page_table, lengths, counts,
            cache._head_dim ** -0.5 if sm_scale is None else float(sm_scale),
            bool(return_softmax_lse))
        if out is not None:
            return out if return_softmax_lse else out[0]
    _require(isinstance(q, torch.Tensor), "q must be a tensor")
    _cache(cache, q.device)
    _rows(q, "q", cache)
    B, Sq, H, D = q.shape
    Hk = cache.num_kv_heads
    _require(H % Hk == 0, lambda: f"query heads ({H}) must be a multiple of the cache's ({Hk})")
    page_table = _table(page_table, B, q.device)
    _require(lengths is not None, "lengths must be an int32 tensor")
    lengths, counts = _counts(lengths, "lengths", B, q.device), _counts(counts, "counts", B, q.device)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    out = torch.empty((B, Sq, H, D), dtype=q.dtype, device=q.device)
    lse = (torch.empty((B, H, Sq), dtype=torch.float32, device=q.device)
           if return_softmax_lse else None)
    if out.numel() == 0:
        return (out, lse) if return_softmax_lse else out
    q = _kernel_ready(q)
    lib = _capi.load()
    with _on_device(q.device):
        stream = _stream_ptr(q.device)
        nbytes = _ws_bytes(lib, B, Sq, H, Hk, D)
        ws = _runtime.workspace(nbytes, q.device, stream) if nbytes else None
        rc = lib.fa_paged_attn(
            q.data_ptr(), cache._struct(page_table.shape[1])[0], page_table.data_ptr(),
            page_table.stride(0), lengths.data_ptr(), _ptr(counts), out.data_ptr(), _ptr(lse),
            _ptr(ws), nbytes, B, Sq, H, D, kernel_strides(q), float(sm_scale),
            _DTYPES[cache.dtype], stream)
    _capi.check(rc, "fa_paged_attn")
    return (out, lse) if return_softmax_lse else out
