"""Paged key / value cache: the writer of new tokens, the attention of one new token per sequence, and eviction.

No counterpart in the reference.  A pool of pages holds the keys and values of all sequences; slot s of sequence b is row
``s % page_size`` of page ``block_table[b, s // page_size]``.  Page tables and lengths are read on the device, so the calls
neither synchronise nor depend on host copies of them, and may be captured into a graph (after one call on the device
outside of a capture).  A page number or length that the cache does not have is left out by the kernels and raised by
``check_status()``, or by the first call after it, outside of a capture, that sees it; a page that a call writes (keys,
weights or positions) must stand in the tables once only, pages that are only read may be shared.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _cabi
from ._cabi import FbaPaged
from .interface import HEAD_DIM, _checked, _monitor, _poisoned, _ptr, _raw_stream, _scale_of
from .window import _window_of

_Strides3, _Strides2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2


@dataclass
class PagedKVCache:
    """The pools (``new_paged_cache`` allocates them).

    ``k``, ``v``: bf16, or uint8 holding e4m3, [n_pages, kv_heads, page_size, 128]; ``k_scale``, ``v_scale``: fp32
    [n_pages, kv_heads, page_size], the value that a row's bytes are to be multiplied by (uint8 pools only).
    ``weight`` (fp32) and ``position`` (int32), both or neither, likewise: the attention weight that the token in a slot
    has received, and its place in its sequence; ``evict_kv`` goes by them.
    """

    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None
    weight: Optional[torch.Tensor] = None
    position: Optional[torch.Tensor] = None

    def dequantize(self):
        """(k, v) in fp32: what the kernels' arithmetic stands for."""
        if self.k.dtype == torch.bfloat16:
            return self.k.float(), self.v.float()
        return (self.k.view(torch.float8_e4m3fn).float() * self.k_scale[..., None],
                self.v.view(torch.float8_e4m3fn).float() * self.v_scale[..., None])


def new_paged_cache(n_pages: int, kv_heads: int, page_size: int, e4m3: bool = False, track: bool = False,
                    device="cuda") -> PagedKVCache:
    """An empty cache of ``n_pages`` pages; ``track``: with weights and positions, for ``evict_kv``."""
    shape = (n_pages, kv_heads, page_size)
    new = lambda dtype, *more: torch.zeros((*shape, *more), dtype=dtype, device=device)  # noqa: E731
    kind = torch.uint8 if e4m3 else torch.bfloat16
    cache = PagedKVCache(new(kind, HEAD_DIM), new(kind, HEAD_DIM))
    if e4m3:
        cache.k_scale, cache.v_scale = new(torch.float32), new(torch.float32)
    if track:
        cache.weight, cache.position = new(torch.float32), new(torch.int32)
    return cache


def _i32(name: str, x: torch.Tensor, B: Optional[int], dev: torch.device) -> int:
    """Pointer of a checked int32 [B]."""
    if x.dtype != torch.int32 or x.dim() != 1 or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous torch.int32 tensor of 1 dimension")
    if x.shape[0] != B:
        raise ValueError(f"{name} has the shape {tuple(x.shape)}, which does not fit")
    if x.device != dev:
        raise RuntimeError(f"{name} must be on the device of the cache")
    return x.data_ptr()


def _table(name: str, x: torch.Tensor, dev: torch.device) -> tuple[int, int, int]:
    """(pointer, sequences, pages per sequence) of a checked int32 [B, pages]."""
    if x.dtype != torch.int32 or x.dim() != 2 or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous torch.int32 tensor of 2 dimensions")
    if x.device != dev:
        raise RuntimeError(f"{name} must be on the device of the cache")
    return x.data_ptr(), *x.shape


def _cache_arg(cache: PagedKVCache, block_table: torch.Tensor) -> tuple[FbaPaged, int, torch.device]:
    """The checked cache with its table as the C entry points take it, the number of sequences, and the device."""
    k, v = cache.k, cache.v
    if not k.is_cuda:
        raise RuntimeError("the cache must be on a CUDA device (there is no CPU path)")
    e4m3 = k.dtype == torch.uint8
    if not e4m3 and k.dtype != torch.bfloat16 or v.dtype != k.dtype:
        raise TypeError("cache.k and cache.v must be torch.bfloat16, or torch.uint8 holding e4m3")
    shape = k.shape
    if len(shape) != 4 or shape[3] != HEAD_DIM or v.shape != shape or not k.is_contiguous() or not v.is_contiguous():
        raise ValueError("cache.k and cache.v must be contiguous, [pages, kv heads, page size, 128]")
    dev = k.device
    if v.device != dev:
        raise RuntimeError("the cache's tensors must be on one device")
    if e4m3 and (cache.k_scale is None or cache.v_scale is None):
        raise ValueError("an e4m3 cache needs k_scale and v_scale")
    if (cache.weight is None) != (cache.position is None):
        raise ValueError("cache.weight and cache.position come together")
    if e4m3 or cache.weight is not None:
        rows = shape[:3]
        for what in ("k_scale", "v_scale", "weight", "position"):
            x = getattr(cache, what)
            if x is not None:
                dtype = torch.int32 if what == "position" else torch.float32
                if x.dtype != dtype or x.shape != rows or not x.is_contiguous():
                    raise ValueError(f"cache.{what} must be a contiguous {dtype} tensor, [pages, kv heads, page size]")
                if x.device != dev:
                    raise RuntimeError("the cache's tensors must be on one device")
    table, B, pages = _table("block_table", block_table, dev)
    return FbaPaged(k.data_ptr(), v.data_ptr(), _ptr(cache.k_scale), _ptr(cache.v_scale), _ptr(cache.weight),
                    _ptr(cache.position), table, shape[0], shape[1], shape[2], pages, e4m3), B, dev


def _strides(name: str, x: torch.Tensor, shape: torch.Size):
    """The strides of all dimensions but the last, as the C entry points take them; one that is never taken counts as 0."""
    *st, last = x.stride()
    if last != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    if 1 in shape:
        st = [0 if d == 1 else s for s, d in zip(st, shape)]
    return (_Strides3 if len(st) == 3 else _Strides2)(*st)


def append_kv(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
              new_lens: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Write new tokens behind the ends of the sequences; returns the new lengths, int32 [B].

    Args:
        k, v: bf16 [B, kv_heads, T, 128], any strides that are multiples of 8 elements (last dimension contiguous)
        block_table: int32 [B, max_pages]; seq_lens: int32 [B], slots in use (left as they are)
        new_lens: int32 [B], how many of the T tokens are real (a padded batch); None = all
        positions: int32 [B], place in the sequence of each first new token, for a cache that tracks weights and has
            been cut; None = seq_lens

    In an e4m3 cache a row gets the scale max|x| / 448 (NaN if it is not finite) and the bytes of x / scale.
    """
    arg, B, dev = _cache_arg(cache, block_table)
    shape = k.shape
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or len(shape) != 4 or shape[0] != B or shape[1] != arg.Hkv or \
            shape[3] != HEAD_DIM:
        raise ValueError("k and v must be torch.bfloat16, [batch, kv heads, tokens, 128]")
    if v.shape != shape:
        raise ValueError("k and v must have the same shape")
    if not k.device == v.device == dev:
        raise RuntimeError("k and v must be on the device of the cache")
    lens = _i32("seq_lens", seq_lens, B, dev)
    new = None if new_lens is None else _i32("new_lens", new_lens, B, dev)
    pos = None if positions is None else _i32("positions", positions, B, dev)
    out = torch.empty_like(seq_lens)
    mon = _monitor(dev)
    mon.poll_mapped()
    rc = _cabi.lib().fba_paged_append(ctypes.byref(arg), k.data_ptr(), v.data_ptr(), _strides("k", k, shape),
                                      _strides("v", v, shape), B, shape[2], lens, new, pos, out.data_ptr(),
                                      mon.mapped_ptr, _raw_stream(dev.index))
    _checked(rc, "fba_paged_append", dev)
    return out


def paged_decode_attn(q: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                      window: Optional[int] = None, sinks: int = 0, softmax_scale=None, need_lse: bool = False,
                      accumulate: bool = False):
    """Attention of one new token per sequence over its cached tokens, its own (the last one) among them.

    Args:
        q: bf16 [B, heads, 128] (heads % kv_heads == 0), even strides, last dimension contiguous
        block_table: int32 [B, max_pages]; seq_lens: int32 [B], the new token counted
        window, sinks: as for ``sliding_window_attn_func``; only the pages that hold visible tokens are read
        accumulate: add to ``cache.weight`` the probability that each token received, summed over the query heads of
            its kv head (no window; at most 16 query heads per kv head).  Takes 4 bytes of scratch per query head and
            slot that the table has room for: pass a table of the pages in use, not of the most there may be

    Returns o, bf16 [B, heads, 128] (and the log-sum-exp, fp32 [B, heads], with ``need_lse``).  A sequence of length 0
    gives zeros and -inf.  Not differentiable.
    """
    w, s = _window_of(window, sinks)
    arg, B, dev = _cache_arg(cache, block_table)
    shape = q.shape
    if q.dtype != torch.bfloat16 or len(shape) != 3 or shape[0] != B or shape[2] != HEAD_DIM:
        raise ValueError("q must be torch.bfloat16, [batch, heads, 128]")
    if q.device != dev:
        raise RuntimeError("q must be on the device of the cache")
    Hq = shape[1]
    if Hq % arg.Hkv != 0 or Hq == 0:
        raise ValueError("the number of query heads must be a multiple of the number of kv heads")
    if accumulate and cache.weight is None:
        raise ValueError("accumulate needs a cache with weights (new_paged_cache(..., track=True))")
    if w and cache.weight is not None:
        raise ValueError("a window goes by slots, which a cache that evict_kv cuts does not keep in order")
    lens = _i32("seq_lens", seq_lens, B, dev)
    lib = _cabi.lib()
    n = ctypes.c_uint64(0)
    rc = lib.fba_paged_decode_workspace_bytes(B, Hq, arg.Hkv, arg.page_size, arg.max_pages, arg.e4m3, accumulate,
                                               ctypes.byref(n))
    _cabi.check(rc, "fba_paged_decode_workspace_bytes")
    o = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    lse = q.new_empty((B, Hq), dtype=torch.float32) if need_lse else None
    # The workspace; with accumulation the kernels want the log-sum-exp, too, also where the caller does not.
    words, own_lse = n.value // 4, accumulate and not need_lse
    ws = q.new_empty((words + own_lse * B * Hq,), dtype=torch.float32) if words else None
    _poisoned(ws, o, lse)
    ws_ptr = _ptr(ws)
    lse_ptr = ws_ptr + n.value if own_lse else _ptr(lse)
    mon = _monitor(dev)
    mon.poll_mapped()
    rc = lib.fba_paged_decode(ctypes.byref(arg), q.data_ptr(), _strides("q", q, shape), o.data_ptr(), lse_ptr, B, Hq,
                              lens, w, s, _scale_of(softmax_scale), accumulate, ws_ptr, n.value, mon.mapped_ptr,
                              _raw_stream(dev.index))
    _checked(rc, "fba_paged_decode", dev)
    return (o, lse) if need_lse else o


def evict_kv(cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor, budget: int, sinks: int = 0,
             recent: int = 0, next_positions: Optional[torch.Tensor] = None,
             out_table: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cut sequences to at most ``budget`` tokens by the attention weight they have received; returns the new lengths.

    Every kv head drops, of its n tokens, the n - budget with the least ``cache.weight`` (of equal ones the lowest slots)
    that are not protected: the first ``sinks`` positions and the last ``recent`` ones stay (sinks + recent <= budget).
    ``next_positions``: int32 [B], how many tokens the sequences have seen; None = seq_lens (never cut before).
    The weights are what ``paged_decode_attn(..., accumulate=True)`` and the caller have put there; ``append_kv`` starts
    with 0, so a prompt that is cut before anything was accumulated loses its first unprotected tokens.

    In place, the staying tokens behind the budget move to the slots that came free before it: the slots are then in no
    order of positions (``cache.position`` keeps them), the pages from ``ceil(budget / page_size)`` on are free, and
    ``paged_decode_attn`` goes on without a window.  With ``out_table`` (int32 [B, pages], pages that ``block_table`` does not
    name) the staying tokens are copied there in slot order instead, and the source, which others may share, is left.
    """
    arg, B, dev = _cache_arg(cache, block_table)
    if cache.weight is None:
        raise ValueError("evict_kv needs a cache with weights (new_paged_cache(..., track=True))")
    for name, x, least in (("budget", budget, 1), ("sinks", sinks, 0), ("recent", recent, 0)):
        if type(x) is not int or not least <= x < 2**31:
            raise ValueError(f"{name} must be an integer from {least} on")
    if sinks + recent > budget:
        raise ValueError("sinks + recent must not exceed budget")
    lens = _i32("seq_lens", seq_lens, B, dev)
    nxt = None if next_positions is None else _i32("next_positions", next_positions, B, dev)
    to, to_pages = None, 0
    if out_table is not None:
        to, to_rows, to_pages = _table("out_table", out_table, dev)
        if to_rows != B:
            raise ValueError("out_table must have a row for every sequence")
    lib = _cabi.lib()
    n = ctypes.c_uint64(0)
    rc = lib.fba_paged_evict_workspace_bytes(B, arg.Hkv, arg.page_size, arg.max_pages, budget, ctypes.byref(n))
    _cabi.check(rc, "fba_paged_evict_workspace_bytes")
    ws = seq_lens.new_empty((n.value // 4,))
    out = torch.empty_like(seq_lens)
    mon = _monitor(dev)
    mon.poll_mapped()
    rc = lib.fba_paged_evict(ctypes.byref(arg), B, lens, budget, sinks, recent, nxt, to, to_pages, out.data_ptr(),
                             ws.data_ptr(), n.value, mon.mapped_ptr, _raw_stream(dev.index))
    _checked(rc, "fba_paged_evict", dev)
    return out
