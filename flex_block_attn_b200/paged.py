"""Paged key / value cache: the writer of new tokens, the attention of one new token per sequence, and eviction.

No counterpart in the reference.  A pool of pages holds the keys and values of all sequences; slot s of sequence b is row
``s % page_size`` of page ``block_table[b, s // page_size]``.  Page tables and lengths are read on the device, so the calls
neither synchronise nor depend on host copies of them, and may be captured into a graph (after one call on the device
outside of a capture).  A page number or length that the cache does not have is left out by the kernels and raised by
``check_status()`` (or by the first attention call after it that sees it); pages that a call writes must belong to one
sequence only, pages that are read may be shared.
"""
from __future__ import annotations

import ctypes
import os
from dataclasses import dataclass
from typing import Optional

import torch

from . import _cabi
from ._cabi import FbaPaged
from .interface import HEAD_DIM, _new, _ptr, _scale_of, _status, _stream_ptr, check_status
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


def _i32(name: str, x: torch.Tensor, shape: tuple, dev: torch.device) -> int:
    if x.dtype != torch.int32 or x.dim() != len(shape) or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous torch.int32 tensor of {len(shape)} dimension(s)")
    if any(want is not None and want != got for want, got in zip(shape, x.shape)):
        raise ValueError(f"{name} has the shape {tuple(x.shape)}, which does not fit")
    if x.device != dev:
        raise RuntimeError(f"{name} must be on the device of the cache")
    return x.data_ptr()


def _cache_arg(cache: PagedKVCache, block_table: torch.Tensor, name: str = "block_table") -> tuple[FbaPaged, int]:
    """The checked cache with its table as the C entry points take it, and the number of sequences."""
    k, v = cache.k, cache.v
    if not k.is_cuda:
        raise RuntimeError("the cache must be on a CUDA device (there is no CPU path)")
    if k.dtype not in (torch.bfloat16, torch.uint8) or v.dtype != k.dtype:
        raise TypeError("cache.k and cache.v must be torch.bfloat16, or torch.uint8 holding e4m3")
    if k.dim() != 4 or k.shape[3] != HEAD_DIM or v.shape != k.shape or not k.is_contiguous() or not v.is_contiguous():
        raise ValueError("cache.k and cache.v must be contiguous, [pages, kv heads, page size, 128]")
    dev, e4m3 = k.device, k.dtype == torch.uint8
    for what, x, dtype, needed in (("k_scale", cache.k_scale, torch.float32, e4m3), ("v_scale", cache.v_scale, torch.float32, e4m3),
                                   ("weight", cache.weight, torch.float32, False), ("position", cache.position, torch.int32, False)):
        if x is None:
            if needed:
                raise ValueError(f"an e4m3 cache needs {what}")
        elif x.dtype != dtype or x.shape != k.shape[:3] or not x.is_contiguous():
            raise ValueError(f"cache.{what} must be a contiguous {dtype} tensor, [pages, kv heads, page size]")
        elif x.device != dev:
            raise RuntimeError("the cache's tensors must be on one device")
    if v.device != dev:
        raise RuntimeError("the cache's tensors must be on one device")
    if (cache.weight is None) != (cache.position is None):
        raise ValueError("cache.weight and cache.position come together")
    table = _i32(name, block_table, (None, None), dev)
    return FbaPaged(k.data_ptr(), v.data_ptr(), _ptr(cache.k_scale), _ptr(cache.v_scale), _ptr(cache.weight),
                    _ptr(cache.position), table, k.shape[0], k.shape[1], k.shape[2], block_table.shape[1],
                    int(e4m3)), block_table.shape[0]


def _strides(name: str, x: torch.Tensor, n: int):
    """The strides of the first ``n`` dimensions; one that is never taken counts as 0."""
    if x.stride(-1) != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    return [x.stride(i) if x.shape[i] > 1 else 0 for i in range(n)]


def _check(rc: int, what: str, dev: torch.device) -> None:
    _cabi.check(rc, what)
    if os.environ.get("FBA_CHECK_STATUS", "0") == "1" and not torch.cuda.is_current_stream_capturing():
        check_status(dev)


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
    arg, B = _cache_arg(cache, block_table)
    dev = cache.k.device
    for name, x in (("k", k), ("v", v)):
        if x.dtype != torch.bfloat16 or x.dim() != 4 or x.shape[:2] != (B, arg.Hkv) or x.shape[3] != HEAD_DIM:
            raise ValueError(f"{name} must be torch.bfloat16, [batch, kv heads, tokens, 128]")
        if x.device != dev:
            raise RuntimeError(f"{name} must be on the device of the cache")
    if k.shape != v.shape:
        raise ValueError("k and v must have the same shape")
    lens = _i32("seq_lens", seq_lens, (B,), dev)
    new = None if new_lens is None else _i32("new_lens", new_lens, (B,), dev)
    pos = None if positions is None else _i32("positions", positions, (B,), dev)
    out = torch.empty_like(seq_lens)
    rc = _cabi.lib().fba_paged_append(ctypes.byref(arg), k.data_ptr(), v.data_ptr(), _Strides3(*_strides("k", k, 3)),
                                      _Strides3(*_strides("v", v, 3)), B, k.shape[2], lens, new, pos, out.data_ptr(),
                                      _status(dev).data_ptr(), _stream_ptr(dev))
    _check(rc, "fba_paged_append", dev)
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
            its kv head (no window; at most 16 query heads per kv head)

    Returns o, bf16 [B, heads, 128] (and the log-sum-exp, fp32 [B, heads], with ``need_lse``).  A sequence of length 0
    gives zeros and -inf.  Not differentiable.
    """
    w, s = _window_of(window, sinks)
    arg, B = _cache_arg(cache, block_table)
    dev = cache.k.device
    if q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[0] != B or q.shape[2] != HEAD_DIM:
        raise ValueError("q must be torch.bfloat16, [batch, heads, 128]")
    if q.device != dev:
        raise RuntimeError("q must be on the device of the cache")
    Hq = q.shape[1]
    if Hq % arg.Hkv != 0 or Hq == 0:
        raise ValueError("the number of query heads must be a multiple of the number of kv heads")
    if accumulate and cache.weight is None:
        raise ValueError("accumulate needs a cache with weights (new_paged_cache(..., track=True))")
    if w and cache.weight is not None:
        raise ValueError("a window goes by slots, which a cache that evict_kv cuts does not keep in order")
    lens = _i32("seq_lens", seq_lens, (B,), dev)
    lib = _cabi.lib()
    n = ctypes.c_uint64(0)
    _cabi.check(lib.fba_paged_decode_workspace_bytes(B, Hq, arg.Hkv, arg.page_size, arg.max_pages, int(accumulate),
                                                     ctypes.byref(n)), "fba_paged_decode_workspace_bytes")
    ws = torch.empty((n.value,), dtype=torch.uint8, device=dev) if n.value else None
    o = _new((B, Hq, HEAD_DIM), torch.bfloat16, dev)
    lse = _new((B, Hq), torch.float32, dev) if need_lse or accumulate else None
    rc = lib.fba_paged_decode(ctypes.byref(arg), q.data_ptr(), _Strides2(*_strides("q", q, 2)), o.data_ptr(), _ptr(lse), B, Hq,
                              lens, w, s, _scale_of(softmax_scale), int(accumulate), _ptr(ws), n.value,
                              _status(dev).data_ptr(), _stream_ptr(dev))
    _check(rc, "fba_paged_decode", dev)
    return (o, lse) if need_lse else o


def evict_kv(cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor, budget: int, sinks: int = 0,
             recent: int = 0, next_positions: Optional[torch.Tensor] = None,
             out_table: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cut sequences to at most ``budget`` tokens by the attention weight they have received; returns the new lengths.

    Every kv head drops, of its n tokens, the n - budget with the least ``cache.weight`` (of equal ones the lowest slots)
    that are not protected: the first ``sinks`` positions and the last ``recent`` ones stay (sinks + recent <= budget).
    ``next_positions``: int32 [B], how many tokens the sequences have seen; None = seq_lens (never cut before).

    In place, the staying tokens behind the budget move to the slots that came free before it: the slots are then in no
    order of positions (``cache.position`` keeps them), the pages from ``ceil(budget / page_size)`` on are free, and
    ``paged_decode_attn`` goes on without a window.  With ``out_table`` (int32 [B, pages], pages that ``block_table`` does not
    name) the staying tokens are copied there in slot order instead, and the source, which others may share, is left.
    """
    arg, B = _cache_arg(cache, block_table)
    dev = cache.k.device
    if cache.weight is None:
        raise ValueError("evict_kv needs a cache with weights (new_paged_cache(..., track=True))")
    for name, x, least in (("budget", budget, 1), ("sinks", sinks, 0), ("recent", recent, 0)):
        if isinstance(x, bool) or not isinstance(x, int) or not least <= x < 2**31:
            raise ValueError(f"{name} must be an integer from {least} on")
    if sinks + recent > budget:
        raise ValueError("sinks + recent must not exceed budget")
    lens = _i32("seq_lens", seq_lens, (B,), dev)
    nxt = None if next_positions is None else _i32("next_positions", next_positions, (B,), dev)
    to = None if out_table is None else _i32("out_table", out_table, (B, None), dev)
    lib = _cabi.lib()
    n = ctypes.c_uint64(0)
    _cabi.check(lib.fba_paged_evict_workspace_bytes(B, arg.Hkv, arg.page_size, arg.max_pages, budget, ctypes.byref(n)),
                "fba_paged_evict_workspace_bytes")
    ws = torch.empty((n.value,), dtype=torch.uint8, device=dev)
    out = torch.empty_like(seq_lens)
    rc = lib.fba_paged_evict(ctypes.byref(arg), B, lens, budget, sinks, recent, nxt, to,
                             0 if out_table is None else out_table.shape[1], out.data_ptr(), ws.data_ptr(), n.value,
                             _status(dev).data_ptr(), _stream_ptr(dev))
    _check(rc, "fba_paged_evict", dev)
    return out
