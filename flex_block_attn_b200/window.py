"""Causal attention under a sliding window with a few first tokens that stay visible (sinks).

No counterpart in the reference, whose masks are made of blocks.  The query of row i stands at position
``i + Skv - Sq`` (the last query and the last key belong to the same token, so a piece of a prompt may follow earlier keys)
and sees key j when ``j <= position and (position - j < window or j < sinks)``.  The kernels are those of
``flex_block_attn_func`` with the tiles derived from the window instead of from lists, and a mask per key at its edges.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _cabi
from .interface import _check_qkv, _maybe_check, _monitor, _new, _ptr, _scale_of, _status, _stream_ptr


def _window_of(window: Optional[int], sinks: int) -> tuple[int, int]:
    """(window, sinks) as the C entry points take them: 0 for no limit."""
    if window is not None and (isinstance(window, bool) or not isinstance(window, int) or window < 1):
        raise ValueError("window must be a positive integer, or None for no limit")
    if isinstance(sinks, bool) or not isinstance(sinks, int) or sinks < 0:
        raise ValueError("sinks must be a non-negative integer")
    most = 2**31 - 1
    return (0 if window is None else min(window, most)), min(sinks, most)


def _check_window_qkv(q, k, v) -> None:
    _check_qkv(q, k, v)
    if min(q.shape[:3]) < 1 or min(k.shape[1:3]) < 1:
        raise ValueError("q, k and v must not be empty")


def forward_with_window(q, k, v, window: Optional[int], sinks: int = 0, softmax_scale=None, need_lse: bool = True):
    """Forward kernel alone; returns (o bf16 [B, Hq, Sq, 128], lse fp32 [B, Hq, Sq] or None).  A row that sees no key
    (possible when Sq > Skv) is zero, its lse -inf."""
    w, s = _window_of(window, sinks)
    _check_window_qkv(q, k, v)
    B, Hq, Sq, _ = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    dev = q.device
    o = _new(q)
    lse = _new((B, Hq, Sq), torch.float32, dev) if need_lse else None
    _monitor(dev).poll()
    with torch.cuda.device(dev):
        rc = _cabi.lib().fba_window_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(lse), B, Hq, Hkv, Sq,
                                        Skv, w, s, _scale_of(softmax_scale), _status(dev).data_ptr(), _stream_ptr(dev))
    _cabi.check(rc, "fba_window_fwd")
    _maybe_check(dev)
    return o, lse


def backward_with_window(q, k, v, o, lse, dout, window: Optional[int], sinks: int = 0, softmax_scale=None):
    """Backward kernels; ``o`` and ``lse`` are the forward's.  Returns (dq, dk, dv) in bf16.  dK and dV are reproducible
    bit by bit; dQ is summed in fp32 in scheduling order."""
    w, s = _window_of(window, sinks)
    _check_window_qkv(q, k, v)
    B, Hq, Sq, _ = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    dev = q.device
    dout = dout.to(torch.bfloat16).contiguous()
    o = o.contiguous()
    lse = lse.reshape(B, Hq, Sq).contiguous()
    if lse.dtype != torch.float32:
        raise TypeError("lse must be torch.float32")
    if dout.shape != q.shape or o.shape != q.shape or o.dtype != torch.bfloat16:
        raise ValueError("o and dout must have the shape of q, and o its type")
    if any(t.device != dev for t in (o, lse, dout)):
        raise RuntimeError("o, lse and dout must be on the device of q")
    lib = _cabi.lib()
    dq, dk, dv = _new(q), _new(k), _new(v)
    n1, n2, n3 = ctypes.c_uint64(0), ctypes.c_uint64(0), ctypes.c_uint64(0)
    _cabi.check(lib.fba_bwd_scratch_bytes(B, Hq, Sq, ctypes.byref(n1), ctypes.byref(n2)), "fba_bwd_scratch_bytes")
    _cabi.check(lib.fba_window_partial_bytes(B, Hq, Hkv, Sq, Skv, w, s, ctypes.byref(n3)), "fba_window_partial_bytes")
    lse_delta = _new((n1.value // 4,), torch.float32, dev)
    dq_accum = _new((n2.value // 4,), torch.float32, dev)
    partial = _new((n3.value // 4,), torch.float32, dev) if n3.value else None
    _monitor(dev).poll()
    with torch.cuda.device(dev):
        rc = lib.fba_window_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), dout.data_ptr(),
                                dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), B, Hq, Hkv, Sq, Skv, w, s,
                                _scale_of(softmax_scale), lse_delta.data_ptr(), dq_accum.data_ptr(), _ptr(partial),
                                n3.value, _status(dev).data_ptr(), _stream_ptr(dev))
    _cabi.check(rc, "fba_window_bwd")
    _maybe_check(dev)
    return dq, dk, dv


class SlidingWindowAttnFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, softmax_scale, is_grad_enabled):
        is_grad = is_grad_enabled and any(x.requires_grad for x in (q, k, v))
        o, lse = forward_with_window(q, k, v, window, sinks, softmax_scale, need_lse=is_grad)
        if is_grad:
            ctx.save_for_backward(q, k, v, o, lse)
            ctx.args = (window, sinks, softmax_scale)
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, o, lse = ctx.saved_tensors
        return *backward_with_window(q, k, v, o, lse, dout, *ctx.args), None, None, None, None


def sliding_window_attn_func(q, k, v, window, sinks=0, softmax_scale=None):
    """Causal attention under a sliding window with sinks.

    Args:
        q: [batch, heads, q_seq_len, 128] bf16 CUDA tensor, contiguous; any length from 1
        k, v: [batch, kv_heads, kv_seq_len, 128], likewise (heads % kv_heads == 0); the values must be finite, those of
            padding behind a sequence's end included
        window: how many last keys a query sees, its own among them; None = all (a causal mask)
        sinks: how many first keys stay visible to every query at or behind them
        softmax_scale: factor applied to q k^T before the softmax; None = 1/sqrt(128)

    The query of row i stands at position i + kv_seq_len - q_seq_len.  In a batch padded at the end (q_seq_len ==
    kv_seq_len) no real token sees the padding; its own rows are to be ignored and their gradients given as zero.

    Returns:
        [batch, heads, q_seq_len, 128] bf16; differentiable (once) w.r.t. q, k and v.
    """
    return SlidingWindowAttnFunc.apply(q, k, v, window, sinks, softmax_scale, torch.is_grad_enabled())
