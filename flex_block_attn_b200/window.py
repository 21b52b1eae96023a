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
from .interface import _check_qkv, _checked, _monitor, _poisoned, _ptr, _raw_stream, _scale_of


def _window_of(window: Optional[int], sinks: int) -> tuple[int, int]:
    """(window, sinks) as the C entry points take them: 0 for no limit."""
    if window is not None and (type(window) is not int or window < 1):
        raise ValueError("window must be a positive integer, or None for no limit")
    if type(sinks) is not int or sinks < 0:
        raise ValueError("sinks must be a non-negative integer")
    most = 2**31 - 1
    return (0 if window is None else min(window, most)), min(sinks, most)


def _sizes(q, k, v) -> tuple[int, int, int, int, int]:
    """(B, Hq, Hkv, Sq, Skv) of checked inputs."""
    _check_qkv(q, k, v)
    (B, Hq, Sq, _), (_, Hkv, Skv, _) = q.shape, k.shape
    if not (B and Hq and Sq and Hkv and Skv):
        raise ValueError("q, k and v must not be empty")
    return B, Hq, Hkv, Sq, Skv


def forward_with_window(q, k, v, window: Optional[int], sinks: int = 0, softmax_scale=None, need_lse: bool = True,
                        need_rest: bool = False):
    """Forward kernel alone; returns (o bf16 [B, Hq, Sq, 128], lse fp32 [B, Hq, Sq] or None), and with ``need_rest`` what the
    rounding of o left, for ``backward_with_window``.  A row that sees no key (possible when Sq > Skv) is zero, its lse
    -inf."""
    w, s = _window_of(window, sinks)
    B, Hq, Hkv, Sq, Skv = _sizes(q, k, v)
    dev = q.device
    o = torch.empty_like(q)
    lse = q.new_empty((B, Hq, Sq), dtype=torch.float32) if need_lse else None
    rest = torch.empty_like(q) if need_rest else None
    _poisoned(o, lse, rest)
    mon = _monitor(dev)
    mon.poll_mapped()
    rc = _cabi.lib().fba_window_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(lse), _ptr(rest), B, Hq, Hkv, Sq,
                                    Skv, w, s, _scale_of(softmax_scale), mon.mapped_ptr, _raw_stream(dev.index))
    _checked(rc, "fba_window_fwd", dev)
    return (o, lse, rest) if need_rest else (o, lse)


def backward_with_window(q, k, v, o, lse, dout, window: Optional[int], sinks: int = 0, softmax_scale=None, rest=None):
    """Backward kernels; ``o``, ``lse`` and, if it was asked for, ``rest`` are the forward's.  Returns (dq, dk, dv) in bf16.
    dK and dV are reproducible bit by bit; dQ is summed in fp32 in scheduling order.  ``rest`` makes the gradients more
    exact, those of rows that see few keys most."""
    w, s = _window_of(window, sinks)
    B, Hq, Hkv, Sq, Skv = _sizes(q, k, v)
    dev = q.device
    if dout.dtype != torch.bfloat16:
        dout = dout.to(torch.bfloat16)
    dout, o, lse = dout.contiguous(), o.contiguous(), lse.reshape(B, Hq, Sq).contiguous()
    if lse.dtype != torch.float32:
        raise TypeError("lse must be torch.float32")
    if dout.shape != q.shape or o.shape != q.shape or o.dtype != torch.bfloat16:
        raise ValueError("o and dout must have the shape of q, and o its type")
    if rest is not None and (rest.shape != q.shape or rest.dtype != torch.bfloat16 or not rest.is_contiguous()):
        raise ValueError("rest must be the forward's")
    if not dout.device == o.device == lse.device == dev or (rest is not None and rest.device != dev):
        raise RuntimeError("o, lse, rest and dout must be on the device of q")
    lib = _cabi.lib()
    n = ctypes.c_uint64(0)
    _cabi.check(lib.fba_window_partial_bytes(B, Hq, Hkv, Sq, Skv, w, s, ctypes.byref(n)), "fba_window_partial_bytes")
    # One buffer: row statistics, 2 floats a padded row; the dQ accumulator, 128; the partial sums.  All parts start at
    # multiples of 1 KiB.
    rows = B * Hq * -(-Sq // 128) * 128
    scratch = q.new_empty((rows * 130 + n.value // 4,), dtype=torch.float32)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    _poisoned(scratch, dq, dk, dv)
    at = scratch.data_ptr()
    mon = _monitor(dev)
    mon.poll_mapped()
    rc = lib.fba_window_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(rest), lse.data_ptr(),
                            dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), B, Hq, Hkv, Sq, Skv, w, s, _scale_of(softmax_scale),
                            at, at + rows * 8, at + rows * 520 if n.value else None, n.value, mon.mapped_ptr,
                            _raw_stream(dev.index))
    _checked(rc, "fba_window_bwd", dev)
    return dq, dk, dv


class SlidingWindowAttnFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, softmax_scale, is_grad_enabled):
        is_grad = is_grad_enabled and any(x.requires_grad for x in (q, k, v))
        if not is_grad:
            return forward_with_window(q, k, v, window, sinks, softmax_scale, need_lse=False)[0]
        o, lse, rest = forward_with_window(q, k, v, window, sinks, softmax_scale, need_rest=True)
        ctx.save_for_backward(q, k, v, o, lse, rest)
        ctx.args = (window, sinks, softmax_scale)
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        *saved, rest = ctx.saved_tensors
        return *backward_with_window(*saved, dout, *ctx.args, rest), None, None, None, None


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
