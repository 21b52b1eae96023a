"""Oracle of the sliding-window attention, the paged cache and what reads and cuts it, in 64 bits with plain loops and
elementary tensor operations.  TEST INFRASTRUCTURE ONLY: the package does not import it."""
from __future__ import annotations

import math
from typing import Optional

import torch


def visible(Sq: int, Skv: int, window: Optional[int], sinks: int, device=None) -> torch.Tensor:
    """Bool [Sq, Skv]: whether the query of row i, at position i + Skv - Sq, sees key j."""
    p = torch.arange(Sq, device=device)[:, None] + (Skv - Sq)
    j = torch.arange(Skv, device=device)[None]
    m = j <= p
    return m if window is None else m & ((p - j < window) | (j < sinks))


def masked_attention(q, k, v, mask, dout=None, softmax_scale: Optional[float] = None):
    """(o, lse) or (o, lse, dq, dk, dv) in 64 bits; q [B, Hq, Sq, D], k, v [B, Hkv, Skv, D], mask [Sq, Skv].

    Rows that see nothing give zeros, lse = -inf and no gradient; grouped heads' dK and dV are summed.
    """
    q, k, v = q.double(), k.double(), v.double()
    B, Hq, Sq, D = q.shape
    Hkv, Skv = k.shape[1:3]
    scale = 1 / math.sqrt(D) if softmax_scale is None else softmax_scale
    qg = q.reshape(B, Hkv, Hq // Hkv, Sq, D)
    s = (qg @ k[:, :, None].transpose(-1, -2) * scale).masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = (s - lse.masked_fill(lse == -math.inf, 0.0)[..., None]).exp()
    o = p @ v[:, :, None]
    if dout is None:
        return o.reshape(q.shape), lse.reshape(B, Hq, Sq)
    do = dout.double().reshape(qg.shape)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = p * (do @ v[:, :, None].transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * scale
    dq = ds @ k[:, :, None]
    dk = (ds.transpose(-1, -2) @ qg).sum(2)
    return o.reshape(q.shape), lse.reshape(B, Hq, Sq), dq.reshape(q.shape), dk, dv
