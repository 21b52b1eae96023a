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


# ------------------------------------------------------------------------------------------------------- paged cache
def quantize_rows(x: torch.Tensor):
    """(e4m3 bytes, fp32 scales) of bf16 rows, as the cache writer defines them."""
    x = x.float()
    most = x.abs().amax(-1)
    scale = torch.where(most > 0, (most * torch.tensor(1 / 448, dtype=torch.float32)).clamp_min(2.0**-126), torch.ones(()))
    bad = ~torch.isfinite(x).all(-1)
    scale = torch.where(bad, torch.full((), math.nan), scale)
    return (x * (1.0 / scale)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), scale


def rows_of(pool: torch.Tensor, table_row, n: int, h: int) -> torch.Tensor:
    """The first n rows of a sequence for kv head h, in slot order: plain loop over its pages."""
    size = pool.shape[2]
    pages = [int(p) for p in table_row[: -(-n // size)]]
    got = [pool[p, h] for p in pages]
    return torch.cat(got)[:n] if got else pool[0, 0][:0]


def decode(q, pools, table, lens, window: Optional[int] = None, sinks: int = 0, softmax_scale: Optional[float] = None):
    """(o, lse, weight per sequence: list of [Hkv, n]) in 64 bits; ``pools``: dict of CPU tensors, k, v and scales."""
    B, Hq, D = q.shape
    Hkv = pools["k"].shape[1]
    G = Hq // Hkv
    scale = 1 / math.sqrt(D) if softmax_scale is None else softmax_scale
    o, lse, weight = torch.zeros((B, Hq, D), dtype=torch.float64), torch.full((B, Hq), -math.inf, dtype=torch.float64), []
    for b, n in enumerate(int(x) for x in lens):
        w = torch.zeros((Hkv, n), dtype=torch.float64)
        j = torch.arange(n)
        vis = torch.ones(n, dtype=torch.bool) if window is None else (n - 1 - j < window) | (j < sinks)
        for h in range(Hkv if n else 0):
            k, v = (rows_of(pools[x], table[b], n, h) for x in "kv")
            if k.dtype == torch.uint8:
                k, v = (x.view(torch.float8_e4m3fn).double() * rows_of(pools[s], table[b], n, h).double()[:, None]
                        for x, s in ((k, "k_scale"), (v, "v_scale")))
            k, v = k.double()[vis], v.double()[vis]
            s = q[b, h * G:(h + 1) * G].double() @ k.T * scale
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(s, -1)
            p = s.softmax(-1)
            o[b, h * G:(h + 1) * G] = p @ v
            w[h, vis] = p.sum(0)
        weight.append(w)
    return o, lse, weight


def evict(pools, table, lens, budget: int, sinks: int = 0, recent: int = 0, next_positions=None, out_table=None):
    """New lengths; ``pools`` (CPU tensors) are changed.  Plain loops over sequences, heads and tokens."""
    size = pools["k"].shape[2]
    fresh = {n: x.clone() for n, x in pools.items()}
    for b, n in enumerate(int(x) for x in lens):
        left = min(n, budget)
        start = (n if next_positions is None else int(next_positions[b])) - recent
        for h in range(pools["k"].shape[1]):
            at = [(int(table[b, j // size]), h, j % size) for j in range(n)]

            def order(j):
                pos, w = int(pools["position"][at[j]]), float(pools["weight"][at[j]])
                return (2 if pos < sinks or pos >= start else 1 if math.isnan(w) else 0, 0.0 if math.isnan(w) else w, j)

            # a protected token's weight does not matter, nor a NaN's sign
            gone = set(sorted(range(n), key=lambda j: order(j) if order(j)[0] == 0 else (order(j)[0], 0.0, j))[: n - left])
            kept = [j for j in range(n) if j not in gone]
            if out_table is not None:
                moves = [(j, (int(out_table[b, i // size]), h, i % size)) for i, j in enumerate(kept)]
            else:
                moves = list(zip((j for j in kept if j >= left), (at[j] for j in range(left) if j in gone)))
            for j, to in moves:
                for name, x in fresh.items():
                    x[to] = pools[name][at[j]]
    for name, x in fresh.items():
        pools[name].copy_(x)
    return [min(int(n), budget) for n in lens]
