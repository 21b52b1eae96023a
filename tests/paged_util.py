"""Paged caches for the tests: random pages in random order, poison wherever no sequence has a row."""
from __future__ import annotations

import math

import torch

from oracle import window_oracle as orc


def make(lens, Hkv, page, e4m3=False, track=False, spare=3, seed=0, std=1.0, max_pages=None):
    """(pools: dict of CPU tensors, table [B, max_pages]); the pages behind a sequence's last are numbered nonsense."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    mp = max_pages or max(1, max(need))
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), mp), -7, dtype=torch.int32)
    table[:, 1::2] = 2**30
    shape = (n_pages, Hkv, page)
    k = torch.full((*shape, 128), math.nan, dtype=torch.bfloat16)
    v = k.clone()
    weight, position = torch.full(shape, math.nan), torch.full(shape, -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        for i in range(need[b]):
            p = int(order[at])
            at += 1
            table[b, i] = p
            rows = min(page, n - i * page)
            k[p, :, :rows] = (torch.randn((Hkv, rows, 128), generator=g) * std).bfloat16()
            v[p, :, :rows] = (torch.randn((Hkv, rows, 128), generator=g) * std).bfloat16()
            weight[p, :, :rows] = torch.rand((Hkv, rows), generator=g) * 8
            position[p, :, :rows] = torch.arange(i * page, i * page + rows, dtype=torch.int32)
    pools = {"k": k, "v": v}
    if e4m3:
        (pools["k"], pools["k_scale"]), (pools["v"], pools["v_scale"]) = orc.quantize_rows(k), orc.quantize_rows(v)
        for x in "kv":   # NaN scales and NaN bytes where there is no row
            pools[x] = torch.where(torch.isnan(pools[x + "_scale"])[..., None], torch.tensor(0x7F, dtype=torch.uint8), pools[x])
    if track:
        pools |= {"weight": weight, "position": position}
    return pools, table


def to_gpu(pools):
    import flex_block_attn_b200 as fba

    return fba.PagedKVCache(**{n: x.cuda() for n, x in pools.items()})


def same(got, want, what=""):
    """Equal, NaN where NaN is."""
    got, want = got.cpu(), want.cpu()
    assert got.dtype == want.dtype and got.shape == want.shape, what
    if got.is_floating_point():
        assert torch.equal(torch.isnan(got), torch.isnan(want)), what
        got, want = torch.nan_to_num(got), torch.nan_to_num(want)
    assert torch.equal(got, want), what
