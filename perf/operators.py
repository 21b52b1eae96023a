"""Attention over a sliding window with sinks, and the paged key / value cache that serves it: what is measured.

Kinds of case:

  window   sliding_window_attn_func: causal attention in which a query sees the last `window` keys and the first `sinks`
           ones; forward and backward (grad), or the forward alone (a prompt, or a piece of one behind earlier keys)
  decode   paged_decode_attn: one new token of every sequence over the sequence's pages, bf16 or e4m3
  append   append_kv: new tokens' keys and values into the pages, as they are or as e4m3 with a scale per row
  evict    evict_kv: the tokens of least accumulated attention weight leave; the others go to the pages of another table
  step     append_kv, paged_decode_attn with accumulation and evict_kv: one step of serving within a fixed budget
"""
import math

import torch

own = False

D = 128
E4M3_MAX = 448.0


def _case(kind, name=None, **kw):
    c = {"kind": kind, "B": 1, "Hq": 8, "Hkv": 8}
    if kind == "window":
        c |= {"Sq": 1, "Skv": 1, "window": 0, "sinks": 0, "grad": False, "std": 1.0, "softmax_scale": 0.0}
    else:
        c |= {"page": 64, "e4m3": False, "L": 1, "ragged": False}
    if kind == "decode":
        c |= {"window": 0, "sinks": 0, "std": 1.0, "softmax_scale": 0.0}
    if kind == "append":
        c |= {"T": 1}
    if kind in ("evict", "step"):
        c |= {"budget": 1, "sinks": 0, "recent": 0}
    c.update(kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # Training on long documents with a local window: grouped heads, the largest work of all.
        _case("window", "window_train_long", Hq=16, Hkv=4, Sq=12288, Skv=12288, window=4096, sinks=4, grad=True),
        # A piece of a long prompt behind the keys of the pieces before it.
        _case("window", "window_prompt_piece", Hq=16, Hkv=2, Sq=4096, Skv=20480, window=8192, sinks=64),
        # Odd length, a window of about two tiles, sinks that end inside the second tile.
        _case("window", "window_train_odd", B=2, Hq=8, Hkv=8, Sq=1531, Skv=1531, window=257, sinks=130, grad=True),
        # A short sample, where launches count.
        _case("window", "window_train_short", Hq=4, Hkv=2, Sq=200, Skv=200, window=64, sinks=4, grad=True),
        # One user, a short conversation: the latency of a call.
        _case("decode", "decode_short", Hq=8, Hkv=2, page=16, L=180),
        # A batch of users with conversations of all lengths.
        _case("decode", "decode_batch", B=64, Hq=32, Hkv=8, page=64, L=8192, ragged=True),
        # Two very long documents in an 8-bit cache: the length is split over the chip.
        _case("decode", "decode_long_e4m3", B=2, Hq=24, Hkv=8, page=128, L=131072, e4m3=True),
        # A model with a local window serving long sequences: most pages are not read.
        _case("decode", "decode_window", B=16, Hq=64, Hkv=8, page=32, L=30011, ragged=True, window=4096, sinks=4),
        # The keys and values of a batch of prompts into an 8-bit cache.
        _case("append", "append_prompts_e4m3", B=4, Hkv=8, page=64, T=8192, L=8192, e4m3=True, ragged=True),
        # One token of every user: the smallest call.
        _case("append", "append_token", B=64, Hkv=8, page=64, T=1, L=4096, ragged=True),
        # Long prompts cut to a budget; their pages stay as they are (others share them).
        _case("evict", "evict_prompts", B=4, Hkv=8, page=64, L=32768, ragged=True, budget=4096, sinks=4, recent=256),
        # Serving with a fixed budget per sequence: a step in, a step out.
        _case("step", "step_budget", B=16, Hq=32, Hkv=8, page=64, L=2049, budget=2048, sinks=4, recent=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["window", "window", "window", "decode", "decode", "append", "evict", "step"])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16])
    B = _log_int(rng, 1, 64)
    if kind == "window":
        Sq = _log_int(rng, 1, 12288)
        Skv = rng.choice([Sq, Sq, Sq + _log_int(rng, 1, 12288), max(1, Sq - _log_int(rng, 1, 200))])
        return _case(kind, B=rng.choice([1, 1, 2, 3]), Hq=Hkv * group, Hkv=Hkv, Sq=Sq, Skv=Skv,
                     window=rng.choice([0, _log_int(rng, 1, Skv), _log_int(rng, 1, Skv)]),
                     sinks=rng.choice([0, 1, 4, rng.randint(2, 300)]), grad=rng.random() < 0.6,
                     std=rng.choice([1.0, 1.0, 0.5]), softmax_scale=rng.choice([0.0, 0.0, 0.07]))
    base = {"B": B, "Hq": Hkv * group, "Hkv": Hkv, "page": rng.choice([16, 32, 64, 128, 256]), "e4m3": rng.random() < 0.5,
            "ragged": rng.random() < 0.7}
    L = _log_int(rng, 1, 131072)
    if kind == "decode":
        return _case(kind, **base, L=L, window=rng.choice([0, 0, _log_int(rng, 1, L)]), sinks=rng.choice([0, 4, 70]),
                     std=rng.choice([1.0, 0.5]), softmax_scale=rng.choice([0.0, 0.0, 0.07]))
    if kind == "append":
        T = rng.choice([1, _log_int(rng, 1, 16384)])
        return _case(kind, **base, T=T, L=T + rng.choice([0, _log_int(rng, 1, 4096)]))
    L = max(2, L)
    recent, sinks = rng.choice([0, 1, 32]), rng.choice([0, 4])
    if kind == "step":
        L = _log_int(rng, 50, 16384)
        return _case(kind, **base, L=L + 1, budget=L, sinks=sinks, recent=recent)
    budget = max(sinks + recent, _log_int(rng, 1, L))
    return _case(kind, **base, L=L, budget=budget, sinks=sinks, recent=recent)


def _cells(c):   # values of the largest array of the plain form
    if c["kind"] == "window":
        return c["B"] * c["Hq"] * c["Sq"] * c["Skv"]
    return c["B"] * c["Hkv"] * D * -(-c["L"] // c["page"]) * c["page"]


def draw(rng):
    cases = listed()
    flops, size = max(work(c)["flops"] for c in cases), max(work(c)["bytes"] for c in cases)
    cells = {k: max(_cells(c) for c in cases if (c["kind"] == "window") == k) for k in (True, False)}
    while True:
        c = _draw(rng)
        w = work(c)
        if w["flops"] <= flops and w["bytes"] <= size and _cells(c) <= cells[c["kind"] == "window"]:
            return c


# ----------------------------------------------------------------------------------------------------------------- inputs
def _quantised(x):
    """e4m3 and fp32 scales of bf16 rows (see append_kv)."""
    x = x.float()
    most = x.abs().amax(-1)
    scale = torch.where(most > 0, (most * torch.tensor(1 / E4M3_MAX, dtype=torch.float32, device=x.device)).clamp_min(2.0**-126), 1.0)
    return (x * (1.0 / scale)[..., None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    rand = lambda *shape: torch.rand(shape, generator=g, device="cuda")  # noqa: E731
    s = {"case": c, "softmax_scale": c.get("softmax_scale") or None}
    if c["kind"] == "window":
        for name, heads, rows in (("q", c["Hq"], c["Sq"]), ("k", c["Hkv"], c["Skv"]), ("v", c["Hkv"], c["Skv"]), ("do", c["Hq"], c["Sq"])):
            s[name] = randn(c["B"], heads, rows, D).mul_(c["std"])
        if c["grad"]:
            for name in "qkv":
                s[name].requires_grad_()
        return s

    B, Hkv, page = c["B"], c["Hkv"], c["page"]
    mp = -(-c["L"] // page)
    tables = 2 if c["kind"] == "evict" else 1
    order = torch.randperm(tables * B * mp, generator=g, device="cuda").to(torch.int32).reshape(tables, B, mp)
    s["table"] = order[0].contiguous()
    shape = (tables * B * mp, Hkv, page)
    k, v = randn(*shape, D).mul_(c.get("std", 1.0)), randn(*shape, D).mul_(c.get("std", 1.0))
    s["k_scale"] = s["v_scale"] = None
    if c["e4m3"]:
        (k, s["k_scale"]), (v, s["v_scale"]) = _quantised(k), _quantised(v)
        k, v = k.view(torch.uint8), v.view(torch.uint8)
    s["k"], s["v"] = k, v
    lens = torch.full((B,), c["L"], dtype=torch.int32, device="cuda")
    if c["ragged"]:
        least = max(1, c["L"] // 16) if c["kind"] == "decode" else max(1, c["L"] // 2)
        lens = (least + (rand(B) * (c["L"] - least + 1)).floor().clamp_max(c["L"] - least)).to(torch.int32)
        lens[B // 2] = c["L"]
    if c["kind"] in ("decode", "step"):
        s["q"] = randn(B, c["Hq"], D).mul_(c.get("std", 1.0))
    if c["kind"] in ("append", "step"):
        T = c.get("T", 1)
        s["new_k"], s["new_v"] = randn(B, T, Hkv, D).transpose(1, 2), randn(B, T, Hkv, D).transpose(1, 2)   # as a projection leaves them
        s["new"] = None
        if T > 1 and c["ragged"]:   # a padded batch of prompts
            s["new"] = (1 + (rand(B) * T).floor().clamp_max(T - 1)).to(torch.int32)
        lens = (lens - T).clamp_min(0)
    if c["kind"] in ("evict", "step"):
        s["weight"] = rand(*shape) * 8   # sums of probabilities over many steps and the heads of a group
        at = torch.arange(mp * page, dtype=torch.int32, device="cuda").reshape(1, mp, page).expand(B, mp, page)
        s["position"] = torch.zeros(shape, dtype=torch.int32, device="cuda")
        s["position"][s["table"].long().reshape(-1)] = at.reshape(B * mp, 1, page).expand(B * mp, Hkv, page).contiguous()
        s["next"] = lens.clone()
    if c["kind"] == "step":   # a cache that has been cut before: its slots are in no order
        s["next"] = lens + 5000
    s["lens"] = lens
    if c["kind"] == "evict":
        s["out_table"] = order[1][:, : -(-min(c["budget"], c["L"]) // page)].contiguous()
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _masked_softmax(x, mask):
    """(probabilities, log of the sum of exponentials) over the last axis; zeros and -inf where a row's mask leaves nothing."""
    x = x.masked_fill(~mask, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m > -math.inf, m, 0.0)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0), (m + torch.log(total)).squeeze(-1)


def _window_plain(s):
    c = s["case"]
    B, Hkv, G, Sq, Skv = c["B"], c["Hkv"], c["Hq"] // c["Hkv"], c["Sq"], c["Skv"]
    scale = s["softmax_scale"] or 1 / math.sqrt(D)
    with torch.no_grad():
        q = s["q"].float().reshape(B, Hkv, G * Sq, D)
        k, v = s["k"].float(), s["v"].float()
        at = torch.arange(Sq, device=q.device)[:, None] + (Skv - Sq)
        j = torch.arange(Skv, device=q.device)[None]
        mask = j <= at
        if c["window"]:
            mask = mask & ((at - j < c["window"]) | (j < c["sinks"]))
        p, _ = _masked_softmax(((q @ k.transpose(-1, -2)) * scale).reshape(B, Hkv, G, Sq, Skv), mask)
        p = p.reshape(B, Hkv, G * Sq, Skv)
        o = p @ v
        out = o.reshape(B, c["Hq"], Sq, D).to(torch.bfloat16)
        if not c["grad"]:
            return {"o": out}
        do = s["do"].float().reshape(B, Hkv, G * Sq, D)
        dv = p.transpose(-1, -2) @ do
        ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * scale
        dq, dk = (ds @ k).reshape(B, c["Hq"], Sq, D), ds.transpose(-1, -2) @ q
        return {"o": out, "dq": dq.to(torch.bfloat16), "dk": dk.to(torch.bfloat16), "dv": dv.to(torch.bfloat16)}


def _rows(s, name):
    """A pool's rows in the order of the sequences' slots, [B, Hkv, slots, ...]."""
    x = s[name][s["table"].long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], x.shape[2] * x.shape[3], *x.shape[4:])


def _values(s, name):
    x = _rows(s, name)
    if not s["case"]["e4m3"]:
        return x.float()
    return x.view(torch.float8_e4m3fn).float() * _rows(s, name + "_scale")[..., None]


def _places(s):
    """(page, kv head, row) of every slot of every sequence, as indices that broadcast to [B, Hkv, slots]."""
    page = s["case"]["page"]
    j = torch.arange(s["table"].shape[1] * page, device=s["table"].device)
    h = torch.arange(s["case"]["Hkv"], device=j.device)
    return s["table"].long()[:, j // page][:, None], h[None, :, None], (j % page)[None, None]


def _decode_plain(s, lens, accumulate=False):
    c = s["case"]
    B, Hkv, G = c["B"], c["Hkv"], c["Hq"] // c["Hkv"]
    k, v = _values(s, "k"), _values(s, "v")
    j = torch.arange(k.shape[2], device=k.device)[None]
    mask = j < lens[:, None]
    if c.get("window"):
        mask = mask & ((lens[:, None] - 1 - j < c["window"]) | (j < c["sinks"]))
    x = (s["q"].float().reshape(B, Hkv, G, D) @ k.transpose(-1, -2)) * (s["softmax_scale"] or 1 / math.sqrt(D))
    p, lse = _masked_softmax(x, mask[:, None, None])
    o = p @ v.masked_fill(~mask[:, None, :, None], 0.0)
    if accumulate:
        at = _places(s)
        s["weight"][at] = s["weight"][at] + p.sum(2)
    return o.reshape(B, c["Hq"], D).to(torch.bfloat16), lse.reshape(B, c["Hq"])


def _append_plain(s):
    c = s["case"]
    T, page = s["new_k"].shape[2], c["page"]
    t = torch.arange(T, device=s["lens"].device)
    b = torch.arange(c["B"], device=t.device)[:, None].expand(-1, T).reshape(-1)
    t = t.expand(c["B"], -1).reshape(-1)
    if s["new"] is not None:
        real = (t < s["new"][b]).nonzero().squeeze(-1)
        b, t = b[real], t[real]
    slot = (s["lens"][b] + t).long()
    pg, row = s["table"].long()[b, slot // page], slot % page
    for name, new in (("k", s["new_k"]), ("v", s["new_v"])):
        x = new[b, :, t]
        if c["e4m3"]:
            x, s[name + "_scale"][pg, :, row] = _quantised(x)
            x = x.view(torch.uint8)
        s[name][pg, :, row] = x
    if "weight" in s:
        s["weight"][pg, :, row] = 0.0
        s["position"][pg, :, row] = (s["next"][b] + t.to(torch.int32))[:, None].expand(-1, c["Hkv"])
    return s["lens"] + (T if s["new"] is None else s["new"])


def _evict_plain(s, lens):
    c = s["case"]
    weight, position = _rows(s, "weight"), _rows(s, "position")
    j = torch.arange(weight.shape[2], device=weight.device)[None, None]
    n, left = lens[:, None, None], lens.clamp_max(c["budget"])[:, None, None]
    stays = (position < c["sinks"]) | (position >= s["next"][:, None, None] - c["recent"]) | (j >= n)
    order = weight.masked_fill(stays, math.inf).sort(dim=-1, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, j.expand_as(order).contiguous())
    kept = (rank >= n - left) & (j < n)
    if "out_table" in s:   # the i-th token that stays goes to slot i
        table = s["out_table"].long()
        source = (~kept).sort(dim=-1, stable=True).indices[:, :, : table.shape[1] * c["page"]]
    else:                  # the i-th token behind the budget goes to the i-th slot that came free
        table = s["table"].long()
        hole = ~kept & (j < left)
        movers = (~(kept & (j >= left))).sort(dim=-1, stable=True).indices
        source = torch.where(hole, movers.gather(-1, (hole.cumsum(-1) - 1).clamp_min(0)), j)
    valid = j[:, :, : source.shape[2]] < left
    for name in ("k", "v", "k_scale", "v_scale", "weight", "position"):
        if s[name] is None:
            continue
        rows, old = _rows(s, name), s[name][table].transpose(1, 2)   # old: [B, Hkv, pages, page, ...]
        wide = (1,) * (rows.dim() - 3)
        rows = rows.gather(2, source.reshape(*source.shape, *wide).expand(*source.shape, *rows.shape[3:]))
        rows = torch.where(valid.reshape(*valid.shape[:2], -1, *wide), rows, old.reshape(rows.shape))
        s[name][table] = rows.reshape(old.shape).transpose(1, 2)
    return left.reshape(-1)


def _pools(s):
    got = {"k": s["k"], "v": s["v"]}
    if s["case"]["e4m3"]:
        got = {n: x.view(torch.float8_e4m3fn) for n, x in got.items()} | {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return got | ({"weight": s["weight"], "position": s["position"]} if "weight" in s else {})


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        import flex_block_attn_b200 as fba

        if kind == "window":
            with torch.set_grad_enabled(c["grad"]):
                o = fba.sliding_window_attn_func(s["q"], s["k"], s["v"], c["window"] or None, c["sinks"], s["softmax_scale"])
            if not c["grad"]:
                return {"o": o}
            dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
            return {"o": o, "dq": dq, "dk": dk, "dv": dv}
        cache = fba.PagedKVCache(s["k"], s["v"], s["k_scale"], s["v_scale"], s.get("weight"), s.get("position"))
        if kind == "decode":
            o, lse = fba.paged_decode_attn(s["q"], cache, s["table"], s["lens"], c["window"] or None, c["sinks"],
                                           s["softmax_scale"], need_lse=True)
            return {"o": o, "lse": lse}
        if kind == "append":
            return {"lens": fba.append_kv(cache, s["new_k"], s["new_v"], s["table"], s["lens"], s["new"])} | _pools(s)
        if kind == "evict":
            lens = fba.evict_kv(cache, s["table"], s["lens"], c["budget"], c["sinks"], c["recent"], s["next"], s["out_table"])
            return {"lens": lens} | _pools(s)
        lens = fba.append_kv(cache, s["new_k"], s["new_v"], s["table"], s["lens"], positions=s["next"])
        s["next"].add_(1)
        o = fba.paged_decode_attn(s["q"], cache, s["table"], lens, accumulate=True)
        lens = fba.evict_kv(cache, s["table"], lens, c["budget"], c["sinks"], c["recent"], s["next"])
        return {"o": o, "lens": lens} | _pools(s)
    if kind == "window":
        return _window_plain(s)
    if kind == "decode":
        o, lse = _decode_plain(s, s["lens"])
        return {"o": o, "lse": lse}
    if kind == "append":
        return {"lens": _append_plain(s)} | _pools(s)
    if kind == "evict":
        return {"lens": _evict_plain(s, s["lens"])} | _pools(s)
    lens = _append_plain(s)
    s["next"].add_(1)
    o, _ = _decode_plain(s, lens, accumulate=True)
    return {"o": o, "lens": _evict_plain(s, lens)} | _pools(s)


# ------------------------------------------------------------------------------------------------------------------- work
def _seen(length, offset, n, window, sinks):
    """Visible (query, key) pairs: queries at positions offset .. offset + n - 1 over `length` keys."""
    at = torch.arange(offset, offset + n, dtype=torch.int64)
    at = at[at >= 0]
    if not window:
        return int((at + 1).sum())
    local = (at + 1).clamp_max(window)
    return int((local + (at + 1 - local).clamp_max(sinks)).sum())


def _mean_len(c):
    if not c["ragged"]:
        return c["L"]
    least = max(1, c["L"] // 16) if c["kind"] == "decode" else max(1, c["L"] // 2)
    return ((c["B"] - 1) * (least + c["L"]) / 2 + c["L"]) / c["B"]


def work(case):
    c = case
    if c["kind"] == "window":
        q, kv = 2 * D * c["B"] * c["Hq"] * c["Sq"], 2 * D * c["B"] * c["Hkv"] * c["Skv"]
        pairs = c["B"] * c["Hq"] * _seen(c["Skv"], c["Skv"] - c["Sq"], c["Sq"], c["window"], c["sinks"])
        if c["grad"]:   # q, k, v, dO in; O, dQ, dK, dV out
            return {"bytes": 4 * q + 4 * kv, "flops": 14 * D * pairs}
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * D * pairs}
    row = D + 4 if c["e4m3"] else 2 * D   # one key or value row of one head
    heads = c["B"] * c["Hkv"]
    length = _mean_len(c)
    if c["kind"] == "append":
        n = c["T"] if c["T"] == 1 or not c["ragged"] else (c["T"] + 1) / 2
        return {"bytes": heads * n * 2 * (2 * D + row) + 12 * c["B"], "flops": 0}
    seen = length if not c.get("window") else min(length, c["window"] + c["sinks"])
    decode = {"bytes": heads * seen * 2 * row + c["B"] * c["Hq"] * 4 * D, "flops": 4 * D * c["B"] * c["Hq"] * seen}
    if c["kind"] == "decode":
        return decode
    left = min(length, c["budget"])
    if c["kind"] == "evict":   # weights and positions in; the rows that stay in and out
        return {"bytes": heads * (length * 8 + left * 2 * (2 * row + 8)), "flops": 0}
    # step: the decode, a row in, weights in and out and in again with the positions, a row over a free slot
    return {"bytes": decode["bytes"] + heads * (2 * (2 * D + row) + length * 16 + 4 * row), "flops": decode["flops"]}


# ------------------------------------------------------------------------------------------------------------------ exact
def _attend64(q, k, v, visible, scale):
    """softmax over the visible keys, times v, and the log of the sum, in 64 bits; q [n, D], k, v [m, D], visible [n, m]."""
    x = (q @ k.T * scale).masked_fill_(~visible, -math.inf)
    lse = torch.logsumexp(x, -1)
    p = (x - lse.masked_fill(lse == -math.inf, 0.0)[:, None]).exp_()
    return p @ v, lse, p


def exact(case, seed):
    c = case
    if c["kind"] == "evict" or (c["kind"] == "append" and not c["e4m3"]):
        return None
    s = prepare(case, seed)
    scale = s["softmax_scale"] or D**-0.5
    G = c["Hq"] // c["Hkv"]
    if c["kind"] == "append":   # the scales that change; the rest stands as it was
        most = {n: s["new_" + n].double().abs().amax(-1) for n in "kv"}
        new = [c["T"]] * c["B"] if s["new"] is None else s["new"].tolist()
        for b, start in enumerate(s["lens"].tolist()):
            slot = torch.arange(start, start + new[b], device="cuda")
            at = s["table"][b].long()[slot // c["page"]], slot % c["page"]
            for n in "kv":
                s[n + "_scale"][at[0], :, at[1]] = (most[n][b, :, : new[b]] / E4M3_MAX).T.float()
        return {"k_scale": s["k_scale"].double(), "v_scale": s["v_scale"].double()}
    if c["kind"] == "window":
        if c["B"] * c["Hq"] * c["Sq"] * c["Skv"] > 6e9:
            return None
        rows = torch.arange(c["Skv"] - c["Sq"], c["Skv"], device="cuda")
        keys = torch.arange(c["Skv"], device="cuda")
        far = rows[:, None] - keys[None]
        visible = far >= 0
        if c["window"]:
            visible &= (far < c["window"]) | (keys[None] < c["sinks"])
        got = {n: torch.zeros_like(s[m], dtype=torch.float64) for n, m in (("o", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
        for b in range(c["B"]):
            for h in range(c["Hq"]):
                q, k, v, do = (s[n].detach()[b, i].double() for n, i in (("q", h), ("k", h // G), ("v", h // G), ("do", h)))
                o, _, p = _attend64(q, k, v, visible, scale)
                got["o"][b, h] = o
                if c["grad"]:
                    got["dv"][b, h // G] += p.T @ do
                    p *= (do @ v.T).sub_((do * o).sum(-1, keepdim=True))
                    got["dq"][b, h] = p @ k * scale
                    got["dk"][b, h // G] += p.T @ q * scale
        return got if c["grad"] else {"o": got["o"]}
    o = torch.zeros((c["B"], c["Hq"], D), dtype=torch.float64, device="cuda")
    lse = torch.zeros((c["B"], c["Hq"]), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, : -(-n // c["page"])].long()
        for h in range(c["Hkv"]):
            k, v = (s[name][pages, h].reshape(-1, D)[:n] for name in "kv")
            if c["e4m3"]:
                k, v = (x.view(torch.float8_e4m3fn).double() * s[name + "_scale"][pages, h].reshape(-1)[:n, None].double()
                        for name, x in (("k", k), ("v", v)))
            k, v = k.double(), v.double()
            if c["kind"] == "step":   # behind the new token's rows
                new = [s["new_" + name][b, h] for name in "kv"]
                if c["e4m3"]:
                    new = [x.double() * r[..., None].double() for x, r in map(_quantised, new)]
                k, v = (torch.cat((x, y.double())) for x, y in zip((k, v), new))
            m = k.shape[0]
            visible = torch.ones((1, m), dtype=torch.bool, device="cuda")
            if c.get("window"):
                visible[0, min(c["sinks"], m): max(0, m - c["window"])] = False
            o[b, h * G: (h + 1) * G], lse[b, h * G: (h + 1) * G], _ = _attend64(
                s["q"][b, h * G: (h + 1) * G].double(), k, v, visible, scale)
    return {"o": o, "lse": lse} if c["kind"] == "decode" else {"o": o}
