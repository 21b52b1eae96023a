"""GPU: the paged cache's writer (exact) and the attention of one new token, against the 64-bit oracle.

Tolerance of o: each probability is rounded to bf16 (relative u = 2^-8) for its product and the result once more, so an
element is off by at most u * (sum p |v| + |o|); the rest is fp32: scores are sums of 128 products, off by at most
128 * 2^-23 * scale * |q| |k| (dq below), which moves a probability by that share.  In an e4m3 cache a weight times its V scale is held in fp16 as a multiple of
2^-7 R, where R is at most twice the largest V scale and the largest weight at least 1: below fp16's normal range it is
off by at most 2^-25 of that, so n keys add at most n * 2^-32 * R * 448 to an element, whatever the key's own weight.
"""
import math

import pytest
import torch

from oracle import window_oracle as orc
from tests.paged_util import make, same, to_gpu

pytestmark = pytest.mark.gpu
U = 2.0**-8


def queries(B, Hq, seed, std=1.0):
    return (torch.randn((B, Hq, 128), generator=torch.Generator().manual_seed(seed)) * std).bfloat16()


def check(q, pools, table, lens, o, lse, window=None, sinks=0, scale=None):
    want, wl, weight = orc.decode(q, pools, table, lens, window, sinks, scale)
    positive = {**pools, "v": (pools["v"] & 0x7F if pools["v"].dtype == torch.uint8 else pools["v"].abs())}
    around = orc.decode(q, positive, table, lens, window, sinks, scale)[0]
    s = 128**-0.5 if scale is None else scale
    kmax = float(values(pools).norm(dim=-1).nan_to_num(0.0, 0.0).max())   # rows of nobody are NaN
    dq = 128 * 2.0**-23 * s * float(q.double().norm(dim=-1).max()) * kmax
    assert torch.isfinite(o.float()).all()
    bound = U * (around + want.abs()) + (2 * dq + 1e-6) * around + 1e-30
    if "v_scale" in pools:
        largest = float(pools["v_scale"].nan_to_num(0.0, 0.0).max())
        bound = bound + torch.tensor([int(n) * 2.0**-31 * largest * 448 for n in lens], dtype=torch.float64)[:, None, None]
    assert ((o.cpu().double() - want).abs() <= bound).all(), float(((o.cpu().double() - want).abs() / bound).max())
    if lse is not None:
        none = wl == -math.inf
        assert torch.equal(lse.cpu() == -math.inf, none)
        assert ((lse.cpu().double() - wl)[~none].abs() <= dq + 1e-6 * wl[~none].abs() + 1e-6).all()
    return weight, dq


def values(pools):
    if pools["k"].dtype == torch.uint8:
        return pools["k"].view(torch.float8_e4m3fn).double() * pools["k_scale"].double()[..., None]
    return pools["k"].double()


# lens, Hq, Hkv, page, window, sinks
CASES = [
    ([1], 1, 1, 16, None, 0),
    ([0], 2, 1, 16, None, 0),
    ([15, 16, 17], 4, 2, 16, None, 0),
    ([0, 100, 0, 1, 33], 6, 2, 32, None, 0),
    ([513], 8, 1, 64, None, 0),              # one sequence over several CTAs
    ([2000, 3, 700], 24, 8, 128, None, 0),
    ([5000], 16, 1, 256, None, 0),           # 16 heads a kv head
    ([300, 1111], 18, 2, 64, None, 0),       # 9
    ([400, 90], 34, 2, 64, None, 0),         # 17: two groups of heads
    ([1000, 20], 5, 1, 64, 100, 0),
    ([1000, 20, 113], 4, 4, 16, 100, 4),
    ([1000, 333], 4, 2, 32, 17, 33),
    ([640], 2, 2, 64, 64, 64),               # window and sinks end at a page
    ([640], 2, 2, 64, 1, 0),                 # only the new token
    ([640, 50], 2, 1, 64, 600, 50),
    ([40] * 150, 4, 2, 16, None, 0),         # many short sequences
    ([700] * 3 + [0] * 40 + [90] * 5, 4, 2, 16, None, 0),
    ([4100, 2900, 0, 600] + [17 * i % 200 for i in range(56)], 16, 8, 64, None, 0),    # 480 rows, of two parts
    ([4100, 2900, 0, 600] + [17 * i % 200 for i in range(60)], 16, 8, 64, 2500, 70),   # 512, with a window
    ([5 * i % 700 for i in range(150)], 8, 8, 64, None, 0),                            # 1200 rows of one part
]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens,Hq,Hkv,page,window,sinks", CASES)
def test_decode(lens, Hq, Hkv, page, window, sinks, e4m3):
    import flex_block_attn_b200 as fba

    pools, table = make(lens, Hkv, page, e4m3, seed=sum(lens) + Hq)
    q = queries(len(lens), Hq, seed=Hq)
    cache, n = to_gpu(pools), torch.tensor(lens, dtype=torch.int32)
    o, lse = fba.paged_decode_attn(q.cuda(), cache, table.cuda(), n.cuda(), window, sinks, need_lse=True)
    check(q, pools, table, lens, o, lse, window, sinks)
    again = fba.paged_decode_attn(q.cuda(), cache, table.cuda(), n.cuda(), window, sinks)
    assert torch.equal(again, o)
    for name, x in pools.items():
        same(getattr(cache, name), x, name)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("std,scale", [(4.0, 1.0), (1.0, 0.01), (1e-3, None)])
def test_decode_large_and_small_scores(std, scale, e4m3):
    import flex_block_attn_b200 as fba

    lens = [1500, 31]
    pools, table = make(lens, 2, 64, e4m3, seed=5, std=std)
    q = queries(2, 8, 6, std)
    o, lse = fba.paged_decode_attn(q.cuda(), to_gpu(pools), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), None, 0,
                                   scale, need_lse=True)
    check(q, pools, table, lens, o, lse, scale=scale)


def test_decode_every_e4m3_value():
    """All finite bytes, subnormals among them, through both products: one key decides, its value row comes out."""
    import flex_block_attn_b200 as fba

    codes = torch.tensor([x for x in range(256) if x & 0x7F != 0x7F], dtype=torch.uint8)
    codes = torch.cat((codes, codes[:2])).reshape(2, 128)
    pools, table = make([2], 1, 16, True, seed=1)
    p = int(table[0, 0])
    pools["k"][p, 0, :2] = codes
    pools["v"][p, 0, :2] = codes
    pools["k_scale"][p, 0, :2] = pools["v_scale"][p, 0, :2] = 1.0
    for d in range(0, 128, 5):   # q picks one dim: scores of +-448 at most, and exact
        q = torch.zeros((1, 1, 128), dtype=torch.bfloat16)
        q[0, 0, d] = 1.0
        o = fba.paged_decode_attn(q.cuda(), to_gpu(pools), table.cuda(), torch.tensor([2], dtype=torch.int32).cuda(), None, 0, 1.0)
        check(q, pools, table, [2], o, None, scale=1.0)


def test_decode_nan_reaches_only_the_heads_that_see_it():
    import flex_block_attn_b200 as fba

    for e4m3 in (False, True):
        pools, table = make([100, 60], 2, 16, e4m3, seed=2)
        page, row = int(table[0, 3]), 5   # slot 53 of sequence 0, kv head 1
        if e4m3:
            pools["k_scale"][page, 1, row] = math.nan
        else:
            pools["k"][page, 1, row, 7] = math.nan
        q = queries(2, 4, 3)
        n = torch.tensor([100, 60], dtype=torch.int32).cuda()
        o, lse = fba.paged_decode_attn(q.cuda(), to_gpu(pools), table.cuda(), n, need_lse=True)
        assert torch.isnan(o[0, 2:]).all() and torch.isnan(lse[0, 2:]).all()
        assert torch.isfinite(o[0, :2]).all() and torch.isfinite(o[1]).all()
        o = fba.paged_decode_attn(q.cuda(), to_gpu(pools), table.cuda(), n, 40, 50)   # sees neither
        assert torch.isfinite(o).all()


@pytest.mark.parametrize("lens,Hq,Hkv,page,e4m3", [([1], 1, 1, 16, False), ([900, 0, 40], 8, 2, 64, False), ([3000], 16, 1, 128, True),
                                                   ([70, 100], 9, 3, 16, True), ([400, 30], 20, 2, 32, False),
                                                   ([4100, 2900, 0] + [13 * i % 150 for i in range(57)], 8, 8, 64, False),
                                                   ([11 * i % 600 for i in range(150)], 16, 8, 32, True)])
def test_accumulated_weights(lens, Hq, Hkv, page, e4m3):
    import flex_block_attn_b200 as fba

    pools, table = make(lens, Hkv, page, e4m3, track=True, seed=9)
    q = queries(len(lens), Hq, 4)
    cache, n = to_gpu(pools), torch.tensor(lens, dtype=torch.int32).cuda()
    plain = fba.paged_decode_attn(q.cuda(), cache, table.cuda(), n)
    same(cache.weight, pools["weight"], "weight")
    o = fba.paged_decode_attn(q.cuda(), cache, table.cuda(), n, accumulate=True)
    assert torch.equal(o, plain)
    weight, dq = check(q, pools, table, lens, o, None)
    got, old = cache.weight.cpu(), pools["weight"]
    rest = torch.ones_like(old, dtype=torch.bool)
    for b, m in enumerate(lens):
        for h in range(Hkv):
            new, was = (orc.rows_of(x, table[b], m, h).double() for x in (got, old))
            # a probability is off by the share dq twice (its score, the sum) and 1e-6, the sum by two fp32 roundings
            assert ((new - was - weight[b][h]).abs() <= (2 * dq + 1e-6) * weight[b][h] + 2.0**-23 * (new + 1)).all()
        for j in range(m):
            rest[table[b, j // page], :, j % page] = False
    same(torch.where(rest, got, 0.0), torch.where(rest, old, 0.0), "rows of nobody")


def test_decode_takes_strided_queries_and_other_streams():
    import flex_block_attn_b200 as fba

    lens = [333, 64]
    pools, table = make(lens, 2, 32, seed=12)
    wide = queries(2, 24, 1).cuda()
    q = wide[:, 4:20:2]   # heads 4, 6, ..., 18 of a wider projection
    stream = torch.cuda.Stream()
    cache, n, tab = to_gpu(pools), torch.tensor(lens, dtype=torch.int32).cuda(), table.cuda()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        o = fba.paged_decode_attn(q, cache, tab, n)
    stream.synchronize()
    check(q.cpu(), pools, table, lens, o, None)


def test_decode_captured_and_replayed_while_lengths_grow():
    import flex_block_attn_b200 as fba

    lens = [900, 64, 0]
    pools, table = make([1100, 300, 300], 2, 32, seed=14)
    cache, n, tab = to_gpu(pools), torch.tensor(lens, dtype=torch.int32).cuda(), table.cuda()
    q = queries(3, 8, 1).cuda()
    fba.paged_decode_attn(q, cache, tab, n)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    with pytest.MonkeyPatch.context() as m:
        m.setenv("FBA_POISON_OUTPUTS", "0")
        for graph, window in zip(graphs, (None, 50)):
            with torch.cuda.graph(graph):
                outs.append(fba.paged_decode_attn(q, cache, tab, n, window))
    for lens in ([901, 65, 1], [1100, 300, 299]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        for graph in graphs:
            graph.replay()
        check(q.cpu(), pools, table, lens, outs[0], None)
        check(q.cpu(), pools, table, lens, outs[1], None, window=50)
    fba.check_status()


def test_bad_pages_and_lengths_are_left_out_and_reported():
    import flex_block_attn_b200 as fba

    with pytest.MonkeyPatch.context() as m:
        m.setenv("FBA_CHECK_STATUS", "0")
        for bad in (-1, 10**9):
            pools, table = make([80], 1, 16, seed=3)
            q = queries(1, 2, 3)
            broken = table.clone()
            broken[0, 2] = bad
            o = fba.paged_decode_attn(q.cuda(), to_gpu(pools), broken.cuda(), torch.tensor([80], dtype=torch.int32).cuda())
            with pytest.raises(RuntimeError, match=f"page number {bad}"):
                fba.check_status()
            fba.check_status()
            kept = torch.cat((table[:, :2], table[:, 3:]), 1)   # the other rows' attention
            check(q, pools, kept, [64], o, None)
        for length in (-5, 81):   # held to nothing, and to the table's 80 slots
            pools, table = make([80], 1, 16, seed=3)
            q = queries(1, 2, 3)
            o = fba.paged_decode_attn(q.cuda(), to_gpu(pools), table.cuda(), torch.tensor([length], dtype=torch.int32).cuda())
            with pytest.raises(RuntimeError, match=f"length {length}"):
                fba.check_status()
            check(q, pools, table, [min(80, max(0, length))], o, None)


# ---------------------------------------------------------------------------------------------------------------- writer
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens,T,new,page,track,layout", [
    ([0], 1, None, 16, False, "bhtd"),
    ([15, 16, 0], 1, None, 16, True, "bthd"),
    ([5, 0, 40], 100, [100, 0, 37], 16, True, "bthd"),
    ([3, 130], 77, [76, 77], 64, False, "wide"),
    ([0, 0], 700, None, 256, True, "bhtd"),
])
def test_append(lens, T, new, page, track, layout, e4m3):
    import flex_block_attn_b200 as fba

    B, Hkv = len(lens), 3
    real = [T] * B if new is None else new
    pools, table = make([a + b for a, b in zip(lens, real)], Hkv, page, e4m3, track, seed=T)
    g = torch.Generator().manual_seed(1)
    width = {"bhtd": 128, "bthd": 128, "wide": 136}[layout]   # wide: slices of one projection with room at the rows' ends
    base = torch.randn((B, 2 * Hkv, T, width) if layout == "bhtd" else (B, T, 2 * Hkv, width), generator=g).bfloat16()

    def views(x):
        x = x if layout == "bhtd" else x.transpose(1, 2)
        return x[:, :Hkv, :, width - 128:], x[:, Hkv:, :, :128]

    k, v = views(base)
    k[0, 0, 0] = 0.0
    if T > 10:
        k[0, 1, 2] *= 2.0**-100
        v[0, 2, 3, 9] = math.inf
        v[0, 1, 3, 9] = math.nan
    cache = to_gpu(pools)
    move = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    pos = [1000 + b for b in range(B)] if track else None
    got = fba.append_kv(cache, *views(base.cuda()), table.cuda(), move(lens), move(new), move(pos))
    assert got.tolist() == [a + b for a, b in zip(lens, real)]
    for name, x in (("k", k), ("v", v)):
        rows, scale = orc.quantize_rows(x) if e4m3 else (x, None)
        for b in range(B):
            for t in range(real[b]):
                at = int(table[b, (lens[b] + t) // page]), slice(None), (lens[b] + t) % page
                pools[name][at] = rows[b, :, t]
                if e4m3:
                    pools[name + "_scale"][at] = scale[b, :, t]
                if track:
                    pools["weight"][at] = 0.0
                    pools["position"][at] = pos[b] + t
    bad = {n: torch.isnan(pools[n + "_scale"]) for n in "kv"} if e4m3 else {}
    for name, x in pools.items():
        got = getattr(cache, name).cpu()
        if name in bad:   # the bytes of a row without a scale stand for nothing
            got, x = (y.masked_fill(bad[name][..., None], 0) for y in (got, x))
        same(got, x, name)


def test_append_beyond_the_table_is_left_out_and_reported():
    import flex_block_attn_b200 as fba

    pools, table = make([32, 32], 2, 16, seed=1)
    cache = to_gpu(pools)
    x = torch.ones((2, 2, 8, 128), dtype=torch.bfloat16, device="cuda")
    with pytest.MonkeyPatch.context() as m:
        m.setenv("FBA_CHECK_STATUS", "0")
        got = fba.append_kv(cache, x, x, table.cuda(), torch.tensor([30, 4], dtype=torch.int32).cuda())
        assert got.tolist() == [32, 12]
        with pytest.raises(RuntimeError, match="for sequence 0"):
            fba.check_status()
    for b, (start, stop) in enumerate(((30, 32), (4, 12))):
        for j in range(start, stop):
            pools["k"][table[b, j // 16], :, j % 16] = 1
    same(cache.k, pools["k"], "k")
    with pytest.MonkeyPatch.context() as m:   # lengths that are none: nothing is written
        m.setenv("FBA_CHECK_STATUS", "0")
        got = fba.append_kv(cache, 2 * x, x, table.cuda(), torch.tensor([-1, 33], dtype=torch.int32).cuda())
        assert got.tolist() == [0, 32]
        with pytest.raises(RuntimeError, match="length"):
            fba.check_status()
    same(cache.k, pools["k"], "k")


def test_prompt_then_tokens_equals_attention_over_the_whole():
    """A padded batch of prompts through sliding_window_attn_func and append_kv, then token by token through append_kv and
    paged_decode_attn: every output is the causal window attention of the whole sequence."""
    import flex_block_attn_b200 as fba

    Hq, Hkv, page, window, sinks, steps = 8, 2, 32, 60, 3, 5
    prompt, T = [150, 97], 150
    g = torch.Generator().manual_seed(3)
    rand = lambda h: torch.randn((2, T + steps, h, 128), generator=g).bfloat16().cuda()  # noqa: E731
    q, k, v = rand(Hq), rand(Hkv), rand(Hkv)
    want = [orc.masked_attention(q[b:b + 1].transpose(1, 2), *(x[b:b + 1].transpose(1, 2) for x in (k, v)),
                                 orc.visible(T + steps, T + steps, window, sinks, "cuda"))[0][0] for b in range(2)]
    most = max(float(x.abs().max()) for x in want)
    cache = fba.new_paged_cache(20, Hkv, page)
    table = torch.randperm(20, generator=g).to(torch.int32)[:12].reshape(2, 6).cuda()
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    o = fba.sliding_window_attn_func(*(x[:, :T].transpose(1, 2).contiguous() for x in (q, k, v)), window, sinks)
    lens = fba.append_kv(cache, k[:, :T].transpose(1, 2), v[:, :T].transpose(1, 2), table, lens, torch.tensor(prompt, dtype=torch.int32).cuda())
    for b, n in enumerate(prompt):
        assert (o[b, :, :n].double() - want[b][:, :n]).abs().max() <= 8 * U * most
    for step in range(steps):
        at = lens.long()
        pick = lambda x: x[torch.arange(2, device="cuda"), at]  # noqa: E731
        lens = fba.append_kv(cache, pick(k)[:, :, None], pick(v)[:, :, None], table, lens)
        o = fba.paged_decode_attn(pick(q), cache, table, lens, window, sinks)
        for b in range(2):
            assert (o[b].double() - want[b][:, prompt[b] + step]).abs().max() <= 8 * U * most
    fba.check_status()


def test_c_callers_with_status_words_on_the_device():
    """The entry points report into device memory as well; fba_check_status reads and clears it."""
    import ctypes

    from flex_block_attn_b200 import _cabi, paged

    lib = _cabi.lib()
    pools, table = make([40], 1, 16, seed=3)
    table[0, 1] = 12345
    tab = table.cuda()
    arg, B, dev = paged._cache_arg(to_gpu(pools), tab)
    status = torch.zeros(8, dtype=torch.int32, device="cuda")
    q, n = queries(1, 2, 3).cuda(), torch.tensor([40], dtype=torch.int32).cuda()
    o = torch.empty_like(q)
    stream = torch.cuda.current_stream().cuda_stream
    rc = lib.fba_paged_decode(ctypes.byref(arg), q.data_ptr(), (ctypes.c_int64 * 2)(256, 128), o.data_ptr(), None, 1, 2,
                              n.data_ptr(), 0, 0, 0.1, 0, None, 0, status.data_ptr(), stream)
    assert rc == 0
    assert lib.fba_check_status(status.data_ptr(), stream) == _cabi.FBA_ERR_BAD_CACHE
    assert b"page number 12345 for sequence 0" in lib.fba_last_error()
    assert lib.fba_check_status(status.data_ptr(), stream) == 0
    check(q.cpu(), pools, torch.cat((table[:, :1], table[:, 2:]), 1), [24], o, None, scale=0.1)


@pytest.mark.parametrize("e4m3", [False, True])
def test_pools_beyond_32_bit_offsets(e4m3):
    """The highest pages of pools of 9 (4.6) GB each: writer, attention and eviction reach the rows they mean."""
    import flex_block_attn_b200 as fba

    n_pages, Hkv, page = 70000, 2, 256
    shape = (n_pages, Hkv, page)
    new = lambda dtype, *more: torch.empty((*shape, *more), dtype=dtype, device="cuda")  # noqa: E731
    kind = torch.uint8 if e4m3 else torch.bfloat16
    cache = fba.PagedKVCache(new(kind, 128), new(kind, 128), weight=new(torch.float32), position=new(torch.int32))
    if e4m3:
        cache.k_scale, cache.v_scale = new(torch.float32), new(torch.float32)
    table = torch.tensor([[n_pages - 1, n_pages - 3, 5]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((1, Hkv, 700, 128), generator=g).bfloat16().cuda() for _ in "kv")
    lens = fba.append_kv(cache, k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    small = fba.new_paged_cache(3, Hkv, page, e4m3, track=True)   # the same in a small pool
    near = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    fba.append_kv(small, k, v, near, torch.zeros(1, dtype=torch.int32, device="cuda"))
    q = queries(1, 8, 2).cuda()
    for step in range(2):
        assert torch.equal(fba.paged_decode_attn(q, cache, table, lens, accumulate=True),
                           fba.paged_decode_attn(q, small, near, lens, accumulate=True))
        for name in ("k", "v", "weight", "position") + (("k_scale", "v_scale") if e4m3 else ()):
            for p, m in zip(table[0].tolist(), near[0].tolist()):
                rows = max(0, min(page, int(lens[0]) - table[0].tolist().index(p) * page))
                assert torch.equal(getattr(cache, name)[p, :, :rows], getattr(small, name)[m, :, :rows]), name
        lens, fewer = fba.evict_kv(cache, table, lens, 300, 4, 10), fba.evict_kv(small, near, lens, 300, 4, 10)
        assert torch.equal(lens, fewer)
