"""GPU: arguments and values at the ends of what the paged cache's entry points take, against the 64-bit oracle."""
import math

import pytest
import torch

from oracle import window_oracle as orc
from tests.paged_util import make, to_gpu
from tests.test_paged_gpu import check, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("window", [None, 1, 40, 2**31 - 1])
@pytest.mark.parametrize("sinks", [2**31 - 1, 2**31 - 16, 2**40])
@pytest.mark.parametrize("lens", [[180], [900, 0, 31], [600 + 7 * i for i in range(20)], [3 * i for i in range(160)]])
def test_sinks_that_cover_everything(lens, sinks, window, e4m3):
    """Every slot is visible then: parts of rows, one list of all tiles (of more than 16 sequences, too), a part a row."""
    import flex_block_attn_b200 as fba

    pools, table = make(lens, 8, 16, e4m3, seed=len(lens))
    q, n = queries(len(lens), 8, 3), torch.tensor(lens, dtype=torch.int32).cuda()
    o, lse = fba.paged_decode_attn(q.cuda(), to_gpu(pools), table.cuda(), n, window, sinks, need_lse=True)
    check(q, pools, table, lens, o, lse)


@pytest.mark.parametrize("lens,Hkv", [([40], 2), ([900, 30], 2), ([3000], 2), ([1100 + i for i in range(60)], 8)])
def test_heads_without_a_finite_score_add_nothing(lens, Hkv):
    """Keys of -inf under queries that are positive there: no probabilities, zeros, lse of -inf, and weights as they were;
    where only some keys are, the others share what there is.  In one part, in several, in several of many rows."""
    import flex_block_attn_b200 as fba

    page = 32
    pools, table = make(lens, Hkv, page, track=True, seed=21)
    q = queries(len(lens), 2 * Hkv, 5)
    q[..., 0] = q[..., 0].abs() + 1
    for b, n in enumerate(lens):
        for j in range(n):   # all keys of kv head 1, every third one of kv head 0
            row = int(table[b, j // page]), slice(None), j % page
            pools["k"][row][1, 0] = -math.inf
            if j % 3 == 1:
                pools["k"][row][0, 0] = -math.inf
    cache, n = to_gpu(pools), torch.tensor(lens, dtype=torch.int32).cuda()
    o, lse = fba.paged_decode_attn(q.cuda(), cache, table.cuda(), n, need_lse=True, accumulate=True)
    assert not o[:, 2:4].any() and (lse[:, 2:4] == -math.inf).all()
    assert torch.isfinite(o.float()).all() and torch.isfinite(lse[:, :2]).all()
    got = cache.weight.cpu()
    for b, m in enumerate(lens):
        new, was = (orc.rows_of(x, table[b], m, 0).double() for x in (got, pools["weight"]))
        none = torch.arange(m) % 3 == 1
        assert torch.equal(new[none], was[none])
        # two heads' probabilities; a score is a sum of 128 products, off by at most dq, a weight by two fp32 roundings
        k = orc.rows_of(pools["k"], table[b], m, 0).double()[~none]
        dq = 128 * 2.0**-23 * 128**-0.5 * float(q[b].double().norm(dim=-1).max()) * float(k.norm(dim=-1).max())
        assert (new >= was).all() and abs(float((new - was).sum()) - 2) <= 2 * (2 * dq + 1e-6) + 2.0**-23 * float((new + 1).sum())
        assert torch.equal(*(orc.rows_of(x, table[b], m, 1) for x in (got, pools["weight"])))


def test_a_report_ahead_of_a_capture_is_raised_behind_it():
    """The call that is captured neither raises it nor records a clearing of the device's status words."""
    import flex_block_attn_b200 as fba
    from flex_block_attn_b200 import interface

    pools, table = make([80], 1, 16, seed=3)
    q, cache, n = queries(1, 2, 3).cuda(), to_gpu(pools), torch.tensor([80], dtype=torch.int32).cuda()
    good, broken = table.cuda(), table.clone()
    broken[0, 2] = 77
    graph = torch.cuda.CUDAGraph()
    with pytest.MonkeyPatch.context() as m:
        m.setenv("FBA_CHECK_STATUS", "0")
        m.setenv("FBA_POISON_OUTPUTS", "0")
        fba.paged_decode_attn(q, cache, good, n)
        fba.paged_decode_attn(q, cache, broken.cuda(), n)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            o = fba.paged_decode_attn(q, cache, good, n)
        words = interface._monitor(q.device).buf
        words[0] = 1
        graph.replay()
        assert words.tolist() == [1] + [0] * 7
        words.zero_()
        check(q.cpu(), pools, table, [80], o, None)
        with pytest.raises(RuntimeError, match="page number 77"):
            fba.check_status()
        fba.check_status()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens,Hkv", [([700, 64, 0], 2), ([20 * i for i in range(60)], 8)])
def test_a_graph_of_many_steps(lens, Hkv, e4m3):
    """Steps with no other kernel in between, in memory that later steps use again: each reads the lengths and rows of the
    step before it, and none later ones."""
    import flex_block_attn_b200 as fba

    steps, page, B = 12, 32, len(lens)
    pools, table = make([n + steps for n in lens], Hkv, page, e4m3, seed=31)
    g = torch.Generator().manual_seed(32)
    q, k, v = (torch.randn((steps, B, h, 1, 128), generator=g).bfloat16() for h in (2 * Hkv, Hkv, Hkv))
    for b, n in enumerate(lens):   # the rows that the steps write
        for i in range(steps):
            at = int(table[b, (n + i) // page]), slice(None), (n + i) % page
            for name, x in (("k", k), ("v", v)):
                if e4m3:
                    pools[name][at], pools[name + "_scale"][at] = orc.quantize_rows(x[i, b, :, 0])
                else:
                    pools[name][at] = x[i, b, :, 0]
    cache = to_gpu(pools)
    for name in pools:   # not there yet
        x = getattr(cache, name)
        for b, n in enumerate(lens):
            for i in range(steps):
                x[int(table[b, (n + i) // page]), :, (n + i) % page] = 0x7F if x.dtype == torch.uint8 else math.nan
    tab, start, dev = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), [x.cuda() for x in (q, k, v)]
    fba.paged_decode_attn(dev[0][0, :, :, 0].contiguous(), cache, tab, start)
    torch.cuda.synchronize()
    graph, outs = torch.cuda.CUDAGraph(), []
    with pytest.MonkeyPatch.context() as m:
        m.setenv("FBA_POISON_OUTPUTS", "0")
        with torch.cuda.graph(graph):
            n = start
            for i in range(steps):
                n = fba.append_kv(cache, dev[1][i], dev[2][i], tab, n)
                outs.append(fba.paged_decode_attn(dev[0][i, :, :, 0], cache, tab, n, need_lse=True))
    for _ in range(2):
        for o, lse in outs:
            o.fill_(math.nan), lse.fill_(math.nan)
        graph.replay()
    for i, (o, lse) in enumerate(outs):
        check(q[i, :, :, 0], pools, table, [x + i + 1 for x in lens], o, lse)
    fba.check_status()
