"""GPU: eviction by accumulated weight moves exactly the rows that the loop oracle moves."""
import math

import pytest
import torch

from oracle import window_oracle as orc
from tests.paged_util import make, same, to_gpu

pytestmark = pytest.mark.gpu

# lens, kv heads, page, budget, sinks, recent
CASES = [
    ([1], 1, 16, 1, 0, 0),
    ([0, 5], 1, 16, 3, 1, 1),
    ([17], 2, 16, 16, 0, 0),             # one token leaves
    ([100, 3, 64], 2, 16, 64, 4, 10),    # one, none and none
    ([500, 501], 3, 64, 33, 0, 33),      # only the last tokens stay
    ([700], 1, 32, 350, 350, 0),         # only the first
    ([2049, 2000], 2, 64, 2048, 4, 64),
    ([9000], 1, 256, 1000, 4, 100),      # several CTAs a head
    ([5000, 1, 300], 2, 128, 4999, 0, 1),
    ([90] * 40, 4, 16, 50, 2, 2),
]


def run(pools, table, lens, budget, sinks, recent, nxt=None, out=None):
    import flex_block_attn_b200 as fba

    gpu = lambda x: None if x is None else torch.as_tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    cache = to_gpu(pools)
    got = fba.evict_kv(cache, table.cuda(), gpu(lens), budget, sinks, recent, gpu(nxt), gpu(out))
    want = orc.evict(pools, table, lens, budget, sinks, recent, nxt, out)
    assert got.tolist() == want
    for name, x in pools.items():
        same(getattr(cache, name), x, name)
    return cache


def out_table(pools, table, lens, budget, page, seed=0):
    """Pages of the pools that no sequence has, in random order."""
    used = {int(p) for b, n in enumerate(lens) for p in table[b, : -(-n // page)]}
    free = torch.tensor([p for p in range(pools["k"].shape[0]) if p not in used], dtype=torch.int32)
    need = -(-min(budget, table.shape[1] * page) // page)
    free = free[torch.randperm(len(free), generator=torch.Generator().manual_seed(seed))]
    return free[: len(lens) * need].reshape(len(lens), need)


@pytest.mark.parametrize("elsewhere", [False, True])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens,Hkv,page,budget,sinks,recent", CASES)
def test_evict(lens, Hkv, page, budget, sinks, recent, e4m3, elsewhere):
    most = max(1, max(-(-n // page) for n in lens))
    need = -(-min(budget, most * page) // page)
    pools, table = make(lens, Hkv, page, e4m3, track=True, spare=2 + len(lens) * need * elsewhere, seed=budget)
    run(pools, table, lens, budget, sinks, recent, out=out_table(pools, table, lens, budget, page) if elsewhere else None)


@pytest.mark.parametrize("lens,budget", [([300], 100), ([6000], 700), ([6000], 5999)])
def test_equal_special_and_negative_weights(lens, budget):
    """Few distinct weights (the lowest slots leave first), zeros of both signs, infinities and NaN of both signs."""
    pools, table = make(lens, 2, 64, track=True, seed=1)
    g = torch.Generator().manual_seed(2)
    odd = torch.tensor([0.0, -0.0, 1.0, -1.0, math.inf, -math.inf, math.nan, -math.nan, 2.0**-140, 0.5])
    odd[7] = torch.tensor([-1], dtype=torch.int32).view(torch.float32)[0]   # a NaN with its sign set
    pools["weight"] = odd[torch.randint(0, 10, pools["weight"].shape, generator=g)]
    run(pools, table, lens, budget, 2, 3)
    pools["weight"] = torch.ones_like(pools["weight"])
    run(pools, table, lens, budget, 0, 0)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("n,max_pages", [(2, 1), (300, 5), (300, 40), (6000, 94), (18001, 283)])   # one to four CTAs a head
def test_one_token_too_many(n, max_pages, e4m3):
    """The one that leaves first, last, in between and among equals."""
    pools, table = make([n], 2, 64, e4m3, track=True, seed=11, max_pages=max_pages)
    for slots in ([0], [n - 1], [n // 2], [n - 1, n // 2], range(n)):
        for h in range(2):   # of the second head always the slot before the last
            for s in slots if h == 0 else [n - 2]:
                pools["weight"][table[0, s // 64], h, s % 64] = -2.0
        run(pools, table, [n], n - 1, 0, 0)


@pytest.mark.parametrize("lens", [[300], [18001]])
def test_weights_of_few_leading_digits(lens):
    """Distinct weights that agree in their first 11 or 22 bits, where the last to leave shares them with others, and where
    it does not."""
    for step in (2.0**-23, 2.0**-12, 2.0**-2):
        pools, table = make(lens, 2, 64, track=True, seed=12)
        g = torch.Generator().manual_seed(13)
        pools["weight"] = 1.0 + step * torch.randint(0, 400, pools["weight"].shape, generator=g)
        for budget in (lens[0] - 3, lens[0] // 2, 7):
            run({k: x.clone() for k, x in pools.items()}, table, lens, budget, 2, 3)


def test_a_cut_cache_is_cut_again_by_positions():
    """Slots in no order of positions; duplicates that protect more than the budget holds."""
    lens, page = [200, 130], 16
    pools, table = make(lens, 2, page, track=True, seed=3)
    g = torch.Generator().manual_seed(4)
    pools["position"] = torch.randint(0, 5000, pools["position"].shape, generator=g, dtype=torch.int32)
    run(pools, table, lens, 100, 50, 50, nxt=[5000, 4000])
    pools["position"] = torch.zeros_like(pools["position"])
    run(pools, table, [100, 100], 60, 10, 0)


def test_a_wide_table_reads_the_weights_again():
    """A table whose capacity is beyond what the keys have room for in shared memory."""
    for e4m3 in (False, True):
        pools, table = make([3000, 40], 2, 256, e4m3, track=True, seed=5, max_pages=2000)
        run(pools, table, [3000, 40], 1111, 4, 32)


def test_bad_pages_and_lengths_are_reported():
    import flex_block_attn_b200 as fba

    lens = torch.tensor([100], dtype=torch.int32).cuda()
    with pytest.MonkeyPatch.context() as m:
        m.setenv("FBA_CHECK_STATUS", "0")
        pools, table = make([100], 1, 16, track=True, seed=6)
        table[0, 3] = 77
        cache = to_gpu(pools)
        assert fba.evict_kv(cache, table.cuda(), lens, 50).tolist() == [50]
        with pytest.raises(RuntimeError, match="page number 77"):
            fba.check_status()
        pools, table = make([100], 1, 16, track=True, seed=6)
        cache = to_gpu(pools)
        assert fba.evict_kv(cache, table.cuda(), lens - 200, 50).tolist() == [0]
        with pytest.raises(RuntimeError, match="length -100"):
            fba.check_status()
        for name, x in pools.items():
            same(getattr(cache, name), x, name)


@pytest.mark.parametrize("e4m3", [False, True])
def test_serving_within_a_budget(e4m3):
    """append_kv, paged_decode_attn with accumulation and evict_kv, captured once and replayed as a program would, against
    the same steps of the oracle on what the cache held."""
    import flex_block_attn_b200 as fba

    Hq, Hkv, page, budget = 8, 2, 16, 70
    pools, table = make([71, 71], Hkv, page, e4m3, track=True, seed=7)
    lens = torch.tensor([70, 55], dtype=torch.int32)
    cache, tab, n = to_gpu(pools), table.cuda(), lens.cuda()
    nxt = torch.tensor([500, 55], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.zeros((2, h, 128), dtype=torch.bfloat16, device="cuda") for h in (Hq, Hkv, Hkv))

    def step():
        grown = fba.append_kv(cache, k[:, :, None], v[:, :, None], tab, n, positions=nxt)
        nxt.add_(1)
        o = fba.paged_decode_attn(q, cache, tab, grown, accumulate=True)
        n.copy_(fba.evict_kv(cache, tab, grown, budget, 2, 8, nxt))
        return o, grown

    saved = {name: getattr(cache, name).clone() for name in pools}, n.clone(), nxt.clone()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.MonkeyPatch.context() as m:
        m.setenv("FBA_POISON_OUTPUTS", "0")
        with torch.cuda.graph(graph):
            o, grown = step()
    for name, x in saved[0].items():
        getattr(cache, name).copy_(x)
    n.copy_(saved[1])
    nxt.copy_(saved[2])
    for i in range(20):
        x = [torch.randn((2, h, 128), generator=g).bfloat16() for h in (Hq, Hkv, Hkv)]
        for to, new in zip((q, k, v), x):
            to.copy_(new)
        before, m0, p0 = {name: getattr(cache, name).cpu() for name in pools}, n.tolist(), nxt.tolist()
        graph.replay()
        assert grown.tolist() == [a + 1 for a in m0]
        for b in range(2):   # the appended rows
            at = int(table[b, m0[b] // page]), slice(None), m0[b] % page
            for name, new in (("k", x[1]), ("v", x[2])):
                before[name][at] = new[b]
                if e4m3:
                    before[name][at], before[name + "_scale"][at] = orc.quantize_rows(new[b])
            before["weight"][at], before["position"][at] = 0.0, p0[b]
        want, _, weight = orc.decode(x[0], before, table, grown.tolist())
        # P and the result rounded to bf16: 2^-8 of the largest value each, which two norms below 4 bound
        assert (o.cpu().double() - want).abs().max() <= 2 * 2.0**-8 * 4.5
        # the weights as the kernels summed them decide; of what left they are gone, so take the moved ones by position
        for b in range(2):
            for h in range(Hkv):
                pos = orc.rows_of(before["position"], table[b], m0[b] + 1, h)
                total = orc.rows_of(before["weight"], table[b], m0[b] + 1, h).double() + weight[b][h]
                kept = orc.rows_of(cache.position.cpu(), table[b], int(n[b]), h)
                has = orc.rows_of(cache.weight.cpu(), table[b], int(n[b]), h).double()
                index = {int(p): j for j, p in enumerate(pos)}
                assert len(set(kept.tolist())) == len(kept)
                j = torch.tensor([index[int(p)] for p in kept])
                assert ((has - total[j]).abs() <= 1e-3 * weight[b][h][j] + 1e-5).all()
                out = sorted(set(index) - set(kept.tolist()))
                for p in out:   # it was not protected, and nobody unprotected who stays has clearly less
                    assert 2 <= p < p0[b] + 1 - 8
                    free = (kept >= 2) & (kept < p0[b] + 1 - 8)
                    assert (has[free] >= total[index[p]] - 1e-3).all()
                rows = orc.rows_of(cache.k.cpu(), table[b], int(n[b]), h)
                same(rows, orc.rows_of(before["k"], table[b], m0[b] + 1, h)[j], "k")
                same(orc.rows_of(cache.v.cpu(), table[b], int(n[b]), h), orc.rows_of(before["v"], table[b], m0[b] + 1, h)[j], "v")
    fba.check_status()
