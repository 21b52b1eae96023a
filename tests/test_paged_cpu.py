"""CPU: refusals of the paged cache's entry points, and the oracle they are tested against."""
import ctypes
import math

import pytest
import torch

import flex_block_attn_b200 as fba
from oracle import window_oracle as orc
from tests.paged_util import make


def test_oracle_decode_is_the_last_row_of_masked_attention():
    lens = [37, 1, 0]
    pools, table = make(lens, 2, 16, seed=4)
    q = torch.randn((3, 6, 128), generator=torch.Generator().manual_seed(0)).bfloat16()
    for window, sinks in ((None, 0), (5, 2)):
        o, lse, weight = orc.decode(q, pools, table, lens, window, sinks)
        for b, n in enumerate(lens[:2]):
            k, v = (torch.stack([orc.rows_of(pools[x], table[b], n, h) for h in range(2)])[None] for x in "kv")
            want = orc.masked_attention(q[b][None, :, None], k, v, orc.visible(1, n, window, sinks))
            assert torch.allclose(o[b], want[0][0, :, 0]) and torch.allclose(lse[b], want[1][0, :, 0])
            assert torch.allclose(weight[b].sum(-1), torch.full((2,), 3.0, dtype=torch.float64))
        assert not o[2].any() and (lse[2] == -math.inf).all()


def test_oracle_rows_in_e4m3():
    x = torch.zeros((4, 128), dtype=torch.bfloat16)
    x[1, 3], x[1, 4] = 2.0, -1.0
    x[2, 0] = math.nan
    x[3, 0] = 2.0**-130
    bytes_, scale = orc.quantize_rows(x)
    assert scale[0] == 1 and not bytes_[0].any() and torch.isnan(scale[2]) and scale[3] == 2.0**-126
    assert abs(float(scale[1]) * 448 - 2) < 1e-6
    assert bytes_[1].view(torch.float8_e4m3fn).float()[[3, 4]].tolist() == [448.0, -224.0]


def cache(**more):
    x = torch.zeros((4, 2, 16, 128), dtype=torch.bfloat16)
    return fba.PagedKVCache(**({"k": x, "v": x.clone()} | more))


def test_cpu_caches_are_refused():
    table, lens = torch.zeros((1, 4), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    new = torch.zeros((1, 2, 1, 128), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fba.append_kv(cache(), new, new, table, lens)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fba.paged_decode_attn(torch.zeros((1, 4, 128), dtype=torch.bfloat16), cache(), table, lens)


def test_new_cache():
    c = fba.new_paged_cache(5, 2, 32, e4m3=True, track=True, device="cpu")
    assert c.k.shape == c.v.shape == (5, 2, 32, 128) and c.k.dtype == torch.uint8
    assert c.k_scale.shape == c.position.shape == c.weight.shape == (5, 2, 32) and c.position.dtype == torch.int32
    c = fba.new_paged_cache(5, 2, 32, device="cpu")
    assert c.k.dtype == torch.bfloat16 and c.k_scale is c.weight is c.position is None
    assert c.dequantize()[0].dtype == torch.float32


@pytest.fixture(scope="module")
def lib():
    from flex_block_attn_b200 import _cabi
    from flex_block_attn_b200.build import build_library

    build_library()
    return _cabi.lib()


def struct(**more):
    from flex_block_attn_b200._cabi import FbaPaged

    fields = {"k": 256, "v": 256, "table": 256, "n_pages": 4, "Hkv": 2, "page_size": 16, "max_pages": 3, "e4m3": 0} | more
    return ctypes.byref(FbaPaged(**fields))


BAD_CACHES = [{"k": None}, {"table": None}, {"n_pages": 0}, {"Hkv": 0}, {"max_pages": 0}, {"page_size": 8}, {"page_size": 48},
              {"page_size": 512}, {"e4m3": 1}, {"weight": 256}, {"position": 256}, {"k": 264}]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_c_entry_points_refuse_bad_caches(lib, bad):
    some, three, two = ctypes.c_void_p(256), (ctypes.c_int64 * 3)(8, 8, 8), (ctypes.c_int64 * 2)(8, 8)
    assert lib.fba_paged_append(struct(**bad), some, some, three, three, 1, 1, some, None, None, None, some, None) == -1
    assert lib.fba_paged_decode(struct(**bad), some, two, some, some, 1, 4, some, 0, 0, 0.1, 0, some, 2**40, some, None) == -1
    assert lib.fba_last_error()


def test_c_append_refuses_bad_arguments(lib):
    some, good = ctypes.c_void_p(256), (ctypes.c_int64 * 3)(8, 8, 8)
    call = lambda k=some, ks=good, vs=good, B=1, T=1, lens=some, out=None, c=None: lib.fba_paged_append(  # noqa: E731
        c or struct(), k, some, ks, vs, B, T, lens, None, None, out, some, None)
    assert call(k=None) == -1 and call(lens=None) == -1 and call(ks=None) == -1
    assert call(B=0) == -1 and call(T=0) == -1 and call(T=-4) == -1
    assert call(out=some) == -1 and b"out_lens" in lib.fba_last_error()
    assert call(ks=(ctypes.c_int64 * 3)(8, 4, 8)) == -1 and call(vs=(ctypes.c_int64 * 3)(8, 8, 1)) == -1
    assert call(k=ctypes.c_void_p(264)) == -1
    assert call(B=70000) == -5 and call(T=2**31 - 1) == -5 and call(T=2**29 + 1) == -5
    assert call(c=struct(max_pages=2**26)) == -5


def test_c_decode_refuses_bad_arguments(lib):
    some, two = ctypes.c_void_p(256), (ctypes.c_int64 * 2)(512, 128)
    n = ctypes.c_uint64()

    def call(c=None, q=some, qs=two, lse=some, B=1, Hq=4, lens=some, window=0, sinks=0, scale=0.1, acc=0, ws=some, n=2**40):
        return lib.fba_paged_decode(c or struct(), q, qs, some, lse, B, Hq, lens, window, sinks, scale, acc, ws, n, some, None)

    assert call(q=None) == -1 and call(lens=None) == -1 and call(Hq=3) == -1 and call(Hq=0) == -1
    assert call(window=-1) == -1 and call(sinks=-1) == -1
    for scale in (0.0, -1.0, math.nan, math.inf):
        assert call(scale=scale) == -1
    assert call(q=ctypes.c_void_p(258)) == -1 and call(qs=(ctypes.c_int64 * 2)(512, 127)) == -1
    track = {"weight": 256, "position": 256}
    assert call(acc=1) == -1 and call(struct(**track), acc=1, window=5) == -1 and call(struct(**track), acc=1, lse=None) == -1
    assert call(struct(**track), acc=1, Hq=34) == -1
    long = {"max_pages": 1000}
    assert lib.fba_paged_decode_workspace_bytes(1, 4, 2, 16, 1000, 0, 0, ctypes.byref(n)) == 0 and n.value > 0
    assert call(struct(**long), ws=None) == -1 and call(struct(**long), n=n.value - 1) == -1
    assert call(struct(**long), ws=ctypes.c_void_p(128)) == -1
    assert b"workspace" in lib.fba_last_error()
    assert lib.fba_paged_decode_workspace_bytes(1, 4, 2, 16, 3, 0, 0, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.fba_paged_decode_workspace_bytes(1, 4, 3, 16, 3, 0, 0, ctypes.byref(n)) == -1
    assert lib.fba_paged_decode_workspace_bytes(1, 4, 2, 16, 3, 0, 0, None) == -1
    assert lib.fba_paged_decode_workspace_bytes(1, 4, 2, 16, 2**26, 0, 0, ctypes.byref(n)) == -5
    assert lib.fba_paged_decode_workspace_bytes(65535, 4, 2, 256, 2**21, 0, 0, ctypes.byref(n)) == -5


@pytest.mark.parametrize("e4m3", [0, 1])
@pytest.mark.parametrize("B,Hq,Hkv,page,mp", [(1, 1, 1, 16, 40), (30, 32, 8, 64, 128), (64, 32, 8, 64, 128), (200, 34, 2, 16, 400),
                                              (300, 34, 2, 16, 100)])
def test_workspace_holds_a_slot_for_every_part(lib, B, Hq, Hkv, page, mp, e4m3):
    """Few rows: a CTA's part of a row goes to slot CTA + row, both counted from 0.  Many: parts of a row side by side."""
    n = ctypes.c_uint64()
    assert lib.fba_paged_decode_workspace_bytes(B, Hq, Hkv, page, mp, e4m3, 0, ctypes.byref(n)) == 0
    group = Hq // Hkv
    nt = 2 if group > 8 else 1
    rows = B * Hkv * -(-group // (8 * nt))
    tiles = mp * page // 16
    slots = min(148 * (3 if e4m3 and nt == 1 else 2), -(-rows * tiles // 16)) + rows
    if rows >= 444:
        slots = rows * max(1, min(-(-1184 // rows), tiles // 128))
        if slots == rows:
            assert n.value == 0   # nothing to join
            return
    assert n.value >= slots * 8 * nt * (128 + 2) * 4


def test_oracle_evict_by_hand():
    pools, table = make([6], 1, 16, track=True, seed=0, spare=2)
    p = int(table[0, 0])
    pools["weight"][p, 0, :6] = torch.tensor([5.0, 1.0, 3.0, 1.0, math.nan, 0.0])
    old = pools["k"].clone()
    assert orc.evict(pools, table, [6], 4, sinks=1, recent=1) == [4]   # 1 and 3 leave (0.0 is the last token's)
    assert torch.equal(pools["k"][p, 0, :4], old[p, 0, [0, 4, 2, 5]])
    assert pools["position"][p, 0, :4].tolist() == [0, 4, 2, 5]
    assert torch.equal(pools["k"][p, 0, 4:6], old[p, 0, 4:6])
    pools, table = make([6], 1, 16, track=True, seed=0, spare=2)
    pools["weight"][p, 0, :6] = torch.tensor([5.0, 1.0, 3.0, 1.0, math.nan, 0.0])
    free = next(x for x in range(3) if x != p)
    assert orc.evict(pools, table, [6], 3, out_table=torch.tensor([[free]])) == [3]
    assert torch.equal(pools["k"][free, 0, :3], old[p, 0, [0, 2, 4]])
    assert torch.equal(pools["k"][p, 0, :6], old[p, 0, :6])


def test_evict_refuses_bad_arguments(lib):
    some = ctypes.c_void_p(256)
    track = {"weight": 256, "position": 256}
    n = ctypes.c_uint64()
    assert lib.fba_paged_evict_workspace_bytes(2, 3, 16, 10, 100, ctypes.byref(n)) == 0 and n.value == 2 * 3 * (100 * 8 + 4)
    assert lib.fba_paged_evict_workspace_bytes(2, 3, 16, 10, 1000, ctypes.byref(n)) == 0 and n.value == 2 * 3 * (160 * 8 + 4)
    for bad in ((0, 3, 16, 10, 100), (2, 0, 16, 10, 100), (2, 3, 16, 10, 0)):
        assert lib.fba_paged_evict_workspace_bytes(*bad, ctypes.byref(n)) == -1
    assert lib.fba_paged_evict_workspace_bytes(2, 3, 256, 2**22, 100, ctypes.byref(n)) == -5

    def call(c=None, B=1, lens=some, budget=20, sinks=0, recent=0, out=None, out_pages=0, out_lens=ctypes.c_void_p(512), ws=some,
             size=2**30):
        return lib.fba_paged_evict(c or struct(**track), B, lens, budget, sinks, recent, None, out, out_pages, out_lens, ws,
                                   size, some, None)

    assert call(struct()) == -1 and b"no weights" in lib.fba_last_error()
    assert call(lens=None) == -1 and call(out_lens=None) == -1 and call(out_lens=some) == -1
    assert call(budget=0) == -1 and call(sinks=-1) == -1 and call(recent=-1) == -1 and call(sinks=15, recent=6) == -1
    assert call(out=some, out_pages=1) == -1 and call(out=some, out_pages=0) == -1
    assert call(ws=None) == -1 and call(ws=ctypes.c_void_p(258)) == -1 and call(size=2 * (20 * 8 + 4) - 1) == -1
    for bad in BAD_CACHES:
        assert call(struct(**(track | bad | ({"weight": None} if "position" in bad else {})
                              | ({"position": None} if "weight" in bad else {})))) == -1
    with pytest.raises(RuntimeError, match="no CPU path"):
        fba.evict_kv(cache(), torch.zeros((1, 4), dtype=torch.int32), torch.ones(1, dtype=torch.int32), 4)
