"""CPU: refusals of the sliding-window entry points, and the oracle they are tested against."""
import ctypes

import pytest
import torch

import flex_block_attn_b200 as fba
from oracle import window_oracle as orc


def test_oracle_mask_by_hand():
    m = orc.visible(3, 5, 2, 1)   # positions 2, 3, 4
    assert m.int().tolist() == [[1, 1, 1, 0, 0], [1, 0, 1, 1, 0], [1, 0, 0, 1, 1]]
    m = orc.visible(3, 2, 1, 1)   # positions -1, 0, 1
    assert m.int().tolist() == [[0, 0], [1, 0], [1, 1]]
    assert torch.equal(orc.visible(4, 4, None, 0), torch.ones(4, 4).tril().bool())


def test_oracle_gradients_against_autograd():
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn((2, h, n, 8), generator=g, dtype=torch.float64) for h, n in ((4, 9), (2, 7), (2, 7), (4, 9)))
    mask = orc.visible(9, 7, 3, 1)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    s = (leaves[0] @ leaves[1].repeat_interleave(2, 1).transpose(-1, -2) * 0.3).masked_fill(~mask, -1e300)
    o = (s.softmax(-1) * mask) @ leaves[2].repeat_interleave(2, 1)
    want = torch.autograd.grad(o, leaves, do)
    got = orc.masked_attention(q, k, v, mask, do, 0.3)
    assert torch.allclose(got[0], o.detach(), atol=1e-12)
    for a, b in zip(got[2:], want):
        assert torch.allclose(a, b, atol=1e-12)


def _qkv(Sq=16, Skv=16, Hq=2, Hkv=1):
    q, k = torch.zeros((1, Hq, Sq, 128), dtype=torch.bfloat16), torch.zeros((1, Hkv, Skv, 128), dtype=torch.bfloat16)
    return q, k, k.clone()


@pytest.mark.parametrize("window,sinks,what", [(0, 0, "window"), (-3, 0, "window"), (2.0, 0, "window"), (True, 0, "window"),
                                               (4, -1, "sinks"), (4, 1.5, "sinks"), (None, True, "sinks")])
def test_bad_windows_are_refused(window, sinks, what):
    with pytest.raises(ValueError, match=what):
        fba.sliding_window_attn_func(*_qkv(), window, sinks)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fba.sliding_window_attn_func(*_qkv(), 4)


def test_c_entry_points_refuse_bad_arguments():
    from flex_block_attn_b200 import _cabi
    from flex_block_attn_b200.build import build_library

    build_library()
    lib = _cabi.lib()
    n = ctypes.c_uint64()
    some = ctypes.c_void_p(256)   # never followed: every call ends before a pointer is
    sizes = (1, 2, 1, 16, 16)

    def fwd(sizes=sizes, window=4, sinks=0, scale=0.1):
        return lib.fba_window_fwd(some, some, some, some, None, None, *sizes, window, sinks, scale, some, None)

    assert lib.fba_window_fwd(None, some, some, some, None, None, *sizes, 4, 0, 0.1, some, None) == -1
    for bad in ((0, 2, 1, 16, 16), (1, 2, 1, 0, 16), (1, 2, 1, 16, 0), (1, 3, 2, 16, 16)):
        assert fwd(bad) == -1
    assert fwd(window=-1) == -1 and fwd(sinks=-1) == -1
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert fwd(scale=scale) == -1
    assert fwd((2, 40000, 1, 16, 16)) == _cabi.FBA_ERR_TOO_LARGE
    assert fwd((1, 2, 1, 2**30, 2**30)) == _cabi.FBA_ERR_TOO_LARGE
    assert lib.fba_window_partial_bytes(1, 2, 1, 16, 16, 4, 0, None) == -1
    assert lib.fba_window_partial_bytes(1, 2, 1, 16, 16, -4, 0, ctypes.byref(n)) == -1
    # enough kv heads for the chip: nothing is split
    for window, sinks in ((100, 0), (0, 5), (5000, 5)):
        assert lib.fba_window_partial_bytes(8, 64, 64, 5000, 5000, window, sinks, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.fba_window_partial_bytes(1, 8, 1, 5000, 5000, 100, 5, ctypes.byref(n)) == 0
    assert 0 < n.value <= 592 * 2**17 and n.value % 2**17 == 0
    assert lib.fba_window_fwd(some, some, some, some, None, ctypes.c_void_p(8), *sizes, 4, 0, 0.1, some, None) == -1   # o_rest
    bwd = [some] * 10 + [1, 8, 1, 5000, 5000, 100, 5, 0.1, some, some]
    assert lib.fba_window_bwd(*bwd, None, 0, some, None) == -1                       # the partial buffer is missing,
    assert lib.fba_window_bwd(*bwd, some, n.value - 1, some, None) == -1             # too small,
    assert lib.fba_window_bwd(*bwd, ctypes.c_void_p(8), n.value, some, None) == -1   # misaligned
    assert b"partial" in lib.fba_last_error()


@pytest.mark.parametrize("B,Hq,Hkv,Sq,Skv,window,sinks", [(1, 8, 1, 5000, 5000, 100, 5), (64, 64, 64, 400, 400, 1, 400),
                                                          (1, 1, 1, 2**20, 2**20, 1, 1), (2, 40, 5, 900, 100000, 7, 3),
                                                          (1, 16, 1, 100000, 300, 10, 300)])
def test_partial_sums_stay_within_their_limit(B, Hq, Hkv, Sq, Skv, window, sinks):
    from flex_block_attn_b200 import _cabi

    n = ctypes.c_uint64()
    assert _cabi.lib().fba_window_partial_bytes(B, Hq, Hkv, Sq, Skv, window, sinks, ctypes.byref(n)) == 0
    assert n.value <= 592 * 2**17


def test_the_same_sizes_are_always_divided_alike():
    """Whatever was asked for in between, and in another thread."""
    import random
    import threading

    from flex_block_attn_b200 import _cabi

    lib, rng = _cabi.lib(), random.Random(5)

    def parts(sizes):
        n = ctypes.c_uint64()
        assert lib.fba_window_partial_bytes(*sizes, ctypes.byref(n)) == 0
        assert n.value <= 592 * 2**17
        return n.value // 2**17

    def draw():
        heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 12, 16])
        rows = rng.randint(150, 444) * 128 // heads
        return 1, heads * group, heads, rows - rng.randint(0, 127), rows, rng.choice([0, rows // 4, rows // 9]), rng.choice([0, 4, 150])

    sizes = [draw() for _ in range(60)]
    first = [parts(x) for x in sizes]
    assert any(first) and first == [parts(x) for x in sizes]
    other = []
    thread = threading.Thread(target=lambda: other.extend(parts(x) for x in reversed(sizes)))
    thread.start()
    thread.join()
    assert first == other[::-1]
