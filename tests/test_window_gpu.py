"""GPU: sliding-window attention with sinks against the 64-bit oracle.

Tolerance, in steps of a bf16 rounding (half a step: u = 2^-8 of a value): O rounds P (relative u, weighted by |V|) and
the result; dV rounds P and the result; dQ and dK round dS, which the rounded O enters through delta, and the result.  So
a 2-norm within 2 u = 7.8e-3 of the expected one's, and no element further off than 8 u of the largest expected one.
Where every row sees one key at most, dS = P (dP - delta) is 0, and what remains of it is the rounding of two fp32 sums of
128 products: at most 2 * 128 * 2^-24 |dO| |V|, times the scale and a key's (a query's) element, over the heads of a group.
LSE: fp32 sums over at most a few thousand scores below 100: 1e-5 absolute.
"""
import math

import pytest
import torch

from oracle import window_oracle as orc
from tests.util import rand_qkv

pytestmark = pytest.mark.gpu
U = 2.0**-8


def close(got, want, what, least=None):
    got, want = got.double().cpu(), want.cpu()
    assert torch.isfinite(got).all(), what
    if least is not None:
        assert not want.any() and got.abs().max() <= least, what
        return
    off, norm, most = (got - want).norm(), want.norm(), want.abs().max()
    assert off <= 2 * U * norm, f"{what}: {off / norm:.3e} of the 2-norm"
    assert (got - want).abs().max() <= 8 * U * most, f"{what}: {((got - want).abs().max() / most):.3e} of the largest"


# B, Hq, Hkv, Sq, Skv, window, sinks
CASES = [
    (1, 1, 1, 1, 1, None, 0),          # one token
    (1, 2, 1, 1, 300, 64, 4),          # one query behind earlier keys
    (2, 2, 2, 5, 5, 1, 0),             # every query sees itself alone
    (1, 2, 2, 127, 127, 127, 1),
    (1, 2, 1, 128, 128, 64, 128),      # sinks cover the whole sequence
    (1, 4, 2, 129, 129, 128, 0),
    (1, 2, 2, 255, 257, 129, 3),
    (1, 2, 1, 256, 256, None, 4),      # causal
    (2, 6, 2, 300, 300, 37, 130),      # sinks end in the second tile
    (1, 3, 1, 777, 777, 256, 4),
    (1, 2, 2, 640, 640, 128, 0),       # window of exactly a tile
    (1, 2, 2, 640, 640, 129, 129),
    (1, 4, 1, 1100, 1100, 300, 300),   # window and sinks meet
    (1, 2, 1, 200, 1000, 150, 7),      # a piece of a prompt
    (1, 2, 1, 515, 1301, 2000, 0),     # the window is longer than the keys
    (1, 2, 2, 900, 400, 100, 5),       # more queries than keys: 500 rows see nothing
    (1, 1, 1, 300, 20, 5, 2),
    (1, 8, 1, 2500, 2500, 200, 5),     # the sinks' key tile is divided over CTAs, heads shared
    (2, 16, 2, 1531, 1531, 64, 200),
]


@pytest.mark.parametrize("B,Hq,Hkv,Sq,Skv,window,sinks", CASES)
def test_forward_and_gradients(B, Hq, Hkv, Sq, Skv, window, sinks):
    import flex_block_attn_b200 as fba

    q, k, v, do = rand_qkv(B, Hq, Hkv, Sq, Skv, seed=Sq + Skv, device="cuda")
    mask = orc.visible(Sq, Skv, window, sinks, q.device)
    want = orc.masked_attention(q, k, v, mask, do)
    for x in (q, k, v):
        x.requires_grad_()
    o = fba.sliding_window_attn_func(q, k, v, window, sinks)
    grads = torch.autograd.grad(o, (q, k, v), do)
    least = None
    if mask.sum(-1).max() <= 1:
        row = lambda x: x.detach().double().norm(dim=-1).max()  # noqa: E731
        least = 2**-16 * row(do) * row(v) * 128**-0.5 * max(q.abs().max(), k.abs().max()) * (Hq // Hkv)
    for got, w, what in zip((o.detach(), *grads), (want[0], *want[2:]), ("O", "dQ", "dK", "dV")):
        close(got, w, what, least if what in ("dQ", "dK") else None)
    dead = ~mask.any(-1)
    assert not o.detach()[:, :, dead].any() and not grads[0][:, :, dead].any()
    unseen = ~mask.any(0)
    assert not grads[1][:, :, unseen].any() and not grads[2][:, :, unseen].any()
    o2, lse = fba.forward_with_window(q.detach(), k.detach(), v.detach(), window, sinks)
    assert torch.equal(o2, o.detach())
    assert torch.equal(lse[:, :, dead], torch.full_like(lse[:, :, dead], -math.inf))
    assert (lse[:, :, ~dead].double() - want[1][:, :, ~dead]).abs().max() <= 1e-5
    o3, none = fba.forward_with_window(q.detach(), k.detach(), v.detach(), window, sinks, need_lse=False)
    assert none is None and torch.equal(o3, o2)


def test_causal_equals_the_block_operator_on_block_masks():
    """The last row of a 128-row tile sees whole key tiles under the causal mask: what the block operator gives it for the
    lower triangle of 128 x 128 blocks, bit for bit."""
    import flex_block_attn_b200 as fba

    q, k, v, _ = rand_qkv(1, 2, 2, 256, 256, seed=3, device="cuda")
    o = fba.sliding_window_attn_func(q, k, v, None)
    mask = orc.visible(256, 256, None, 0, q.device)
    close(o, orc.masked_attention(q, k, v, mask)[0], "causal")
    full = fba.flex_block_attn_func(q, k, v, 128, 128, torch.tensor([[True, False], [True, True]], device="cuda"))
    # rows 127 and 255 see every key of their listed tiles
    assert torch.equal(o[:, :, [127, 255]], full[:, :, [127, 255]])


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_softmax_scale_and_large_scores(scale):
    import flex_block_attn_b200 as fba

    q, k, v, do = rand_qkv(1, 2, 1, 400, 400, seed=11, device="cuda")
    want = orc.masked_attention(q, k, v, orc.visible(400, 400, 100, 3, q.device), do, scale)
    for x in (q, k, v):
        x.requires_grad_()
    o = fba.sliding_window_attn_func(q, k, v, 100, 3, scale)
    grads = torch.autograd.grad(o, (q, k, v), do)
    for got, w, what in zip((o.detach(), *grads), (want[0], *want[2:]), ("O", "dQ", "dK", "dV")):
        close(got, w, what)


def test_gradient_against_differences():
    """The directional derivative of sum(O * dO) against central differences of the 64-bit forward."""
    import flex_block_attn_b200 as fba

    q, k, v, do = rand_qkv(1, 2, 1, 150, 150, seed=5, device="cuda")
    mask = orc.visible(150, 150, 40, 2, q.device)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(fba.sliding_window_attn_func(*leaves, 40, 2), leaves, do)
    eps = 1e-5
    g = torch.Generator().manual_seed(1)
    for n in range(3):
        step = torch.randn(leaves[n].shape, generator=g, dtype=torch.float64).cuda()
        at = [x.double() for x in (q, k, v)]
        f = []
        for sign in (1, -1):
            moved = list(at)
            moved[n] = at[n] + sign * eps * step
            f.append((orc.masked_attention(*moved, mask)[0] * do.double()).sum())
        want = (f[0] - f[1]) / (2 * eps)
        got = (grads[n].double() * step).sum()
        # the step's entries are independent of the gradient's errors (2 u of its norm, as above); 4 deviations
        assert (got - want).abs() <= 4 * 2 * U * grads[n].double().norm() + 1e-6, n


def test_gradients_of_some_inputs_and_none():
    import flex_block_attn_b200 as fba

    q, k, v, do = rand_qkv(1, 2, 2, 200, 200, seed=9, device="cuda")
    v2 = v.clone().requires_grad_()
    o = fba.sliding_window_attn_func(q, k, v2, 50, 1)
    (dv,) = torch.autograd.grad(o, (v2,), do)
    close(dv, orc.masked_attention(q, k, v, orc.visible(200, 200, 50, 1, q.device), do)[4], "dV")
    assert not fba.sliding_window_attn_func(q, k, v, 50, 1).requires_grad
    with torch.no_grad():
        assert not fba.sliding_window_attn_func(q, k, v2, 50, 1).requires_grad


def test_dk_dv_are_reproducible_and_rows_of_a_padded_batch_do_not_matter():
    import flex_block_attn_b200 as fba

    q, k, v, do = rand_qkv(2, 8, 2, 1000, 1000, seed=21, device="cuda")
    runs = []
    for fill in (0.0, 7.0):   # sequence 1 ends at row 600
        qq, kk, vv, dd = (x.clone() for x in (q, k, v, do))
        for x in (qq, kk, vv):
            x[1, :, 600:] = fill
        dd[1, :, 600:] = 0
        o, lse = fba.forward_with_window(qq, kk, vv, 90, 4)
        runs.append((o, *fba.backward_with_window(qq, kk, vv, o, lse, dd, 90, 4)[1:]))
    assert torch.equal(runs[0][0][0], runs[1][0][0]) and torch.equal(runs[0][0][1, :, :600], runs[1][0][1, :, :600])
    for a, b in zip(runs[0][1:], runs[1][1:]):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1, :, :600], b[1, :, :600])


def test_captured_and_replayed_on_new_inputs():
    import flex_block_attn_b200 as fba

    bufs = [x.clone() for x in rand_qkv(1, 4, 2, 700, 700, seed=1, device="cuda")]

    def step():
        o, lse = fba.forward_with_window(*bufs[:3], 200, 4)
        return (o, *fba.backward_with_window(*bufs[:3], o, lse, bufs[3], 200, 4))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.MonkeyPatch.context() as m:
        m.setenv("FBA_CHECK_STATUS", "0")
        m.setenv("FBA_POISON_OUTPUTS", "0")
        with torch.cuda.graph(graph):
            outs = step()
    for seed in (2, 3):
        fresh = rand_qkv(1, 4, 2, 700, 700, seed=seed, device="cuda")
        for b, x in zip(bufs, fresh):
            b.copy_(x)
        graph.replay()
        want = orc.masked_attention(*fresh[:3], orc.visible(700, 700, 200, 4, "cuda"), fresh[3])
        for got, w, what in zip(outs, (want[0], *want[2:]), ("O", "dQ", "dK", "dV")):
            close(got, w, what)
    fba.check_status()


def test_two_streams_at_once():
    import flex_block_attn_b200 as fba

    sets = [rand_qkv(1, 2, 1, 900, 900, seed=s, device="cuda") for s in (31, 32)]
    streams = [torch.cuda.Stream() for _ in sets]
    outs = []
    with pytest.MonkeyPatch.context() as m:
        m.setenv("FBA_CHECK_STATUS", "0")
        for s, (q, k, v, do) in zip(streams, sets):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                o, lse = fba.forward_with_window(q, k, v, 100, 2)
                outs.append((o, *fba.backward_with_window(q, k, v, o, lse, do, 100, 2)))
    torch.cuda.synchronize()
    for (q, k, v, do), got in zip(sets, outs):
        want = orc.masked_attention(q, k, v, orc.visible(900, 900, 100, 2, "cuda"), do)
        for g, w, what in zip(got, (want[0], *want[2:]), ("O", "dQ", "dK", "dV")):
            close(g, w, what)


def test_training_step_captured_with_autograd():
    """Forward and torch.autograd.grad inside a capture, as make_graphed_callables does it."""
    import flex_block_attn_b200 as fba

    bufs = [x.clone() for x in rand_qkv(1, 4, 2, 500, 500, seed=41, device="cuda")]
    leaves = [x.requires_grad_() for x in bufs[:3]]

    def step():
        o = fba.sliding_window_attn_func(*leaves, 100, 4)
        return (o.detach(), *torch.autograd.grad(o, leaves, bufs[3]))

    with pytest.MonkeyPatch.context() as m:
        m.setenv("FBA_POISON_OUTPUTS", "0")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
    fresh = rand_qkv(1, 4, 2, 500, 500, seed=42, device="cuda")
    with torch.no_grad():
        for b, x in zip(bufs, fresh):
            b.copy_(x)
    graph.replay()
    want = orc.masked_attention(*fresh[:3], orc.visible(500, 500, 100, 4, "cuda"), fresh[3])
    for got, w, what in zip(outs, (want[0], *want[2:]), ("O", "dQ", "dK", "dV")):
        close(got, w, what)


@pytest.mark.parametrize("B,Hq,Hkv,Sq,Skv,window,sinks", [(1, 16, 1, 1500, 1500, 300, 5), (1, 8, 1, 1100, 1300, None, 0),
                                                          (1, 1, 1, 4000, 4000, None, 0), (2, 6, 1, 900, 700, 200, 3)])
def test_divided_key_tiles(B, Hq, Hkv, Sq, Skv, window, sinks):
    """Few kv heads: the steps of many key tiles are divided over CTAs; dK and dV stay reproducible."""
    import ctypes

    import flex_block_attn_b200 as fba
    from flex_block_attn_b200 import _cabi

    n = ctypes.c_uint64()
    assert _cabi.lib().fba_window_partial_bytes(B, Hq, Hkv, Sq, Skv, window or 0, sinks, ctypes.byref(n)) == 0 and n.value > 0
    q, k, v, do = rand_qkv(B, Hq, Hkv, Sq, Skv, seed=Sq, device="cuda")
    want = orc.masked_attention(q, k, v, orc.visible(Sq, Skv, window, sinks, "cuda"), do)
    o, lse = fba.forward_with_window(q, k, v, window, sinks)
    grads = fba.backward_with_window(q, k, v, o, lse, do, window, sinks)
    for got, w, what in zip((o, *grads), (want[0], *want[2:]), ("O", "dQ", "dK", "dV")):
        close(got, w, what)
    again = fba.backward_with_window(q, k, v, o, lse, do, window, sinks)
    assert torch.equal(grads[1], again[1]) and torch.equal(grads[2], again[2])


@pytest.mark.parametrize("B,Hq,Hkv,Sq,Skv,window,sinks", [(1, 48, 4, 4900, 4900, 1000, 3), (2, 40, 2, 4700, 4700, None, 0),
                                                          (1, 96, 3, 6500, 6500, 500, 140)])
def test_key_tiles_divided_to_pack_the_grid(B, Hq, Hkv, Sq, Skv, window, sinks):
    """Long lists, one to three an SM: the first few tiles of every kv head are divided."""
    import ctypes

    import flex_block_attn_b200 as fba
    from flex_block_attn_b200 import _cabi

    n = ctypes.c_uint64()
    assert _cabi.lib().fba_window_partial_bytes(B, Hq, Hkv, Sq, Skv, window or 0, sinks, ctypes.byref(n)) == 0 and n.value > 0
    q, k, v, do = rand_qkv(B, Hq, Hkv, Sq, Skv, seed=Sq, device="cuda")
    o, lse, rest = fba.forward_with_window(q, k, v, window, sinks, need_rest=True)
    grads = fba.backward_with_window(q, k, v, o, lse, do, window, sinks, rest=rest)
    mask, group = orc.visible(Sq, Skv, window, sinks, "cuda"), Hq // Hkv
    for b in range(B):
        for h in range(Hkv):
            ours, one = (slice(b, b + 1), slice(h * group, (h + 1) * group)), (slice(b, b + 1), slice(h, h + 1))
            want = orc.masked_attention(q[ours], k[one], v[one], mask, do[ours])
            for got, w, what in zip((o[ours], grads[0][ours], grads[1][one], grads[2][one]), (want[0], *want[2:]),
                                    ("O", "dQ", "dK", "dV")):
                close(got, w, what)
    again = fba.backward_with_window(q, k, v, o, lse, do, window, sinks, rest=rest)
    assert torch.equal(grads[1], again[1]) and torch.equal(grads[2], again[2])


@pytest.mark.parametrize("S,window,sinks", [(2, None, 0), (3, None, 0), (300, 2, 0), (300, 2, 1), (300, 5, 0)])
def test_gradients_of_rows_that_see_few_keys(S, window, sinks):
    """dS is the difference of nearly equal values there; what the rounding of O left keeps it exact.  Element by element:
    dS and the result are rounded (u each), and dP - delta is off by the rounding of P in O = P V (u of each p |dO V|; O's own
    rounding would add u |dO| |O|) and of fp32 sums of 128 products and O's second part (2^-16 of |dO| |V| + |dO| |O|),
    times P, the scale and a key (a query)."""
    import flex_block_attn_b200 as fba

    q, k, v, do = rand_qkv(2, 4, 2, S, S, seed=S + (window or 0), device="cuda")
    mask = orc.visible(S, S, window, sinks, "cuda")
    _, lse, dq, dk, _ = orc.masked_attention(q, k, v, mask, do)
    o = orc.masked_attention(q, k, v, mask)[0]
    ke, ve = (x.double().repeat_interleave(2, 1) for x in (k, v))
    scale, Q, dO = 128**-0.5, q.double(), do.double()
    p = ((Q @ ke.transpose(-1, -2) * scale).masked_fill(~mask, -math.inf) - lse[..., None]).exp()
    dp = dO @ ve.transpose(-1, -2)
    ds = p * (dp - (dO * o).sum(-1, keepdim=True)) * scale
    norm = lambda x: x.norm(dim=-1)  # noqa: E731
    noise = p * scale * 2.0**-16 * norm(dO)[..., None] * (norm(ve)[..., None, :] + norm(o)[..., None])
    off = (U + 2.0**-18) * ds.abs() + U * scale * p * (p * dp.abs()).sum(-1, keepdim=True) + noise
    leaves = [x.requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(fba.sliding_window_attn_func(*leaves, window, sinks), leaves, do)
    around = (off @ ke.abs(), (off.transpose(-1, -2) @ Q.abs()).unflatten(1, (2, 2)).sum(2))
    for g, w, a, what in zip(got, (dq, dk), around, ("dQ", "dK")):
        assert ((g.double() - w).abs() <= (1 + U) * a + U * w.abs()).all(), what
