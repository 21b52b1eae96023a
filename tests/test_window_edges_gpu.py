"""GPU: the window operator where a softmax has nothing to choose from."""
import pytest
import torch

pytestmark = pytest.mark.gpu


# B, Hq, Hkv, Sq, Skv, window, sinks
ONE_KEY = [(1, 20, 4, 1, 1, 1, 165), (2, 8, 4, 1, 1, None, 0), (1, 3, 1, 150, 1, None, 4), (1, 4, 2, 300, 300, 1, 0),
           (2, 2, 2, 1, 90, 1, 0), (1, 8, 1, 1000, 1300, 1, 0)]


@pytest.mark.parametrize("B,Hq,Hkv,Sq,Skv,window,sinks", ONE_KEY)
def test_one_visible_key_gives_exact_zeros(B, Hq, Hkv, Sq, Skv, window, sinks):
    """A probability of 1 does not depend on the scores: dQ and dK are zeros, O is the value row and dV the sum of dO."""
    import flex_block_attn_b200 as fba

    g = torch.Generator().manual_seed(Sq + Skv)
    q, do = (torch.randn((B, Hq, Sq, 128), generator=g).bfloat16().cuda() for _ in range(2))
    k, v = (torch.randn((B, Hkv, Skv, 128), generator=g).bfloat16().cuda() for _ in range(2))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = fba.sliding_window_attn_func(*leaves, window, sinks)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    assert not dq.any() and not dk.any()
    n = min(Sq, Skv)   # the rows that see a key, and the keys that are seen
    group = Hq // Hkv
    assert torch.equal(o[:, :, Sq - n:], v[:, :, Skv - n:].repeat_interleave(group, 1)) and not o[:, :, : Sq - n].any()
    seen = do.double()[:, :, Sq - n:].reshape(B, Hkv, group, n, 128)
    # sums of `group` values in fp32, rounded once to bf16
    bound = 2.0**-8 * seen.sum(2).abs() * (1 + 2.0**-8) + group * 2.0**-23 * seen.abs().sum(2)
    assert ((dv.double()[:, :, Skv - n:] - seen.sum(2)).abs() <= bound).all() and not dv[:, :, : Skv - n].any()
