"""CPU: the backward entry points refuse pointers that their kernels could not follow: o, dq and the scratch buffers are read
and written 16 bytes at a time, and no tensor map (whose making checks q, k, v, dO, dK and dV) covers them."""
import ctypes

import pytest

from tests.test_cabi_cpu import lib  # noqa: F401

BAD = [2, 8, 264, 1028]


def pointers(**at):
    names = ("q", "k", "v", "o", "rest", "lse", "dout", "dq", "dk", "dv", "lse_delta", "dq_accum")
    return {n: ctypes.c_void_p(at.get(n, 1024)) for n in names}


@pytest.mark.parametrize("at", BAD)
@pytest.mark.parametrize("name", ["o", "rest", "dq", "lse_delta", "dq_accum"])
def test_window_backward_refuses_misaligned_pointers(lib, name, at):  # noqa: F811
    p = pointers(**{name: at})
    some = ctypes.c_void_p(1024)
    rc = lib.fba_window_bwd(p["q"], p["k"], p["v"], p["o"], p["rest"], p["lse"], p["dout"], p["dq"], p["dk"], p["dv"], 1, 2, 1, 200,
                            200, 50, 4, 0.1, p["lse_delta"], p["dq_accum"], some, 2**30, some, None)
    assert rc == -1 and b"16-byte aligned" in lib.fba_last_error()


@pytest.mark.parametrize("at", BAD)
@pytest.mark.parametrize("mode,name", [(0, "o"), (0, "dq"), (0, "lse_delta"), (0, "dq_accum"), (1, "o"), (1, "dq"), (1, "lse_delta")])
def test_block_backward_refuses_misaligned_pointers(lib, mode, name, at):  # noqa: F811
    from flex_block_attn_b200._cabi import FbaList

    p = pointers(**{name: at})
    some = 1024
    whole = ctypes.byref(FbaList(some, some, None, 2, 2, 2, 1, 1))   # two tiles by two, one list for every head
    p = {n: x for n, x in p.items() if n != "rest"}
    common = [p[n] for n in ("q", "k", "v", "o", "lse", "dout", "dq", "dk", "dv")] + [1, 2, 1, 256, 256, whole]
    rc = lib.fba_bwd_ex(*common, whole, 0.1, mode, p["lse_delta"], p["dq_accum"], ctypes.c_void_p(some), None)
    assert rc == -1 and b"16-byte aligned" in lib.fba_last_error()
    if mode == 0:
        assert lib.fba_bwd(*common, p["lse_delta"], p["dq_accum"], ctypes.c_void_p(some), None) == -1
        assert b"16-byte aligned" in lib.fba_last_error()
