"""CPU: pointers that the paged cache's entry points must refuse on the host, as no kernel could follow them."""
import ctypes

import pytest

from tests.test_paged_cpu import lib, struct  # noqa: F401


@pytest.mark.parametrize("at", [2, 4, 258, 260])
def test_decode_refuses_a_misaligned_output(lib, at):  # noqa: F811
    """The kernel writes 8 bytes at a time."""
    some, two = ctypes.c_void_p(256), (ctypes.c_int64 * 2)(512, 128)
    rc = lib.fba_paged_decode(struct(), some, two, ctypes.c_void_p(at), some, 1, 4, some, 0, 0, 0.1, 0, some, 2**40, some, None)
    assert rc == -1 and b"o must be 8-byte aligned" in lib.fba_last_error()


TRACK = {"weight": 256, "position": 256}


@pytest.mark.parametrize("name", ["seq_lens", "new_lens", "positions"])
@pytest.mark.parametrize("B,offset", [(1, 0), (5, 0), (5, 16), (5, -16)])
def test_append_refuses_lengths_over_its_inputs(lib, name, B, offset):  # noqa: F811
    """A sequence's other CTAs may still read them when its new length is written."""
    some, three = ctypes.c_void_p(256), (ctypes.c_int64 * 3)(8, 8, 8)
    at = {"seq_lens": 4096, "new_lens": 8192, "positions": 12288}
    p = {n: ctypes.c_void_p(x) for n, x in at.items()}
    rc = lib.fba_paged_append(struct(**TRACK), some, some, three, three, B, 1, p["seq_lens"], p["new_lens"], p["positions"],
                              ctypes.c_void_p(at[name] + offset), some, None)
    assert rc == -1 and b"out_lens must not overlap" in lib.fba_last_error()


@pytest.mark.parametrize("name", ["seq_lens", "next_positions"])
@pytest.mark.parametrize("B,offset", [(1, 0), (5, 0), (5, 16), (5, -16)])
def test_evict_refuses_lengths_over_its_inputs(lib, name, B, offset):  # noqa: F811
    some = ctypes.c_void_p(256)
    at = {"seq_lens": 4096, "next_positions": 8192}
    rc = lib.fba_paged_evict(struct(**TRACK), B, ctypes.c_void_p(4096), 20, 0, 0, ctypes.c_void_p(8192), None, 0,
                             ctypes.c_void_p(at[name] + offset), some, 2**30, some, None)
    assert rc == -1 and b"out_lens must not overlap" in lib.fba_last_error()


def test_evict_refuses_its_own_table_as_the_new_one(lib):  # noqa: F811
    """Rows would be written over others that are still to be read."""
    some, table = ctypes.c_void_p(256), ctypes.c_void_p(4096)
    rc = lib.fba_paged_evict(struct(**TRACK, table=4096), 1, some, 20, 0, 0, None, table, 3, ctypes.c_void_p(512), some, 2**30,
                             some, None)
    assert rc == -1 and b"out_table must not be the cache's table" in lib.fba_last_error()
