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
