"""What the packed operators refuse and how they size themselves, on the host: no GPU needed."""
import ctypes
import os

import pytest


@pytest.fixture(scope="module")
def lib():
    from nkipy_amd import _lib, build
    if not os.path.exists(build.LIB_PATH):
        build.build()
    return _lib.load()


Z = ctypes.c_void_p(0)
P = ctypes.c_void_p(4096)          # an aligned address that nothing dereferences: the calls below are refused before a launch


def test_rows_beyond_the_positions_of_32_bits(lib):
    def call(nq, nk):
        return lib.pa_packed_prefill(P, P, P, 128, 128, 128, P, P, Z, Z, P, Z, 0, 2, nq, nk, 1, 1, 128, 0, 0.1, 1, Z, 0, Z)
    assert call((1 << 31) - (1 << 17), 1 << 17) == -1 and b"2^31 together" in lib.pa_last_error()
    assert call(0, 1 << 17) == 0
