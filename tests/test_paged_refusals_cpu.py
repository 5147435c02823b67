"""Calls of the paged cache's C ABI that are refused on the host, before anything is launched."""

import ctypes

import pytest

from cab_attention import _lib
from test_paged_cpu import fake_cache


@pytest.fixture(scope="module")
def lib():
    import cab_build
    cab_build.build()
    return _lib.lib()


FAKE = ctypes.c_void_p(256)


def update(lib, c, dst=None, n=2, copies=1):
    return lib.cab_pages_update(c, None, dst, n, None, -1, None, 0, 0, 0, None, 0, None, 0, copies, FAKE, 1 << 20, None)


def test_other_rows_without_copies(lib):
    assert update(lib, fake_cache(), dst=FAKE, copies=0) == 1
    assert b"copies" in lib.cab_last_error_string()
