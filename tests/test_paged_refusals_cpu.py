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


@pytest.mark.parametrize("page,width,ok", [(16, (1 << 27) - 2, False), (16, (1 << 27) - 33, True),
                                           (8, (1 << 28) - 2, False), (128, (1 << 24) - 5, True)])
def test_rows_whose_tiles_would_pass_31_bits(lib, page, width, ok):
    """Tile arithmetic rounds a row's length up to tiles of 128 and looks two tiles ahead."""
    size = _lib._c_size(0)
    c = fake_cache(page_size=page, width=width, table_stride=width)
    assert lib.cab_tree_attn_workspace_size(c, 1, 4, 1, ctypes.byref(size)) == (0 if ok else 2)


@pytest.mark.parametrize("strides", [(0, 1024, 64), (2048, 0, 64), (2048, 1024, 0)])
def test_outputs_in_one_place(lib, strides):
    """An expanded output: several rows would be stored over one another."""
    s3 = _lib._i64_3(2048, 1024, 64)
    rc = lib.cab_tree_attn_fwd(fake_cache(), 0, FAKE, FAKE, None, 2, 4, 2, s3, _lib._i64_3(*strides), None, None, None, 0, None,
                               0, 0.1, FAKE, 1 << 30, None)
    assert rc == 1 and b"output" in lib.cab_last_error_string()
