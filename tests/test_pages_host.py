"""Pages of a key/value cache on the host: the layout of a book, and what the
entry points refuse before they touch a GPU (include/mi355_blit.h)."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def capi_host(pkg):
    import torch  # noqa: F401  (one HIP runtime per process: torch's first)
    pkg.capi.load()
    return pkg.capi


def _up(n):
    return (n + 63) // 64 * 64


@pytest.mark.parametrize("pages,seqs,width", [(1, 1, 1), (64, 64, 64), (65, 63, 7), (100000, 1000, 512),
                                              (4194240, 65536, 33)])
def test_book_layout(capi_host, pages, seqs, width):
    b = capi_host.book_layout(pages, seqs, width)
    assert b.lengths == 64
    assert b.ref_counts == 64 + _up(seqs)
    assert b.free_bits == b.ref_counts + _up(pages)
    assert b.tables == b.free_bits + _up((pages + 31) // 32)
    assert b.words == b.tables + _up(seqs * width)


def test_book_limits(capi_host):
    lib, b = capi_host.load(), capi_host.Book()
    inv, res = capi_host.ERROR_INVALID_ARGUMENT, capi_host.ERROR_OUT_OF_RESOURCES
    for args in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        assert lib.mi355_blit_pages_book(*args, C.byref(b)) == inv
    assert lib.mi355_blit_pages_book(1, 1, 1, None) == inv
    assert lib.mi355_blit_pages_book(capi_host.PAGES_MAX_PAGES + 1, 1, 1, C.byref(b)) == res
    assert lib.mi355_blit_pages_book(1, capi_host.PAGES_MAX_SEQS + 1, 1, C.byref(b)) == res
    assert lib.mi355_blit_pages_book(1, 1, capi_host.PAGES_MAX_PAGES + 1, C.byref(b)) == res


def test_struct_layouts_match_header(capi_host):
    assert C.sizeof(capi_host.Plane) == 24 and C.sizeof(capi_host.PagesDesc) == 40 and C.sizeof(capi_host.Book) == 40
    assert capi_host.PagesDesc.book.offset == 32


def test_missing_objects_are_refused(capi_host):
    lib, inv = capi_host.load(), capi_host.ERROR_INVALID_ARGUMENT
    p = C.c_void_p(1)
    desc = capi_host.PagesDesc()
    assert lib.mi355_blit_pages_create(None, C.byref(desc), C.byref(p)) == inv and not p.value
    assert lib.mi355_blit_pages_create(None, C.byref(desc), None) == inv
    assert lib.mi355_blit_pages_destroy(None) == inv
    assert lib.mi355_blit_pages_reset(None, None) == inv
    assert lib.mi355_blit_pages_copy(None, 16, None, 16, None, 1, 0, None) == inv
    assert lib.mi355_blit_pages_reserve(None, 16, 16, 1, None, None) == inv
    assert lib.mi355_blit_pages_fork(None, 16, 16, 1, None, None) == inv
    assert lib.mi355_blit_pages_free(None, 16, None, 1, None) == inv
    assert lib.mi355_blit_pages_compact(None, 1, None, None) == inv
