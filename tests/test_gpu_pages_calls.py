"""Calls on the pages of a key/value cache that the header allows and the lives of
tests/test_gpu_pages.py do not make."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def ok(capi, status):
    assert status == capi.SUCCESS, "0x%x" % status


@pytest.fixture(scope="module")
def engine(capi):
    b = capi.Blit(0)
    yield b
    b.close()


def ints(torch, values):
    t = torch.tensor(values, dtype=torch.int32, device="cuda:0")
    torch.cuda.synchronize()
    return t


@pytest.mark.parametrize("held", [False, True])
def test_compaction_of_a_single_page_says_that_nothing_moved(torch_cuda, capi, engine, held):
    torch = torch_cuda
    pool = torch.zeros(64, dtype=torch.uint8, device="cuda:0")
    at = capi.book_layout(1, 2, 1)
    book = torch.zeros(at.words, dtype=torch.int32, device="cuda:0")
    lists, moves = ints(torch, [1, 3]), ints(torch, [-9] * 6)
    with capi.Pages(engine, [(pool.data_ptr(), 64, 16, 1)], 1, 4, 2, 1, book.data_ptr()) as p:
        ok(capi, p.reset())
        if held:
            ok(capi, p.reserve(lists.data_ptr(), lists.data_ptr() + 4, 1))
        ok(capi, engine.synchronize())
        book[0] = 7  # as a compaction of another book's copy may have left it
        torch.cuda.synchronize()
        want = book.clone()
        want[0] = 0
        torch.cuda.synchronize()
        ok(capi, p.compact(3, moves.data_ptr()))
        ok(capi, engine.synchronize())
        assert torch.equal(book, want) and moves.tolist() == [-9] * 6
        assert int(book[at.ref_counts]) == int(held)
        # no budget, no launch: the head stays
        book[0] = 7
        torch.cuda.synchronize()
        ok(capi, p.compact(0))
        ok(capi, engine.synchronize())
        assert int(book[0]) == 7
