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


def test_default_stream_by_its_name(torch_cuda, capi, engine):
    """torch's default stream has the handle 0, which means the handle's own; HIP's name for it,
    hipStreamLegacy, puts the calls behind and in front of torch's work."""
    torch, legacy = torch_cuda, 1
    assert torch.cuda.default_stream().cuda_stream == 0
    rows, row_bytes, pages = 16, 256, 64
    pool = torch.zeros((pages, rows * row_bytes), dtype=torch.uint8, device="cuda:0")
    at = capi.book_layout(pages, 8, 8)
    book = torch.zeros(at.words, dtype=torch.int32, device="cuda:0")
    ids, more = ints(torch, range(8)), ints(torch, [20] * 8)
    src, dst = torch.zeros(8, dtype=torch.int32, device="cuda:0"), torch.zeros(8, dtype=torch.int32, device="cuda:0")
    with capi.Pages(engine, [(pool.data_ptr(), rows * row_bytes, row_bytes, 1)], pages, rows, 8, 8,
                    book.data_ptr()) as p:
        for turn in range(1, 6):
            torch.cuda.synchronize()
            torch.cuda._sleep(1 << 21)
            book.fill_(turn)
            ok(capi, p.reset(legacy))
            ok(capi, p.reserve(ids.data_ptr(), more.data_ptr(), 8, None, legacy))
            # pages 0 .. 15 are held; the first page of each goes to one behind them
            pool.fill_(turn)
            src.copy_(book[at.tables:at.tables + 64].view(8, 8)[:, 0])
            dst.copy_(src + 30)
            pool[:16] += 100
            ok(capi, p.copy(dst.data_ptr(), src.data_ptr(), 8, stream=legacy))
            got = pool[:, 0].clone()
            held = book[at.ref_counts:at.ref_counts + pages].clone()
            want = [turn + 100 if q < 16 or (30 <= q < 46 and q % 2 == 0) else turn for q in range(pages)]
            assert got.tolist() == want and held.tolist() == [1] * 16 + [0] * 48
