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


def test_pools_of_two_handles(torch_cuda, capi, engine):
    """A pool made on one handle, copied from and to from a pool of another; the stream that NULL
    means is the destination's."""
    torch = torch_cuda
    rows, row_bytes, n = 7, 72, 30
    a, b = (torch.randint(0, 256, (40, rows * row_bytes), dtype=torch.uint8, device="cuda:0") for _ in range(2))
    src, dst = (torch.randperm(40, device="cuda:0", dtype=torch.int32)[:n].contiguous() for _ in range(2))
    want = b.clone()
    want[dst.long()] = a[src.long()]
    back = a.clone()
    back[src.long()] = want[dst.long()]
    torch.cuda.synchronize()
    other = capi.Blit(0)
    here = capi.Pages(engine, [(a.data_ptr(), rows * row_bytes, row_bytes, 1)], 40, rows)
    there = capi.Pages(other, [(b.data_ptr(), rows * row_bytes, row_bytes, 1)], 40, rows)
    try:
        ok(capi, there.copy(dst.data_ptr(), src.data_ptr(), n, src=here))
        ok(capi, other.synchronize())
        assert torch.equal(b, want)
        ok(capi, here.copy(src.data_ptr(), dst.data_ptr(), n, src=there))
        ok(capi, engine.synchronize())
        assert torch.equal(a, back)
    finally:
        here.close(), there.close(), other.close()


def test_as_many_sequences_as_a_book_can_have(torch_cuda, capi, engine):
    """Sequences with the highest numbers, in lists long enough to be taken in turns; numbers
    just out of range beside them."""
    torch = torch_cuda
    seqs, pages, n = capi.PAGES_MAX_SEQS, 20000, 3000
    pool = torch.zeros(pages * 16, dtype=torch.uint8, device="cuda:0")
    at = capi.book_layout(pages, seqs, 2)
    book = torch.zeros(at.words, dtype=torch.int32, device="cuda:0")
    lengths = book[at.lengths:at.lengths + seqs]
    refs = book[at.ref_counts:at.ref_counts + pages]
    ids = torch.arange(seqs - n, seqs, dtype=torch.int32, device="cuda:0")
    ids = torch.cat([ids, ids[:1] * 0 + seqs, ids])         # out of range, then all of them once more
    more = torch.full_like(ids, 3)
    granted = torch.full_like(ids, 7)
    kids = torch.arange(n, dtype=torch.int32, device="cuda:0")
    torch.cuda.synchronize()
    with capi.Pages(engine, [(pool.data_ptr(), 16, 8, 1)], pages, 2, seqs, 2, book.data_ptr()) as p:
        ok(capi, p.reset())
        ok(capi, p.reserve(ids.data_ptr(), more.data_ptr(), ids.numel(), granted.data_ptr()))
        ok(capi, engine.synchronize())
        assert granted.tolist() == [1] * n + [0] * (n + 1)
        assert lengths.tolist() == [0] * (seqs - n) + [3] * n
        assert refs.tolist() == [1] * (2 * n) + [0] * (pages - 2 * n)
        ok(capi, p.fork(ids.data_ptr(), kids.data_ptr(), n, granted.data_ptr()))
        ok(capi, p.free(ids.data_ptr(), ids.numel()))
        ok(capi, engine.synchronize())
        assert granted[:n].tolist() == [1] * n
        assert lengths.tolist() == [3] * n + [0] * (seqs - n)
        assert refs.tolist() == [1] * (2 * n) + [0] * (pages - 2 * n)


def test_copies_recorded_into_a_graph(torch_cuda, capi, engine):
    """Whole pages and first rows, recorded once, replayed with other lists (a padded one
    among them) and eager work in between."""
    torch = torch_cuda
    rows, row_bytes, runs, n = 16, 40, 3, 20
    page = rows * row_bytes * runs
    a, b = (torch.randint(0, 256, (60, page), dtype=torch.uint8, device="cuda:0") for _ in range(2))
    lists = torch.full((5, n), -1, dtype=torch.int32, device="cuda:0")
    with capi.Pages(engine, [(a.data_ptr(), page, row_bytes, runs)], 60, rows) as from_, \
            capi.Pages(engine, [(b.data_ptr(), page, row_bytes, runs)], 60, rows) as to:
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            s = torch.cuda.current_stream().cuda_stream
            ok(capi, to.copy(lists[0].data_ptr(), lists[1].data_ptr(), n, src=from_, stream=s))
            ok(capi, to.copy(lists[2].data_ptr(), lists[3].data_ptr(), n, lists[4].data_ptr(), from_, stream=s))
        want = b.clone()
        for replay in range(5):
            pages_to, pages_from = torch.randperm(60)[:2 * n].view(2, n), torch.randperm(60)[:2 * n].view(2, n)
            valid = torch.randint(0, rows + 1, (n,))
            here = torch.stack([pages_to[0], pages_from[0], pages_to[1], pages_from[1], valid]).int()
            here[:4, n - replay:] = -1
            lists.copy_(here)
            for d, f in zip(here[0].tolist(), here[1].tolist()):
                if d >= 0:
                    want[d] = a[f]
            for d, f, v in zip(*(here[k].tolist() for k in (2, 3, 4))):
                if d >= 0:
                    want[d].view(runs, rows, row_bytes)[:, :v] = a[f].view(runs, rows, row_bytes)[:, :v]
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(b, want), replay
            a.add_(1)  # eager work between the replays
        del graph


def test_long_tables_with_a_sequence_named_again(torch_cuda, capi, engine):
    """Tables that several workgroups share: entries that name a sequence twice, with other
    lengths to keep, in the second stretch of a table and at its ends."""
    torch = torch_cuda
    width, seqs, pages, rows = 10007, 5, 30000, 2
    pool = torch.zeros(pages * 4, dtype=torch.uint8, device="cuda:0")
    at = capi.book_layout(pages, seqs, width)
    book = torch.zeros(at.words, dtype=torch.int32, device="cuda:0")
    lengths = book[at.lengths:at.lengths + seqs]
    refs = book[at.ref_counts:at.ref_counts + pages]
    bits = book[at.free_bits:at.free_bits + -(-pages // 32)]
    calls = [ints(torch, v) for v in ([0, 1], [2 * width, 9000], [0, 0, 1, 0], [2, 3, 2, 1],
                                      [0, 2, 0, 9, 1, 2], [8193, 16386, 16383, 0, -1, 20000])]
    at_ = [c.data_ptr() for c in calls]
    with capi.Pages(engine, [(pool.data_ptr(), 4, 2, 1)], pages, rows, seqs, width, book.data_ptr()) as p:
        ok(capi, p.reset())
        ok(capi, p.reserve(at_[0], at_[1], 2))
        ok(capi, p.fork(at_[2], at_[3], 4))      # 0 -> 2 and 0 -> 3; the other two are refused
        ok(capi, p.free(at_[4], 6, at_[5]))
        ok(capi, engine.synchronize())
        # (the third names a child again, and a parent that is named as a child; the child of the
        # fourth has tokens)
        assert lengths.tolist() == [8193, 9000, 16386, 2 * width, 0]
        count = np.zeros(pages, dtype=np.int64)
        count[:width] += 1                       # 3
        count[:4097] += 1                        # 0
        count[:8193] += 1                        # 2
        count[width:width + 4500] += 1           # 1
        assert np.array_equal(refs.cpu().numpy(), count)
        free = np.unpackbits(bits.cpu().numpy().view(np.uint8), bitorder="little")[:pages]
        assert np.array_equal(free, count == 0)
