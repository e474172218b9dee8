"""Pages of a key/value cache (mi355_blit_pages_*) through the C ABI, against a
book that is kept one entry at a time in numpy.  Everything is whole numbers and
bytes: equal or wrong."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

I32 = np.int32


def ok(capi, status):
    assert status == capi.SUCCESS, "0x%x" % status


class Model:
    """The book by its definition."""

    def __init__(self, pages, rows, seqs, width):
        self.rows, self.width = rows, width
        self.lengths = np.zeros(seqs, dtype=np.int64)
        self.refs = np.zeros(pages, dtype=np.int64)
        self.tables = np.full((seqs, width), -1, dtype=np.int64)

    def held(self, tokens):
        return int(-(-int(tokens) // self.rows))

    def pages(self, s):
        return self.tables[s, :self.held(self.lengths[s])]

    def reserve(self, seqs, more):
        """-> (granted, [(from, to, rows)])"""
        granted, moves, named = [0] * len(seqs), [], set()
        free = list(np.nonzero(self.refs == 0)[0][::-1])
        for i, (s, a) in enumerate(zip(seqs, more)):
            if not 0 <= s < len(self.lengths) or s in named:
                continue
            named.add(s)
            o, m = self.held(self.lengths[s]), self.held(self.lengths[s] + a)
            if a < 0 or m > self.width:
                continue
            fill = int(self.lengths[s]) % self.rows
            apart = a > 0 and fill != 0 and self.refs[self.tables[s, o - 1]] > 1
            if m - o + apart > len(free):
                break
            if apart:
                old = self.tables[s, o - 1]
                self.refs[old] -= 1
                moves.append((int(old), int(free[-1]), fill))
            for slot in range(o - int(apart), m):
                q = free.pop()
                self.tables[s, slot] = q
                self.refs[q] = 1
            self.lengths[s] += a
            granted[i] = 1
        return granted, moves

    def fork(self, parents, children):
        granted, named = [0] * len(parents), set()
        for i, (p, c) in enumerate(zip(parents, children)):
            if not 0 <= c < len(self.lengths):
                continue
            first = c not in named
            named.add(c)
            if not 0 <= p < len(self.lengths) or not first or p in children or self.lengths[c]:
                continue
            held = self.pages(p)
            self.tables[c, :len(held)] = held
            self.refs[held] += 1
            self.lengths[c] = self.lengths[p]
            granted[i] = 1
        return granted

    def free(self, seqs, keep=None):
        for s, k in zip(seqs, keep if keep is not None else [0] * len(seqs)):
            if 0 <= s < len(self.lengths) and 0 <= k < self.lengths[s]:
                np.subtract.at(self.refs, self.tables[s, self.held(k):self.held(self.lengths[s])], 1)
                self.lengths[s] = k

    def compact(self, most):
        """-> [(from, to)]"""
        holes, movers = np.nonzero(self.refs == 0)[0], np.nonzero(self.refs > 0)[0][::-1]
        n = min(most, len(holes), len(movers))
        pairs = [(int(m), int(h)) for m, h in zip(movers[:n], holes[:n]) if h < m]
        now = np.arange(len(self.refs))
        for m, h in pairs:
            now[m] = h
            self.refs[h], self.refs[m] = self.refs[m], 0
        for s in range(len(self.lengths)):
            held = self.pages(s)
            held[:] = now[held]
        return pairs


class Cache:
    """A pool of random bytes with its book, and the model of both.  planes: (row_bytes,
    runs, gap behind each page, offset of the first page)."""

    def __init__(self, torch, capi, blit, rand, pages, rows, seqs, width, planes, seed=1, stream=None):
        self.torch, self.capi, self.stream = torch, capi, stream
        self.n_pages, self.rows = pages, rows
        self.model = Model(pages, rows, seqs, width)
        self.planes, self.mem, self.want = planes, [], []
        spec = []
        for k, (row_bytes, runs, gap, at) in enumerate(planes):
            page = rows * row_bytes * runs
            host = rand(at + pages * (page + gap), 0xCAC40000 + 16 * seed + k)
            dev = torch.from_numpy(host).to("cuda:0")
            self.mem.append(dev)
            self.want.append(host)
            spec.append((dev.data_ptr() + at, page + gap, row_bytes, runs))
        self.at = capi.book_layout(pages, seqs, width)
        self.book = torch.full((self.at.words,), 0x5A5A5A5A, dtype=torch.int32, device="cuda:0")
        torch.cuda.synchronize()
        self.pages = capi.Pages(blit, spec, pages, rows, seqs, width, self.book.data_ptr())
        ok(capi, self.pages.reset(stream))

    def close(self):
        self.pages.close()

    def list(self, values):
        """int32 on the device, ready for any stream."""
        t = self.torch.tensor(list(values), dtype=self.torch.int32, device="cuda:0")
        self.torch.cuda.synchronize()
        return t

    def part(self, name, n):
        start = getattr(self.at, name)
        return self.book[start:start + n].cpu().numpy()

    def page_view(self, k, q):
        """Page q of plane k of the wanted bytes: [runs][rows][row_bytes]."""
        row_bytes, runs, gap, at = self.planes[k]
        page = self.rows * row_bytes * runs
        start = at + q * (page + gap)
        return self.want[k][start:start + page].reshape(runs, self.rows, row_bytes)

    def move(self, moves):
        taken = [[(self.page_view(k, f).copy()) for k in range(len(self.planes))] for f, _, _ in moves]
        for (_, t, n), pages in zip(moves, taken):
            for k, page in enumerate(pages):
                self.page_view(k, t)[:, :n] = page[:, :n]

    def check(self, what):
        self.torch.cuda.synchronize()
        m = self.model
        assert np.array_equal(self.part("lengths", len(m.lengths)), m.lengths), what
        refs = self.part("ref_counts", self.n_pages)
        assert np.array_equal(refs, m.refs), what
        assert np.array_equal(self.part("tables", m.tables.size), m.tables.reshape(-1)), what
        bits = np.unpackbits(self.part("free_bits", -(-self.n_pages // 32)).view(np.uint8), bitorder="little")
        assert np.array_equal(bits[:self.n_pages], m.refs == 0) and not bits[self.n_pages:].any(), what
        for k in range(len(self.mem)):
            assert np.array_equal(self.mem[k].cpu().numpy(), self.want[k]), "%s: bytes of plane %d" % (what, k)

    def reserve(self, seqs, more):
        granted = self.list([7] * len(seqs))
        s, a = self.list(seqs), self.list(more)
        ok(self.capi, self.pages.reserve(s.data_ptr(), a.data_ptr(), len(seqs), granted.data_ptr(), self.stream))
        want, moves = self.model.reserve(seqs, more)
        self.move(moves)
        self.check("reserve")
        assert granted.tolist() == want
        return want

    def fork(self, parents, children):
        granted = self.list([7] * len(parents))
        p, c = self.list(parents), self.list(children)
        ok(self.capi, self.pages.fork(p.data_ptr(), c.data_ptr(), len(parents), granted.data_ptr(), self.stream))
        want = self.model.fork(parents, children)
        self.check("fork")
        assert granted.tolist() == want
        return want

    def free(self, seqs, keep=None):
        s, k = self.list(seqs), None if keep is None else self.list(keep)
        ok(self.capi, self.pages.free(s.data_ptr(), len(seqs), None if k is None else k.data_ptr(), self.stream))
        self.model.free(seqs, keep)
        self.check("free")

    def compact(self, most):
        moves = self.list([-9] * (2 * most + 2))
        ok(self.capi, self.pages.compact(most, moves.data_ptr(), self.stream))
        want = self.model.compact(most)
        self.move([(f, t, self.rows) for f, t in want])
        self.check("compact")
        assert int(self.book[0]) == len(want)
        assert moves.tolist() == [x for pair in want for x in pair] + [-9] * (2 * most + 2 - 2 * len(want))
        return want


@pytest.fixture(scope="module")
def engine(capi):
    b = capi.Blit(0)
    yield b
    b.close()


# ------------------------------------------------------------------ the copies

PLANES = [
    [(64, 1, 0, 0)],                                  # whole vectors
    [(2, 1, 0, 0), (30, 3, 5, 1)],                    # rows and runs that end inside a vector
    [(1024, 1, 0, 0), (512, 8, 256, 64), (4, 8, 0, 0)],  # a quantised cache with its scales
    [(5000, 1, 7, 3)],                                # rows longer than a wave's segment, odd addresses
]


@pytest.mark.parametrize("planes", PLANES, ids=["plain", "odd", "scales", "long"])
@pytest.mark.parametrize("rows", [1, 7, 16])
def test_copy_between_pools_and_within(torch_cuda, capi, engine, rand, planes, rows):
    torch = torch_cuda
    rng = np.random.default_rng(rows)
    a = Cache(torch, capi, engine, rand, 37, rows, 2, 5, planes, seed=1)
    b = Cache(torch, capi, engine, rand, 21, rows, 2, 5, [(r, n, g + 16, at) for r, n, g, at in planes], seed=2)
    try:
        for within in (False, True):
            for cut in (False, True):
                to = a if within else b
                n = 10
                src = rng.integers(0, 37, n)
                dst = rng.permutation(21)[:n]
                if within:  # sources are even pages, destinations odd ones
                    src, dst = src // 2 * 2, rng.permutation(18)[:n] * 2 + 1
                src[3], dst[4], dst[5] = -1, -1, to.n_pages  # entries to pass over
                valid = rng.integers(-1, rows + 2, n) if cut else np.full(n, rows)
                ls, ld, lv = a.list(src), a.list(dst), a.list(valid)
                ok(capi, to.pages.copy(ld.data_ptr(), ls.data_ptr(), n, lv.data_ptr() if cut else None, a.pages))
                for s, d, v in zip(src, dst, valid):
                    if 0 <= s < a.n_pages and 0 <= d < to.n_pages:
                        for k in range(len(planes)):
                            to.page_view(k, d)[:, :max(0, min(rows, v))] = a.page_view(k, s)[:, :max(0, min(rows, v))]
                a.check("source"), b.check("destination")
    finally:
        a.close(), b.close()


def test_copy_of_many_pages_streams(torch_cuda, capi, engine):
    """More than the few MiB from which on loads and stores bypass the caches, and more
    segments than the grid has waves."""
    torch = torch_cuda
    pages, rows, planes, row_bytes = 700, 16, 6, 2056
    pool = torch.randint(0, 256, (planes, pages, rows * row_bytes), dtype=torch.uint8, device="cuda:0")
    src = torch.randperm(350, device="cuda:0", dtype=torch.int32)
    dst = 350 + torch.randperm(350, device="cuda:0", dtype=torch.int32)
    want = pool.clone()
    want[:, dst.long()] = pool[:, src.long()]
    torch.cuda.synchronize()
    with capi.Pages(engine, [(pool[p].data_ptr(), rows * row_bytes, row_bytes, 1) for p in range(planes)], pages,
                    rows) as p:
        ok(capi, p.copy(dst.data_ptr(), src.data_ptr(), 350))
        ok(capi, engine.synchronize())
        assert torch.equal(pool, want)


def test_copy_to_host_memory_and_back(torch_cuda, capi, engine):
    torch = torch_cuda
    pages, rows, row_bytes = 300, 16, 2048
    pool = torch.randint(0, 256, (2, pages, rows * row_bytes), dtype=torch.uint8, device="cuda:0")
    host = torch.zeros((2, 256, rows * row_bytes), dtype=torch.uint8, pin_memory=True)
    there = torch.randperm(256, device="cuda:0", dtype=torch.int32)
    held = torch.randperm(pages, device="cuda:0", dtype=torch.int32)[:256].contiguous()
    want = pool[:, held.long()].clone()
    torch.cuda.synchronize()

    def spec(t):
        return [(t[k].data_ptr(), rows * row_bytes, row_bytes, 1) for k in range(2)]
    with capi.Pages(engine, spec(pool), pages, rows) as dev, capi.Pages(engine, spec(host), 256, rows) as out:
        for n in (3, 256):  # below and beyond the size from which on stores bypass the caches
            ok(capi, out.copy(there.data_ptr(), held.data_ptr(), n, src=dev, route=capi.ROUTE_DEVICE_TO_HOST))
            ok(capi, engine.synchronize())
            assert torch.equal(host[:, there[:n].cpu().long()], want[:, :n].cpu())
            pool[:, held[:n].long()] = 0
            torch.cuda.synchronize()
            ok(capi, dev.copy(held.data_ptr(), there.data_ptr(), n, src=out, route=capi.ROUTE_HOST_TO_DEVICE))
            ok(capi, engine.synchronize())
            assert torch.equal(pool[:, held.long()], want)


def test_copy_of_first_rows_to_host_memory_and_back(torch_cuda, capi, engine):
    """Rows behind the valid ones stay as they are on either side, for pages of one run and
    of several, in rows that are whole vectors and rows that are not."""
    torch = torch_cuda
    for runs, row_bytes in ((1, 2048), (6, 80), (3, 25)):
        pages, rows, n = 120, 9, 100
        dev = torch.randint(0, 256, (pages, runs, rows, row_bytes), dtype=torch.uint8, device="cuda:0")
        host = torch.full((pages, runs, rows, row_bytes), 7, dtype=torch.uint8, pin_memory=True)
        src = torch.randperm(pages, device="cuda:0", dtype=torch.int32)[:n].contiguous()
        dst = torch.randperm(pages, device="cuda:0", dtype=torch.int32)[:n].contiguous()
        valid = torch.randint(0, rows + 1, (n,), device="cuda:0", dtype=torch.int32)
        torch.cuda.synchronize()
        kept = (torch.arange(rows, device="cuda:0") < valid[:, None])[:, None, :, None]
        spec = [(dev.data_ptr(), runs * rows * row_bytes, row_bytes, runs)]
        with capi.Pages(engine, spec, pages, rows) as d, \
                capi.Pages(engine, [(host.data_ptr(),) + spec[0][1:]], pages, rows) as h:
            ok(capi, h.copy(dst.data_ptr(), src.data_ptr(), n, valid.data_ptr(), d, capi.ROUTE_DEVICE_TO_HOST))
            ok(capi, engine.synchronize())
            want = torch.full_like(dev, 7)
            want[dst.long()] = torch.where(kept, dev[src.long()], want[dst.long()])
            assert torch.equal(host, want.cpu())
            before = dev.clone()
            torch.cuda.synchronize()
            ok(capi, d.copy(src.data_ptr(), dst.data_ptr(), n, valid.data_ptr(), h, capi.ROUTE_HOST_TO_DEVICE))
            ok(capi, engine.synchronize())
            assert torch.equal(dev, before)   # what went out came back, the rest was left
            dev.zero_()
            torch.cuda.synchronize()
            ok(capi, d.copy(src.data_ptr(), dst.data_ptr(), n, valid.data_ptr(), h, capi.ROUTE_HOST_TO_DEVICE))
            ok(capi, engine.synchronize())
            back = torch.zeros_like(dev)
            back[src.long()] = torch.where(kept, before[src.long()], back[src.long()])
            assert torch.equal(dev, back)


def test_pages_beyond_32_bits(torch_cuda, capi, engine):
    """Pages 3 GiB apart: the last one starts beyond 2^33."""
    torch = torch_cuda
    pitch, rows, row_bytes = (3 << 30) + 48, 16, 272
    pool = torch.empty(4 * pitch, dtype=torch.uint8, device="cuda:0")
    book_at = capi.book_layout(4, 4, 3)
    book = torch.zeros(book_at.words, dtype=torch.int32, device="cuda:0")
    views = [pool[q * pitch:q * pitch + rows * row_bytes] for q in range(4)]
    for q in range(4):
        views[q].copy_(torch.randint(0, 256, (rows * row_bytes,), dtype=torch.uint8, device="cuda:0"))
    want = views[0].clone()
    lists = torch.tensor([0, 3, 1, 2], dtype=torch.int32, device="cuda:0")
    more = torch.tensor([48, 16], dtype=torch.int32, device="cuda:0")
    torch.cuda.synchronize()
    at = lists.data_ptr()
    with capi.Pages(engine, [(pool.data_ptr(), pitch, row_bytes, 1)], 4, rows, 4, 3, book.data_ptr()) as p:
        ok(capi, p.copy(at + 4, at, 1))
        ok(capi, engine.synchronize())
        assert torch.equal(views[3], want)
        # pages 0, 1, 2 to sequence 0, page 3 to sequence 1; then 0 ends and 1 moves down
        ok(capi, p.reset())
        ok(capi, p.reserve(at, more.data_ptr(), 1))
        ok(capi, p.reserve(at + 8, more.data_ptr() + 4, 1))
        ok(capi, p.free(at, 1))
        ok(capi, p.compact(4))
        ok(capi, engine.synchronize())
        assert int(book[book_at.tables + 3]) == 0 and torch.equal(views[0], want)


# ------------------------------------------------------------------- the book

CACHES = [
    # pages, rows, seqs, width, planes
    (1, 1, 1, 1, [(16, 1, 0, 0)]),
    (50, 16, 12, 9, [(64, 1, 0, 0), (30, 3, 5, 1)]),
    (400, 5, 40, 30, [(7, 2, 3, 1)]),
    (3000, 33, 300, 20, [(128, 1, 0, 0)]),
    (5000, 16, 2600, 4, [(4, 1, 0, 0)]),
]


@pytest.mark.parametrize("case", range(len(CACHES)))
@pytest.mark.parametrize("seed", [1, 2])
def test_life_of_a_cache(torch_cuda, capi, engine, rand, case, seed):
    """Random calls with clean lists, and with lists that name sequences twice, out of
    range or beyond what fits."""
    pages, rows, seqs, width, planes = CACHES[case]
    rng = np.random.default_rng(100 * case + seed)
    c = Cache(torch_cuda, capi, engine, rand, pages, rows, seqs, width, planes, seed=seed)
    try:
        c.check("reset")
        for step in range(30):
            n = int(rng.integers(1, min(2600, 2 * seqs) + 1))
            if rng.random() < 0.5:
                ids = [int(x) for x in rng.permutation(seqs)[:n]]
            else:
                ids = [int(x) for x in rng.integers(-1, seqs + 1, n)]
            what = rng.integers(0, 6)
            if what < 3:
                most = rows * width + 2 if rng.random() < 0.3 else 2 * rows + 1
                c.reserve(ids, [int(x) for x in rng.integers(-1 if rng.random() < 0.3 else 0, most, len(ids))])
            elif what == 3:
                if len(ids) > 1:
                    c.fork(ids[:len(ids) // 2], ids[len(ids) // 2:len(ids) // 2 * 2])
            elif what == 4:
                keep = [int(x) for x in rng.integers(-1, rows * width + 2, len(ids))] if rng.random() < 0.6 else None
                c.free(ids[:max(1, len(ids) // 2)], keep)
            elif pages > 1:
                c.compact(int(rng.choice([pages, 1, 5])))
    finally:
        c.close()


def test_forks_part_ways_and_the_last_holder_keeps_the_page(torch_cuda, capi, engine, rand):
    c = Cache(torch_cuda, capi, engine, rand, 40, 16, 10, 6, [(64, 1, 0, 0), (48, 2, 16, 4)])
    try:
        assert c.reserve([0, 1], [20, 32]) == [1, 1]
        assert c.fork([0] * 4 + [1] * 2, [2, 3, 4, 5, 6, 7]) == [1] * 6
        shared = int(c.model.tables[0, 1])
        assert c.model.refs[shared] == 5
        # 0 and its four children grow together: four copy, the last keeps the page
        assert c.reserve([3, 0, 5, 2, 4], [1] * 5) == [1] * 5
        assert c.model.refs[shared] == 1 and c.model.tables[4, 1] == shared
        # a full last page is not copied, and one that is not written either
        assert c.reserve([6, 7, 1], [1, 0, 0]) == [1] * 3
        assert c.model.refs[int(c.model.tables[1, 1])] == 3
        # rolled back into a page that others hold, then grown: the rows in use are copied
        c.free([7], [19])
        assert c.reserve([7], [3]) == [1]
        assert c.model.tables[7, 1] != c.model.tables[1, 1]
    finally:
        c.close()


def test_pool_runs_out(torch_cuda, capi, engine, rand):
    c = Cache(torch_cuda, capi, engine, rand, 10, 4, 8, 8, [(16, 1, 0, 0)])
    try:
        # nine pages fit; the third entry ends the call, the fourth would have fitted
        assert c.reserve([0, 1, 2, 3], [16, 20, 8, 4]) == [1, 1, 0, 0]
        assert c.reserve([3], [4]) == [1]
        assert c.reserve([0, 1], [0, 1]) == [1, 0]
        c.free([0])
        assert c.reserve([2], [4 * 8 + 1]) == [0]   # no room in the table
        assert c.reserve([2], [16]) == [1]
    finally:
        c.close()


def test_a_list_of_the_longest_kind(torch_cuda, capi, engine, rand):
    n = capi.PAGES_MAX_LIST
    c = Cache(torch_cuda, capi, engine, rand, 20000, 16, 2 * n, 2, [(4, 1, 0, 0)])
    try:
        c.reserve(list(range(n)), [1 + i % 20 for i in range(n)])
        c.fork(list(range(n)), list(range(n, 2 * n)))
        c.reserve(list(range(n)), [1] * n)
        c.free(list(range(0, 2 * n, 2)))
        c.compact(10000)
    finally:
        c.close()


def test_holders_of_a_page_far_apart_in_a_list(torch_cuda, capi, engine, rand):
    """A list is taken 1024 entries at a time: what the first have left of a page's holders is
    what later ones find."""
    n = 2600
    c = Cache(torch_cuda, capi, engine, rand, 12000, 16, 3 * n, 2, [(4, 1, 0, 0)])
    try:
        c.reserve(list(range(n)), [1 + i % 20 for i in range(n)])
        c.fork(list(range(n)), list(range(n, 2 * n)))
        c.fork(list(range(0, n, 3)), list(range(2 * n, 2 * n + len(range(0, n, 3)))))
        # parents first, then the children in another order: the last to come keeps the page
        c.reserve(list(range(n)) + list(range(2 * n - 1, n - 1, -1)) + list(range(2 * n, 3 * n))[:900], [1] * (2 * n + 900))
        c.free(list(range(0, 3 * n, 2)) + list(range(0, 300)), [i % 7 for i in range(len(range(0, 3 * n, 2)) + 300)])
    finally:
        c.close()


def test_a_large_pool(torch_cuda, capi, engine, rand):
    """More pages than one tile of the free bits covers, sequences of tens of thousands."""
    pages = 131072 + 70001
    c = Cache(torch_cuda, capi, engine, rand, pages, 1, 6, 120000, [(1, 1, 0, 0)])
    try:
        c.reserve([0, 1, 2], [90000, 50000, 61000])
        c.reserve([3], [100])
        c.free([1])
        c.fork([2], [4])
        c.free([0], [33333])
        c.compact(1000)
        c.compact(pages)
        c.reserve([5, 3], [120000, 1])
    finally:
        c.close()


# ---------------------------------------------------- streams, graphs, refusals

def test_other_streams(torch_cuda, capi, engine, rand):
    torch = torch_cuda
    side = torch.cuda.Stream()
    c = Cache(torch, capi, engine, rand, 60, 16, 8, 8, [(64, 1, 0, 0)], stream=side.cuda_stream)
    try:
        c.reserve([0, 1], [40, 50])
        c.fork([0], [2])
        c.reserve([0, 2], [5, 6])
        c.free([1])
        c.compact(10)
    finally:
        c.close()


def test_two_caches_at_once(torch_cuda, capi, engine, rand):
    """Two threads, each with a cache and a stream of its own, calling the same handle."""
    import threading
    torch = torch_cuda
    streams = [torch.cuda.Stream() for _ in range(2)]
    caches = [Cache(torch, capi, engine, rand, 300, 16, 24, 12, [(64, 1, 0, 0), (30, 3, 5, 1)], seed=k,
                    stream=streams[k].cuda_stream) for k in range(2)]
    failed = []

    def live(k):
        try:
            rng = np.random.default_rng(40 + k)
            for _ in range(25):
                ids = [int(x) for x in rng.permutation(24)[:8]]
                caches[k].reserve(ids, [int(x) for x in rng.integers(0, 40, 8)])
                caches[k].fork(ids[:4], ids[4:])
                caches[k].free(ids[2:5], [int(x) for x in rng.integers(0, 60, 3)])
                caches[k].compact(int(rng.integers(1, 60)))
        except BaseException as e:  # an assertion of another thread
            failed.append((k, repr(e)))
    try:
        threads = [threading.Thread(target=live, args=(k,)) for k in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not failed, failed
    finally:
        for c in caches:
            c.close()


def test_graphs_of_two_caches_replayed_together(torch_cuda, capi, engine, rand):
    """Each cache has work memory of its own: their graphs may run side by side."""
    torch = torch_cuda
    caches = [Cache(torch, capi, engine, rand, 5000, 4, 64, 60, [(64, 1, 0, 0)], seed=k) for k in range(2)]
    try:
        n = 40
        seqs, more, keep = (caches[0].list(v) for v in (range(n), [70 + i for i in range(n)], [33 + i for i in range(n)]))
        graphs = []
        for c in caches:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
                s = torch.cuda.current_stream().cuda_stream
                ok(capi, c.pages.reserve(seqs.data_ptr(), more.data_ptr(), n, None, s))
                ok(capi, c.pages.free(seqs.data_ptr(), n, keep.data_ptr(), s))
                ok(capi, c.pages.compact(400, None, s))
            graphs.append(graph)
        streams = [torch.cuda.Stream() for _ in range(2)]
        for replay in range(4):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
            for c in caches:
                m = c.model
                c.move(m.reserve(list(range(n)), [70 + i for i in range(n)])[1])
                m.free(list(range(n)), [33 + i for i in range(n)])
                c.move([(f, t, c.rows) for f, t in m.compact(400)])
            for c in caches:
                c.check("replay %d" % replay)
            for k, c in enumerate(caches):  # eager calls between the replays
                c.free([5 + k, 11], [0, 3 * replay])
        del graphs
    finally:
        for c in caches:
            c.close()


def test_calls_recorded_into_a_graph(torch_cuda, capi, engine, rand):
    """One decode step -- reserve, roll back, fork, free, compact a little -- recorded once
    and replayed with other lists, eager calls in between, against the model."""
    torch = torch_cuda
    c = Cache(torch, capi, engine, rand, 90, 4, 16, 12, [(64, 1, 0, 0), (24, 2, 0, 8)])
    try:
        c.reserve(list(range(6)), [9, 17, 4, 30, 1, 12])
        n = 6
        lists = {k: c.list([-1] * n) for k in ("seqs", "more", "granted", "parents", "children", "gone", "keep")}
        at = {k: v.data_ptr() for k, v in lists.items()}
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            s = torch.cuda.current_stream().cuda_stream
            ok(capi, c.pages.reserve(at["seqs"], at["more"], n, at["granted"], s))
            ok(capi, c.pages.fork(at["parents"], at["children"], n, None, s))
            ok(capi, c.pages.free(at["gone"], n, at["keep"], s))
            ok(capi, c.pages.compact(3, None, s))
        c.check("capture")
        rng = np.random.default_rng(5)
        for replay in range(6):
            v = {"seqs": rng.permutation(16)[:n], "more": rng.integers(0, 6, n), "parents": rng.integers(0, 16, n),
                 "children": rng.permutation(16)[:n], "gone": rng.integers(-1, 16, n), "keep": rng.integers(0, 20, n)}
            v = {k: [int(y) for y in x] for k, x in v.items()}
            for k, x in v.items():
                lists[k].copy_(torch.tensor(x, dtype=torch.int32))
            torch.cuda.synchronize()
            graph.replay()
            granted, moves = c.model.reserve(v["seqs"], v["more"])
            c.move(moves)
            c.model.fork(v["parents"], v["children"])
            c.model.free(v["gone"], v["keep"])
            c.move([(f, t, c.rows) for f, t in c.model.compact(3)])
            c.check("replay %d" % replay)
            assert lists["granted"].tolist() == granted
            c.reserve([replay], [3])  # an eager call in between
        del graph
    finally:
        c.close()


def test_a_snapshot_of_the_book_is_the_state(torch_cuda, capi, engine, rand):
    c = Cache(torch_cuda, capi, engine, rand, 60, 16, 8, 8, [(64, 1, 0, 0)])
    try:
        c.reserve([0, 1], [40, 50])
        saved = c.book.clone()
        before = [x.copy() for x in (c.model.lengths, c.model.refs, c.model.tables)]
        torch_cuda.cuda.synchronize()
        c.free([0])
        c.reserve([3], [90])
        ok(capi, engine.copy(c.book.data_ptr(), saved.data_ptr(), 4 * saved.numel()))
        ok(capi, engine.synchronize())
        c.model.lengths, c.model.refs, c.model.tables = before
        c.check("restored")
        c.reserve([1, 2], [20, 7])
    finally:
        c.close()


def test_refusals(torch_cuda, capi, engine, rand):
    torch = torch_cuda
    inv, res = capi.ERROR_INVALID_ARGUMENT, capi.ERROR_OUT_OF_RESOURCES
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda:0")
    book = torch.zeros(4096, dtype=torch.int32, device="cuda:0")
    base = buf.data_ptr()

    def status(planes, pages=4, rows=4, seqs=0, width=0, where=None):
        try:
            capi.Pages(engine, planes, pages, rows, seqs, width, where).close()
        except capi.BlitError as e:
            return e.status
        return capi.SUCCESS
    good = [(base, 64, 16, 1)]
    assert status(good) == capi.SUCCESS
    assert status(good, seqs=2, width=2, where=book.data_ptr()) == capi.SUCCESS
    assert status([]) == inv and status([(0, 64, 16, 1)]) == inv
    assert status([(base, 63, 16, 1)]) == inv                      # pages overlap
    assert status([(base, 0, 16, 1)], pages=1) == capi.SUCCESS     # a single page needs no pitch
    assert status([(base, 64, 0, 1)]) == inv and status([(base, 64, 16, 0)]) == inv
    assert status(good, pages=0) == inv and status(good, rows=0) == inv
    assert status(good, seqs=2, width=2) == inv                    # no book
    assert status(good, where=book.data_ptr()) == inv              # no sequences
    assert status(good, seqs=2, where=book.data_ptr()) == inv
    assert status(good, seqs=2, width=2, where=book.data_ptr() + 4) == inv
    assert status([(base, 1 << 63, 16, 1)]) == inv                 # beyond the address space
    assert status(good * 4097) == res
    assert status([(base, 1 << 40, 1 << 30, 2)], rows=1, pages=1) == res
    assert status([(base, 1 << 40, 1 << 30, 1)] * 5, rows=1, pages=1) == res
    assert status(good, pages=capi.PAGES_MAX_PAGES + 1) == res
    assert status(good, seqs=capi.PAGES_MAX_SEQS + 1, width=2, where=book.data_ptr()) == res
    assert status(good, rows=4, seqs=2, width=1 << 29, where=book.data_ptr()) == res

    lists = torch.zeros(16, dtype=torch.int32, device="cuda:0").data_ptr()
    with capi.Pages(engine, good, 4, 4) as pool, capi.Pages(engine, [(base, 64, 8, 2)], 4, 4) as other, \
            capi.Pages(engine, good, 4, 4, 2, 2, book.data_ptr()) as p:
        assert pool.copy(None, lists, 1) == inv and pool.copy(lists, None, 1) == inv
        assert pool.copy(lists, lists, 1, route=3) == inv
        assert pool.copy(lists, lists, 1, src=other) == inv        # another geometry
        assert pool.copy(lists, lists, 1 << 32) == res
        assert pool.copy(None, None, 0) == capi.SUCCESS
        for bare in (pool.reset(), pool.reserve(lists, lists, 1), pool.fork(lists, lists, 1), pool.free(lists, 1),
                     pool.compact(1)):
            assert bare == inv                                     # no book
        too_many = capi.PAGES_MAX_LIST + 1
        assert p.reserve(None, lists, 1) == inv and p.reserve(lists, None, 1) == inv
        assert p.reserve(lists, lists, too_many) == res and p.reserve(None, None, 0) == capi.SUCCESS
        assert p.fork(None, lists, 1) == inv and p.fork(lists, None, 1) == inv
        assert p.fork(lists, lists, too_many) == res and p.fork(None, None, 0) == capi.SUCCESS
        assert p.free(None, 1) == inv and p.free(lists, too_many) == res and p.free(None, 0) == capi.SUCCESS
        assert p.compact(0) == capi.SUCCESS
        # lists at addresses that are no multiple of 4
        assert pool.copy(lists + 2, lists, 1) == inv and pool.copy(lists, lists + 1, 1) == inv
        assert pool.copy(lists, lists, 1, valid=lists + 3) == inv
        assert p.reserve(lists + 1, lists, 1) == inv and p.reserve(lists, lists + 2, 1) == inv
        assert p.reserve(lists, lists, 1, granted=lists + 2) == inv
        assert p.fork(lists + 2, lists, 1) == inv and p.fork(lists, lists + 2, 1) == inv
        assert p.fork(lists, lists, 1, granted=lists + 1) == inv
        assert p.free(lists + 2, 1) == inv and p.free(lists, 1, keep=lists + 2) == inv
        assert p.compact(1, moves=lists + 2) == inv
        # the handle stays while something uses it
        assert capi.load().mi355_blit_destroy(engine.handle) == inv
        assert engine.synchronize() == capi.SUCCESS
    torch.cuda.synchronize()
    assert int(buf.sum()) == 0 and int(book.sum()) == 0


# -------------------------------------------------------------- all of it at work

def test_serving_run(torch_cuda, capi, engine):
    """A small server: prompts come in, answers grow a token at a time, prompts are sampled
    several times over, drafts are rolled back, answers end, the pool is compacted, and
    a sequence goes to host memory and comes back.  Every token's rows carry a
    stamp; whatever the pages went through, each sequence has to read back as its own tokens."""
    torch = torch_cuda
    rng = np.random.default_rng(11)
    pages, rows, seqs, width, planes, words = 220, 16, 24, 20, 3, 20
    pool = torch.zeros((planes, pages, rows, words), dtype=torch.int32, device="cuda:0")
    host = torch.zeros((planes, width, rows, words), dtype=torch.int32, pin_memory=True)
    at = capi.book_layout(pages, seqs, width)
    book = torch.zeros(at.words, dtype=torch.int32, device="cuda:0")
    lengths = book[at.lengths:at.lengths + seqs]
    tables = book[at.tables:at.tables + seqs * width].view(seqs, width)
    side = torch.cuda.Stream()
    told = {}   # sequence -> stamps of its tokens
    stamp = [1]

    def spec(t):
        return [(t[k].data_ptr(), rows * words * 4, words * 4, 1) for k in range(planes)]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda:0")

    torch.cuda.synchronize()
    with torch.cuda.stream(side), capi.Pages(engine, spec(pool), pages, rows, seqs, width, book.data_ptr()) as cache, \
            capi.Pages(engine, spec(host), width, rows) as out:
        s = side.cuda_stream
        ok(capi, cache.reset(s))

        def grow(ids, more):
            """Reserves, and writes the new tokens' rows where the tables say, as a model's kernels do."""
            granted = torch.zeros(len(ids), dtype=torch.int32, device="cuda:0")
            a, b = ints(ids), ints(more)
            ok(capi, cache.reserve(a.data_ptr(), b.data_ptr(), len(ids), granted.data_ptr(), s))
            for i, (q, m, g) in enumerate(zip(ids, more, granted.tolist())):
                if not g or not m:
                    continue
                have = len(told.setdefault(q, []))
                new = list(range(stamp[0], stamp[0] + m))
                stamp[0] += m
                told[q] += new
                where = torch.arange(have, have + m, device="cuda:0")
                for k in range(planes):
                    pool[k, tables[q, where // rows].long(), where % rows] = (ints(new) * 8 + k)[:, None]

        def read_back():
            got = lengths.tolist()
            for q in range(seqs):
                mine = told.get(q, [])
                assert got[q] == len(mine), q
                if mine:
                    where = torch.arange(len(mine), device="cuda:0")
                    for k in range(planes):
                        rows_of = pool[k, tables[q, where // rows].long(), where % rows]
                        assert torch.equal(rows_of, (ints(mine) * 8 + k)[:, None].expand(-1, words)), (q, k)

        def end(ids):
            a = ints(ids)
            ok(capi, cache.free(a.data_ptr(), len(ids), None, s))
            for q in ids:
                told.pop(q, None)
            side.synchronize()

        for step in range(40):
            idle = [q for q in range(seqs) if q not in told]
            busy = sorted(told)
            if idle and rng.random() < 0.5:
                new = idle[:int(rng.integers(1, 4))]
                grow(new, [int(x) for x in rng.integers(1, 100, len(new))])
            if busy and len(idle) > 4 and rng.random() < 0.6:
                parents = [int(rng.choice(busy)) for _ in range(3)]
                children = [q for q in range(seqs) if q not in told][-3:]
                a, b, g = ints(parents), ints(children), ints([0] * 3)
                ok(capi, cache.fork(a.data_ptr(), b.data_ptr(), 3, g.data_ptr(), s))
                for x, y, z in zip(parents, children, g.tolist()):
                    if z and told.get(x):
                        told[y] = list(told[x])
            if told:
                grow(sorted(told), [int(x) for x in rng.integers(0, 4, len(told))])
            if told and rng.random() < 0.5:   # a draft that was not accepted
                q = int(rng.choice(sorted(told)))
                keep = max(1, len(told[q]) - int(rng.integers(1, 20)))
                a, b = ints([q]), ints([keep])
                ok(capi, cache.free(a.data_ptr(), 1, b.data_ptr(), s))
                told[q] = told[q][:keep]
                side.synchronize()
            if len(told) > 6 and rng.random() < 0.7:
                end([int(x) for x in rng.permutation(sorted(told))[:4]])
            if rng.random() < 0.4:
                ok(capi, cache.compact(int(rng.choice([2, pages])), None, s))
            if step % 10 == 9 and told:       # out to the host, its pages given to others, and in again
                q = sorted(told)[0]
                mine, n = told[q], -(-len(told[q]) // rows)
                there = torch.arange(width, dtype=torch.int32, device="cuda:0")
                ok(capi, out.copy(there.data_ptr(), tables[q].data_ptr(), n, src=cache,
                                  route=capi.ROUTE_DEVICE_TO_HOST, stream=s))
                end([q])
                ok(capi, cache.compact(pages, None, s))
                a, b, g = ints([q]), ints([len(mine)]), ints([0])
                ok(capi, cache.reserve(a.data_ptr(), b.data_ptr(), 1, g.data_ptr(), s))
                assert g.tolist() == [1]
                ok(capi, cache.copy(tables[q].data_ptr(), there.data_ptr(), n, src=out,
                                    route=capi.ROUTE_HOST_TO_DEVICE, stream=s))
                side.synchronize()
                told[q] = mine
            read_back()
        assert stamp[0] > 1500
