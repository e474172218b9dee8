"""Workloads for the operators on the pages of a key/value cache: copying,
reserving, forking, freeing and compacting.

A cache keeps its keys and values in pages of `rows` tokens.  A pool has `planes`
planes (one for the keys and one for the values of every layer); page q of a plane
is `runs` runs of `rows` rows of `row_bytes` bytes: one run for the layout [token]
[head][dim], one for each head for [head][token][dim].  A book says who holds which
page, all of it int32 in one device buffer:

  lengths[s]      tokens of sequence s, 0 for an empty one
  ref_counts[q]   sequences that hold page q
  free_bits       bit q % 32 of word q / 32 is 1 where ref_counts[q] is 0
  tables[s][j]    the page of tokens [j * rows, (j + 1) * rows) of sequence s

Lists (of pages, of sequences) are on the GPU too.  What each operator does:

  copy      the first valid[i] rows of every run of page src[i], or whole pages, to page dst[i], in all planes
  reserve   add[i] more tokens for sequence seqs[i]: the lowest free pages, in the list's order; a last page that
            others hold too is left to them and its tokens are copied to a page of the sequence's own, unless it is
            the last to hold it; the first entry that does not fit ends the call
  fork      children[i] becomes a sequence of parents[i]'s tokens that holds the same pages
  free      sequence seqs[i] keeps its first keep[i] tokens (none without `keep`); a page that nobody holds is free
  compact   the highest pages in use move to the lowest free ones, as long as that moves them down and at most
            `budget` of them; the tables follow

The operators that change a book start every pass from the same book: a pass begins by
copying a snapshot over it, as a program does that runs a step speculatively.
"""
import math
import weakref

import numpy as np
import torch

own = False

ALIGN = 64  # words: each part of a book starts at a multiple of it


# ---------------------------------------------------------------------- cases

def listed():
    return [
        # one page of a small cache: what a prefix that is extended by one request costs before anything moves
        {"name": "copy 1 page", "op": "copy", "type": "bf16", "planes": 4, "pages": 64, "rows": 16, "runs": 1, "row_bytes": 512, "n": 1, "ragged": False, "pools": 1},
        # half-filled pages handed to another pool, head-major fp8, an odd head count and row length
        {"name": "copy ragged fp8 heads", "op": "copy", "type": "fp8", "planes": 24, "pages": 400, "rows": 33, "runs": 5, "row_bytes": 80, "n": 190, "ragged": True, "pools": 2},
        # a long prompt's pages to the pool that decodes it: 64 planes of 32 KiB, 1 GiB read and 1 GiB written
        {"name": "copy 512 pages", "op": "copy", "type": "bf16", "planes": 64, "pages": 1100, "rows": 16, "runs": 1, "row_bytes": 2048, "n": 512, "ragged": False, "pools": 1},
        # one decode step of 48 sequences: one token each
        {"name": "reserve 1 token each", "op": "reserve", "type": "bf16", "planes": 2, "pages": 4096, "rows": 16, "runs": 1, "row_bytes": 64, "seqs": 64, "live": 48, "width": 256, "lo": 1, "hi": 1000, "group": 1, "n": 48, "add_lo": 1, "add_hi": 1},
        # prompts of many requests admitted at once: some twenty thousand pages in one call
        {"name": "reserve prompts", "op": "reserve", "type": "bf16", "planes": 2, "pages": 65536, "rows": 16, "runs": 1, "row_bytes": 64, "seqs": 400, "live": 300, "width": 600, "lo": 0, "hi": 700, "group": 1, "n": 300, "add_lo": 1, "add_hi": 2000},
        # parallel samples of 32 prompts part ways: their shared last pages are copied
        {"name": "reserve after forks", "op": "reserve", "type": "bf16", "planes": 32, "pages": 3000, "rows": 16, "runs": 1, "row_bytes": 1024, "seqs": 300, "live": 256, "width": 130, "lo": 200, "hi": 1200, "group": 8, "n": 256, "add_lo": 1, "add_hi": 4},
        # a beam step over 8 requests of 8 beams
        {"name": "fork beams", "op": "fork", "type": "bf16", "planes": 2, "pages": 4096, "rows": 16, "runs": 1, "row_bytes": 64, "seqs": 150, "live": 64, "width": 160, "lo": 100, "hi": 2100, "group": 4, "n": 64},
        # many samples of long prompts: a thousand children of up to 16,000 tokens
        {"name": "fork long prompts", "op": "fork", "type": "bf16", "planes": 2, "pages": 100000, "rows": 16, "runs": 1, "row_bytes": 64, "seqs": 1100, "live": 90, "width": 1024, "lo": 2000, "hi": 16000, "group": 1, "n": 1000},
        # a few answers that ended
        {"name": "free 5 sequences", "op": "free", "type": "bf16", "planes": 2, "pages": 4096, "rows": 16, "runs": 1, "row_bytes": 64, "seqs": 64, "live": 48, "width": 256, "lo": 1, "hi": 1100, "group": 1, "n": 5, "keep": False},
        # drafts rolled back and forks dropped over a large batch
        {"name": "free tails", "op": "free", "type": "bf16", "planes": 2, "pages": 200000, "rows": 16, "runs": 1, "row_bytes": 64, "seqs": 1000, "live": 900, "width": 700, "lo": 500, "hi": 11000, "group": 3, "n": 850, "keep": True},
        # a bounded slice of compaction between two decode steps
        {"name": "compact 24 pages", "op": "compact", "type": "fp8", "planes": 16, "pages": 3000, "rows": 16, "runs": 1, "row_bytes": 1000, "seqs": 100, "live": 60, "width": 100, "lo": 1, "hi": 400, "group": 1, "budget": 24},
        # a pool two thirds empty packed into its lower part
        {"name": "compact pool", "op": "compact", "type": "bf16", "planes": 16, "pages": 3500, "rows": 32, "runs": 8, "row_bytes": 256, "seqs": 200, "live": 110, "width": 100, "lo": 1, "hi": 700, "group": 1, "budget": 3500},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("copy", "reserve", "fork", "free", "compact"))
    c = {"op": op, "type": rng.choice(("bf16", "fp16", "fp8")), "rows": rng.choice((1, 7, 8, 16, 16, 32, 33, 64))}
    size = 1 if c["type"] == "fp8" else 2
    if op in ("copy", "compact"):
        c["runs"] = rng.choice((1, 1, rng.randint(2, 16)))
        c["row_bytes"] = size * _log(rng, 16, 2048 if c["runs"] == 1 else 256)
        page = c["rows"] * c["runs"] * c["row_bytes"]
        c["planes"] = _log(rng, 2, max(2, min(80, (1 << 20) // page)))
        most = max(4, min(1000, (400 << 20) // (page * c["planes"])))
        if op == "copy":
            c.update(n=_log(rng, 1, most), ragged=rng.random() < 0.5, pools=rng.choice((1, 2)))
            c["pages"] = c["n"] * 2 + rng.randint(1, 100)
            return c
        c.update(live=_log(rng, 2, 100), lo=1, group=rng.choice((1, 1, 2, 5)))
        c["width"] = max(2, most // c["live"])
        c["hi"] = c["width"] * c["rows"]
        c["pages"] = int(c["live"] * c["width"] * rng.uniform(1.0, 2.5)) + 8
        c["seqs"] = c["live"] + rng.randint(0, 50)
        c["budget"] = rng.choice((c["pages"], _log(rng, 1, c["pages"])))
        return c
    c.update(runs=1, row_bytes=size * rng.randint(8, 64), planes=rng.choice((2, 2, 5, 16)), live=_log(rng, 2, 800), group=rng.choice((1, 1, 2, 4, 7)), lo=0)
    c["width"] = _log(rng, 2, max(4, min(800, 150000 // c["live"])))
    c["hi"] = max(1, c["width"] * c["rows"] // 2)
    c["seqs"] = c["live"] + rng.randint(0, 100)
    c["n"] = rng.randint(1, c["live"])
    if op == "reserve":
        c.update(add_lo=1, add_hi=rng.choice((1, 5, c["hi"])))
    elif op == "fork":
        c["n"] = _log(rng, 1, 800)
        c["seqs"] = c["live"] + c["n"] + rng.randint(0, 50)
        c["hi"] *= 2
    else:
        c["keep"] = rng.random() < 0.5
    leaders = -(-c["live"] // c["group"])
    c["pages"] = leaders * (-(-c["hi"] // c["rows"])) + c["n"] * (2 + (-(-c.get("add_hi", 0) // c["rows"]))) + rng.randint(0, 1000)
    # at most about a quarter of a GiB of pages: these operators move few of them
    c["planes"] = max(1, min(c["planes"], (1 << 28) // (c["pages"] * c["rows"] * c["row_bytes"])))
    return c


# --------------------------------------------------------------------- inputs

def _up(words):
    return -(-words // ALIGN) * ALIGN


def _layout(case):
    """Where the parts of a book start, in words, and how many words it has."""
    s, n = case["seqs"], case["pages"]
    lengths = ALIGN
    refs = lengths + _up(s)
    bits = refs + _up(n)
    tables = bits + _up(-(-n // 32))
    return lengths, refs, bits, tables, tables + _up(s * case["width"])


class _Book:
    """int32 views of the parts of a book's buffer."""

    def __init__(self, buf, case):
        lengths, refs, bits, tables, end = _layout(case)
        self.buf = buf
        self.lengths = buf[lengths:lengths + case["seqs"]]
        self.refs = buf[refs:refs + case["pages"]]
        self.bits = buf[bits:bits + -(-case["pages"] // 32)]
        self.tables = buf[tables:tables + case["seqs"] * case["width"]].view(case["seqs"], case["width"])


def _bits(free):
    """Truth values -> int32 words, value 32 * w + b in bit b of word w."""
    n = -(-free.numel() // 32)
    wide = torch.zeros(n * 32, dtype=torch.int64, device=free.device)
    wide[:free.numel()] = free
    words = (wide.view(n, 32) << torch.arange(32, device=free.device)).sum(1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _pool(case, g):
    shape = (case["planes"], case["pages"], case["runs"], case["rows"])
    if case["type"] == "fp8":  # the bytes of e4m3 values, no NaN among them
        p = torch.randint(0, 126, shape + (case["row_bytes"],), generator=g, device="cuda", dtype=torch.uint8)
        return p
    t = torch.bfloat16 if case["type"] == "bf16" else torch.float16
    return torch.randn(shape + (case["row_bytes"] // 2,), generator=g, device="cuda", dtype=t)


def _filled_book(case, g):
    """`live` sequences of lo..hi tokens on pages picked at random, `group` of them at a time
    holding the same pages."""
    dev, rows = "cuda", case["rows"]
    live, group = case["live"], case["group"]
    book = _Book(torch.zeros(_layout(case)[4], dtype=torch.int32, device=dev), case)
    lead = torch.arange(live, device=dev) // group * group
    tokens = torch.randint(case["lo"], case["hi"] + 1, (live,), generator=g, device=dev)[lead]
    count = (tokens + rows - 1) // rows
    ends = torch.cumsum(torch.where(lead == torch.arange(live, device=dev), count, 0), 0)
    place = torch.randperm(case["seqs"], generator=g, device=dev)[:live]  # sequences are scattered over the slots
    order = torch.randperm(case["pages"], generator=g, device=dev).to(torch.int32)
    at = torch.arange(case["width"], device=dev)
    held = at < count[:, None]
    pages = order[((ends - torch.where(lead == torch.arange(live, device=dev), count, 0))[lead][:, None] + at).clamp(max=case["pages"] - 1)]
    book.tables.fill_(-1)
    book.tables[place] = torch.where(held, pages, -1)
    book.lengths[place] = tokens.to(torch.int32)
    book.refs.copy_(torch.bincount(pages[held].long(), minlength=case["pages"]))
    book.bits.copy_(_bits(book.refs == 0))
    return book, place


_engine = {}


def _blit():
    if not _engine:
        import __graft_entry__
        _engine["pkg"] = __graft_entry__.load_package()
        _engine["blit"] = _engine["pkg"].capi.Blit(0)
    return _engine["pkg"].capi, _engine["blit"]


def _own_pages(case, pool, book=None):
    """The framework's handle of a pool, or of a pool and its book."""
    capi, blit = _blit()
    pitch = pool.stride(1) * pool.element_size()
    planes = [(pool[p].data_ptr(), pitch, case["row_bytes"], case["runs"]) for p in range(case["planes"])]
    if book is None:
        pages = capi.Pages(blit, planes, case["pages"], case["rows"])
    else:
        where = capi.book_layout(case["pages"], case["seqs"], case["width"])
        assert (where.lengths, where.ref_counts, where.free_bits, where.tables, where.words) == _layout(case)
        pages = capi.Pages(blit, planes, case["pages"], case["rows"], case["seqs"], case["width"], book.buf.data_ptr())
    # closed with the state that holds it; at the end of the process it goes with the process
    weakref.finalize(pages, pages.lib.mi355_blit_pages_destroy, pages.handle).atexit = False
    return pages


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = dict(case, pool=_pool(case, g))
    n = case.get("n", 0)
    i32 = torch.int32
    if case["op"] == "copy":
        st["other"] = _pool(case, g) if case["pools"] == 2 else st["pool"]
        order = torch.randperm(case["pages"], generator=g, device="cuda").to(i32)
        st["src"], st["dst"] = order[:n].clone(), order[n:2 * n].clone()
        st["valid"] = torch.randint(1, case["rows"] + 1, (n,), generator=g, device="cuda", dtype=i32) if case["ragged"] else None
        if own:
            st["from"] = _own_pages(case, st["pool"])
            st["to"] = _own_pages(case, st["other"]) if case["pools"] == 2 else st["from"]
        return st
    st["book"], place = _filled_book(case, g)
    st["snapshot"] = st["book"].buf.clone()
    pick = place[torch.randperm(case["live"], generator=g, device="cuda")].to(i32)
    if case["op"] == "reserve":
        st["list"] = pick[:n].clone()
        st["add"] = torch.randint(case["add_lo"], case["add_hi"] + 1, (n,), generator=g, device="cuda", dtype=i32)
    elif case["op"] == "fork":
        st["list"] = pick[torch.randint(0, case["live"], (n,), generator=g, device="cuda")].clone()
        empty = torch.ones(case["seqs"], dtype=torch.bool, device="cuda")
        empty[place] = False
        empty = empty.nonzero().flatten().to(i32)
        st["children"] = empty[torch.randperm(empty.numel(), generator=g, device="cuda")[:n]].clone()
    elif case["op"] == "free":
        st["list"] = pick[:n].clone()
        u = torch.rand(n, generator=g, device="cuda")
        st["keep"] = (st["book"].lengths[st["list"].long()] * u).to(i32) if case["keep"] else None
    st["granted"] = torch.zeros(n, dtype=i32, device="cuda")
    if own:
        st["pages_of"] = _own_pages(case, st["pool"], st["book"])
    return st


# ---------------------------------------------------------------- plain forms

def _held(tokens, rows):
    return (tokens + (rows - 1)) // rows


def _move(to, dst, frm, src, valid, rows):
    """Pages src of `frm` to pages dst of `to`, the first valid rows of each run; whole pages without `valid`."""
    if valid is None:
        to[:, dst] = frm[:, src]
    else:
        kept = (torch.arange(rows, device=to.device) < valid[:, None])[None, :, None, :, None]
        to[:, dst] = torch.where(kept, frm[:, src], to[:, dst])


def _first(ids, ok, size):
    """Where an entry is the first of the list that names its id."""
    at = torch.arange(ids.numel(), device=ids.device)
    first = torch.full((size + 1,), ids.numel(), dtype=torch.int64, device=ids.device)
    first.scatter_reduce_(0, torch.where(ok, ids, size), at, "amin")
    return first[ids] == at


def _plain_reserve(st, b):
    rows, n_pages, n_seqs, width = st["rows"], st["pages"], st["seqs"], st["width"]
    dev = b.buf.device
    ids, add = st["list"].long(), st["add"].long()
    at = torch.arange(ids.numel(), device=dev)
    named = (ids >= 0) & (ids < n_seqs)
    s = torch.where(named, ids, 0)
    tokens = b.lengths[s].long()
    old, new = _held(tokens, rows), _held(tokens + add, rows)
    ok = named & _first(s, named, n_seqs) & (add >= 0) & (new <= width)
    # a last page with room, held by others too
    partial = ok & (add > 0) & (tokens % rows != 0)
    tail = torch.where(partial, b.tables[s, (old - 1).clamp(min=0)].long(), n_pages)
    holders = torch.cat([b.refs, b.refs.new_zeros(1)])[tail].long()
    shared = partial & (holders > 1)
    spot = torch.where(shared, tail, n_pages)
    askers = torch.zeros(n_pages + 1, dtype=torch.int64, device=dev).index_add_(0, spot, torch.ones_like(spot))
    last = torch.zeros(n_pages + 1, dtype=torch.int64, device=dev).scatter_reduce_(0, spot, at, "amax")
    copies = shared & ~((askers[tail] == holders) & (last[tail] == at))
    need = torch.where(ok, new - old + copies, 0)
    end = torch.cumsum(need, 0)
    free = b.refs == 0
    granted = ok & (end <= free.sum())
    copies = copies & granted
    need = torch.where(granted, need, 0)
    end = torch.cumsum(need, 0)
    # the k-th lowest free page goes to the entry that has the k-th page to get
    rank = torch.cumsum(free, 0) - 1
    page = (free & (rank < end[-1])).nonzero().flatten()
    rank = rank[page]
    owner = torch.searchsorted(end, rank, right=True)
    nth = rank - (end - need)[owner]
    slot = old[owner] + nth - copies[owner].long()
    b.tables[s[owner], slot] = page.to(torch.int32)
    b.refs[page] = 1
    b.refs.index_add_(0, tail.clamp(max=n_pages - 1), -copies.to(torch.int32))
    b.lengths.index_add_(0, s, torch.where(granted, add, 0).to(torch.int32))
    st["granted"].copy_(granted)
    c = copies.nonzero().flatten()
    _move(st["pool"], b.tables[s[c], old[c] - 1].long(), st["pool"], tail[c], tokens[c] % rows, rows)


def _plain_fork(st, b):
    rows, n_seqs = st["rows"], st["seqs"]
    parents, children = st["list"].long(), st["children"].long()
    some = (children >= 0) & (children < n_seqs)
    ok = some & (parents >= 0) & (parents < n_seqs)
    p, c = torch.where(ok, parents, 0), torch.where(some, children, 0)
    named = torch.zeros(n_seqs + 1, dtype=torch.bool, device=p.device).index_fill_(0, torch.where(some, children, n_seqs), True)
    ok = ok & _first(c, some, n_seqs) & ~named[p] & (b.lengths[c] == 0)
    st["granted"].copy_(ok)
    p, c = p[ok], c[ok]
    tokens = b.lengths[p]
    held = torch.arange(st["width"], device=p.device) < _held(tokens, rows)[:, None]
    pages = b.tables[p]
    b.tables[c] = torch.where(held, pages, b.tables[c])
    b.refs.index_add_(0, torch.where(held, pages, 0).flatten().long(), held.flatten().to(torch.int32))
    b.lengths[c] = tokens


def _plain_free(st, b):
    rows, n_seqs = st["rows"], st["seqs"]
    ids = st["list"].long()
    keep = st["keep"] if st["keep"] is not None else torch.zeros_like(st["list"])
    ok = (ids >= 0) & (ids < n_seqs) & (keep >= 0)
    s = torch.where(ok, ids, n_seqs)
    before = torch.cat([b.lengths, b.lengths.new_zeros(1)])
    after = before.scatter_reduce(0, s, torch.where(ok, keep, 0), "amin")
    once = ok & _first(torch.where(ok, ids, 0), ok, n_seqs)
    j = torch.arange(st["width"], device=ids.device)
    given = once[:, None] & (j >= _held(after[s], rows)[:, None]) & (j < _held(before[s], rows)[:, None])
    pages = b.tables[s.clamp(max=n_seqs - 1)]
    b.refs.index_add_(0, torch.where(given, pages, 0).flatten().long(), -given.flatten().to(torch.int32))
    b.lengths.copy_(after[:n_seqs])


def _plain_compact(st, b):
    live = b.refs > 0
    at = torch.arange(st["pages"], device=live.device)
    low = at < live.sum()
    holes = (~live & low).nonzero().flatten()[:st["budget"]]
    movers = (live & ~low).nonzero().flatten().flip(0)[:st["budget"]]
    st["pool"][:, holes] = st["pool"][:, movers]
    b.refs[holes] = b.refs[movers]
    b.refs[movers] = 0
    now = at.to(torch.int32)
    now[movers] = holes.to(torch.int32)
    held = torch.arange(st["width"], device=at.device) < _held(b.lengths, st["rows"])[:, None]
    b.tables.copy_(torch.where(held, now[b.tables.clamp(min=0).long()], b.tables))


# ------------------------------------------------------------------- one pass

def _bits_of(pool):
    return pool if pool.dtype == torch.uint8 else pool.view(torch.int16)


def _stream():
    """The stream that torch's work is on, so that the calls come behind what made their inputs and in
    front of what reads their outputs.  torch names its default stream 0, which the calls take
    for the handle's own; HIP's name for it is hipStreamLegacy, 1.  (torch.cuda.current_stream() makes a
    Python object for it, 2.7 us, as long as a call; this is the number alone, as code that torch
    generates asks for it.)"""
    return torch._C._cuda_getCurrentRawStream(0) or 1


def run(st):
    op = st["op"]
    stream = _stream() if own else None
    if op == "copy":
        if own:
            valid = st["valid"].data_ptr() if st["valid"] is not None else None
            _ok(st["to"].copy(st["dst"].data_ptr(), st["src"].data_ptr(), st["n"], valid=valid, src=st["from"], stream=stream))
        else:
            _move(st["other"], st["dst"].long(), st["pool"], st["src"].long(), st["valid"], st["rows"])
        return {"pool": _bits_of(st["other"])}
    b = st["book"]
    if own:
        blit = _engine["blit"]
        pages = st["pages_of"]
        _ok(blit.copy(b.buf.data_ptr(), st["snapshot"].data_ptr(), 4 * b.buf.numel(), stream=stream))
        if op == "reserve":
            _ok(pages.reserve(st["list"].data_ptr(), st["add"].data_ptr(), st["n"], granted=st["granted"].data_ptr(), stream=stream))
        elif op == "fork":
            _ok(pages.fork(st["list"].data_ptr(), st["children"].data_ptr(), st["n"], granted=st["granted"].data_ptr(), stream=stream))
        elif op == "free":
            _ok(pages.free(st["list"].data_ptr(), st["n"], keep=st["keep"].data_ptr() if st["keep"] is not None else None, stream=stream))
        else:
            _ok(pages.compact(st["budget"], stream=stream))
    else:
        b.buf.copy_(st["snapshot"])
        {"reserve": _plain_reserve, "fork": _plain_fork, "free": _plain_free, "compact": _plain_compact}[op](st, b)
    out = {"lengths": b.lengths, "refs": b.refs, "tables": b.tables}
    if op in ("reserve", "fork"):
        out["granted"] = st["granted"]
    if op in ("reserve", "compact"):
        out["pool"] = _bits_of(st["pool"])
    return out


def _ok(status):
    if status:
        raise RuntimeError("the call was refused: 0x%x" % status)


# ----------------------------------------------------------------------- work

def work(case):
    """Expected over the seeds; lists and book words 4 bytes each, rows read once and written once."""
    page = case["planes"] * case["runs"] * case["row_bytes"]  # bytes of one row of a page over all planes
    rows, n = case["rows"], case.get("n", 0)
    if case["op"] == "copy":
        mean = (rows + 1) / 2 if case["ragged"] else rows
        return {"bytes": n * (2 * mean * page + 8 + (4 if case["ragged"] else 0)), "flops": 0}
    tokens = (case["lo"] + case["hi"]) / 2
    held = tokens / rows + 0.5  # pages of a sequence
    if case["op"] == "reserve":
        fresh = n * ((case["add_lo"] + case["add_hi"]) / 2) / rows
        shared = 0.0
        if case["group"] > 1:  # nearly all holders of a last page with room copy it
            shared = n * (1 - 1 / case["group"]) * (1 - 1 / rows)
        moved = shared * (rows - 1) / 2 * 2 * page
        return {"bytes": n * 28 + case["pages"] / 8 + (fresh + shared) * 8 + moved, "flops": 0}
    if case["op"] == "fork":
        return {"bytes": n * (20 + held * 16), "flops": 0}
    if case["op"] == "free":
        gone = held * (0.5 if case["keep"] else 1.0)
        return {"bytes": n * (16 + gone * 12), "flops": 0}
    in_use = min(case["pages"], -(-case["live"] // case["group"]) * held)
    moves = min(case["budget"], in_use * (1 - in_use / case["pages"]))
    return {"bytes": case["pages"] / 8 + moves * (2 * rows * page + 24) + case["live"] * held * 4, "flops": 0}


# ------------------------------------------------------- the definitions again

def exact(case, seed):
    """The book that the operator's definition gives, one entry after the other; nothing for
    the bytes that are moved, which are equal or not."""
    if case["op"] == "copy":
        return None
    st = prepare(case, seed)
    b = st["book"]
    rows, width = case["rows"], case["width"]
    lengths, refs = b.lengths.cpu().numpy().astype(np.int64), b.refs.cpu().numpy().astype(np.int64)
    tables = b.tables.cpu().numpy().astype(np.int64)
    ids = st["list"].tolist() if "list" in st else []
    granted, named = [0] * len(ids), set()
    if case["op"] == "reserve":
        free, taken = np.nonzero(refs == 0)[0], 0
        for i, (s, a) in enumerate(zip(ids, st["add"].tolist())):
            again, named = s in named, named | {s}
            if not 0 <= s < case["seqs"] or again or a < 0 or -(-(lengths[s] + a) // rows) > width:
                continue
            o, m = -(-lengths[s] // rows), -(-(lengths[s] + a) // rows)
            apart = a > 0 and lengths[s] % rows != 0 and refs[tables[s, o - 1]] > 1
            if m - o + apart > len(free) - taken:
                break
            if apart:
                refs[tables[s, o - 1]] -= 1
            for slot in range(o - int(apart), m):
                tables[s, slot] = free[taken]
                refs[free[taken]] = 1
                taken += 1
            lengths[s] += a
            granted[i] = 1
    elif case["op"] == "fork":
        children = st["children"].tolist()
        for i, (p, c) in enumerate(zip(ids, children)):
            again, named = c in named, named | {c}
            if not (0 <= p < case["seqs"] and 0 <= c < case["seqs"]) or again or p in children or lengths[c]:
                continue
            held = tables[p, :-(-lengths[p] // rows)]
            tables[c, :len(held)] = held
            refs[held] += 1
            lengths[c] = lengths[p]
            granted[i] = 1
    elif case["op"] == "free":
        keep = st["keep"].tolist() if st["keep"] is not None else [0] * len(ids)
        for s, k in zip(ids, keep):
            if not 0 <= s < case["seqs"] or not 0 <= k < lengths[s]:
                continue
            refs[tables[s, -(-k // rows):-(-lengths[s] // rows)]] -= 1
            lengths[s] = k
    else:
        holes, movers = np.nonzero(refs == 0)[0], np.nonzero(refs > 0)[0][::-1]
        now = np.arange(case["pages"])
        for k in range(min(case["budget"], len(holes), len(movers))):
            if holes[k] > movers[k]:
                break
            now[movers[k]] = holes[k]
            refs[holes[k]], refs[movers[k]] = refs[movers[k]], 0
        for s in range(case["seqs"]):
            held = -(-lengths[s] // rows)
            tables[s, :held] = now[tables[s, :held]]
    out = {"lengths": torch.from_numpy(lengths), "refs": torch.from_numpy(refs), "tables": torch.from_numpy(tables)}
    if case["op"] in ("reserve", "fork"):
        out["granted"] = torch.tensor(granted)
    if case["op"] in ("reserve", "compact"):
        out["pool"] = None
    return out
