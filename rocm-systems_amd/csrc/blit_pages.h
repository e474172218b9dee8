// Pages of a key/value cache: argument blocks of their kernels, and the host
// arithmetic in front of them (the layout of a book, the check of a pool's
// geometry, the table of its planes, launch sizes).  Plain C++, no HIP.
//
// A pool is a set of planes; page q of plane p is at base_p + q * pitch_p and
// is runs_p runs of `rows` rows of row_bytes_p bytes, one behind the other.  A
// book is int32 words in one device buffer: how long every sequence is, which
// pages it holds, how many sequences hold each page, which pages nobody holds.
#ifndef MI355_BLIT_PAGES_H_
#define MI355_BLIT_PAGES_H_

#include <stdint.h>

#include "blit_args.h"
#include "blit_plan.h"
#include "mi355_blit.h"

namespace mi355 {

// A wave moves a piece of a page at a time: 16 bytes for each lane, or four
// times that where the first rows of the pages are moved only, so that fewer
// waves go through the longer chain of loads in front of such a move, and fewer find
// nothing to do (4 KiB against 1 KiB: 190 pages of 24 planes, half of their 33 rows
// of 80 bytes in 5 runs, 13.5 us against 19.5; 600 pages of 1 MiB, half of their
// rows, 137 against 482; whole pages, 800 of 1 MiB: 285 us with 1 KiB, 330 with
// 4 KiB).
constexpr unsigned kPieceUnrolls[] = {1, 4};
constexpr uint32_t piece_bytes(unsigned unroll) { return kWave * 16 * unroll; }

// What a wave needs to know of a plane.  The tables of a pool, made once, one for
// each size of piece, have a record for each piece of a page, counted through all
// planes, and all records of a plane are the same: work item w of n moves belongs
// to the plane of piece w / n, whatever n is.
struct __attribute__((aligned(64))) PagePlane {
  uint8_t* base;
  uint64_t pitch;
  uint64_t magic_pieces;  // magic_divisor(pieces)
  uint32_t pieces;        // of a page in this plane
  uint32_t first;         // pieces of the planes before it
  uint32_t bytes;         // of a page in this plane
  uint32_t run_bytes;     // rows * row_bytes; 0 where the page is one run
  uint32_t row_bytes;
  uint32_t runs;
  uint32_t pad[2];
};
static_assert(sizeof(PagePlane) == 64, "one s_load_dwordx16");

// The number of moves that a call has decided on the device, with what it takes
// to divide by it.
struct PageMoveCount {
  uint32_t n;
  uint32_t pad;
  uint64_t magic;  // magic_divisor(n)
};

// Pages src[i] to pages dst[i], in all planes.
struct PageMoveArgs {
  const PagePlane* dst_planes;
  const PagePlane* src_planes;
  const int32_t* dst;
  const int32_t* src;
  const int32_t* valid;        // rows of every run that are moved; null: all
  const PageMoveCount* count;  // the number of moves, at most n; null: n
  uint64_t magic_n;            // magic_divisor(n)
  uint64_t magic_even;         // magic_divisor(even_pieces)
  uint32_t n;
  uint32_t pieces;       // of a page, over all planes
  uint32_t even_pieces;  // of a page in one plane, where all planes have the same number; 0 otherwise
  uint32_t pad;
  uint32_t dst_pages;  // pages of each pool: others are not moved
  uint32_t src_pages;
  uint32_t rows;
  uint32_t n_waves;
};

// The parts of a book on the device.
struct BookPtrs {
  int32_t* head;     // [0]: moves of the last compaction
  int32_t* lengths;
  int32_t* refs;
  uint32_t* bits;    // 16-byte aligned
  int32_t* tables;
  uint32_t num_pages;
  uint32_t max_seqs;
  uint32_t width;    // pages a sequence can hold
  uint32_t rows;
  uint64_t magic_rows;  // magic_divisor(rows)
};

// Moves that a call decides on the device, for the launches behind it.
struct PageMoveList {
  int32_t* src;
  int32_t* dst;
  int32_t* valid;   // reserve only
  int32_t* remap;   // compact only: the new number of a page that moved
  PageMoveCount* count;
};

// What the first launch of a reservation leaves for the second: for each entry
// how many pages the entries before it get, the sequence (and whether its first
// page takes the place of a shared one) and the first table slot, and for each
// two words of the free bits how many free pages are in front of them.
struct PageReserveWork {
  uint32_t* start;
  uint32_t* who;  // sequence, top bit: copies
  uint32_t* slot;
  uint32_t* pairs;
  uint32_t* wanted;  // pages that the second launch hands out
};

struct PageReserveArgs {
  BookPtrs book;
  PageMoveList moves;
  PageReserveWork work;
  const int32_t* seqs;
  const int32_t* add;
  int32_t* granted;  // may be null
  uint32_t n;
  uint32_t lane_vecs;  // 16-byte vectors of free bits for each of 1024 lanes: a power of two
};

struct PageFinishArgs {
  PageMoveArgs moves;
  BookPtrs book;
  PageReserveWork work;
  uint32_t n;
  uint32_t n_pairs;
  uint32_t assign_wgs;  // workgroups that hand out pages; those behind them move
  uint32_t pad;
};

struct PageForkArgs {
  BookPtrs book;
  const int32_t* parents;
  const int32_t* children;
  int32_t* granted;  // may be null
  uint32_t* made;    // not null: the children's lengths for the second launch
  uint32_t n;
  uint32_t wg_size;
  uint32_t chunk;    // pages of a table that one workgroup goes through
  uint32_t pad;
};

struct PageFreeArgs {
  BookPtrs book;
  const int32_t* seqs;
  const int32_t* keep;  // null: 0
  uint32_t n;
  uint32_t wg_size;
  uint32_t chunk;       // as in PageForkArgs
  uint32_t pad;
};

struct PageCompactArgs {
  BookPtrs book;
  PageMoveList moves;
  uint32_t* pairs;  // free pages in front of each two words of the free bits
  uint32_t* live;   // pages in use
  int32_t* out;     // [max_moves][2]: from, to; may be null
  uint32_t max_moves;
  uint32_t lane_vecs;  // as in PageReserveArgs
  uint32_t n_pairs;
  uint32_t pair_wgs;   // workgroups that go through the pairs
};

struct PageCompactFinishArgs {
  PageMoveArgs moves;
  PageCompactArgs compact;
};

struct PageResetArgs {
  BookPtrs book;
  uint64_t words;  // of the whole buffer
  uint64_t lanes;  // of the launch
};

// The free bits as the first launch of a reservation or a compaction takes
// them: one stretch of 16-byte vectors for each of 1024 lanes.
inline uint32_t reserve_lane_vecs(uint32_t num_pages) {
  uint32_t v = 1;
  while (static_cast<uint64_t>(v) * 1024 * 128 < num_pages) v *= 2;
  return v;
}

// Sequences that one call can name, sequences and pages that a book can have.
constexpr uint32_t kMaxList = MI355_BLIT_PAGES_MAX_LIST;
constexpr uint32_t kMaxSeqs = MI355_BLIT_PAGES_MAX_SEQS;
constexpr uint32_t kMaxPages = MI355_BLIT_PAGES_MAX_PAGES;
static_assert(1024ull * (kMaxPages + 1) < 1ull << 32, "what 1024 sequences ask for is summed up in 32 bits");
constexpr uint32_t kMaxPlanes = 4096;
constexpr uint64_t kMaxPieces = 1u << 22;  // a page of 4 GiB over all planes
// Every part of a book starts at a multiple of this many words.
constexpr uint64_t kBookAlign = 64;

inline uint64_t book_up(uint64_t words) { return (words + kBookAlign - 1) / kBookAlign * kBookAlign; }

inline int pages_book_layout(uint32_t num_pages, uint32_t max_seqs, uint32_t width, mi355_blit_book_t* out) {
  if (!out || num_pages == 0 || max_seqs == 0 || width == 0) return MI355_BLIT_ERROR_INVALID_ARGUMENT;
  if (num_pages > kMaxPages || max_seqs > kMaxSeqs || width > kMaxPages) return MI355_BLIT_ERROR_OUT_OF_RESOURCES;
  out->lengths = kBookAlign;
  out->ref_counts = out->lengths + book_up(max_seqs);
  out->free_bits = out->ref_counts + book_up(num_pages);
  out->tables = out->free_bits + book_up((num_pages + 31ull) / 32);
  out->words = out->tables + book_up(static_cast<uint64_t>(max_seqs) * width);
  return MI355_BLIT_SUCCESS;
}

inline BookPtrs pages_book_ptrs(int32_t* book, const mi355_blit_book_t& at, uint32_t num_pages, uint32_t max_seqs,
                                uint32_t width, uint32_t rows) {
  return {book, book + at.lengths, book + at.ref_counts, reinterpret_cast<uint32_t*>(book + at.free_bits),
          book + at.tables, num_pages, max_seqs, width, rows, magic_divisor(rows)};
}

// The work memory of a book's calls, in words.  Every word that a launch reads
// was written by one before it in the same call.
struct PageWorkLayout {
  uint64_t move_src, move_dst, move_valid, remap, start, who, slot, pairs, words;
};

inline PageWorkLayout pages_work_layout(uint32_t num_pages) {
  // a move for each entry of a reservation, or for each two pages of a compaction
  const uint64_t moves = book_up(num_pages > 2 * kMaxList ? num_pages / 2 : kMaxList);
  PageWorkLayout w;
  w.move_src = kBookAlign;  // the count of moves and that of pages to hand out are in front
  w.move_dst = w.move_src + moves;
  w.move_valid = w.move_dst + moves;
  w.remap = w.move_valid + kMaxList;
  w.start = w.remap + book_up(num_pages);
  w.who = w.start + kMaxList;
  w.slot = w.who + kMaxList;
  w.pairs = w.slot + kMaxList;
  w.words = w.pairs + book_up((num_pages + 127ull) / 128 * 2);
  return w;
}

inline PageMoveList pages_move_list(uint32_t* work, const PageWorkLayout& w) {
  int32_t* p = reinterpret_cast<int32_t*>(work);
  return {p + w.move_src, p + w.move_dst, p + w.move_valid, p + w.remap, reinterpret_cast<PageMoveCount*>(work)};
}

inline PageReserveWork pages_reserve_work(uint32_t* work, const PageWorkLayout& w) {
  return {work + w.start, work + w.who, work + w.slot, work + w.pairs, work + 16};
}

inline uint64_t plane_page_bytes(const mi355_blit_plane_t& p, uint32_t rows) {
  // each factor below 2^32; the product of two of them fits in 64 bits
  const uint64_t run = static_cast<uint64_t>(rows) * p.row_bytes;
  if (run > 0x7fffffffull || run * p.runs > 0x7fffffffull) return ~0ull;
  return run * p.runs;
}

// What mi355_blit_pages_create takes; *pieces gets the number of the smallest pieces of a page.
inline int pages_check(const mi355_blit_pages_desc_t* d, uint64_t* pieces) {
  if (!d || !d->planes || d->n_planes == 0 || d->num_pages == 0 || d->rows == 0)
    return MI355_BLIT_ERROR_INVALID_ARGUMENT;
  if ((d->max_seqs == 0) != (d->book == nullptr) || (d->max_seqs == 0) != (d->max_pages_per_seq == 0))
    return MI355_BLIT_ERROR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(d->book) & 15) return MI355_BLIT_ERROR_INVALID_ARGUMENT;
  if (d->n_planes > kMaxPlanes || d->num_pages > kMaxPages || d->max_seqs > kMaxSeqs)
    return MI355_BLIT_ERROR_OUT_OF_RESOURCES;
  // a sequence's tokens are counted in 31 bits
  if (static_cast<uint64_t>(d->max_pages_per_seq) * d->rows > 0x7fffffffull) return MI355_BLIT_ERROR_OUT_OF_RESOURCES;
  uint64_t total = 0;
  for (uint32_t i = 0; i < d->n_planes; ++i) {
    const mi355_blit_plane_t& p = d->planes[i];
    if (!p.base || p.row_bytes == 0 || p.runs == 0) return MI355_BLIT_ERROR_INVALID_ARGUMENT;
    const uint64_t page = plane_page_bytes(p, d->rows);
    if (page == ~0ull) return MI355_BLIT_ERROR_OUT_OF_RESOURCES;
    if (d->num_pages > 1 && p.pitch < page) return MI355_BLIT_ERROR_INVALID_ARGUMENT;
    // the last byte of the plane has an address
    const unsigned __int128 end = static_cast<unsigned __int128>(d->num_pages - 1) * p.pitch + page +
                                  reinterpret_cast<uintptr_t>(p.base);
    if (end >> 64) return MI355_BLIT_ERROR_INVALID_ARGUMENT;
    total += (page + piece_bytes(1) - 1) / piece_bytes(1);
  }
  // work items are counted in 32 bits; the tables have a record for each piece
  if (total > kMaxPieces || total * d->num_pages > 0xffffffffull) return MI355_BLIT_ERROR_OUT_OF_RESOURCES;
  *pieces = total;
  return MI355_BLIT_SUCCESS;
}

// The table of a pool for one size of piece; returns the number of its records.
// `out` may be null, and has room for what pages_check counted otherwise.
inline uint32_t pages_planes(const mi355_blit_pages_desc_t& d, unsigned unroll, PagePlane* out) {
  uint32_t first = 0;
  for (uint32_t i = 0; i < d.n_planes; ++i) {
    const mi355_blit_plane_t& p = d.planes[i];
    PagePlane r{};
    r.base = static_cast<uint8_t*>(p.base);
    r.pitch = p.pitch;
    r.bytes = static_cast<uint32_t>(plane_page_bytes(p, d.rows));
    r.pieces = (r.bytes + piece_bytes(unroll) - 1) / piece_bytes(unroll);
    r.magic_pieces = magic_divisor(r.pieces);
    r.first = first;
    r.run_bytes = p.runs > 1 ? d.rows * p.row_bytes : 0;
    r.row_bytes = p.row_bytes;
    r.runs = p.runs;
    for (uint32_t k = 0; out && k < r.pieces; ++k) out[first + k] = r;
    first += r.pieces;
  }
  return first;
}

// Lanes for each entry of a call that goes through tables of `width` pages, four
// at a time.
inline uint32_t table_wg_size(uint32_t width) { return width <= 1024 ? 256 : 1024; }
// Pages of a table that one workgroup goes through where an entry has several
// (64 of them at most, so that a grid for the longest list has a size), and the
// width from which on it has.
constexpr uint32_t kTableChunk = 4096;
constexpr uint32_t kSplitWidth = 2 * kTableChunk;
inline uint32_t table_chunk(uint32_t width) {
  const uint32_t share = (width / 64 + 4) / 4 * 4;
  return share > kTableChunk ? share : kTableChunk;
}
inline uint32_t table_chunks(uint32_t width) { return (width + table_chunk(width) - 1) / table_chunk(width); }
static_assert(64ull * kMaxList * 1024 <= kMaxGridWorkItems, "work-items of a grid are counted in 31 bits");

// From so many pages that a list can free on, the free bits are made from the
// counts: 256 sequences of 375 pages (width 512) 14.4 us with an atomic for each
// page's bit, 10.8 so; 128 sequences 12.3 and 11.1; 100 in tables of 700 8.5 and 11.5.
constexpr uint64_t kFreeByCounts = 1u << 17;

// Moves that a compaction may make: each takes a page that is in use and a free
// one.  (One page: none, but the launches say so in the book's head.)
inline uint32_t most_page_moves(uint32_t max_moves, uint32_t num_pages) {
  const uint32_t pairs = num_pages > 1 ? num_pages / 2 : 1;
  return max_moves < pairs ? max_moves : pairs;
}

// Moves of a compaction that its first launch finds by itself.
constexpr uint32_t kListedAtOnce = 1024;

// Workgroups that go through all pages, 256 at a time.
inline uint32_t page_pairs(uint32_t num_pages) { return (num_pages + 63) / 64; }
inline uint32_t page_pair_wgs(uint32_t num_pages) {
  const uint32_t want = (num_pages + 255) / 256;
  return want < 1024 ? want : 1024;
}

struct PageMovePlan {
  uint32_t table;  // index into kPieceUnrolls
  uint32_t nt_load, store_policy, grid;
};

// How n moves are launched; most_per_cu not 0: n is what a list has room for,
// the device knows how many there are, and this many workgroups for each CU are
// the most.  pieces: of a page, for each size of piece.
//
// Cache policy, by the bytes that are likely moved (half of the pages where only
// their first rows are).  Measured, pages of 32 planes of 32 KiB, loads and
// stores cached / non-temporal loads with stores written through / with
// non-temporal stores: 64 MiB 22.8 / 22.0 / 27.7 us, 128 MiB 42.9 / 41.9 / 51.0,
// 192 MiB 79.2 / 61.0 / 74.2, 256 MiB 106.7 / 83.1 / 98.5, 384 MiB 156 / 153 / 143,
// 600 MiB 237 / 239 / 221.
//
// A wave for each piece: the dispatcher hands pieces out in order, which keeps
// what is in flight close together (1 GiB, 32 KiB a page and plane: 369 us; with 32
// workgroups for each CU whose waves stride 425, and 422 with the next piece's
// loads in front of the stores).  A list of unknown length is as long as its
// room: a wave too many costs 0.05 ns, so kMostListed workgroups for each CU (26
// us of them at most), and strides beyond (800 MiB 292 us; with 128 for each CU
// 325).  A reservation's list is as long as the call's and mostly empty:
// kMostReserved for each CU (256 copies of 16 KiB in 32 planes 27.5 us; a wave
// for each piece 25.5, and 6 us where nothing is copied).  Over the host link at
// most link_grid workgroups, as for the linear copy (57 GB/s either way); what
// goes to the host is written through at once.
constexpr uint32_t kMoveWaves = 4;
constexpr uint32_t kMostListed = 512, kMostReserved = 16;
constexpr uint64_t kMoveStreams = 128ull << 20, kMoveNtStores = 320ull << 20;

inline PageMovePlan plan_page_moves(uint64_t n, uint32_t most_per_cu, bool cut, const uint32_t (&pieces)[2],
                                    uint64_t page_bytes, uint32_t num_cus, uint32_t route, uint32_t link_grid) {
  PageMovePlan p;
  p.table = cut ? 1 : 0;
  const uint64_t bytes = cut ? n * page_bytes / 2 : n * page_bytes;
  p.nt_load = bytes >= kMoveStreams;
  p.store_policy = route == MI355_BLIT_ROUTE_DEVICE_TO_HOST ? MI355_BLIT_STORE_SYSTEM_WT
                   : bytes >= kMoveNtStores ? MI355_BLIT_STORE_NT
                   : bytes >= kMoveStreams ? MI355_BLIT_STORE_AGENT_WT : MI355_BLIT_STORE_CACHED;
  const uint64_t want = (n * pieces[p.table] + kMoveWaves - 1) / kMoveWaves;
  const uint64_t most = route != MI355_BLIT_ROUTE_DEVICE ? link_grid
                        : most_per_cu ? static_cast<uint64_t>(num_cus) * most_per_cu
                                      : kMaxGridWorkItems / (kMoveWaves * kWave);
  p.grid = static_cast<uint32_t>(want < most ? want : most);
  return p;
}

}  // namespace mi355

#endif  // MI355_BLIT_PAGES_H_
