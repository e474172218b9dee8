// Pages of a key/value cache: argument blocks of their kernels, and the host
// arithmetic in front of them (the layout of a book, the check of a pool's
// geometry, the cut of a page into segments, launch sizes).  Plain C++, no HIP.
//
// A pool is a set of planes; page q of plane p is at base_p + q * pitch_p and
// is runs_p runs of `rows` rows of row_bytes_p bytes, one behind the other.  A
// book is int32 words in one device buffer: how long every sequence is, which
// pages it holds, how many sequences hold each page, which pages nobody holds.
#ifndef MI355_BLIT_PAGES_H_
#define MI355_BLIT_PAGES_H_

#include <stdint.h>

#include "blit_args.h"
#include "mi355_blit.h"

namespace mi355 {

// 16-byte vectors each lane keeps in flight, and with that the bytes of a page
// that one wave moves at a time.
constexpr unsigned kPageUnroll = 4;
constexpr uint32_t kSegmentBytes = kWave * 16 * kPageUnroll;

// One wave's share of a page: `bytes` bytes at `offset` of the page of one
// plane.  The table of all segments of a page, over all planes, is made once
// for a pool; a wave of a move reads one record from it and needs nothing else
// than the number of the page.
struct __attribute__((aligned(32))) PageSegment {
  uint8_t* base;  // the segment in page 0 (the plane's base + offset)
  uint64_t pitch;
  uint32_t offset;
  uint32_t bytes;      // <= kSegmentBytes
  uint32_t run_bytes;  // rows * row_bytes; 0 where the page is one run
  uint32_t row_bytes;
};
static_assert(sizeof(PageSegment) == 32, "one s_load_dwordx8");

// Pages src[i] to pages dst[i], in all planes: work item w is segment w % segs
// of move w / segs.
struct PageMoveArgs {
  const PageSegment* dst_segs;
  const PageSegment* src_segs;
  const int32_t* dst;
  const int32_t* src;
  const int32_t* valid;   // rows of every run that are moved; null: all
  const uint32_t* count;  // the number of moves, at most n; null: n
  uint32_t n;
  uint32_t segs;
  uint64_t magic_segs;  // magic_divisor(segs)
  uint32_t dst_pages;   // pages of each pool: others are not moved
  uint32_t src_pages;
  uint32_t rows;
  uint32_t waves_per_wg;
  uint32_t n_waves;
  uint32_t pad;
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
  uint32_t* count;
};

struct PageReserveArgs {
  BookPtrs book;
  PageMoveList moves;
  const int32_t* seqs;
  const int32_t* add;
  int32_t* granted;  // may be null
  uint32_t n;
  uint32_t pad;
};

struct PageForkArgs {
  BookPtrs book;
  const int32_t* parents;
  const int32_t* children;
  int32_t* granted;  // may be null
  uint32_t n;
  uint32_t pad;
};

struct PageFreeArgs {
  BookPtrs book;
  const int32_t* seqs;
  const int32_t* keep;  // null: 0
  uint32_t n;
  uint32_t pad;
};

struct PageCompactArgs {
  BookPtrs book;
  PageMoveList moves;
  int32_t* out;  // [max_moves][2]: from, to; may be null
  uint32_t max_moves;
  uint32_t pad;
};

struct PageResetArgs {
  BookPtrs book;
  uint64_t words;  // of the whole buffer
};

// Sequences that one call can name, sequences and pages that a book can have.
constexpr uint32_t kMaxList = MI355_BLIT_PAGES_MAX_LIST;
constexpr uint32_t kMaxSeqs = MI355_BLIT_PAGES_MAX_SEQS;
constexpr uint32_t kMaxPages = MI355_BLIT_PAGES_MAX_PAGES;
static_assert(1024ull * (kMaxPages + 1) < 1ull << 32, "what 1024 sequences ask for is summed up in 32 bits");
constexpr uint32_t kMaxPlanes = 4096;
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

inline uint64_t plane_page_bytes(const mi355_blit_plane_t& p, uint32_t rows) {
  // each factor below 2^32; the product of two of them fits in 64 bits
  const uint64_t run = static_cast<uint64_t>(rows) * p.row_bytes;
  if (run > 0x7fffffffull || run * p.runs > 0x7fffffffull) return ~0ull;
  return run * p.runs;
}

// What mi355_blit_pages_create takes; *segs gets the number of segments of a page.
inline int pages_check(const mi355_blit_pages_desc_t* d, uint64_t* segs) {
  if (!d || !d->planes || d->n_planes == 0 || d->num_pages == 0 || d->rows == 0) return MI355_BLIT_ERROR_INVALID_ARGUMENT;
  if ((d->max_seqs == 0) != (d->book == nullptr) || (d->max_seqs == 0) != (d->max_pages_per_seq == 0))
    return MI355_BLIT_ERROR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(d->book) & 15) return MI355_BLIT_ERROR_INVALID_ARGUMENT;
  if (d->n_planes > kMaxPlanes || d->num_pages > kMaxPages || d->max_seqs > kMaxSeqs) return MI355_BLIT_ERROR_OUT_OF_RESOURCES;
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
    total += (page + kSegmentBytes - 1) / kSegmentBytes;
  }
  // work items are counted in 32 bits
  if (total * d->num_pages > 0xffffffffull) return MI355_BLIT_ERROR_OUT_OF_RESOURCES;
  *segs = total;
  return MI355_BLIT_SUCCESS;
}

// The segments of a page, plane by plane; `out` has room for what pages_check counted.
inline void pages_segments(const mi355_blit_pages_desc_t& d, PageSegment* out) {
  for (uint32_t i = 0; i < d.n_planes; ++i) {
    const mi355_blit_plane_t& p = d.planes[i];
    const uint32_t page = static_cast<uint32_t>(plane_page_bytes(p, d.rows));
    for (uint32_t at = 0; at < page; at += kSegmentBytes) {
      PageSegment s;
      s.base = static_cast<uint8_t*>(p.base) + at;
      s.pitch = p.pitch;
      s.offset = at;
      s.bytes = page - at < kSegmentBytes ? page - at : kSegmentBytes;
      s.run_bytes = p.runs > 1 ? d.rows * p.row_bytes : 0;
      s.row_bytes = p.row_bytes;
      *out++ = s;
    }
  }
}

struct PageMovePlan {
  uint32_t nt_load, store_policy, wg_size, grid;
};

// A wave for every segment, up to a grid that fills the device: the list of a
// call that decides its moves on the device is as long as it could be, and
// mostly empty.  Over the host link at most kLinkGrid workgroups, as for the
// linear copy; what goes to the host is written through at once.
constexpr uint32_t kMoveWaves = 4;
inline PageMovePlan plan_page_moves(uint64_t n, uint64_t segs, uint64_t page_bytes, uint32_t num_cus, uint32_t route,
                                    uint32_t link_grid) {
  PageMovePlan p;
  const bool large = n * page_bytes >= (4ull << 20);
  p.nt_load = large;
  p.store_policy = route == MI355_BLIT_ROUTE_DEVICE_TO_HOST ? MI355_BLIT_STORE_SYSTEM_WT
                   : large ? MI355_BLIT_STORE_AGENT_WT : MI355_BLIT_STORE_CACHED;
  p.wg_size = kMoveWaves * kWave;
  const uint64_t want = (n * segs + kMoveWaves - 1) / kMoveWaves;
  const uint64_t most = route == MI355_BLIT_ROUTE_DEVICE ? static_cast<uint64_t>(num_cus) * 8 : link_grid;
  p.grid = static_cast<uint32_t>(want < most ? want : most);
  return p;
}

}  // namespace mi355

#endif  // MI355_BLIT_PAGES_H_
