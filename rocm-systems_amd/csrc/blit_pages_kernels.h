// Kernels for the pages of a key/value cache (blit_pages.h has their arguments).
//
// What they have in common: lists, tables and counts stay on the device, so a
// call needs no answer from it before the next one can be submitted, and all of
// them can be recorded into a graph.  No workgroup waits for another; what one
// launch decides for many workgroups, the next launch reads.  Numbers of pages
// and of sequences come from memory that the caller can write, so every one of
// them is checked before it becomes an address.
#ifndef MI355_BLIT_PAGES_KERNELS_H_
#define MI355_BLIT_PAGES_KERNELS_H_

#include "blit_kernels.h"
#include "blit_pages.h"

namespace mi355 {

// ---------------------------------------------------------------------------
// Moves.  One wave moves one piece of a page.  Work items go through the
// planes one after the other, in each through the moves, and in each move through
// the pieces of the page: what is in flight then lies in one plane, some tens of
// MiB, and not in all of them (512 pages of 64 planes of 32 KiB, 1 GiB each way: 369 us,
// 5.8 TB/s, against 403 us in the order move, plane, piece; a linear copy of as many bytes 313).
// Bound by memory: the counters show as many bytes read and written as the pages have.
// First rows are bound by latency instead (below, and 600 pages of 1 MiB, half of
// their rows, 629 MB: 137 us, 4.6 TB/s): a lane's four vectors each have a
// condition of their own, and the compiler waits for each before the next.
// ---------------------------------------------------------------------------

// A page of several runs of which only the first rows are moved, `limit` bytes
// of each run; dp and sp are the pages.  The units of work are the vectors of the
// moved bytes alone, one run's behind the other's, so that no lane is idle; the
// last vector of a run ends where its rows end, and moves again some bytes of the one in
// front of it (fewer bytes than a vector go one by one).  The waves of a page
// take at least as many units each as their piece has, the last ones none.  246
// pages of 12 planes, half of their 32 rows of 42 bytes in 7 runs: 7.5 us, and 24.5
// where vectors that lie across an end go byte by byte; 190 pages of 24
// planes in 5 runs of 33 rows of 80 bytes 14.6, and 15.5 over all vectors of the page.
// Bound by latency: the waves of the latter spend three quarters of their time
// waiting, behind the loads that lead to their rows and then for up to four vectors a lane
// one after the other, and half of them find nothing to do; 34.8 MB are read and 32.9
// written for 31.8.  (As many bytes of whole pages take 13.4 us, a linear copy 9.3; a variant
// with four vectors a lane on the way at once was slower, 17.1.)
template <int U, bool NTL, int ST>
MI355_DEVICE void move_cut_runs(uint8_t* dp, const uint8_t* sp, const PagePlane& g, unsigned piece, unsigned pieces,
                                unsigned limit, unsigned lane) {
  const unsigned per_run = limit < 16 ? limit : (limit + 15) / 16;
  const unsigned all = g.runs * per_run;
  unsigned share = (all + pieces - 1) / pieces;
  if (share < U * kWave) share = U * kWave;
  // (no more than a page's bytes, and 2^19 pieces beyond them: 32 bits)
  const unsigned begin = piece * share;
  const unsigned end = begin + share < all ? begin + share : all;
  for (unsigned i = begin + lane; i < end; i += kWave) {
    const unsigned run = i / per_run;
    const unsigned k = i - run * per_run;
    if (limit < 16) {
      const unsigned at = run * g.run_bytes + k;
      st_u8(dp + at, ld_u8(sp + at));
    } else {
      const unsigned at = run * g.run_bytes + (16 * k + 16 <= limit ? 16 * k : limit - 16);
      st_v4_any<ST>(reinterpret_cast<uintptr_t>(dp + at), ld_v4_any<NTL>(sp + at));
    }
  }
}

template <int U, bool NTL, int ST>
MI355_DEVICE void page_move_body(const PageMoveArgs& a, uint64_t first_wave) {
  constexpr bool kCut = U == kPieceUnrolls[1];  // a.valid is not null
  const unsigned lane = thread_in_workgroup() & (kWave - 1);
  uint32_t n = a.n;
  uint64_t magic_n = a.magic_n;
  if (a.count) {
    const PageMoveCount found = ld_uniform_count(a.count);
    if (found.n < n) n = found.n, magic_n = found.magic;
  }
  // fits in 32 bits (checked on the host); the sum with n_waves may not
  const uint64_t total = static_cast<uint64_t>(n) * a.pieces;
  for (uint64_t w = first_wave; w < total; w += a.n_waves) {
    const uint32_t item = static_cast<uint32_t>(w);
    // (the limits on piece and move here and below hold, unless another call on
    // the book has changed the count meanwhile: then the wave moves some piece of some
    // page of the lists, and touches nothing outside the pool.  Selections: a branch costs 9 % of
    // a compaction, these less than 1 % of any workload)
    uint32_t some_piece = div_magic(item, magic_n);
    some_piece = some_piece < a.pieces ? some_piece : 0;
    uint32_t first = 0, pieces = a.even_pieces;
    uint64_t magic_pieces = a.magic_even;
    if (pieces) {
      // the same number in all planes: the list can be read together with the planes
      first = div_magic(some_piece, magic_pieces) * pieces;
      some_piece = first;
    } else {
      const PagePlane p = ld_uniform_plane(a.dst_planes + some_piece);
      first = p.first, pieces = p.pieces, magic_pieces = p.magic_pieces;
    }
    const uint32_t in_plane = item - n * first;
    uint32_t move = div_magic(in_plane, magic_pieces);
    move = move < n ? move : n - 1;
    uint32_t piece = in_plane - move * pieces;
    piece = piece < pieces ? piece : 0;
    const uint32_t offset = piece * piece_bytes(U);
    const uint32_t to = ld_uniform_u32(reinterpret_cast<const uint32_t*>(a.dst + move));
    const uint32_t from = ld_uniform_u32(reinterpret_cast<const uint32_t*>(a.src + move));
    const PagePlane d = ld_uniform_plane(a.dst_planes + some_piece);
    const PagePlane s = ld_uniform_plane(a.src_planes + some_piece);
    uint32_t valid = a.rows;
    if constexpr (kCut) {
      const int32_t v = static_cast<int32_t>(ld_uniform_u32(reinterpret_cast<const uint32_t*>(a.valid + move)));
      if (v < static_cast<int32_t>(a.rows)) valid = v > 0 ? v : 0;
    }
    // a negative number is a large unsigned one
    if (to >= a.dst_pages || from >= a.src_pages || valid == 0) continue;
    uint8_t* dp = d.base + to * d.pitch + offset;
    const uint8_t* sp = s.base + from * s.pitch + offset;
    unsigned bytes = d.bytes - offset < piece_bytes(U) ? d.bytes - offset : piece_bytes(U);
    if constexpr (kCut) {
      if (valid < a.rows) {
        const unsigned limit = valid * d.row_bytes;
        if (d.run_bytes) {
          move_cut_runs<U, NTL, ST>(dp - offset, sp - offset, d, piece, pieces, limit, lane);
          continue;
        }
        if (limit <= offset) continue;
        if (limit - offset < bytes) bytes = limit - offset;
      }
    }
    const unsigned vecs = bytes / 16;
    v4u x[U];
#pragma unroll
    for (unsigned u = 0; u < U; ++u)
      if (lane + u * kWave < vecs) x[u] = ld_v4_any<NTL>(sp + 16 * (lane + u * kWave));
#pragma unroll
    for (unsigned u = 0; u < U; ++u)
      if (lane + u * kWave < vecs) st_v4_any<ST>(reinterpret_cast<uintptr_t>(dp + 16 * (lane + u * kWave)), x[u]);
    const unsigned tail = bytes & 15;
    if (lane < tail) st_u8(dp + 16 * vecs + lane, ld_u8(sp + 16 * vecs + lane));
  }
}

// ---------------------------------------------------------------------------
// The book.
// ---------------------------------------------------------------------------

// Pages that `tokens` tokens take.
MI355_DEVICE uint32_t pages_held(uint32_t tokens, const BookPtrs& b) {
  return div_magic(tokens, b.magic_rows) + (tokens - div_magic(tokens, b.magic_rows) * b.rows ? 1 : 0);
}

// Four words of the free bits.
struct BitTile {
  uint32_t word[4];
};

MI355_DEVICE uint32_t count_bits(const BitTile& t) {
  return popcount32(t.word[0]) + popcount32(t.word[1]) + popcount32(t.word[2]) + popcount32(t.word[3]);
}

// A table in LDS that finds equal keys among the 1024 entries of a turn: open
// addressing over twice as many slots, so that a free one is always found.
constexpr uint32_t kSlots = 2048;
constexpr uint32_t kNoKey = ~0u;

MI355_DEVICE uint32_t hash_slot(uint32_t* keys, uint32_t key) {
  uint32_t at = (key * 2654435761u) >> 21;  // 11 bits
  for (;;) {
    const uint32_t was = lds_compare_swap(keys + at, kNoKey, key);
    if (was == kNoKey || was == key) return at;
    at = (at + 1) & (kSlots - 1);
  }
}

// A word of the free bits without the pages that do not exist.
MI355_DEVICE uint32_t existing_bits(const BookPtrs& b, uint32_t word, uint32_t index) {
  const uint32_t first = 32 * index;
  if (first >= b.num_pages) return 0;
  return b.num_pages - first >= 32 ? word : word & ((1u << (b.num_pages - first)) - 1);
}

// Vector v of the free bits, which may lie behind them.
MI355_DEVICE BitTile load_bits_vec(const BookPtrs& b, uint32_t v) {
  BitTile t{};
  if (128 * v < b.num_pages) {
    const v4u x = ld_v4<false>(reinterpret_cast<const v4u_a4*>(b.bits + 4 * v));
    t.word[0] = existing_bits(b, x.x, 4 * v);
    t.word[1] = existing_bits(b, x.y, 4 * v + 1);
    t.word[2] = existing_bits(b, x.z, 4 * v + 2);
    t.word[3] = existing_bits(b, x.w, 4 * v + 3);
  }
  return t;
}

// Place of the bit of `word` that has `r` set bits below it.
MI355_DEVICE uint32_t nth_bit(uint32_t word, uint32_t r) {
  uint32_t at = 0;
#pragma unroll
  for (uint32_t half = 16; half >= 1; half >>= 1) {
    const uint32_t below = popcount32(word >> at & ((1u << half) - 1));
    if (r >= below) r -= below, at += half;
  }
  return at;
}

// The free page (FREE; otherwise the page in use) that has `rank` such pages
// below it; groups[g] is the number of free pages in front of lane g's stretch.
template <bool FREE>
MI355_DEVICE uint32_t select_page(const BookPtrs& b, const uint32_t* groups, uint32_t lane_vecs, uint32_t rank) {
  const uint32_t stretch = 128 * lane_vecs;
  uint32_t g = 0;  // the last stretch that starts at or in front of it
#pragma unroll
  for (uint32_t step = 512; step >= 1; step >>= 1) {
    const uint32_t front = FREE ? groups[g + step] : (g + step) * stretch - groups[g + step];
    if (front <= rank && (FREE || (g + step) * stretch < b.num_pages)) g += step;
  }
  uint32_t r = rank - (FREE ? groups[g] : g * stretch - groups[g]);
  for (uint32_t v = g * lane_vecs; v < (g + 1) * lane_vecs; ++v) {
    const BitTile bits = load_bits_vec(b, v);
#pragma unroll
    for (unsigned k = 0; k < 4; ++k) {
      const uint32_t word = FREE ? bits.word[k] : existing_bits(b, ~bits.word[k], 4 * v + k);
      const uint32_t here = popcount32(word);
      if (r < here) return 32 * (4 * v + k) + nth_bit(word, r);
      r -= here;
    }
  }
  return 0;  // not reached: the rank is below the number of such pages
}

// The page with rank nth goes to the entry whose share of the running sum of
// needs nth falls into.
MI355_DEVICE void hand_out(const BookPtrs& b, uint32_t page, uint32_t nth, uint32_t start, uint32_t who, uint32_t slot) {
  const uint32_t seq = who & 0x7fffffffu;
  const uint32_t at = slot + (nth - start);
  // not so, unless another call on the book has changed the list meanwhile
  if (seq >= b.max_seqs || at >= b.width) return;
  st_obj(b.tables + static_cast<uint64_t>(seq) * b.width + at, static_cast<int32_t>(page));
  st_obj(b.refs + page, 1);
}

// An entry of a reservation with what the book says of its sequence.
struct ReserveEntry {
  uint32_t seq, tokens, old_pages, new_pages;
  int32_t more;
  bool valid;      // but for an earlier entry of the sequence
  uint32_t fill;   // rows in use on the last page
  uint32_t tail;   // the last page, where it has room and rows are to be added
  uint32_t holders;  // of the tail; 0 where there is none
};

// `changed`: earlier turns of the call may have changed the counts.
MI355_DEVICE ReserveEntry load_reserve_entry(const PageReserveArgs& a, uint32_t i, bool changed) {
  const BookPtrs& b = a.book;
  ReserveEntry e{~0u, 0, 0, 0, 0, false, 0, 0, 0};
  if (i >= a.n) return e;
  e.seq = static_cast<uint32_t>(ld_obj(a.seqs + i));
  e.more = ld_obj(a.add + i);
  if (e.seq >= b.max_seqs) return e;
  e.tokens = ld_obj(b.lengths + e.seq);
  if (e.more < 0 || static_cast<int32_t>(e.tokens) < 0) return e;
  // both below 2^31, so the sum is below 2^32
  e.old_pages = pages_held(e.tokens, b);
  e.new_pages = pages_held(e.tokens + e.more, b);
  if (e.new_pages > b.width) return e;
  e.valid = true;
  e.fill = e.tokens - div_magic(e.tokens, b.magic_rows) * b.rows;
  if (e.more == 0 || e.fill == 0) return e;
  e.tail = ld_obj(b.tables + static_cast<uint64_t>(e.seq) * b.width + e.old_pages - 1);
  if (e.tail >= b.num_pages) {
    e.valid = false;  // not a page
    return e;
  }
  e.holders = changed ? ld_agent_u32(reinterpret_cast<const uint32_t*>(b.refs + e.tail))
                      : static_cast<uint32_t>(ld_obj(b.refs + e.tail));
  return e;
}

// Room for new tokens, in two launches, so that the result is that of taking
// the entries one by one.
//
// The first, one workgroup of 1024 lanes, takes the entries 1024 at a time:
// which of them name a sequence first (a table in LDS, and a bit for each
// sequence that an earlier turn named), which of them have to copy a last page
// that others hold as well, how many pages each needs and how many the entries
// before it get, out of how many free ones.  The k-th lowest free page goes to the
// entry whose share of the running sum k falls into.  Where the pages are no
// more than the lanes (a decode step), it hands them out itself, a lane for each page; otherwise
// the second launch does, over the whole device, next to the copies.
//
// Bound by latency: a chain of dependent loads (entry, length, last page,
// its count, free bits) and a dozen barriers.  48 sequences that get a token each
// 5.6 us and 2 for the second launch; 300 prompts, 19,000 pages 7.1 and 4.9 (one
// workgroup that hands out all of them itself 244); 256 forks of 32 prompts of which 224
// copy their last page 9.0, and 18.3 for 115 MB of copies (6.3 TB/s).  In pools of
// more than 131,072 pages a lane goes through its stretch of the free bits one vector
// after the other: for 48 sequences that get a page each the first launch takes 7.0 us
// with 4,096 and with 131,072 pages, 22 with 2,000,000, 47 with 4,194,240.  8,192
// entries take 58 us, 1024 at a time.
MI355_DEVICE void page_reserve_body(const PageReserveArgs& a) {
  MI355_LDS uint32_t scan_a[16], scan_b[16];
  MI355_LDS uint32_t keys[kSlots], first[kSlots], asked[kSlots];
  MI355_LDS uint32_t seen[kMaxSeqs / 32];
  MI355_LDS uint32_t start[1024], who[1024], slot_of[1024], groups[1024];
  MI355_LDS uint32_t any_shared, any_refused, handed, n_moves;
  const BookPtrs& b = a.book;
  const uint32_t t = thread_in_workgroup();

  // The first entries' loads are under way while the free bits are summed up.
  ReserveEntry mine = load_reserve_entry(a, t, false);
  // the free bits, a stretch for each lane
  const BitTile kept = load_bits_vec(b, t * a.lane_vecs);
  uint32_t bits_here = count_bits(kept);
  for (uint32_t k = 1; k < a.lane_vecs; ++k) bits_here += count_bits(load_bits_vec(b, t * a.lane_vecs + k));
  for (uint32_t k = t; k < kSlots; k += 1024) keys[k] = kNoKey, first[k] = ~0u;
  if (a.n > 1024)
    for (uint32_t k = t; k < kMaxSeqs / 32; k += 1024) seen[k] = 0;
  if (t == 0) n_moves = 0, handed = 0, any_shared = 0, any_refused = 0;
  uint32_t free_pages;
  const uint32_t in_front = block_scan_1024(bits_here, scan_b, &free_pages);
  groups[t] = in_front;

  bool stopped = false;  // the same in all lanes, as are the next two
  uint32_t carry = 0;    // pages that earlier turns get
  uint32_t left_over = 0;  // pages that the second launch hands out
  for (uint32_t base = 0; base < a.n; base += 1024) {
    const uint32_t i = base + t;
    if (stopped) {
      if (i < a.n) {
        if (a.granted) st_obj(a.granted + i, 0);
        st_u32(a.work.start + i, ~0u);
      }
      continue;
    }
    if (base) {
      mine = load_reserve_entry(a, i, true);
      for (uint32_t k = t; k < kSlots; k += 1024) keys[k] = kNoKey, first[k] = ~0u;
      if (t == 0) any_shared = 0, any_refused = 0;
      workgroup_barrier();
    }
    const uint32_t s = mine.seq, tokens = mine.tokens, fill = mine.fill, tail = mine.tail, holders = mine.holders;
    const int32_t more = mine.more;
    const bool named = s < b.max_seqs;
    uint32_t slot = 0;
    bool again = false;
    if (named) {
      again = base && (seen[s / 32] >> (s % 32) & 1);
      slot = hash_slot(keys, s);
      lds_min(first + slot, t);
    }
    // (perhaps by an entry that is refused)
    if (static_cast<int32_t>(holders) > 1) any_shared = 1;
    workgroup_barrier();
    if (named) {
      again = again || first[slot] != t;
      if (a.n > 1024) lds_or(seen + s / 32, 1u << (s % 32));
    }
    const uint32_t old_pages = mine.old_pages, new_pages = mine.new_pages;
    const bool ok = mine.valid && !again;
    const bool shared = ok && static_cast<int32_t>(holders) > 1;
    bool copies = shared;
    uint32_t leavers = 0;  // not 0 in one of the askers of a page: how many of them copy it
    if (any_shared) {
      // With as many askers as holders, the last of them finds the page its own.
      workgroup_barrier();  // the table of sequences has been read
      for (uint32_t k = t; k < kSlots; k += 1024) keys[k] = kNoKey, first[k] = 0, asked[k] = 0;
      workgroup_barrier();
      if (shared) {
        slot = hash_slot(keys, tail);
        lds_max(first + slot, t);
        lds_add(asked + slot, 1);
      }
      workgroup_barrier();
      if (shared && first[slot] == t) {
        leavers = asked[slot];
        if (leavers == holders) copies = false, --leavers;
      }
    }
    uint32_t need = ok ? new_pages - old_pages + (copies ? 1 : 0) : 0;
    // more than the pool has is as good as one more: the sum over 1024 entries
    // stays below 2^32 (kMaxPages)
    if (need > b.num_pages) need = b.num_pages + 1;
    uint32_t total;
    const uint32_t before = block_scan_1024(need, scan_a, &total);
    const bool granted = ok && before + need <= free_pages - carry;
    if (ok && !granted) any_refused = 1;
    if (granted && need) lds_max(&handed, carry + before + need);
    start[t] = carry + before;
    who[t] = s | (copies ? 1u << 31 : 0);
    slot_of[t] = old_pages - (copies ? 1 : 0);
    // the table of last pages is not needed any more (the sum has two barriers)
    uint32_t *tail_of = keys, *fill_of = keys + 1024;
    tail_of[t] = tail;
    fill_of[t] = fill;
    workgroup_barrier();
    stopped = any_refused != 0;
    const uint32_t wanted = handed;  // up to here
    const bool at_once = a.n <= 1024 && wanted <= 1024;
    uint32_t page = 0, copy_of = ~0u;  // the entry whose last page is copied to `page`
    if (at_once && t < wanted) {
      uint32_t e = 0;  // the last entry that starts at or in front of the lane's page
#pragma unroll
      for (uint32_t step = 512; step >= 1; step >>= 1)
        if (start[e + step] <= t) e += step;
      page = select_page<true>(b, groups, a.lane_vecs, t);
      hand_out(b, page, t, start[e], who[e], slot_of[e]);
      if (t == start[e] && who[e] >> 31) copy_of = e;
    } else if (!at_once && granted && copies) {
      page = select_page<true>(b, groups, a.lane_vecs, carry + before);
      copy_of = t;
    }
    // a place in the list of moves, one addition for each wave
    const uint64_t copying = wave_ballot(copy_of != ~0u);
    uint32_t m = 0;
    if (t % kWave == 0 && copying) m = lds_add(&n_moves, popcount64(copying));
    m = lane_read(m, 0) + popcount64(copying & ((1ull << (t % kWave)) - 1));
    if (copy_of != ~0u) {
      st_obj(a.moves.src + m, static_cast<int32_t>(tail_of[copy_of]));
      st_obj(a.moves.dst + m, static_cast<int32_t>(page));
      st_obj(a.moves.valid + m, static_cast<int32_t>(fill_of[copy_of]));
      if (stopped) add_agent_i32(b.refs + tail_of[copy_of], -1);
    }
    if (!stopped && leavers) st_obj(b.refs + tail, static_cast<int32_t>(holders - leavers));
    if (granted && more > 0) st_obj(b.lengths + s, static_cast<int32_t>(tokens + more));
    if (i < a.n && a.granted) st_obj(a.granted + i, granted ? 1 : 0);
    if (at_once) {
      // every lane has read the bits it needs; each takes the lowest ones out of its own stretch
      workgroup_barrier();
      uint32_t left = in_front < wanted ? wanted - in_front : 0;
      for (uint32_t v = t * a.lane_vecs; left && v < (t + 1) * a.lane_vecs; ++v) {
        const BitTile bits = v == t * a.lane_vecs ? kept : load_bits_vec(b, v);
#pragma unroll
        for (unsigned k = 0; k < 4; ++k) {
          const uint32_t here = popcount32(bits.word[k]);
          if (left == 0 || here == 0) continue;
          const uint32_t kept_from = here <= left ? 0 : nth_bit(bits.word[k], left);
          st_u32(b.bits + 4 * v + k, here <= left ? 0 : bits.word[k] >> kept_from << kept_from);
          left -= here <= left ? here : left;
        }
      }
    } else {
      if (i < a.n) {
        st_u32(a.work.start + i, start[t]);
        st_u32(a.work.who + i, who[t]);
        st_u32(a.work.slot + i, slot_of[t]);
      }
      carry = left_over = wanted;
      // the next turn reads counts that this one wrote
      if (base + 1024 < a.n) wait_for_memory();
      workgroup_barrier();
    }
  }
  if (left_over) {
    uint32_t front = in_front;
    for (uint32_t k = 0; k < a.lane_vecs; ++k) {
      const uint32_t v = t * a.lane_vecs + k;
      if (128 * v >= b.num_pages) break;
      const BitTile bits = k == 0 ? kept : load_bits_vec(b, v);
      st_u32(a.work.pairs + 2 * v, front);
      front += popcount32(bits.word[0]) + popcount32(bits.word[1]);
      st_u32(a.work.pairs + 2 * v + 1, front);
      front += popcount32(bits.word[2]) + popcount32(bits.word[3]);
    }
  }
  if (t == 0) {
    st_obj(a.moves.count, PageMoveCount{n_moves, 0, magic_divisor(n_moves)});
    st_u32(a.work.wanted, left_over);
  }
}

// A wave's 64 pages: each lane has the free bit of its page and how many free
// pages are below it, of which pair_front are below all of them.
struct PageLane {
  uint32_t page, word, front;
  bool exists, free;
};

MI355_DEVICE PageLane load_page_lane(const BookPtrs& b, uint32_t pair, uint32_t pair_front) {
  const unsigned lane = thread_in_workgroup() & (kWave - 1);
  const uint32_t index = 2 * pair + lane / 32;
  PageLane p;
  p.page = 64 * pair + lane;
  p.exists = p.page < b.num_pages;
  p.word = 32 * index < b.num_pages ? existing_bits(b, ld_u32<false>(b.bits + index), index) : 0;
  const uint32_t low = lane_read(p.word, 0);
  p.front = pair_front + (lane < 32 ? 0 : popcount32(low)) + popcount32(p.word & ((1u << (lane % 32)) - 1));
  p.free = p.word >> (lane % 32) & 1;
  return p;
}

// The second launch hands out what the first has left, a wave for 64 pages at
// a time, a lane for each; the entry that a page goes to is found by bisection
// of the running sum.
MI355_DEVICE void page_assign_body(const PageFinishArgs& a) {
  const BookPtrs& b = a.book;
  const unsigned lane = thread_in_workgroup() & (kWave - 1);
  const uint32_t wanted = ld_uniform_u32(a.work.wanted);
  uint32_t pair = static_cast<uint32_t>(global_wave(kMoveWaves));
  for (; pair < a.n_pairs; pair += a.assign_wgs * kMoveWaves) {
    if (wanted == 0) return;
    const uint32_t front = ld_uniform_u32(a.work.pairs + pair);
    if (front >= wanted) return;  // and so it is for every later pair
    const PageLane p = load_page_lane(b, pair, front);
    const bool taken = p.free && p.front < wanted;
    if (taken) {
      uint32_t e = 0;
#pragma unroll
      for (uint32_t step = kMaxList / 2; step >= 1; step >>= 1)
        if (e + step < a.n && ld_u32<false>(a.work.start + e + step) <= p.front) e += step;
      hand_out(b, p.page, p.front, ld_u32<false>(a.work.start + e), ld_u32<false>(a.work.who + e),
               ld_u32<false>(a.work.slot + e));
    }
    const uint64_t gone = wave_ballot(taken);
    const uint32_t mine = lane < 32 ? static_cast<uint32_t>(gone) : static_cast<uint32_t>(gone >> 32);
    if (lane % 32 == 0 && mine) st_u32(b.bits + p.page / 32, p.word & ~mine);
  }
}

template <bool NTL, int ST>
MI355_DEVICE void page_finish_body(const PageFinishArgs& a) {
  if (workgroup_index() < a.assign_wgs)
    page_assign_body(a);
  else
    page_move_body<4, NTL, ST>(a.moves, global_wave(kMoveWaves) - a.assign_wgs * kMoveWaves);
}

// Entries j .. j + 3 of a table or a list, those below `end` (~0 for the others).
struct FourPages {
  uint32_t page[4];
};

MI355_DEVICE FourPages load_four(const int32_t* table, uint32_t j, uint32_t end) {
  FourPages f;
  if (end - j >= 4) {
    const v4u v = ld_v4<false>(reinterpret_cast<const v4u_a4*>(table + j));
    f.page[0] = v.x, f.page[1] = v.y, f.page[2] = v.z, f.page[3] = v.w;
  } else {
#pragma unroll
    for (unsigned k = 0; k < 4; ++k) f.page[k] = j + k < end ? static_cast<uint32_t>(ld_obj(table + j + k)) : ~0u;
  }
  return f;
}

// A sequence that holds its parent's pages.  A workgroup for each entry.  Each
// reads the whole list (it is short and in L2), and so decides without what
// another may already have written: a child that an earlier entry names too is
// left alone, and so is one whose parent is named as a child.
//
// The atomic additions are what takes time (at addresses that differ the device does
// up to 50 of them in a nanosecond, those to one cache line follow each other 2 to 5 ns
// apart), so the first entry that names a parent adds to its pages' counts for all
// that do; an entry that is refused for its child's sake, which the others cannot
// see, takes its own share off again.
// 1000 children of 90 parents, 560 pages each: 7.6 us, and 27.5 with an addition
// for each child and page; 64 children of 16 parents 3.8.
//
// Where tables are long (a.made not null) an entry has a workgroup for each
// a.chunk pages, nobody writes a length, and another launch does (one child of
// 98,000 pages: 11 us together).
MI355_DEVICE void page_fork_body(const PageForkArgs& a) {
  MI355_LDS uint32_t parent_named, again, first, holders;
  const BookPtrs& b = a.book;
  const uint32_t t = thread_in_workgroup();
  const uint32_t i = workgroup_index() % a.n, chunk = workgroup_index() / a.n;
  const uint32_t parent = static_cast<uint32_t>(ld_obj(a.parents + i));
  const uint32_t child = static_cast<uint32_t>(ld_obj(a.children + i));
  if (parent >= b.max_seqs || child >= b.max_seqs) {
    if (t == 0 && chunk == 0) {
      if (a.granted) st_obj(a.granted + i, 0);
      if (a.made) st_u32(a.made + i, 0);
    }
    return;
  }
  // what is needed behind the barriers is under way in front of them: the
  // lists, and the parent's table as if it were full
  uint32_t k = 4 * t;
  FourPages ps, cs, f;
  if (k < a.n) ps = load_four(a.parents, k, a.n), cs = load_four(a.children, k, a.n);
  const int32_t* from = b.tables + static_cast<uint64_t>(parent) * b.width;
  uint32_t j = chunk * a.chunk + 4 * t;
  if (j < b.width) f = load_four(from, j, b.width);
  if (t == 0) parent_named = 0, again = 0, first = ~0u, holders = 0;
  const uint32_t tokens = ld_obj(b.lengths + parent);
  // only the first entry that names the child writes it, after the barriers
  const bool in_use = ld_obj(b.lengths + child) != 0;
  uint32_t held = pages_held(tokens, b);
  if (held > b.width) held = 0;  // not a length
  if (chunk != 0 && chunk * a.chunk >= held) return;
  workgroup_barrier();
  uint32_t mine = 0;
  while (k < a.n) {
#pragma unroll
    for (unsigned u = 0; u < 4; ++u) {
      if (cs.page[u] == parent) parent_named = 1;
      if (cs.page[u] == child && k + u < i) again = 1;
      if (ps.page[u] == parent && cs.page[u] < b.max_seqs) {
        if (mine++ == 0) lds_min(&first, k + u);
      }
    }
    k += 4 * a.wg_size;
    if (k < a.n) ps = load_four(a.parents, k, a.n), cs = load_four(a.children, k, a.n);
  }
  if (mine) lds_add(&holders, mine);
  workgroup_barrier();
  const bool made = !parent_named && !again && !in_use;
  if (!parent_named) {
    const int32_t more = (first == i ? static_cast<int32_t>(holders) : 0) - (made ? 0 : 1);
    int32_t* to = b.tables + static_cast<uint64_t>(child) * b.width;
    uint32_t end = held;
    if (a.made && end > (chunk + 1) * a.chunk) end = (chunk + 1) * a.chunk;
    while (j < end) {
#pragma unroll
      for (unsigned u = 0; u < 4; ++u) {
        if (j + u >= end) continue;
        if (made) st_obj(to + j + u, static_cast<int32_t>(f.page[u]));
        if (more && f.page[u] < b.num_pages) add_agent_i32(b.refs + f.page[u], more);
      }
      j += 4 * a.wg_size;
      if (j < end) f = load_four(from, j, end);
    }
  }
  if (t != 0 || chunk != 0) return;
  const uint32_t length = made && held ? tokens : 0;
  if (a.made) st_u32(a.made + i, length);
  else if (length) st_obj(b.lengths + child, static_cast<int32_t>(length));
  if (a.granted) st_obj(a.granted + i, made ? 1 : 0);
}

MI355_DEVICE void page_fork_lengths_body(const PageForkArgs& a) {
  const uint32_t i = workgroup_index() * 256 + thread_in_workgroup();
  if (i >= a.n) return;
  const uint32_t length = ld_u32<false>(a.made + i);
  const uint32_t child = static_cast<uint32_t>(ld_obj(a.children + i));
  if (length && child < a.book.max_seqs) st_obj(a.book.lengths + child, static_cast<int32_t>(length));
}

// The end of a sequence, or of its tokens from `keep` on.  A workgroup for each
// entry; lane 0 takes the sequence's tokens with an atomic minimum, so that of
// two entries for one sequence each gives back what the other has not.  Bound by
// latency: entry, minimum, table, count, free bits (5 sequences 4.2 us).
MI355_DEVICE void page_free_body(const PageFreeArgs& a) {
  MI355_LDS uint32_t before;
  const BookPtrs& b = a.book;
  const uint32_t t = thread_in_workgroup();
  const uint32_t i = workgroup_index();
  const uint32_t s = static_cast<uint32_t>(ld_obj(a.seqs + i));
  const int32_t keep = a.keep ? ld_obj(a.keep + i) : 0;
  if (s >= b.max_seqs || keep < 0) return;
  // the table as if it were full, while the minimum is under way
  const int32_t* table = b.tables + static_cast<uint64_t>(s) * b.width;
  uint32_t j = pages_held(keep, b) + 4 * t;
  FourPages f;
  if (j < b.width) f = load_four(table, j, b.width);
  if (t == 0) before = static_cast<uint32_t>(min_agent_i32(b.lengths + s, keep));
  workgroup_barrier();
  const uint32_t was = before;
  if (static_cast<int32_t>(was) <= keep) return;
  uint32_t end = pages_held(was, b);
  if (end > b.width) end = b.width;
  while (j < end) {
    int32_t holders[4];
#pragma unroll
    for (unsigned k = 0; k < 4; ++k)
      holders[k] = j + k < end && f.page[k] < b.num_pages ? add_agent_i32(b.refs + f.page[k], -1) : 0;
    // pages that were handed out together often share a word
    uint32_t word = ~0u, bits = 0;
#pragma unroll
    for (unsigned k = 0; k < 4; ++k) {
      if (holders[k] != 1) continue;
      if (f.page[k] / 32 != word) {
        if (bits) or_agent_u32(b.bits + word, bits);
        word = f.page[k] / 32, bits = 0;
      }
      bits |= 1u << (f.page[k] % 32);
    }
    if (bits) or_agent_u32(b.bits + word, bits);
    j += 4 * a.wg_size;
    if (j < end) f = load_four(table, j, end);
  }
}

// The same for many pages, in two launches.  Atomics are what takes time (see the
// fork), so there is one for each page, whose result nobody waits for, and
// the second launch makes the free bits from the counts and shortens the
// sequences (306,000 pages of 850 sequences: 28 us with the free bits by atomics,
// 17 so; the tails of 850 sequences that share their pages, 150,000 pages in all,
// 9.5 and 2.3 us).  Where many hold the same few pages the counts are in a few cache
// lines, and the additions follow each other: 1000 sequences of one prefix of 300
// pages 78 us, of 300 pages each 6.1; 8192 sequences of one prefix of 10 pages 378.  A
// workgroup for each entry and a.chunk pages of its table; the first entry that
// names a sequence acts for all that do, with the smallest keep of theirs.
MI355_DEVICE void page_free_counts_body(const PageFreeArgs& a) {
  MI355_LDS uint32_t again, least;
  const BookPtrs& b = a.book;
  const uint32_t t = thread_in_workgroup();
  const uint32_t i = workgroup_index() % a.n, chunk = workgroup_index() / a.n;
  const uint32_t s = static_cast<uint32_t>(ld_obj(a.seqs + i));
  if (s >= b.max_seqs) return;
  const int32_t tokens = ld_obj(b.lengths + s);
  if (tokens <= 0) return;
  uint32_t end = pages_held(tokens, b);
  if (end > b.width) end = b.width;
  if (chunk * a.chunk >= end) return;
  if (t == 0) again = 0, least = ~0u;
  workgroup_barrier();
  if (end > (chunk + 1) * a.chunk) end = (chunk + 1) * a.chunk;
  const int32_t* table = b.tables + static_cast<uint64_t>(s) * b.width;
  // the first entries of the stretch are under way while the list is read
  uint32_t j = chunk * a.chunk + 4 * t;
  FourPages f;
  if (j < end) f = load_four(table, j, end);
  for (uint32_t k = 4 * t; k < a.n; k += 4 * a.wg_size) {
    const FourPages named = load_four(a.seqs, k, a.n);
#pragma unroll
    for (unsigned u = 0; u < 4; ++u) {
      if (named.page[u] != s) continue;
      // a negative number is a large unsigned one
      lds_min(&least, a.keep ? static_cast<uint32_t>(ld_obj(a.keep + k + u)) : 0);
      if (k + u < i) again = 1;
    }
  }
  workgroup_barrier();
  if (again || least >= static_cast<uint32_t>(tokens)) return;
  const uint32_t from = pages_held(least, b);
  while (j < end) {
#pragma unroll
    for (unsigned k = 0; k < 4; ++k)
      if (j + k >= from && f.page[k] < b.num_pages) add_agent_i32(b.refs + f.page[k], -1);
    j += 4 * a.wg_size;
    if (j < end) f = load_four(table, j, end);
  }
}

MI355_DEVICE void page_free_finish_body(const PageFreeArgs& a) {
  const BookPtrs& b = a.book;
  const unsigned lane = thread_in_workgroup() & (kWave - 1);
  const uint32_t page = workgroup_index() * 256 + thread_in_workgroup();
  const bool free = page < b.num_pages && ld_obj(b.refs + page) == 0;
  const uint64_t all = wave_ballot(free);
  const uint32_t word = lane < 32 ? static_cast<uint32_t>(all) : static_cast<uint32_t>(all >> 32);
  if (lane % 32 == 0 && page < b.num_pages) st_u32(b.bits + page / 32, word);
  const uint32_t i = page;
  if (i >= a.n) return;
  const uint32_t s = static_cast<uint32_t>(ld_obj(a.seqs + i));
  const int32_t keep = a.keep ? ld_obj(a.keep + i) : 0;
  if (s < b.max_seqs && keep >= 0) min_agent_i32(b.lengths + s, keep);
}

// Compaction.  With L pages in use, a page below L that is free is a hole and a
// page from L on that is in use has to move; there are as many of the one as
// of the other.  The i-th hole from below takes the i-th page from above, as far
// as the caller's budget goes.
//
// Up to 1024 moves take two launches: one workgroup of 1024 lanes counts, and
// finds by rank the hole and the page of each move, a lane for each; the second
// moves the bytes, next to workgroups that rewrite the tables and the free bits.
// Beyond, the first launch leaves the free pages in front of each two words of
// the free bits and how many pages move, and one between the two, over the
// whole device, finds for each hole the page that comes to it.  Bound by memory
// where much moves (3,500 pages of 1 MiB of which 815 move: 4.6, 4.7 and 274 us,
// 6.2 TB/s), by the launches otherwise (24 of 3,000 pages: 4.8 and 5.0 us; the first
// launch in a pool of 2,000,000 pages 49).

// Move k, of page `from` to page `to`: the list, the counts, and what the caller wants to know.
MI355_DEVICE void list_move(const PageCompactArgs& a, uint32_t k, uint32_t from, uint32_t to) {
  const BookPtrs& b = a.book;
  st_obj(a.moves.src + k, static_cast<int32_t>(from));
  st_obj(a.moves.dst + k, static_cast<int32_t>(to));
  st_obj(a.moves.remap + from, static_cast<int32_t>(to));
  st_obj(b.refs + to, ld_obj(b.refs + from));
  st_obj(b.refs + from, 0);
  if (a.out) {
    st_obj(a.out + 2 * static_cast<uint64_t>(k), static_cast<int32_t>(from));
    st_obj(a.out + 2 * static_cast<uint64_t>(k) + 1, static_cast<int32_t>(to));
  }
}

MI355_DEVICE void page_compact_plan_body(const PageCompactArgs& a) {
  MI355_LDS uint32_t scan[16], groups[1024];
  MI355_LDS uint32_t holes;
  const BookPtrs& b = a.book;
  const uint32_t t = thread_in_workgroup();
  uint32_t mine = 0;
  for (uint32_t k = 0; k < a.lane_vecs; ++k) mine += count_bits(load_bits_vec(b, t * a.lane_vecs + k));
  if (t == 0) holes = 0;
  uint32_t free_pages;
  uint32_t front = block_scan_1024(mine, scan, &free_pages);
  groups[t] = front;
  const uint32_t live = b.num_pages - free_pages;
  for (uint32_t k = 0; k < a.lane_vecs; ++k) {
    const uint32_t v = t * a.lane_vecs + k;
    if (128 * v >= b.num_pages) break;
    const BitTile bits = load_bits_vec(b, v);
    uint32_t at = front;
#pragma unroll
    for (unsigned c = 0; c < 4; ++c) {
      const uint32_t page = 128 * v + 32 * c;
      if (c % 2 == 0) st_u32(a.pairs + 2 * v + c / 2, at);
      // the word that page L is in: the free pages below it are the holes
      if (page <= live && live - page < 32) holes = at + popcount32(bits.word[c] & ((1u << (live - page)) - 1));
      at += popcount32(bits.word[c]);
    }
    front = at;
  }
  workgroup_barrier();
  const uint32_t n = holes < a.max_moves ? holes : a.max_moves;
  if (t == 0) {
    st_obj(a.moves.count, PageMoveCount{n, 0, magic_divisor(n)});
    st_u32(a.live, live);
    st_obj(b.head, static_cast<int32_t>(n));
  }
  if (a.max_moves <= kListedAtOnce && t < n)
    list_move(a, t, select_page<false>(b, groups, a.lane_vecs, live - 1 - t),
              select_page<true>(b, groups, a.lane_vecs, t));
}

// The moves that the first launch has counted; never more than there is room
// for, whatever another call on the book may have left there.
MI355_DEVICE uint32_t compact_moves(const PageCompactArgs& a) {
  const uint32_t n = ld_uniform_u32(&a.moves.count->n);
  return n < a.max_moves ? n : a.max_moves;
}

// The counts of the pages that move and where they go.
MI355_DEVICE void page_compact_list_body(const PageCompactArgs& a) {
  const BookPtrs& b = a.book;
  const uint32_t n = compact_moves(a);
  const uint32_t live = ld_uniform_u32(a.live);
  uint32_t pair = static_cast<uint32_t>(global_wave(kMoveWaves));
  for (; pair < a.n_pairs; pair += a.pair_wgs * kMoveWaves) {
    if (64 * pair >= live) return;
    const uint32_t front = ld_uniform_u32(a.pairs + pair);
    if (front >= n) return;  // the pages that move are all further down
    const PageLane p = load_page_lane(b, pair, front);
    const uint32_t k = p.front;
    if (!p.free || p.page >= live || k >= n) continue;
    // the page in use with live - 1 - k of them below it: the last pair with
    // no more in front of it, and in it the bit
    const uint32_t rank = live - 1 - k;
    uint32_t lo = 0, hi = a.n_pairs;  // [lo, hi) holds it
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (64 * mid - ld_u32<false>(a.pairs + mid) <= rank) lo = mid;
      else hi = mid;
    }
    uint32_t r = rank - (64 * lo - ld_u32<false>(a.pairs + lo));
    const uint32_t w0 = ~ld_u32<false>(b.bits + 2 * lo);
    uint32_t from;
    if (r < popcount32(w0)) {
      from = 64 * lo + nth_bit(w0, r);
    } else {
      r -= popcount32(w0);
      from = 64 * lo + 32 + nth_bit(~ld_u32<false>(b.bits + 2 * lo + 1), r);
    }
    if (from >= b.num_pages) from = p.page;  // not reached
    list_move(a, k, from, p.page);
  }
}

// The tables, a workgroup of 256 lanes for each sequence, whatever its length: 200
// sequences of 500 pages 3.2 us, one of 98,000 109.  The pages that moved
// are the highest ones, so every held page from the lowest of them on has moved.
MI355_DEVICE void page_compact_tables_body(const PageCompactArgs& a, uint32_t n, uint32_t s) {
  const BookPtrs& b = a.book;
  const uint32_t lowest = ld_uniform_u32(reinterpret_cast<const uint32_t*>(a.moves.src + n - 1));
  uint32_t held = pages_held(ld_obj(b.lengths + s), b);
  if (held > b.width) held = 0;
  int32_t* table = b.tables + static_cast<uint64_t>(s) * b.width;
  for (uint32_t j = thread_in_workgroup(); j < held; j += 256) {
    const uint32_t page = static_cast<uint32_t>(ld_obj(table + j));
    if (page >= lowest && page < b.num_pages) st_obj(table + j, ld_obj(a.moves.remap + page));
  }
}

// The free bits: the first n holes are taken, the last n pages in use are free.
MI355_DEVICE void page_compact_bits_body(const PageCompactArgs& a, uint32_t n, uint32_t first_wave) {
  const BookPtrs& b = a.book;
  const unsigned lane = thread_in_workgroup() & (kWave - 1);
  const uint32_t live = ld_uniform_u32(a.live);
  for (uint32_t pair = first_wave; pair < a.n_pairs; pair += a.pair_wgs * kMoveWaves) {
    const PageLane p = load_page_lane(b, pair, ld_uniform_u32(a.pairs + pair));
    bool free = p.free;
    if (p.exists && p.page < live && p.front < n) free = false;
    // page - front pages in use are below it
    if (p.exists && p.page >= live && live - (p.page - p.front) <= n) free = true;
    const uint64_t all = wave_ballot(free);
    const uint32_t word = lane < 32 ? static_cast<uint32_t>(all) : static_cast<uint32_t>(all >> 32);
    if (lane % 32 == 0 && p.exists && word != p.word) st_u32(b.bits + p.page / 32, word);
  }
}

template <bool NTL, int ST>
MI355_DEVICE void page_compact_finish_body(const PageCompactFinishArgs& f) {
  const PageCompactArgs& a = f.compact;
  const uint32_t wg = workgroup_index();
  const uint32_t n = compact_moves(a);
  if (n == 0) return;
  if (wg < a.pair_wgs)
    page_compact_bits_body(a, n, static_cast<uint32_t>(global_wave(kMoveWaves)));
  else if (wg < a.pair_wgs + a.book.max_seqs)
    page_compact_tables_body(a, n, wg - a.pair_wgs);
  else
    page_move_body<1, NTL, ST>(f.moves, global_wave(kMoveWaves) -
                                            static_cast<uint64_t>(kMoveWaves) * (a.pair_wgs + a.book.max_seqs));
}

// An empty book: no tokens, no holders, every page free, no table entry.
MI355_DEVICE void page_reset_body(const PageResetArgs& a) {
  const BookPtrs& b = a.book;
  const int64_t bits_at = reinterpret_cast<int32_t*>(b.bits) - b.head;
  const int64_t tables_at = b.tables - b.head;
  for (uint64_t i = static_cast<uint64_t>(workgroup_index()) * 256 + thread_in_workgroup(); i < a.words; i += a.lanes) {
    uint32_t v = 0;
    if (static_cast<int64_t>(i) >= tables_at) {
      v = ~0u;
    } else if (static_cast<int64_t>(i) >= bits_at) {
      const uint64_t page = 32 * (i - bits_at);
      if (page < b.num_pages) v = b.num_pages - page >= 32 ? ~0u : (1u << (b.num_pages - page)) - 1;
    }
    st_obj(b.head + i, static_cast<int32_t>(v));
  }
}

}  // namespace mi355

// Entry points, named as those of blit_kernels.h:
//   mi355_pages_move_u<16-byte vectors a lane>_l<nt loads>_s<store policy>
#define MI355_PAGE_MOVE_LS_(X, U) X(U, 0, 0) X(U, 1, 1) X(U, 1, 2) X(U, 0, 3) X(U, 1, 3)
#define MI355_FOR_EACH_PAGE_MOVE_KERNEL(X) MI355_PAGE_MOVE_LS_(X, 1) MI355_PAGE_MOVE_LS_(X, 4)
#define MI355_DEFINE_PAGE_MOVE(U, L, S)                                                       \
  MI355_KERNEL(256) void mi355_pages_move_u##U##_l##L##_s##S(mi355::PageMoveArgs a) {         \
    mi355::page_move_body<U, L != 0, S>(a, mi355::global_wave(mi355::kMoveWaves));            \
  }
MI355_FOR_EACH_PAGE_MOVE_KERNEL(MI355_DEFINE_PAGE_MOVE)

//   mi355_pages_reserve_finish_l<nt loads>_s<store policy>
#define MI355_FOR_EACH_PAGE_FINISH_KERNEL(X) X(0, 0) X(1, 1) X(1, 2)
#define MI355_DEFINE_PAGE_FINISH(L, S)                                                        \
  MI355_KERNEL(256) void mi355_pages_reserve_finish_l##L##_s##S(mi355::PageFinishArgs a) {    \
    mi355::page_finish_body<L != 0, S>(a);                                                    \
  }
MI355_FOR_EACH_PAGE_FINISH_KERNEL(MI355_DEFINE_PAGE_FINISH)

MI355_KERNEL(1024) void mi355_pages_reserve(mi355::PageReserveArgs a) { mi355::page_reserve_body(a); }
MI355_KERNEL(1024) void mi355_pages_fork(mi355::PageForkArgs a) { mi355::page_fork_body(a); }
MI355_KERNEL(256) void mi355_pages_fork_lengths(mi355::PageForkArgs a) { mi355::page_fork_lengths_body(a); }
MI355_KERNEL(1024) void mi355_pages_free(mi355::PageFreeArgs a) { mi355::page_free_body(a); }
MI355_KERNEL(1024) void mi355_pages_free_counts(mi355::PageFreeArgs a) { mi355::page_free_counts_body(a); }
MI355_KERNEL(256) void mi355_pages_free_finish(mi355::PageFreeArgs a) { mi355::page_free_finish_body(a); }
MI355_KERNEL(1024) void mi355_pages_compact_plan(mi355::PageCompactArgs a) { mi355::page_compact_plan_body(a); }
MI355_KERNEL(256) void mi355_pages_compact_list(mi355::PageCompactArgs a) { mi355::page_compact_list_body(a); }
//   mi355_pages_compact_finish_l<nt loads>_s<store policy>
#define MI355_DEFINE_PAGE_COMPACT_FINISH(L, S)                                                       \
  MI355_KERNEL(256) void mi355_pages_compact_finish_l##L##_s##S(mi355::PageCompactFinishArgs a) {    \
    mi355::page_compact_finish_body<L != 0, S>(a);                                                   \
  }
MI355_FOR_EACH_PAGE_FINISH_KERNEL(MI355_DEFINE_PAGE_COMPACT_FINISH)
MI355_KERNEL(256) void mi355_pages_reset(mi355::PageResetArgs a) { mi355::page_reset_body(a); }

#endif  // MI355_BLIT_PAGES_KERNELS_H_
