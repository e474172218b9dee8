// The page kernels (csrc/blit_pages_kernels.h, compiled unchanged) run on the
// CPU lane by lane, launched with the argument blocks of the product's own host
// code, against a book that is kept one entry at a time.  After every call the
// whole book, what was granted and the bytes of the pool (gaps between its
// pages included) have to be equal, and no access may leave the pool, the book, the
// lists and the work memory; random books and lists, which name no book that the calls
// would have made, may give any result but no access outside either.
//
//   test_pages_on_cpu [--shard I/N]       exit status 0 = all checks passed
#include <cinttypes>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <memory>
#include <set>
#include <string>
#include <vector>

#define MI355_BLIT_DEVICE_HEADER "lane_emulation_pages.h"
#include "blit_pages_kernels.h"

namespace {

using namespace mi355;
using lane_emu::g_check;
using lane_emu::g_m;

uint64_t g_state = 0x9E3779B97F4A7C15ull;
uint64_t rnd() {  // splitmix64
  uint64_t z = (g_state += 0x9E3779B97F4A7C15ull);
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
uint64_t below(uint64_t n) { return n ? rnd() % n : 0; }
uint64_t between(uint64_t lo, uint64_t hi) { return lo + below(hi - lo + 1); }

uint64_t g_calls = 0, g_failures = 0;
std::string g_at;
void fail(const char* what) {
  if (g_failures++ < 20) std::printf("FAIL %s: %s\n", g_at.c_str(), what);
}

// What happens in front of every launch (nothing, usually).
std::function<void()> g_meanwhile;

struct Config {
  uint32_t pages, rows, seqs, width;
  std::vector<mi355_blit_plane_t> planes;  // base unset
};

// A heap block that ends where its last byte ends.
struct Bytes {
  std::unique_ptr<uint8_t[]> raw;
  uint8_t* p = nullptr;
  size_t n = 0;
  void make(size_t bytes, size_t residue) {
    raw.reset(new uint8_t[bytes + residue + 32]);
    p = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw.get()) + 15) / 16 * 16) + residue;
    n = bytes;
    for (size_t i = 0; i < n; ++i) p[i] = static_cast<uint8_t>(rnd());
  }
};

// A pool with the product's table, and the same bytes once more.
struct Pool {
  Config c;
  std::vector<Bytes> mem;
  std::vector<std::vector<uint8_t>> want;
  PagePlane* table[2] = {nullptr, nullptr};
  uint32_t pieces[2] = {0, 0};
  uint64_t page_bytes = 0;
  bool even = true;
  Pool() {}
  Pool(const Pool&) = delete;
  ~Pool() { std::free(table[0]), std::free(table[1]); }
  bool make(const Config& config, bool fresh_pitch) {
    c = config;
    mem.resize(c.planes.size());
    want.resize(c.planes.size());
    for (size_t i = 0; i < c.planes.size(); ++i) {
      const uint64_t page = plane_page_bytes(c.planes[i], c.rows);
      if (fresh_pitch) c.planes[i].pitch = page + below(40);
      mem[i].make((c.pages - 1) * c.planes[i].pitch + page, below(2) ? 0 : below(16));
      c.planes[i].base = mem[i].p;
      want[i].assign(mem[i].p, mem[i].p + mem[i].n);
      page_bytes += page;
      if (page != plane_page_bytes(c.planes[0], c.rows)) even = false;
    }
    mi355_blit_pages_desc_t d = desc(nullptr);
    uint64_t counted = 0;
    if (pages_check(&d, &counted) != MI355_BLIT_SUCCESS) return false;
    for (int k = 0; k < 2; ++k) {
      pieces[k] = pages_planes(d, kPieceUnrolls[k], nullptr);
      if (pieces[k] > counted) return false;
      void* q = nullptr;
      if (posix_memalign(&q, 64, pieces[k] * sizeof(PagePlane))) std::abort();
      table[k] = static_cast<PagePlane*>(q);
      pages_planes(d, kPieceUnrolls[k], table[k]);
    }
    return true;
  }
  mi355_blit_pages_desc_t desc(int32_t* book) const {
    return {c.planes.data(), static_cast<uint32_t>(c.planes.size()), c.pages, c.rows, book ? c.seqs : 0,
            book ? c.width : 0, 0, book};
  }
  void allow(bool write) {
    for (auto& m : mem) {
      g_check.allow_read(m.p, m.n);
      if (write) g_check.allow_write(m.p, m.n);
    }
    for (int k = 0; k < 2; ++k) g_check.allow_read(table[k], pieces[k] * sizeof(PagePlane));
  }
  // what a copy of the first `valid` rows of page `from` of pool `src` leaves
  void move(const Pool& src, uint32_t from, uint32_t to, uint32_t valid, const std::vector<std::vector<uint8_t>>& before) {
    for (size_t i = 0; i < c.planes.size(); ++i) {
      const mi355_blit_plane_t &d = c.planes[i], &s = src.c.planes[i];
      for (uint32_t r = 0; r < d.runs; ++r) {
        const uint64_t run = static_cast<uint64_t>(r) * c.rows * d.row_bytes;
        std::memcpy(want[i].data() + to * d.pitch + run, before[i].data() + from * s.pitch + run, static_cast<uint64_t>(valid) * d.row_bytes);
      }
    }
  }
  void check(const char* what) {
    for (size_t i = 0; i < mem.size(); ++i)
      if (std::memcmp(mem[i].p, want[i].data(), mem[i].n)) return fail(what);
  }
};

typedef std::vector<int32_t> List;

// n words in a block of their own
struct Words {
  std::unique_ptr<int32_t[]> p;
  size_t n;
  explicit Words(const List& v) : p(new int32_t[v.size() ? v.size() : 1]), n(v.size()) {
    if (n) std::memcpy(p.get(), v.data(), 4 * n);
  }
};

struct Cache {
  Pool pool;
  mi355_blit_book_t at;
  int32_t* book = nullptr;
  BookPtrs ptrs;
  PageMoveList moves;
  PageReserveWork reserving;
  uint32_t* work = nullptr;
  uint64_t work_words = 0;
  // the book as it should be
  List lengths, refs, tables;
  int32_t head = 0;

  ~Cache() { std::free(book), std::free(work); }

  bool make(const Config& c) {
    if (!pool.make(c, true)) return false;
    if (pages_book_layout(c.pages, c.seqs, c.width, &at) != MI355_BLIT_SUCCESS) return false;
    void* q = nullptr;
    if (posix_memalign(&q, 16, at.words * 4)) std::abort();
    book = static_cast<int32_t*>(q);
    for (uint64_t i = 0; i < at.words; ++i) book[i] = static_cast<int32_t>(rnd());
    ptrs = pages_book_ptrs(book, at, c.pages, c.seqs, c.width, c.rows);
    const PageWorkLayout w = pages_work_layout(c.pages);
    work_words = w.words;
    if (posix_memalign(&q, 256, work_words * 4)) std::abort();
    work = static_cast<uint32_t*>(q);
    for (uint64_t i = 0; i < work_words; ++i) work[i] = static_cast<uint32_t>(rnd());
    moves = pages_move_list(work, w);
    reserving = pages_reserve_work(work, w);
    start();
    const uint32_t grid = 1 + static_cast<uint32_t>(below((at.words + 255) / 256));
    run(mi355_pages_reset, PageResetArgs{ptrs, at.words, grid * 256ull}, grid, 256);
    lengths.assign(c.seqs, 0);
    refs.assign(c.pages, 0);
    tables.assign(static_cast<size_t>(c.seqs) * c.width, -1);
    check("reset");
    return true;
  }

  uint32_t held(int64_t tokens) const { return static_cast<uint32_t>((tokens + pool.c.rows - 1) / pool.c.rows); }
  int32_t* row(uint32_t s) { return tables.data() + static_cast<size_t>(s) * pool.c.width; }

  void start() {
    g_check.clear();
    g_check.allow_read(book, at.words * 4);
    g_check.allow_write(book, at.words * 4);
    g_check.allow_read(work, work_words * 4);
    g_check.allow_write(work, work_words * 4);
    pool.allow(true);
  }
  void reads(const Words& w) { g_check.allow_read(w.p.get(), w.n * 4); }
  void writes(const Words& w) { g_check.allow_write(w.p.get(), w.n * 4); }

  template <typename Args>
  static void run(void (*kernel)(Args), const Args& args, uint32_t grid, uint32_t wg) {
    if (g_meanwhile) g_meanwhile();
    g_check.seal();
    g_reverse_grid = rnd() & 1 ? grid : 0;
    lane_emu::launch(kernel, args, grid, wg);
    g_reverse_grid = 0;
    if (g_check.violations) fail(g_check.first), g_check.violations = 0, g_check.first[0] = 0;
    if (g_m.errors) fail(g_m.first_error), g_m.errors = 0;
  }

  static PageMoveArgs move_args(const Pool& to, const Pool& from, const PageMovePlan& p, const int32_t* dst,
                                const int32_t* src, const int32_t* valid, const PageMoveCount* count, uint64_t n) {
    const uint32_t even = to.even && below(2) ? to.pieces[p.table] / static_cast<uint32_t>(to.c.planes.size()) : 0;
    return {to.table[p.table], from.table[p.table], dst, src, valid, count, magic_divisor(static_cast<uint32_t>(n)),
            magic_divisor(even), static_cast<uint32_t>(n), to.pieces[p.table], even, 0, to.c.pages, from.c.pages,
            to.c.rows, p.grid * kMoveWaves};
  }

  static void run_moves(const Pool& to, const Pool& from, const int32_t* dst, const int32_t* src, const int32_t* valid,
                        uint64_t n, uint32_t route, uint32_t cus) {
    PageMovePlan p = plan_page_moves(n, 0, valid != nullptr, to.pieces, to.page_bytes, cus, route, 3);
    // the sizes here are small: the policies of large moves, and grids that stride
    if (p.store_policy == MI355_BLIT_STORE_CACHED && below(2)) p.nt_load = 1, p.store_policy = 1 + below(2);
    if (p.store_policy == MI355_BLIT_STORE_SYSTEM_WT) p.nt_load = below(2);
    if (below(2) && p.grid > 3) p.grid = 1 + below(p.grid);
    const PageMoveArgs a = move_args(to, from, p, dst, src, valid, nullptr, n);
#define TRY(U, L, S) \
  if (kPieceUnrolls[p.table] == U && p.nt_load == L && p.store_policy == S) \
    return run(mi355_pages_move_u##U##_l##L##_s##S, a, p.grid, kMoveWaves * kWave);
    MI355_FOR_EACH_PAGE_MOVE_KERNEL(TRY)
#undef TRY
    fail("no kernel for the plan");
  }

  void run_reserve(const Words& seqs, const Words& more, int32_t* granted, uint32_t n) {
    if (!n) return;
    run(mi355_pages_reserve, PageReserveArgs{ptrs, moves, reserving, seqs.p.get(), more.p.get(), granted, n,
                                             reserve_lane_vecs(pool.c.pages)}, 1, 1024);
    const uint64_t copies = n < pool.c.pages ? n : pool.c.pages;
    const PageMovePlan p = plan_page_moves(copies, 2, true, pool.pieces, pool.page_bytes, 1 + below(3), 0, 3);
    const uint32_t n_pairs = (pool.c.pages + 63) / 64;
    const PageFinishArgs f{move_args(pool, pool, p, moves.dst, moves.src, moves.valid, moves.count, copies), ptrs, reserving, n, n_pairs, 1 + static_cast<uint32_t>(below((n_pairs + 3) / 4)), 0};
    switch (below(3)) {
      case 0: return run(mi355_pages_reserve_finish_l0_s0, f, f.assign_wgs + p.grid, 256);
      case 1: return run(mi355_pages_reserve_finish_l1_s1, f, f.assign_wgs + p.grid, 256);
      default: return run(mi355_pages_reserve_finish_l1_s2, f, f.assign_wgs + p.grid, 256);
    }
  }

  void run_fork(const Words& parents, const Words& children, int32_t* granted, uint32_t n) {
    const uint32_t wg = below(2) ? table_wg_size(pool.c.width) : 128;
    const bool split = below(2);
    const PageForkArgs a{ptrs, parents.p.get(), children.p.get(), granted, split ? reserving.start : nullptr, n, wg,
                         table_chunk(pool.c.width), 0};
    run(mi355_pages_fork, a, split ? n * table_chunks(pool.c.width) : n, wg);
    if (split) run(mi355_pages_fork_lengths, a, (n + 255) / 256, 256);
  }

  void run_free(const Words& seqs, const int32_t* keep, uint32_t n) {
    const uint32_t wg = below(2) ? table_wg_size(pool.c.width) : 64;
    const PageFreeArgs a{ptrs, seqs.p.get(), keep, n, wg, table_chunk(pool.c.width), 0};
    if (below(2)) return run(mi355_pages_free, a, n, wg);
    run(mi355_pages_free_counts, a, n * table_chunks(pool.c.width), wg);
    run(mi355_pages_free_finish, a, ((pool.c.pages > n ? pool.c.pages : n) + 255) / 256, 256);
  }

  void run_compact(uint32_t most, int32_t* out) {
    const uint32_t wgs = page_pair_wgs(pool.c.pages);
    const PageCompactArgs a{ptrs, moves, reserving.pairs, reserving.wanted, out, most, reserve_lane_vecs(pool.c.pages),
                            page_pairs(pool.c.pages), 1 + static_cast<uint32_t>(below(wgs))};
    const PageMovePlan p = plan_page_moves(most, 2, false, pool.pieces, pool.page_bytes, 1 + below(3), 0, 3);
    const PageCompactFinishArgs f{move_args(pool, pool, p, moves.dst, moves.src, nullptr, moves.count, most), a};
    const uint32_t grid = a.pair_wgs + pool.c.seqs + p.grid;
    run(mi355_pages_compact_plan, a, 1, 1024);
    if (most > kListedAtOnce) run(mi355_pages_compact_list, a, a.pair_wgs, 256);
    switch (below(3)) {
      case 0: return run(mi355_pages_compact_finish_l0_s0, f, grid, 256);
      case 1: return run(mi355_pages_compact_finish_l1_s1, f, grid, 256);
      default: return run(mi355_pages_compact_finish_l1_s2, f, grid, 256);
    }
  }

  void check(const char* what) {
    ++g_calls;
    if (std::memcmp(ptrs.lengths, lengths.data(), 4 * lengths.size())) fail((std::string(what) + ": lengths").c_str());
    if (std::memcmp(ptrs.refs, refs.data(), 4 * refs.size())) fail((std::string(what) + ": counts").c_str());
    if (std::memcmp(ptrs.tables, tables.data(), 4 * tables.size())) fail((std::string(what) + ": tables").c_str());
    if (ptrs.head[0] != head) fail((std::string(what) + ": head").c_str());
    for (uint32_t q = 0; q < (pool.c.pages + 31) / 32 * 32; ++q) {
      const bool bit = ptrs.bits[q / 32] >> (q % 32) & 1;
      if (bit != (q < pool.c.pages && refs[q] == 0)) return fail((std::string(what) + ": free bits").c_str());
    }
    pool.check((std::string(what) + ": bytes").c_str());
  }

  void reserve(const List& seqs, const List& more) {
    const uint32_t n = static_cast<uint32_t>(seqs.size());
    Words s(seqs), m(more), granted(List(n, 77));
    start(), reads(s), reads(m), writes(granted);
    const bool tell = rnd() % 4 != 0;
    run_reserve(s, m, tell ? granted.p.get() : nullptr, n);
    // one entry after the other
    const auto before = pool.want;
    std::set<int32_t> named;
    List want(n, 0);
    std::vector<uint32_t> free_pages;
    for (uint32_t q = 0; q < pool.c.pages; ++q)
      if (refs[q] == 0) free_pages.push_back(q);
    size_t taken = 0;
    for (uint32_t i = 0; i < n; ++i) {
      const int32_t id = seqs[i];
      if (id < 0 || static_cast<uint32_t>(id) >= pool.c.seqs || !named.insert(id).second || more[i] < 0) continue;
      const uint32_t o = held(lengths[id]), e = held(static_cast<int64_t>(lengths[id]) + more[i]);
      if (e > pool.c.width) continue;
      const uint32_t fill = lengths[id] % pool.c.rows;
      const bool apart = more[i] > 0 && fill && refs[row(id)[o - 1]] > 1;
      if (e - o + apart > free_pages.size() - taken) break;
      uint32_t slot = o;
      if (apart) {
        --slot;
        --refs[row(id)[slot]];
        pool.move(pool, row(id)[slot], free_pages[taken], fill, before);
      }
      for (; slot < e; ++slot) {
        row(id)[slot] = static_cast<int32_t>(free_pages[taken]);
        refs[free_pages[taken++]] = 1;
      }
      lengths[id] += more[i];
      want[i] = 1;
    }
    if (tell && n && std::memcmp(granted.p.get(), want.data(), 4 * n)) fail("reserve: granted");
    check("reserve");
  }

  void fork(const List& parents, const List& children) {
    const uint32_t n = static_cast<uint32_t>(parents.size());
    if (!n) return;
    Words p(parents), c(children), granted(List(n, 77));
    start(), reads(p), reads(c), writes(granted);
    run_fork(p, c, granted.p.get(), n);
    std::set<int32_t> named, all(children.begin(), children.end());
    for (uint32_t i = 0; i < n; ++i) {
      const int32_t a = parents[i], b = children[i];
      const auto in = [this](int32_t s) { return s >= 0 && static_cast<uint32_t>(s) < pool.c.seqs; };
      const bool first = !in(b) || named.insert(b).second;
      const bool ok = in(a) && in(b) && first && !all.count(a) && lengths[b] == 0;
      if (granted.p[i] != ok) fail("fork: granted");
      if (!ok) continue;
      for (uint32_t j = 0; j < held(lengths[a]); ++j) {
        row(b)[j] = row(a)[j];
        ++refs[row(a)[j]];
      }
      lengths[b] = lengths[a];
    }
    check("fork");
  }

  void free_tokens(const List& seqs, const List* keep) {
    const uint32_t n = static_cast<uint32_t>(seqs.size());
    if (!n) return;
    Words s(seqs), k(keep ? *keep : List());
    start(), reads(s), reads(k);
    run_free(s, keep ? k.p.get() : nullptr, n);
    for (uint32_t i = 0; i < n; ++i) {
      const int32_t id = seqs[i], left = keep ? (*keep)[i] : 0;
      if (id < 0 || static_cast<uint32_t>(id) >= pool.c.seqs || left < 0 || left >= lengths[id]) continue;
      for (uint32_t j = held(left); j < held(lengths[id]); ++j) --refs[row(id)[j]];
      lengths[id] = left;
    }
    check("free");
  }

  void compact(uint32_t max_moves) {
    const uint32_t most = max_moves < pool.c.pages / 2 ? max_moves : pool.c.pages / 2;
    if (!most) return;
    Words out(List(2 * static_cast<size_t>(most), -5));
    start(), writes(out);
    run_compact(most, out.p.get());
    const auto before = pool.want;
    uint32_t k = 0, lo = 0, hi = pool.c.pages;
    for (;;) {
      while (lo < pool.c.pages && refs[lo]) ++lo;
      while (hi > 0 && !refs[hi - 1]) --hi;
      if (hi == 0 || lo > hi - 1 || k == most) break;
      refs[lo] = refs[hi - 1];
      refs[hi - 1] = 0;
      pool.move(pool, hi - 1, lo, pool.c.rows, before);
      for (uint32_t s = 0; s < pool.c.seqs; ++s)
        for (uint32_t j = 0; j < held(lengths[s]); ++j)
          if (row(s)[j] == static_cast<int32_t>(hi - 1)) row(s)[j] = static_cast<int32_t>(lo);
      if (out.p[2 * k] != static_cast<int32_t>(hi - 1) || out.p[2 * k + 1] != static_cast<int32_t>(lo)) fail("compact: moves");
      ++k;
    }
    head = static_cast<int32_t>(k);
    for (uint32_t i = 2 * k; i < 2 * most; ++i)
      if (out.p[i] != -5) fail("compact: a pair behind the last move");
    check("compact");
  }

  List some_seqs(size_t n, bool clean) {
    List v;
    std::vector<int32_t> order(pool.c.seqs);
    for (uint32_t i = 0; i < pool.c.seqs; ++i) order[i] = static_cast<int32_t>(i);
    for (uint32_t i = 0; i + 1 < pool.c.seqs; ++i) std::swap(order[i], order[i + below(pool.c.seqs - i)]);
    for (size_t i = 0; i < n; ++i) {
      if (clean && i < order.size()) v.push_back(order[i]);
      else if (!clean && below(8) == 0) v.push_back(static_cast<int32_t>(rnd()));
      else if (!clean) v.push_back(static_cast<int32_t>(below(pool.c.seqs)));
    }
    return v;
  }
};

Config some_config(bool wide) {
  Config c;
  static const uint32_t kRows[] = {1, 2, 5, 16, 33};
  c.rows = kRows[below(5)];
  c.seqs = static_cast<uint32_t>(wide ? between(1000, 2600) : between(1, 40));
  c.width = static_cast<uint32_t>(between(1, wide ? 6 : 30));
  c.pages = static_cast<uint32_t>(between(1, wide ? 5000 : 400));
  const size_t n = between(1, 3);
  for (size_t i = 0; i < n; ++i) {
    const uint32_t runs = below(2) ? 1 : static_cast<uint32_t>(between(2, 4));
    c.planes.push_back({nullptr, 0, static_cast<uint32_t>(between(1, wide ? 3 : below(4) ? 40 : 600)), runs});
    if (below(2)) c.planes.back() = c.planes[0];
  }
  return c;
}

void random_life(unsigned steps, bool wide) {
  Cache cache;
  if (!cache.make(some_config(wide))) return fail("a configuration was refused");
  const Config& c = cache.pool.c;
  for (unsigned step = 0; step < steps; ++step) {
    const bool clean = below(2);
    const size_t n = between(0, wide ? 2500 : 50);
    switch (below(6)) {
      case 0: case 1: case 2: {
        const List seqs = cache.some_seqs(n, clean);
        List more;
        for (size_t i = 0; i < seqs.size(); ++i)
          more.push_back(static_cast<int32_t>(below(10) == 0 ? below(c.rows * c.width * 2) : below(40) == 0 ? rnd() : below(2 * c.rows + 2)));
        cache.reserve(seqs, more);
        break;
      }
      case 3: {
        const List all = cache.some_seqs(2 * (n / 2), clean);
        cache.fork(List(all.begin(), all.begin() + all.size() / 2), List(all.begin() + all.size() / 2, all.begin() + all.size() / 2 * 2));
        break;
      }
      case 4: {
        const List seqs = cache.some_seqs(n / 2, clean);
        List keep;
        for (size_t i = 0; i < seqs.size(); ++i) keep.push_back(static_cast<int32_t>(below(c.rows * c.width + 3)) - 2);
        cache.free_tokens(seqs, below(3) ? &keep : nullptr);
        break;
      }
      default:
        cache.compact(static_cast<uint32_t>(below(3) ? c.pages : 1 + below(5)));
    }
  }
}

void random_copies() {
  Config c = some_config(false);
  Pool a, b;
  if (!a.make(c, true) || !b.make(c, true)) return fail("a pool was refused");
  for (int turn = 0; turn < 6; ++turn) {
    const bool within = below(2);
    Pool& to = within ? a : b;
    // sources and destinations of one pool are disjoint: even pages to odd ones
    List src, dst, valid;
    std::set<uint32_t> used;
    for (uint32_t k = static_cast<uint32_t>(between(1, 30)); k; --k) {
      int32_t s = static_cast<int32_t>(below(c.pages)), d = static_cast<int32_t>(below(c.pages));
      if (within) s &= ~1, d |= 1;
      if (below(9) == 0) s = below(2) ? -1 : static_cast<int32_t>(c.pages + below(9));
      if (below(9) == 0) d = below(2) ? -1 : static_cast<int32_t>(rnd());
      if (static_cast<uint32_t>(d) < c.pages && !used.insert(d).second) continue;
      src.push_back(s), dst.push_back(d);
      valid.push_back(below(4) ? static_cast<int32_t>(below(c.rows + 1)) : static_cast<int32_t>(rnd()));
    }
    const bool cut = below(3);
    Words ws(src), wd(dst), wv(valid);
    g_check.clear();
    a.allow(true), b.allow(true);
    for (const Words* w : {&ws, &wd, &wv}) g_check.allow_read(w->p.get(), w->n * 4);
    if (src.empty()) continue;
    Cache::run_moves(to, a, wd.p.get(), ws.p.get(), cut ? wv.p.get() : nullptr, src.size(), below(3), 1 + below(3));
    const auto before = a.want;
    for (size_t i = 0; i < src.size(); ++i) {
      if (static_cast<uint32_t>(src[i]) >= c.pages || static_cast<uint32_t>(dst[i]) >= c.pages) continue;
      const int64_t v = !cut || valid[i] > static_cast<int64_t>(c.rows) ? c.rows : valid[i] < 0 ? 0 : valid[i];
      to.move(a, src[i], dst[i], static_cast<uint32_t>(v), before);
    }
    ++g_calls;
    a.check("copy: source pool"), b.check("copy: bytes");
  }
}

// A book and lists of random words: any result, no access outside.
void random_words() {
  Cache cache;
  if (!cache.make(some_config(false))) return fail("a configuration was refused");
  const Config& c = cache.pool.c;
  for (int turn = 0; turn < 4; ++turn) {
    for (uint64_t i = 0; i < cache.at.words; ++i)
      cache.book[i] = static_cast<int32_t>(below(3) ? below(2 * c.pages + 2) : rnd());
    const uint32_t n = static_cast<uint32_t>(between(1, 40));
    List x, y;
    for (uint32_t i = 0; i < n; ++i)
      x.push_back(static_cast<int32_t>(below(4) ? below(c.seqs) : rnd())), y.push_back(static_cast<int32_t>(below(4) ? below(c.seqs) : rnd()));
    Words a(x), b(y), granted(List(n, 0)), out(List(c.pages + 2, 0));
    cache.start(), cache.reads(a), cache.reads(b), cache.writes(granted), cache.writes(out);
    cache.run_reserve(a, b, granted.p.get(), n);
    cache.run_fork(a, b, granted.p.get(), n);
    cache.run_free(a, b.p.get(), n);
    if (c.pages / 2) {
      cache.run_compact(c.pages / 2, out.p.get());
    }
    ++g_calls;
  }
}

// Another call on the same book, which nobody has ordered with this one, may change the
// work memory between two launches, or in the middle of one: any result, no access
// outside.
void work_memory_changes() {
  Cache cache;
  if (!cache.make(some_config(false))) return fail("a configuration was refused");
  const Config& c = cache.pool.c;
  const auto some_word = [&] {
    return static_cast<uint32_t>(below(3) ? below(2 * c.pages + 2) : below(2) ? below(50) : rnd());
  };
  for (int turn = 0; turn < 4; ++turn) {
    const uint32_t n = static_cast<uint32_t>(between(1, 40));
    List x, y;
    for (uint32_t i = 0; i < n; ++i)
      x.push_back(static_cast<int32_t>(below(c.seqs))), y.push_back(static_cast<int32_t>(below(3 * c.rows)));
    Words a(x), b(y), granted(List(n, 0)), out(List(c.pages + 2, 0));
    cache.start(), cache.reads(a), cache.reads(b), cache.writes(granted), cache.writes(out);
    g_meanwhile = [&] {
      for (uint64_t i = 0; i < cache.work_words; ++i)
        if (below(2)) cache.work[i] = some_word();
      // a number of moves with the divisor of another
      if (below(2)) *cache.moves.count = {static_cast<uint32_t>(between(1, 40)), 0, magic_divisor(some_word())};
    };
    cache.run_reserve(a, b, granted.p.get(), n);
    cache.run_fork(a, b, granted.p.get(), n);
    if (c.pages / 2) cache.run_compact(c.pages / 2, out.p.get());
    g_meanwhile = nullptr;
    ++g_calls;
  }
}

// More pages than one vector of free bits for each lane covers, and more than one
// round of entries that ask for them.
void large_pool() {
  Config c;
  c.rows = 1, c.seqs = 1500, c.width = 400, c.pages = 131072 + 70001;
  c.planes.push_back({nullptr, 0, 1, 1});
  Cache cache;
  if (!cache.make(c)) return fail("a configuration was refused");
  List seqs, more;
  for (int32_t i = 0; i < 1500; ++i) seqs.push_back(1499 - i), more.push_back(i % 7 == 0 ? 0 : 100 + i % 90);
  cache.reserve(seqs, more);
  List gone;
  for (int32_t i = 0; i < 1500; i += 3) gone.push_back(i);
  cache.free_tokens(gone, nullptr);
  cache.compact(1000);
  cache.compact(c.pages);
  cache.reserve(gone, List(gone.size(), 300));  // does not fit to its end
}

// The rule that picks a kernel, on both sides of each of its limits; for first
// rows half of the pages' bytes count.
void launch_rule() {
  const uint32_t pieces[2] = {1024, 256};
  const uint64_t page = 1 << 20;
  const uint32_t streams = kMoveStreams / page, nt = kMoveNtStores / page;
  for (unsigned cut = 0; cut < 2; ++cut)
    for (uint32_t route = 0; route < 3; ++route)
      for (uint32_t pages : {1u, streams - 1, streams, nt - 1, nt, 4 * nt}) {
        const uint64_t n = static_cast<uint64_t>(pages) * (cut ? 2 : 1);
        const PageMovePlan p = plan_page_moves(n, 0, cut, pieces, page, 256, route, 128);
        const uint32_t store = route == MI355_BLIT_ROUTE_DEVICE_TO_HOST ? MI355_BLIT_STORE_SYSTEM_WT
                               : pages >= nt                            ? MI355_BLIT_STORE_NT
                               : pages >= streams                       ? MI355_BLIT_STORE_AGENT_WT
                                                                        : MI355_BLIT_STORE_CACHED;
        if (p.table != cut || p.nt_load != (pages >= streams) || p.store_policy != store) fail("rule of kernels");
        const uint64_t want = n * pieces[cut] / kMoveWaves;
        if (p.grid != (route ? (want < 128 ? want : 128) : want)) fail("rule of grids");
      }
  // a list of unknown length: its room, up to so many workgroups for each CU
  if (plan_page_moves(500, kMostListed, false, pieces, page, 256, 0, 128).grid != 500 * 256 ||
      plan_page_moves(513, kMostListed, false, pieces, page, 256, 0, 128).grid != kMostListed * 256)
    fail("rule of grids for lists");
}

// A pool of one page has nowhere to move it: no moves, and the head says so.
void one_page() {
  Config c;
  c.rows = 4, c.seqs = 2, c.width = 1, c.pages = 1;
  c.planes.push_back({nullptr, 0, 24, 1});
  Cache cache;
  if (!cache.make(c)) return fail("a configuration was refused");
  for (int turn = 0; turn < 2; ++turn) {
    cache.book[0] = 7;
    Words out(List(2, -5));
    cache.start(), cache.writes(out);
    cache.run_compact(most_page_moves(9, c.pages), out.p.get());
    cache.check("compact of one page");
    if (out.p[0] != -5) fail("compact of one page: moves");
    cache.reserve({1}, {3});
  }
  if (most_page_moves(9, 1) != 1 || most_page_moves(9, 2) != 1 || most_page_moves(9, 7) != 3 ||
      most_page_moves(9, 100) != 9 || most_page_moves(0, 1) != 0 || most_page_moves(0, 100) != 0)
    fail("room for moves");
}

// Tables of several stretches of kTableChunk pages.
void long_sequences() {
  Config c;
  c.rows = 3, c.seqs = 6, c.width = 3 * kTableChunk + 5, c.pages = 4 * kTableChunk;
  c.planes.push_back({nullptr, 0, 1, 1});
  Cache cache;
  if (!cache.make(c)) return fail("a configuration was refused");
  cache.reserve({0, 1}, {static_cast<int32_t>(3 * c.width - 1), static_cast<int32_t>(3 * kTableChunk)});
  for (int turn = 0; turn < 6; ++turn) {
    cache.fork({0, 1, 0, 9}, {2, 3, 2, 4});
    const List keep = {static_cast<int32_t>(3 * kTableChunk + 7 * turn), 5, 100, 3};
    cache.free_tokens({2, 3, 2, 5}, &keep);
    cache.free_tokens({3, 2}, nullptr);
  }
}

}  // namespace

int main(int argc, char** argv) {
  unsigned shard = 0, shards = 1;
  for (int i = 1; i < argc; ++i)
    if (!std::strcmp(argv[i], "--shard") && i + 1 < argc && std::sscanf(argv[++i], "%u/%u", &shard, &shards) != 2) return 2;
  for (unsigned k = shard; k < 302; k += shards) {
    g_state = 0x9E3779B97F4A7C15ull * (k + 1);
    g_at = "case " + std::to_string(k);
    if (k == 0) large_pool();
    else if (k == 1) long_sequences();
    else if (k == 300) one_page();
    else if (k == 301) launch_rule();
    else if (k >= 240) work_memory_changes();
    else if (k % 12 == 1) random_life(4, true);
    else if (k % 4 == 2) random_copies();
    else if (k % 4 == 3) random_words();
    else random_life(14, false);
  }
  std::printf("%" PRIu64 " calls, %" PRIu64 " failures\n", g_calls, g_failures);
  return g_failures ? 1 : 0;
}
