// lane_emulation.h with what the page kernels use beyond it: scalar loads
// of their records, atomics on memory and on LDS, bit counts, and workgroups that run in
// the reverse order on request (the result of a launch may not depend on it).
#ifndef MI355_TESTS_LANE_EMULATION_PAGES_H_
#define MI355_TESTS_LANE_EMULATION_PAGES_H_

#define workgroup_index launch_order_index
#include "lane_emulation.h"
#undef workgroup_index

#include "blit_pages.h"

namespace mi355 {

inline unsigned g_reverse_grid = 0;  // not 0: workgroup b of so many is run as the (grid - 1 - b)th
MI355_DEVICE unsigned workgroup_index() {
  return g_reverse_grid ? g_reverse_grid - 1 - launch_order_index() : launch_order_index();
}

MI355_DEVICE PagePlane ld_uniform_plane(const PagePlane* p) { return lane_emu::checked_load<PagePlane>(p, 64); }
MI355_DEVICE PageMoveCount ld_uniform_count(const PageMoveCount* p) { return lane_emu::checked_load<PageMoveCount>(p, 8); }

// A lane runs until its next lane move or barrier, so these are atomic.
template <typename T, typename F>
MI355_DEVICE T checked_change(T* p, F f) {
  const T was = lane_emu::checked_load<T>(p, sizeof(T));
  lane_emu::checked_store(p, static_cast<T>(f(was)), sizeof(T));
  return was;
}
MI355_DEVICE uint32_t ld_agent_u32(const uint32_t* p) { return lane_emu::checked_load<uint32_t>(p, 4); }
MI355_DEVICE int32_t add_agent_i32(int32_t* p, int32_t v) {
  return checked_change(p, [v](int32_t w) { return static_cast<int32_t>(static_cast<uint32_t>(w) + static_cast<uint32_t>(v)); });
}
MI355_DEVICE int32_t min_agent_i32(int32_t* p, int32_t v) {
  return checked_change(p, [v](int32_t w) { return w < v ? w : v; });
}
MI355_DEVICE uint32_t or_agent_u32(uint32_t* p, uint32_t v) {
  return checked_change(p, [v](uint32_t w) { return w | v; });
}
MI355_DEVICE void wait_for_memory() {}

// LDS is ordinary memory here (AddressSanitizer watches it)
MI355_DEVICE uint32_t lds_compare_swap(uint32_t* p, uint32_t expected, uint32_t v) {
  const uint32_t was = *p;
  if (was == expected) *p = v;
  return was;
}
MI355_DEVICE uint32_t lds_add(uint32_t* p, uint32_t v) { const uint32_t was = *p; *p += v; return was; }
MI355_DEVICE uint32_t lds_min(uint32_t* p, uint32_t v) { const uint32_t was = *p; if (v < was) *p = v; return was; }
MI355_DEVICE uint32_t lds_max(uint32_t* p, uint32_t v) { const uint32_t was = *p; if (v > was) *p = v; return was; }
MI355_DEVICE uint32_t lds_or(uint32_t* p, uint32_t v) { const uint32_t was = *p; *p |= v; return was; }

MI355_DEVICE uint64_t wave_ballot(bool v) {
  const unsigned parity = lane_emu::lane_move_arrive(v);
  const lane_emu::Wave& w = lane_emu::g_m.waves[lane_emu::g_m.cur / kWave];
  uint64_t all = 0;
  for (unsigned i = 0; i < kWave; ++i)
    if (w.deposited[parity] >> i & 1 && w.operand[parity][i]) all |= 1ull << i;
  return all;
}

MI355_DEVICE unsigned popcount32(uint32_t v) { return static_cast<unsigned>(__builtin_popcount(v)); }
MI355_DEVICE unsigned popcount64(uint64_t v) { return static_cast<unsigned>(__builtin_popcountll(v)); }

}  // namespace mi355

#endif  // MI355_TESTS_LANE_EMULATION_PAGES_H_
