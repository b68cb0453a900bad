// wl_paged_device.h - a launch's entries and items, for the paged kernels.
#pragma once
#include "wl_fmma_codec.h"
#include "wl_paged.h"

namespace wl {

// An entry as a launch takes it: its items begin at off; the rest by what the launch needs.
struct __attribute__((aligned(16))) PageEntry {
  int off, row0, pos, seq;
  int rows, per, rec, runs;
};
struct PageItems {
  PageEntry e[kPgRows + 1];  // a prefix' rows are one more
  int n = 0, items = 0;
  // The next entry, of `count` items.
  void add(const PageRows &r, int i, int count, int per = 0, int rec = 0, int runs = 0) {
    if (!count) return;
    e[n++] = PageEntry{items, r.row0[i], r.pos[i], r.seq[i], r.rows(i), per, rec, runs};
    items += count;
  }
};

#ifdef __HIPCC__
// The entry of item x, uniform; every lane active. One load by lanes and its choice, not a search and then loads that wait for
// it (few rows of a shared prefix 8.4 -> 7.8 us); a single entry by scalar loads.
__device__ __forceinline__ PageEntry entry_of(const PageItems &I, int x) {
  if (I.n == 1) return I.e[0];
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  static_assert(kPgRows < 128, "two lanes' worth");
  const int lane = threadIdx.x & 63, n = I.n;
  const i32x4 *p = reinterpret_cast<const i32x4 *>(I.e + (lane < n ? lane : n - 1));
  i32x4 a = p[0], b = p[1];
  int i = __popcll(__ballot(lane < n && a.x <= x)) - 1;
  if (n > 64 && i == 63) {  // uniform
    const i32x4 *h = reinterpret_cast<const i32x4 *>(I.e + (lane + 64 < n ? lane + 64 : n - 1));
    const i32x4 c = h[0], d = h[1];
    const int more = __popcll(__ballot(lane + 64 < n && c.x <= x));
    if (more) {
      a = c;
      b = d;
      i = more - 1;
    }
  }
  auto at = [&](int v) { return __builtin_amdgcn_readlane(v, i); };
  return PageEntry{at(a.x), at(a.y), at(a.z), at(a.w), at(b.x), at(b.y), at(b.z), at(b.w)};
}
#endif

}  // namespace wl
