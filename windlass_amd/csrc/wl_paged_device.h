// wl_paged_device.h - device-side helpers of the paged kernels.
#pragma once
#include "wl_fmma_codec.h"
#include "wl_paged.h"

namespace wl {

// The entry whose items off[i] .. off[i + 1] - 1 hold item x (n entries, kPgRows at most); uniform. Every lane active.
__device__ __forceinline__ int entry_of(const int *off, int n, int x) {
  static_assert(kPgRows == 128, "two ballots");
  const int lane = threadIdx.x & 63;
  const int a = __popcll(__ballot(lane < n && off[lane < n ? lane + 1 : 0] <= x));
  const int b = n > 64 ? __popcll(__ballot(lane + 64 < n && off[lane + 64 < n ? lane + 65 : 0] <= x)) : 0;
  return __builtin_amdgcn_readfirstlane(a + b);
}

}  // namespace wl
