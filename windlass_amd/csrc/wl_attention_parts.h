// wl_attention_parts.h - what the attention kernels on the matrix cores share: queries and probabilities as two fp16
// parts, and sums under a running maximum.
#pragma once
#include "wl_fmma_codec.h"

namespace wl {

typedef float sf4 __attribute__((ext_vector_type(4)));
// A running maximum is raised only by scores more than 2^6 past it, so nearly never after a wave's first tile: the
// exponentials reach 2^6, and 2^8 of them are fp16 parts: 23 bits of what is 2^-10 or more, and off by 2^-33 at most below.
constexpr float kSpUp = 0x1p8f, kSpPast = 6.f;
// In the scores' units: finite where those are the smallest there are, so that a lane without a key yet keeps -inf as what
// raises its maximum.
__device__ __forceinline__ float past_of(float c2) { return fminf(kSpPast / c2, 3.4028235e38f); }

__device__ __forceinline__ fh8 as_fh8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(fh8, u32x4_t{a, b, c, d});
}

// Two probabilities, times kSpUp, as their fp16 parts.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t &hi, uint32_t &lo) {
  hi = __builtin_bit_cast(uint32_t, fh2{(_Float16)__builtin_fmaf(a, kSpUp, 0.f), (_Float16)__builtin_fmaf(b, kSpUp, 0.f)});
  asm("" : "+v"(hi));  // rounded once: the compiler made the halves again for the low parts
  lo = __builtin_bit_cast(uint32_t, fh2{(_Float16)__builtin_fmaf(a, kSpUp, -half_lo(hi)),
                                        (_Float16)__builtin_fmaf(b, kSpUp, -half_hi(hi))});  // exact but for their rounding
}

// What sums under the maximum M weigh under a larger one. Scores of -inf alone leave M at -inf and sums of zeros (or NaN, from
// a NaN score): a factor of zero, also where no other sums have a maximum, and 0 / 0 is such a row's output.
__device__ __forceinline__ float weight_of(float M, float m, float c2) {
  return M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((M - m) * c2);
}

typedef float f4a4 __attribute__((ext_vector_type(4), aligned(4)));  // at any float's address

}  // namespace wl
