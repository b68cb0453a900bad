// wl_kv4.h - the KV cache in 4 bits: its blocks, its tiles, and the host interface of wl_kv4.hip.
//
// A block is 32 consecutive values of a head's row at one position: a scale d and sixteen levels,
// the values (n - 8) d with n = 0..15. d is -m / 8 for m the value of largest magnitude (the first
// of several), rounded to 8 significant bits and to a multiple of 2^-24, at most 2720 in magnitude;
// n = rint(x / d) + 8, held to 0..15. With 8 bits of d and 3 of n - 8 every value is an fp16 number, so
// the matrix cores take the cache exactly: no product with a scale is rounded on the way. A block with an
// infinity or NaN holds NaN.
//
// The scale is kept as s = 16 d in fp16 (exact: a multiple of 2^-20 of 8 bits): with the level in the
// four top bits of the mantissa of 1.0, fma(1 + n / 16, s, -1.5 s) is (n - 8) d in one rounding
// that has nothing to round (1.5 s is exact too: at most 10 bits, at most 65280).
//
// A cache holds kv_heads times ceil(positions / 32) tiles of 18 HD bytes: 32 positions of a head,
// 16 HD bytes of levels, then 2 HD of scales. Inside, the order is the one in which a wave's
// lanes give them to v_mfma_f32_16x16x32_f16, so that every load of a tile is 16 consecutive bytes of a
// lane and 1 KB of a wave, and no level is moved between lanes (E = HD / 64, NB = HD / 32):
//   keys    words [position r'][HD / 8]: value 2 p + h of the word's 8 at bit 16 h + 4 p;
//           scales [r' % 16][NB][r' / 16]
//   values  words [e][kq][x][jp]: bit 16 h + 4 i holds value 4 E x + 4 e + i of position
//           16 t + 4 kq + r, where 4 t + r = 2 jp + h; scales [kq][NB][4 t + r]
// A position's values fill 16-bit halves of their own: two positions share no byte.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace wl {

constexpr int kKv4Tile = 32;   // positions per tile
constexpr int kKv4Rows = 64;   // rows of a batch call that one launch takes

constexpr int kKv4Row = 1 << 24;  // values of a position's keys at most

// Bytes of one cache; 0 for head dims other than 64 and 128, and for more KV heads than the calls take.
inline int64_t kv4_bytes(int64_t positions, int64_t kv_heads, int hd) {
  if (positions <= 0 || kv_heads <= 0 || (hd != 64 && hd != 128) || kv_heads * hd > kKv4Row) return 0;
  return kv_heads * ((positions + kKv4Tile - 1) / kKv4Tile) * 18 * hd;
}

// The rows of a call: T consecutive positions pos0.. of one sequence (batch = 0), or row i at
// position pos[i] of slot slot[i].
struct KvRows {
  int n = 0, pos0 = 0, batch = 0;
  int pos[kKv4Rows] = {}, slot[kKv4Rows] = {};
  __host__ __device__ int position(int t) const { return batch ? pos[t] : pos0 + t; }
  __host__ __device__ int slot_of(int t) const { return batch ? slot[t] : 0; }
};

// k, v [rows][KH * HD] into the caches (of `positions` positions; slot_bytes apart).
hipError_t kv4_store_launch(const float *k, const float *v, int KH, int HD, uint8_t *K, uint8_t *V, int64_t positions,
                            int64_t slot_bytes, const KvRows &rows, hipStream_t st);
// Positions pos0 .. pos0 + T - 1 as fp32 rows k, v [T][KH * HD].
hipError_t kv4_read_launch(const uint8_t *K, const uint8_t *V, int KH, int HD, int64_t positions, int pos0, int T,
                           float *k, float *v, hipStream_t st);

#ifdef __HIPCC__
// Word of a tile that holds values 8 c .. 8 c + 7 of key r'.
__device__ __forceinline__ int kv4_key_word(int r, int c, int HD) { return r * (HD / 8) + c; }
__device__ __forceinline__ int kv4_key_scale(int r, int blk, int HD) { return ((r & 15) * (HD / 32) + blk) * 2 + (r >> 4); }
// The 16-bit half of a tile that holds values 4 f .. 4 f + 3 of value row r'.
__device__ __forceinline__ int kv4_val_half(int r, int f, int HD) {
  const int E = HD / 64, x = f / E, e = f % E, kq = (r & 15) >> 2, j = 4 * (r >> 4) + (r & 3);
  return (((e * 4 + kq) * 16 + x) * 4 + (j >> 1)) * 2 + (j & 1);
}
__device__ __forceinline__ int kv4_val_scale(int r, int blk, int HD) {
  return (((r & 15) >> 2) * (HD / 32) + blk) * 8 + 4 * (r >> 4) + (r & 3);
}
__device__ __forceinline__ float kv4_value(uint32_t n, uint16_t s) {
  return ((float)(int)n - 8.f) * ((float)__builtin_bit_cast(_Float16, s) * 0.0625f);  // exact
}

// A block's scale d from its value m of largest magnitude: -m / 8 to 8 significant bits and a
// multiple of 2^-24 (round to nearest even: adding 1.5 2^(e + 23) leaves multiples of 2^e).
__device__ __forceinline__ float kv4_scale(float m) {
#pragma clang fp contract(off)
  const float d = fminf(fmaxf(m * -0.125f, -2720.f), 2720.f);
  int e = (int)((__float_as_uint(d) >> 23) & 255u) - 127 - 7;
  e = e < -24 ? -24 : e;
  const float c = __uint_as_float((uint32_t)(e + 23 + 127) << 23 | 0x400000u);
  return (d + c) - c;
}

// Values 8 c8 .. 8 c8 + 7 of a head's row into position r' of its tile, four neighbouring lanes a block (all four of them
// active): of values (val) or of keys.
__device__ __forceinline__ void kv4_put(const float (&a)[8], bool val, int c8, uint8_t *tile, int r, int HD) {
#pragma clang fp contract(off)
  float m = a[0];
  int bad = !__builtin_isfinite(a[0]);
#pragma unroll
  for (int i = 1; i < 8; i++) {
    m = fabsf(a[i]) > fabsf(m) ? a[i] : m;
    bad |= !__builtin_isfinite(a[i]);
  }
#pragma unroll
  for (int s = 1; s <= 2; s <<= 1) {  // of equals the lower lane's
    const float o = __shfl_xor(m, s, 64);
    bad |= __shfl_xor(bad, s, 64);
    const bool lower = threadIdx.x & s;
    m = fabsf(o) > fabsf(m) || (fabsf(o) == fabsf(m) && lower) ? o : m;
  }
  const float d = bad ? 0.f : kv4_scale(m);
  uint32_t n[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float q = d != 0.f ? rintf(a[i] / d) + 8.f : 8.f;
    n[i] = (uint32_t)fminf(fmaxf(q, 0.f), 15.f);
  }
  const uint16_t s = bad ? (uint16_t)0x7e00 : __builtin_bit_cast(uint16_t, (_Float16)(16.f * d));
  uint16_t *sc = reinterpret_cast<uint16_t *>(tile + 16 * HD);
  if (!val) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) w |= n[i] << (16 * (i & 1) + 4 * (i >> 1));
    reinterpret_cast<uint32_t *>(tile)[kv4_key_word(r, c8, HD)] = w;
    if ((c8 & 3) == 0) sc[kv4_key_scale(r, c8 >> 2, HD)] = s;
  } else {
#pragma unroll
    for (int f = 0; f < 2; f++)
      reinterpret_cast<uint16_t *>(tile)[kv4_val_half(r, 2 * c8 + f, HD)] =
          (uint16_t)(n[4 * f] | n[4 * f + 1] << 4 | n[4 * f + 2] << 8 | n[4 * f + 3] << 12);
    if ((c8 & 3) == 0) sc[kv4_val_scale(r, c8 >> 2, HD)] = s;
  }
}
#endif

}  // namespace wl
