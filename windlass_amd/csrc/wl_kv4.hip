// wl_kv4.hip - rows of keys and values into the 4-bit caches and back (wl_kv4.h).
//
// What bounds it: 8 bytes read and 1.125 written per key and value pair; a decode step's row is a
// launch's latency, a prompt's rows HBM.
#include "wl_kv4.h"

#include "wl_device.h"

#pragma clang fp contract(off)

namespace wl {

typedef float f4a4 __attribute__((ext_vector_type(4), aligned(4)));  // float4 at any float's address

// A block's scale d from its value m of largest magnitude: -m / 8 to 8 significant bits and a
// multiple of 2^-24 (round to nearest even: adding 1.5 2^(e + 23) leaves multiples of 2^e).
__device__ __forceinline__ float kv4_scale(float m) {
  const float d = fminf(fmaxf(m * -0.125f, -2720.f), 2720.f);
  int e = (int)((__float_as_uint(d) >> 23) & 255u) - 127 - 7;
  e = e < -24 ? -24 : e;
  const float c = __uint_as_float((uint32_t)(e + 23 + 127) << 23 | 0x400000u);
  return (d + c) - c;
}

// Four lanes per block, eight values each; the keys' threads, then the values'.
__global__ __launch_bounds__(256) void kv4_store_kernel(const float *__restrict__ k, const float *__restrict__ v,
                                                        int KH, int HD, uint8_t *__restrict__ K,
                                                        uint8_t *__restrict__ V, int64_t tiles, int64_t slot_bytes,
                                                        KvRows R) {
  const int per = KH * HD / 8;  // threads of a row of keys
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, half = (int64_t)R.n * per;
  if (id >= 2 * half) return;  // whole blocks of four lanes: half is a multiple of 4
  const bool val = id >= half;
  const int64_t at = val ? id - half : id;
  const int t = (int)(at / per), c = (int)(at % per), kvh = c / (HD / 8), c8 = c % (HD / 8);
  const float *x = (val ? v : k) + at * 8;
  const f4a4 xa = *reinterpret_cast<const f4a4 *>(x), xb = *reinterpret_cast<const f4a4 *>(x + 4);
  const float a[8] = {xa.x, xa.y, xa.z, xa.w, xb.x, xb.y, xb.z, xb.w};
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
  const int p = R.position(t), r = p % kKv4Tile;
  uint8_t *tile = (val ? V : K) + R.slot_of(t) * slot_bytes + ((int64_t)kvh * tiles + p / kKv4Tile) * (18 * HD);
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

__global__ __launch_bounds__(256) void kv4_read_kernel(const uint8_t *__restrict__ K, const uint8_t *__restrict__ V,
                                                       int KH, int HD, int64_t tiles, int pos0, int T,
                                                       float *__restrict__ k, float *__restrict__ v) {
  const int per = KH * HD / 8;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, half = (int64_t)T * per;
  if (id >= 2 * half) return;
  const bool val = id >= half;
  const int64_t at = val ? id - half : id;
  const int t = (int)(at / per), c = (int)(at % per), kvh = c / (HD / 8), c8 = c % (HD / 8);
  const int p = pos0 + t, r = p % kKv4Tile;
  const uint8_t *tile = (val ? V : K) + ((int64_t)kvh * tiles + p / kKv4Tile) * (18 * HD);
  const uint16_t *sc = reinterpret_cast<const uint16_t *>(tile + 16 * HD);
  float o[8];
  if (!val) {
    const uint32_t w = reinterpret_cast<const uint32_t *>(tile)[kv4_key_word(r, c8, HD)];
    const uint16_t s = sc[kv4_key_scale(r, c8 >> 2, HD)];
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = kv4_value((w >> (16 * (i & 1) + 4 * (i >> 1))) & 15u, s);
  } else {
    const uint16_t s = sc[kv4_val_scale(r, c8 >> 2, HD)];
#pragma unroll
    for (int f = 0; f < 2; f++) {
      const uint32_t w = reinterpret_cast<const uint16_t *>(tile)[kv4_val_half(r, 2 * c8 + f, HD)];
#pragma unroll
      for (int i = 0; i < 4; i++) o[4 * f + i] = kv4_value((w >> (4 * i)) & 15u, s);
    }
  }
  float *y = (val ? v : k) + at * 8;
  *reinterpret_cast<f4a4 *>(y) = f4a4{o[0], o[1], o[2], o[3]};
  *reinterpret_cast<f4a4 *>(y + 4) = f4a4{o[4], o[5], o[6], o[7]};
}

static int64_t tiles_of(int64_t positions) { return (positions + kKv4Tile - 1) / kKv4Tile; }

hipError_t kv4_store_launch(const float *k, const float *v, int KH, int HD, uint8_t *K, uint8_t *V, int64_t positions,
                            int64_t slot_bytes, const KvRows &rows, hipStream_t st) {
  if (rows.n <= 0) return hipSuccess;
  const int64_t threads = (int64_t)rows.n * KH * (HD / 8) * 2;
  hipLaunchKernelGGL(kv4_store_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, k, v, KH, HD, K, V,
                     tiles_of(positions), slot_bytes, rows);
  return hipGetLastError();
}

hipError_t kv4_read_launch(const uint8_t *K, const uint8_t *V, int KH, int HD, int64_t positions, int pos0, int T,
                           float *k, float *v, hipStream_t st) {
  if (T <= 0) return hipSuccess;
  const int64_t threads = (int64_t)T * KH * (HD / 8) * 2;
  hipLaunchKernelGGL(kv4_read_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, K, V, KH, HD,
                     tiles_of(positions), pos0, T, k, v);
  return hipGetLastError();
}

}  // namespace wl
