// wl_kv4.hip - rows of keys and values into the 4-bit caches and back (wl_kv4.h).
//
// What bounds it: 8 bytes read and 1.125 written per key and value pair. A decode step's row is a launch's latency (1.7-2.5
// us of GPU time); a prompt's rows HBM (2,000 rows of 8 heads of 128, 18.7 MB each way: stored in 7.2 us, read back in
// 6.3, 2.6 and 3.0 TB/s, half of it the launch's ends). Four lanes share a block because its largest value is a maximum
// over 32; 16 bytes a lane and load keep the reads whole.
#include "wl_kv4.h"

#include "wl_device.h"

#pragma clang fp contract(off)

namespace wl {

typedef float f4a4 __attribute__((ext_vector_type(4), aligned(4)));  // float4 at any float's address

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
  const int p = R.position(t);
  kv4_put(a, val, c8, (val ? V : K) + R.slot_of(t) * slot_bytes + ((int64_t)kvh * tiles + p / kKv4Tile) * (18 * HD),
          p % kKv4Tile, HD);
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
