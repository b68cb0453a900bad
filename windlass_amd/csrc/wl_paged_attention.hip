// wl_paged_attention.hip - attention over KV caches in pages (wl_paged.h).
#include "wl_paged.h"

#include "wl_paged_device.h"

#pragma clang fp contract(off)

namespace wl {

// One wave per row and head, a lane per position for the scores and per channel for the outputs.
template <int HD>
__global__ __launch_bounds__(64) void paged_attention_kernel(PagePool P, PageRows R, const float *__restrict__ q, int H,
                                                             int prefix, const int32_t *__restrict__ blocks, int most,
                                                             float scale, float *__restrict__ out) {
  __shared__ float qs[HD];
  const int h = blockIdx.x, row = blockIdx.y, lane = threadIdx.x, kvh = h / (H / P.KH);
  const int i = entry_of(R.row0, R.n, row);
  const int p = R.pos[i] + row - R.row0[i];
  const int64_t at = ((int64_t)row * H + h) * HD;
  for (int d = lane; d < HD; d += 64) qs[d] = q[at + d];
  __syncthreads();
  float M = -INFINITY, O[HD / 64] = {};
  double L = 0.0;
  const int nb = blocks ? most : (p >> P.shift) + 1;
  for (int b = 0; b < nb; b++) {
    const int j = blocks ? blocks[((int64_t)row * P.KH + kvh) * most + b] : b;
    if (j < 0) break;
    const int id = P.id((j << P.shift) < prefix ? R.seq[0] : R.seq[i], j);
    if (id < 0) continue;
    const uint16_t *K = P.K + P.at(id, kvh), *V = P.V + P.at(id, kvh);
    for (int o0 = 0; o0 < P.page; o0 += 64) {
      const int off = o0 + lane;
      const bool in = off < P.page && (j << P.shift) + off <= p;
      float s = 0.f;
      if (in)
        for (int d = 0; d < HD; d++) s += qs[d] * (float)__builtin_bit_cast(_Float16, K[pg_key(off, d, HD)]);
      s = in ? s * scale : -INFINITY;
      float m = s;
      for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
      m = fmaxf(m, M);
      const float al = M == -INFINITY ? 0.f : expf(M - m), w = s == -INFINITY ? 0.f : expf(s - m);
      M = m;
      double l = w;
      for (int x = 32; x; x >>= 1) l += __shfl_xor(l, x, 64);
      L = L * al + l;
      for (int e = 0; e < HD / 64; e++) O[e] *= al;
      const unsigned long long seen = __ballot(in);
      for (int x = 0; x < 64; x++)
        if (seen >> x & 1) {
          const float wx = __shfl(w, x, 64);
          for (int e = 0; e < HD / 64; e++)
            O[e] += wx * (float)__builtin_bit_cast(_Float16, V[pg_val(o0 + x, lane + 64 * e, HD)]);
        }
    }
  }
  for (int e = 0; e < HD / 64; e++) out[at + lane + 64 * e] = L == 0.0 ? 0.f : (float)((double)O[e] / L);
}

int64_t paged_attention_scratch_floats(const PagePool &, const PageRows &, int, int, int) { return 0; }

hipError_t paged_attention_launch(const PagePool &p, const PageRows &r, const float *q, int H, int prefix,
                                  const int32_t *blocks, int most, float scale, float *, float *out, hipStream_t st) {
  const int rows = r.row0[r.n];
  if (rows <= 0) return hipSuccess;
  if (p.HD == 64)
    hipLaunchKernelGGL(paged_attention_kernel<64>, dim3(H, rows), dim3(64), 0, st, p, r, q, H, prefix, blocks, most, scale,
                       out);
  else
    hipLaunchKernelGGL(paged_attention_kernel<128>, dim3(H, rows), dim3(64), 0, st, p, r, q, H, prefix, blocks, most, scale,
                       out);
  return hipGetLastError();
}

}  // namespace wl
