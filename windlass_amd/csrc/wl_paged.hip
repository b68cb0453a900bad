// wl_paged.hip - rows rotated into the pages of a KV cache, and back (wl_paged.h).
#include "wl_paged.h"

#include "wl_paged_device.h"
#include "wl_rope.h"

#include <math.h>

#pragma clang fp contract(off)

namespace wl {

struct StoreArgs {
  PagePool p;
  PageRope e;
  const float *q, *k, *v;
  float *qr;
  int H;
};

__device__ __forceinline__ uint16_t half_of(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }

// A workgroup per row.
__global__ __launch_bounds__(256) void paged_store_kernel(StoreArgs A, PageRows R) {
  __shared__ float2 angle[64];
  const int row = blockIdx.x, tid = threadIdx.x, HD = A.p.HD, KH = A.p.KH, half = A.e.n / 2;
  const int i = entry_of(R.row0, R.n, row);
  const int p = R.pos[i] + row - R.row0[i];
  const int id = A.p.id(R.seq[i], p >> A.p.shift), off = p & (A.p.page - 1);
  if (tid < 64) {
    float c = 1.f, s = 0.f;
    if (half) rope_cs(p, tid < half ? tid : 0, half, A.e.theta_scale, A.e.freq_scale, A.e.freqs, c, s);
    if (tid < half) angle[tid] = make_float2(c, s);
  }
  __syncthreads();
  auto turned = [&](const float *x, int d) {
    if (d >= A.e.n) return x[d];
    const int j = A.e.neox ? d % half : d / 2;
    const int a = A.e.neox ? j : 2 * j, b = A.e.neox ? j + half : 2 * j + 1;
    const float2 cs = angle[j];
    return d == a ? x[a] * cs.x - x[b] * cs.y : x[a] * cs.y + x[b] * cs.x;
  };
  // a pair per thread, so that q may be rotated in place
  for (int j = tid; j < A.H * HD / 2; j += 256) {
    const int h = j / (HD / 2), x = j % (HD / 2);
    const int a = x < half ? (A.e.neox ? x : 2 * x) : 2 * x, b = x < half ? (A.e.neox ? x + half : 2 * x + 1) : 2 * x + 1;
    const float *xp = A.q + ((int64_t)row * A.H + h) * HD;
    float *o = A.qr + ((int64_t)row * A.H + h) * HD;
    const float ya = turned(xp, a), yb = turned(xp, b);
    o[a] = ya;
    o[b] = yb;
  }
  if (id < 0) return;
  for (int j = tid; j < KH * HD; j += 256) {
    const int kvh = j / HD, d = j % HD;
    const int64_t at = A.p.at(id, kvh), r = (int64_t)row * KH * HD;
    A.p.K[at + pg_key(off, d, HD)] = half_of(turned(A.k + r + kvh * HD, d));
    A.p.V[at + pg_val(off, d, HD)] = half_of(A.v[r + j]);
  }
}

// The bounds of the pages written to: a workgroup per page and KV head, 16 bytes of keys a thread and step.
struct BoundsItems {
  int off[kPgRows + 1];  // pages before entry i's
};
__global__ __launch_bounds__(256) void paged_bounds_kernel(PagePool P, PageRows R, BoundsItems B) {
  __shared__ _Float16 lo[4][128], hi[4][128];
  const int kvh = blockIdx.x % P.KH, item = blockIdx.x / P.KH, tid = threadIdx.x, HD = P.HD, oct = tid / 8 % (HD / 8);
  const int i = entry_of(B.off, R.n, item);
  const int j = (R.pos[i] >> P.shift) + item - B.off[i];
  const int id = P.id(R.seq[i], j);
  if (id < 0) return;  // uniform
  const int last = R.pos[i] + R.rows(i) - 1 - (j << P.shift);  // of the page; past it where the page is full
  const uint16_t *K = P.K + P.at(id, kvh);
  _Float16 l[8], h[8];
  const _Float16 inf = (_Float16)INFINITY;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    l[e] = inf;
    h[e] = -inf;
  }
  auto take = [](_Float16 &m, _Float16 x, bool less) {  // a NaN stays
    m = (less ? x < m : x > m) || x != x ? x : m;
  };
  for (int c = tid; c < P.page * HD / 8; c += 256) {
    const int u = c / (2 * HD), t = c / HD & 1, s = c & 7;
    if (16 * u + 8 * (s >> 2) + 4 * t + (s & 3) > last) continue;
    const fh8 x = *reinterpret_cast<const fh8 *>(K + 8 * c);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      take(l[e], x[e], true);
      take(h[e], x[e], false);
    }
  }
  // the eight positions of a piece, then the waves that hold the same channels
#pragma unroll
  for (int m = 1; m <= 4; m <<= 1)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      take(l[e], (_Float16)__shfl_xor((float)l[e], m, 64), true);
      take(h[e], (_Float16)__shfl_xor((float)h[e], m, 64), false);
    }
  const int part = tid / HD;  // 2 or 4 threads a piece
  if ((tid & 7) == 0)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      lo[part][8 * oct + e] = l[e];
      hi[part][8 * oct + e] = h[e];
    }
  __syncthreads();
  if (tid >= 2 * HD) return;
  const int d = tid % HD;
  const bool up = tid >= HD;
  _Float16 m = up ? hi[0][d] : lo[0][d];
  for (int e = 1; e < 256 / HD; e++) take(m, up ? hi[e][d] : lo[e][d], !up);
  P.bounds[(((int64_t)id * P.KH + kvh) * 2 + up) * HD + d] = __builtin_bit_cast(uint16_t, m);
}

__global__ __launch_bounds__(256) void paged_read_kernel(PagePool P, int seq, int pos0, int T, float *__restrict__ k,
                                                         float *__restrict__ v) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int KD = P.KH * P.HD;
  if (e >= (int64_t)T * KD) return;
  const int p = pos0 + (int)(e / KD), j = (int)(e % KD), kvh = j / P.HD, d = j % P.HD, off = p & (P.page - 1);
  const int id = P.id(seq, p >> P.shift);
  const int64_t at = P.at(id < 0 ? 0 : id, kvh);
  k[e] = id < 0 ? 0.f : (float)__builtin_bit_cast(_Float16, P.K[at + pg_key(off, d, P.HD)]);
  v[e] = id < 0 ? 0.f : (float)__builtin_bit_cast(_Float16, P.V[at + pg_val(off, d, P.HD)]);
}

PageRope page_rope(int n, int neox, double base, double freq_scale, const float *freqs) {
  return PageRope{n, neox != 0, n ? pow(base, -2.0 / n) : 1.0, freq_scale, freqs};
}

hipError_t paged_store_launch(const PagePool &p, const PageRows &r, const float *q, int H, const float *k, const float *v,
                              const PageRope &rope, float *qr, hipStream_t st) {
  const int rows = r.row0[r.n];
  if (rows <= 0) return hipSuccess;
  hipLaunchKernelGGL(paged_store_kernel, dim3(rows), dim3(256), 0, st, StoreArgs{p, rope, q, k, v, qr, H}, r);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.bounds) return e;
  BoundsItems b;
  b.off[0] = 0;
  for (int i = 0; i < r.n; i++)
    b.off[i + 1] = b.off[i] + (r.rows(i) ? ((r.pos[i] + r.rows(i) - 1) >> p.shift) - (r.pos[i] >> p.shift) + 1 : 0);
  hipLaunchKernelGGL(paged_bounds_kernel, dim3(b.off[r.n] * p.KH), dim3(256), 0, st, p, r, b);
  return hipGetLastError();
}

hipError_t paged_read_launch(const PagePool &p, int seq, int pos0, int T, float *k, float *v, hipStream_t st) {
  const int64_t n = (int64_t)T * p.KH * p.HD;
  if (n <= 0) return hipSuccess;
  hipLaunchKernelGGL(paged_read_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p, seq, pos0, T, k, v);
  return hipGetLastError();
}

}  // namespace wl
