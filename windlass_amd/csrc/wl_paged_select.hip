// wl_paged_select.hip - the pages that a row and KV head attends to, by a bound of their scores (wl_paged.h).
#include "wl_paged.h"

#include "wl_paged_device.h"

#pragma clang fp contract(off)

namespace wl {

// One workgroup per row and KV head: the scores, then the pages one after the other.
__global__ __launch_bounds__(256) void paged_select_kernel(PagePool P, PageRows R, const float *__restrict__ q, int H,
                                                           PageSelect S, double *__restrict__ scores, int64_t width,
                                                           int32_t *__restrict__ blocks) {
  __shared__ double best[256];
  __shared__ int at[256];
  const int kvh = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, HD = P.HD, G = H / P.KH;
  const int i = entry_of(R.row0, R.n, row);
  const int cur = (R.pos[i] + row - R.row0[i]) >> P.shift;
  const int from = S.first < cur + 1 ? S.first : cur + 1;
  const int to = S.recent > cur + 1 - from ? from : cur + 1 - S.recent;
  double *sc = scores + ((int64_t)row * P.KH + kvh) * width;
  int32_t *o = blocks + ((int64_t)row * P.KH + kvh) * S.most();
  const float *qp = q + ((int64_t)row * H + kvh * G) * HD;
  for (int j = from + tid; j < to; j += 256) {
    const int id = P.id(R.seq[i], j);
    double m = -INFINITY;
    if (id >= 0) {
      const uint16_t *b = P.bounds + ((int64_t)id * P.KH + kvh) * 2 * HD;
      for (int g = 0; g < G; g++) {
        double s = 0.0;
        for (int d = 0; d < HD; d++) {
          const double x = qp[g * HD + d];
          const double l = (double)(float)__builtin_bit_cast(_Float16, b[d]);
          const double h = (double)(float)__builtin_bit_cast(_Float16, b[HD + d]);
          s += fmax(x, 0.0) * h + fmin(x, 0.0) * l;
        }
        s = __builtin_isfinite(s) ? s : INFINITY;
        m = s > m ? s : m;
      }
    }
    sc[j] = m;
  }
  __syncthreads();
  // the largest, `top` times; taken pages become NaN
  for (int k = 0; k < S.top; k++) {
    double m = -INFINITY;
    int a = -1;
    for (int j = from + tid; j < to; j += 256)
      if (sc[j] > m) {
        m = sc[j];
        a = j;
      }
    best[tid] = m;
    at[tid] = a;
    __syncthreads();
    if (tid == 0) {
      for (int t = 1; t < 256; t++)
        if (at[t] >= 0 && (a < 0 || best[t] > m || (best[t] == m && at[t] < a))) {
          m = best[t];
          a = at[t];
        }
      at[0] = a;
      if (a >= 0) sc[a] = __builtin_nan("");
    }
    __syncthreads();
    if (at[0] < 0) break;  // uniform
    __syncthreads();
  }
  __syncthreads();
  if (tid == 0) {
    int n = 0;
    for (int j = 0; j <= cur; j++)
      if (j < from || j >= to || sc[j] != sc[j]) o[n++] = j;
    for (; n < S.most(); n++) o[n] = -1;
  }
}

static int64_t select_width(const PagePool &p, const PageRows &r) {
  int64_t w = 1;
  for (int i = 0; i < r.n; i++)
    if (r.rows(i)) w = w > ((r.pos[i] + r.rows(i) - 1) >> p.shift) + 1 ? w : ((r.pos[i] + r.rows(i) - 1) >> p.shift) + 1;
  return w;
}

int64_t paged_select_scratch_bytes(const PagePool &p, const PageRows &r, const PageSelect &) {
  return (int64_t)r.row0[r.n] * p.KH * select_width(p, r) * 8;
}

hipError_t paged_select_launch(const PagePool &p, const PageRows &r, const float *q, int H, const PageSelect &s,
                               void *scratch, int32_t *blocks, hipStream_t st) {
  const int rows = r.row0[r.n];
  if (rows <= 0) return hipSuccess;
  hipLaunchKernelGGL(paged_select_kernel, dim3(p.KH, rows), dim3(256), 0, st, p, r, q, H, s, (double *)scratch,
                     select_width(p, r), blocks);
  return hipGetLastError();
}

}  // namespace wl
