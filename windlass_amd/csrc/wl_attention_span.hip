// wl_attention_span.hip - attention over 4-bit caches (wl_kv4.h), and over fp16 caches with a sliding
// window and first tokens that stay visible (Attention, src/Transformer.cs:351-393, over the
// positions Span names).
#include "wl_attention_span.h"

#include "wl_device.h"

#pragma clang fp contract(off)

namespace wl {

struct F16Rows {
  const uint16_t *K, *V;
  int64_t kv_dim;
  __device__ float key(int64_t j, int i) const { return (float)__builtin_bit_cast(_Float16, K[j * kv_dim + i]); }
  __device__ float val(int64_t j, int i) const { return (float)__builtin_bit_cast(_Float16, V[j * kv_dim + i]); }
};

struct Kv4Rows {
  const uint8_t *K, *V;  // the head's tiles
  int HD;
  __device__ float key(int64_t j, int i) const {
    const uint8_t *t = K + j / kKv4Tile * (18 * HD);
    const int r = (int)(j % kKv4Tile);
    const uint32_t w = reinterpret_cast<const uint32_t *>(t)[kv4_key_word(r, i >> 3, HD)];
    return kv4_value((w >> (16 * (i & 1) + 4 * ((i & 7) >> 1))) & 15u,
                     reinterpret_cast<const uint16_t *>(t + 16 * HD)[kv4_key_scale(r, i >> 5, HD)]);
  }
  __device__ float val(int64_t j, int i) const {
    const uint8_t *t = V + j / kKv4Tile * (18 * HD);
    const int r = (int)(j % kKv4Tile);
    const uint32_t w = reinterpret_cast<const uint16_t *>(t)[kv4_val_half(r, i >> 2, HD)];
    return kv4_value((w >> (4 * (i & 3))) & 15u,
                     reinterpret_cast<const uint16_t *>(t + 16 * HD)[kv4_val_scale(r, i >> 5, HD)]);
  }
};

// Block-wide sum and maximum of 256 threads.
__device__ double span_sum(double v, double *sh) {
  v = wave_sum_d(v);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (sh[0] + sh[1]) + (sh[2] + sh[3]);
  __syncthreads();
  return v;
}
__device__ float span_max(float v, float *sh) {
  v = wave_max_f(v);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
  __syncthreads();
  return v;
}

// One workgroup per (head, row): scores, their maximum, exponentials, sums.
template <class C>
__device__ void span_row(const C &c, const float *qp, int HD, int p, const Span &s, float scale, float *sp, float *op) {
  __shared__ double shd[4];
  __shared__ float shf[4];
  const int first = s.first(p), lead = s.lead(p), n = s.seen(p);
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int64_t j = i < lead ? i : first + (i - lead);
    float d = 0.f;
    for (int e = 0; e < HD; e++) d += qp[e] * c.key(j, e);
    d *= scale;
    sp[i] = d;
    mx = fmaxf(mx, d);
  }
  mx = span_max(mx, shf);
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) {
    const float e = (float)exp((double)(sp[i] - mx));
    sp[i] = e;
    sum += (double)e;
  }
  sum = span_sum(sum, shd);  // its barriers also order the writes of sp before the reads below
  for (int d = threadIdx.x; d < HD; d += 256) {
    float o = 0.f;
    for (int i = 0; i < n; i++) o += sp[i] * c.val(i < lead ? i : first + (i - lead), d);
    op[d] = (float)((double)o / sum);
  }
}

__global__ __launch_bounds__(256) void span_rows_kernel(const float *__restrict__ q, int H, KvCache c, Span s, KvRows R,
                                                        float scale, float *__restrict__ scores, int64_t max_n,
                                                        float *__restrict__ out) {
  const int h = blockIdx.x, t = blockIdx.y, kvh = h / (H / c.KH), HD = c.HD;
  const int64_t row = ((int64_t)t * H + h), off = (int64_t)R.slot_of(t) * c.slot_bytes;
  const float *qp = q + row * HD;
  if (c.bits == 4) {
    const int64_t head = off + (int64_t)kvh * ((c.positions + kKv4Tile - 1) / kKv4Tile) * (18 * HD);
    span_row(Kv4Rows{c.K + head, c.V + head, HD}, qp, HD, R.position(t), s, scale, scores + row * max_n, out + row * HD);
  } else {
    const int64_t head = off + (int64_t)kvh * HD * 2;
    span_row(F16Rows{(const uint16_t *)(c.K + head), (const uint16_t *)(c.V + head), (int64_t)c.KH * HD}, qp, HD,
             R.position(t), s, scale, scores + row * max_n, out + row * HD);
  }
}

static int64_t span_max_n(const Span &s, const KvRows &R) {
  int64_t m = 0;
  if (!R.batch) return s.seen(R.pos0 + R.n - 1);
  for (int i = 0; i < R.n; i++) m = s.seen(R.pos[i]) > m ? s.seen(R.pos[i]) : m;
  return m;
}

int64_t attention_span_scratch_floats(const KvCache &c, int H, const Span &s, const KvRows &R) {
  return R.n > 0 ? (int64_t)R.n * H * span_max_n(s, R) : 0;
}

hipError_t attention_span_launch(const float *q, int H, const KvCache &c, const Span &s, const KvRows &R, float scale,
                                 float *scratch, float *out, hipStream_t st) {
  if (R.n <= 0) return hipSuccess;
  hipLaunchKernelGGL(span_rows_kernel, dim3(H, R.n), dim3(256), 0, st, q, H, c, s, R, scale, scratch, span_max_n(s, R),
                     out);
  return hipGetLastError();
}

}  // namespace wl
