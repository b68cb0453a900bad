// wl_attention_span.hip - attention over 4-bit caches (wl_kv4.h), and over fp16 caches with a sliding
// window and first tokens that stay visible (Attention, src/Transformer.cs:351-393, over the
// positions Span names).
#include "wl_attention_span.h"

#include "wl_fmma_codec.h"

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

// ------------------------------------------------------------------------------- few rows
// Rows of up to 15 tokens and batch rows: head dims 64 and 128 on v_mfma_f32_16x16x32_f16.
//
// S^T = K Q^T of 16 keys: the 16 columns are eight query heads of the KV head, each row of q as two
// fp16 parts (hi in column 2 g, lo in 2 g + 1: 22 bits of the largest value, exact products, fp32 sums),
// which one addition of neighbouring lanes joins. O^T = V^T P^T of 32 keys: the probabilities are where the
// scores were (lane l has keys 16 t + 4 (l / 16) + i of column l % 16), again in two parts, and V's
// operand holds those keys in that order: 4-bit tiles are stored so, fp16 rows are paired by byte
// permutes. So no value passes through LDS, and a lane's loads are its operands.
//
// A workgroup of W waves takes a run of a row's tiles (32 positions each), the waves one tile in turn, each
// with its own running maximum, sum and output; they are added through LDS. Long rows are cut in runs by a rule
// on the row's own tiles, so that a row's bits do not depend on the rows beside it.
typedef float sf4 __attribute__((ext_vector_type(4)));
// A running maximum is raised only by scores more than 2^6 past it, so nearly never after a wave's first tile: the
// exponentials reach 2^6, and 2^8 of them are fp16 parts (22 bits down to 2^-22 of the row's largest, 2^-33 of it below).
constexpr float kSpUp = 0x1p8f, kSpPast = 6.f;
constexpr int kSpWaves = 4;
constexpr int kSpRuns = 256;      // runs of a row at most

// The tiles a row at p reads, in order: those of the first tokens, then the window's.
struct SpanTiles {
  int lead, from, n;
  __host__ __device__ SpanTiles(const Span &s, int p) {
    lead = (s.lead(p) + kKv4Tile - 1) / kKv4Tile;
    from = s.first(p) / kKv4Tile;
    from = from < lead ? lead : from;
    n = lead + p / kKv4Tile - from + 1;
    if (p / kKv4Tile < from) n = lead;  // the first tokens' tiles reach the row
  }
  __host__ __device__ int tile(int i) const { return i < lead ? i : from + (i - lead); }
};

// 16-bit pairs to fp16 values: levels at bits 4 i of both halves, their scales s and -1.5 s.
template <int I>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w, fh2 s, fh2 s15, uint32_t ones) {
  const uint32_t at = I == 0 ? w << 6 : I == 1 ? w << 2 : I == 2 ? w >> 2 : w >> 6;
  const fh2 n = as_fh2((at & 0x03c003c0u) | ones);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n, s, s15));
}
// Two fp16 ones, in a register: as a constant they cost the mask and the ones an instruction each.
__device__ __forceinline__ uint32_t fp16_ones() {
  uint32_t o;
  asm("v_mov_b32 %0, 0x3c003c00" : "=v"(o));
  return o;
}
__device__ __forceinline__ fh8 as_fh8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(fh8, u32x4_t{a, b, c, d});
}
__device__ __forceinline__ fh2 scale15(fh2 s) { return s * fh2{(_Float16)-1.5f, (_Float16)-1.5f}; }

// Tiles of 4-bit caches. hide(m): bit j set where key j of the lane (keys 16 (j / 4) + 4 kq + j % 4) is not seen:
// its values become zeros.
template <int HD>
struct TileKv4 {
  static constexpr int E = HD / 64, NB = HD / 32;
  u32x4_t v[E], vs;
  uint32_t k[2][4 * E / 2], ks;
  __device__ __forceinline__ void load(const uint8_t *K, const uint8_t *V, int64_t, int64_t tile, int, int lane) {
    const uint8_t *kt = K + tile * (18 * HD), *vt = V + tile * (18 * HD);
    const int r = lane & 15, q = lane >> 4;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const uint8_t *kp = kt + (16 * t + r) * (HD / 2) + q * (HD / 8);
      if constexpr (E == 2) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t *>(kp);
        k[t][0] = w.x, k[t][1] = w.y, k[t][2] = w.z, k[t][3] = w.w;
      } else {
        const u32x2_t w = *reinterpret_cast<const u32x2_t *>(kp);
        k[t][0] = w.x, k[t][1] = w.y;
      }
    }
    ks = reinterpret_cast<const uint32_t *>(kt + 16 * HD)[r * NB + (E == 2 ? q : q >> 1)];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = reinterpret_cast<const u32x4_t *>(vt)[e * 64 + lane];
    vs = *reinterpret_cast<const u32x4_t *>(vt + 16 * HD + (q * NB + (lane & 15) * NB / 16) * 16);
  }
  // step i of the scores of keys 16 t ..: values q HD / 4 + 8 i .. of key r
  __device__ __forceinline__ fh8 key(int t, int i, uint32_t ones) const {
    const fh2 s2 = as_fh2(ks);
    const fh2 s = t ? fh2{s2.y, s2.y} : fh2{s2.x, s2.x}, s15 = scale15(s);
    const uint32_t w = k[t][i];
    return as_fh8(kv4_pair<0>(w, s, s15, ones), kv4_pair<1>(w, s, s15, ones), kv4_pair<2>(w, s, s15, ones),
                  kv4_pair<3>(w, s, s15, ones));
  }
  // value 4 E x + 4 e + I of the lane's eight keys
  template <int I>
  __device__ __forceinline__ fh8 val(int e, uint32_t ones) const {
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const fh2 s = as_fh2(vs[j]);
      o[j] = kv4_pair<I>(v[e][j], s, scale15(s), ones);
    }
    return as_fh8(o[0], o[1], o[2], o[3]);
  }
  __device__ __forceinline__ void hide(uint32_t m) {
#pragma unroll
    for (int j = 0; j < 4; j++)
      vs[j] &= (m >> (2 * j) & 1u ? 0u : 0xffffu) | (m >> (2 * j + 1) & 1u ? 0u : 0xffff0000u);
  }
  static constexpr bool kInf = false;  // every value is finite or NaN
  static constexpr int kOcc = 4;  // waves per SIMD
};

// Tiles of fp16 rows [position][kv_dim]; positions past `last` are read as `last`.
template <int HD>
struct TileF16 {
  static constexpr int E = HD / 64;
  u32x4_t k[2][2 * E];
  uint32_t v[8][2 * E];
  __device__ __forceinline__ void load(const uint8_t *K, const uint8_t *V, int64_t stride, int64_t tile, int last,
                                       int lane) {
    const int r = lane & 15, q = lane >> 4;
    const int64_t p0 = tile * kKv4Tile;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const int64_t p = p0 + 16 * t + r < last ? p0 + 16 * t + r : last;
      const u32x4_t *kp = reinterpret_cast<const u32x4_t *>(K + p * stride + q * (HD / 2));
#pragma unroll
      for (int i = 0; i < 2 * E; i++) k[t][i] = kp[i];
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int64_t at = p0 + 16 * (j >> 2) + 4 * q + (j & 3), p = at < last ? at : last;
      const uint8_t *vp = V + p * stride + r * (HD / 8);
      if constexpr (E == 2) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t *>(vp);
        v[j][0] = w.x, v[j][1] = w.y, v[j][2] = w.z, v[j][3] = w.w;
      } else {
        const u32x2_t w = *reinterpret_cast<const u32x2_t *>(vp);
        v[j][0] = w.x, v[j][1] = w.y;
      }
    }
  }
  __device__ __forceinline__ fh8 key(int t, int i, uint32_t) const { return __builtin_bit_cast(fh8, k[t][i]); }
  template <int I>
  __device__ __forceinline__ fh8 val(int e, uint32_t) const {
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
      o[j] = __builtin_amdgcn_perm(v[2 * j + 1][2 * e + I / 2], v[2 * j][2 * e + I / 2], I & 1 ? 0x07060302u : 0x05040100u);
    return as_fh8(o[0], o[1], o[2], o[3]);
  }
  __device__ __forceinline__ void hide(uint32_t m) {
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
      for (int i = 0; i < 2 * E; i++) v[j][i] = m >> j & 1u ? 0u : v[j][i];
  }
  static constexpr bool kInf = true;
  static constexpr int kOcc = HD == 64 ? 3 : 2;
};

// The runs of a launch's rows: row t's begin at off[t], of per[t] tiles each.
struct SpanRuns {
  int off[kKv4Rows + 1], per[kKv4Rows];
  int most;  // of a row
};

__device__ __forceinline__ float lane_xor1(float v) {
  return __builtin_bit_cast(float, dpp32<0xB1>(__builtin_bit_cast(uint32_t, v)));
}
// hi + lo of neighbouring lanes; past an infinity the low part's product with it means nothing.
template <bool INF>
__device__ __forceinline__ float join_parts(float v, bool low) {
  const float o = lane_xor1(v);
  if constexpr (INF) {
    const float hi = low ? o : v;
    return __builtin_isfinite(hi) ? v + o : hi;
  }
  return v + o;
}

typedef float f4a4 __attribute__((ext_vector_type(4), aligned(4)));  // at any float's address

// A row's outputs lie in LDS and in the runs' records as the matrix cores leave them: values 16 d + 4 kq + e, for
// value HD / 16 (4 kq + e) + d of the head. Four of them to their places in the head's row.
template <int HD>
__device__ __forceinline__ void span_store(float *o, int four, sf4 v) {
#pragma unroll
  for (int e = 0; e < 4; e++) o[HD / 16 * (4 * (four & 3) + e) + (four >> 2)] = v[e];
}

template <int HD, class Tile>
__global__ __launch_bounds__(64 * kSpWaves, Tile::kOcc) void span_decode_kernel(const float *__restrict__ q, int H, int G,
                                                                       KvCache c, Span s, KvRows R, SpanRuns U,
                                                                       float scale, float *__restrict__ part,
                                                                       float *__restrict__ out) {
  constexpr int NK = HD / 32, ND = HD / 16, E = HD / 64, W = kSpWaves;
  __shared__ sf4 so[W][8][HD / 4 + 4];  // a head's rows 16 floats past a multiple of the banks
  __shared__ float sm[W][8], sc2[8];
  __shared__ double sl[W][8];
  __shared__ fh8 qs[NK][64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kq = lane >> 4;
  const int kvh = blockIdx.x, run = blockIdx.y, cb = blockIdx.z;
  const int t = __builtin_amdgcn_readfirstlane(
      __popcll(__ballot(lane < R.n && U.off[lane < R.n ? lane : 0] <= run)) - 1);
  const int runs = U.off[t + 1] - U.off[t], mine = run - U.off[t], per = U.per[t];
  const int p = R.position(t), first = s.first(p), lead = s.lead(p);
  const SpanTiles tl(s, p);
  const int i0 = mine * per, i1 = i0 + per < tl.n ? i0 + per : tl.n;
  const uint8_t *K, *V;
  int64_t stride = 0;
  if constexpr (Tile::kInf) {
    stride = (int64_t)c.KH * HD * 2;
    K = c.K + (int64_t)R.slot_of(t) * c.slot_bytes + kvh * (HD * 2);
    V = c.V + (int64_t)R.slot_of(t) * c.slot_bytes + kvh * (HD * 2);
  } else {
    const int64_t head = (int64_t)R.slot_of(t) * c.slot_bytes + (int64_t)kvh * ((c.positions + 31) / 32) * (18 * HD);
    K = c.K + head;
    V = c.V + head;
  }
  constexpr int NT = 2;  // tiles in registers: two or three loaded ahead were no faster, and cost a wave per SIMD
  Tile T[NT];
  int i = i0 + wv;
#pragma unroll
  for (int a = 0; a < NT - 1; a++)
    if (i + a * W < i1) T[a].load(K, V, stride, tl.tile(i + a * W), p, lane);
  // the query's parts: head cb * 8 + col / 2, part col % 2, values kq HD / 4 + 8 step + 0..7. A wave makes the parts of
  // the steps wv, wv + W, ..; all read them from LDS.
  const bool low = col & 1;
  const int g = cb * 8 + (col >> 1) < G ? cb * 8 + (col >> 1) : G - 1;
  const uint32_t ones = fp16_ones();
  float c2;
  {
    const float *qp = q + ((int64_t)t * H + kvh * G + g) * HD + kq * (HD / 4);
    sf4 x[HD / 16];
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < HD / 16; e++) x[e] = *reinterpret_cast<const f4a4 *>(qp + 4 * e);
#pragma unroll
    for (int e = 0; e < HD / 16; e++)
      m = fmaxf(m, fmaxf(fmaxf(fabsf(x[e].x), fabsf(x[e].y)), fmaxf(fabsf(x[e].z), fabsf(x[e].w))));
    if (__any(m == INFINITY)) {  // an infinity is all in its high part, and takes no part in the scale
      m = 0.f;
#pragma unroll
      for (int e = 0; e < HD / 16; e++)
#pragma unroll
        for (int j = 0; j < 4; j++) m = fabsf(x[e][j]) < INFINITY ? fmaxf(m, fabsf(x[e][j])) : m;
    }
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    float f, inv;
    unit_scale(m, f, inv);
    // scores in units of log2: c2 > 0 (a negative scale negates the query)
    c2 = fmaxf(fabsf(scale) * 1.4426950408889634f * inv, 1.1754944e-38f);
    f = scale < 0.f ? -f : f;
    if (scale != scale) c2 = scale;
#pragma unroll
    for (int k = 0; k < NK; k++) {
      if (k % W != wv) continue;  // uniform
      fh8 b;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float X = x[2 * k + e / 4][e % 4] * f;
        const _Float16 a = (_Float16)X;
        b[e] = low ? (_Float16)(__builtin_isinf(X) ? 0.f : X - (float)a) : a;
      }
      qs[k][lane] = b;
    }
  }
  __syncthreads();
  fh8 qb[NK];
#pragma unroll
  for (int k = 0; k < NK; k++) qb[k] = qs[k][lane];
  sf4 O[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) O[d] = sf4{0.f, 0.f, 0.f, 0.f};
  float M = -INFINITY, top = -INFINITY;  // the running maximum, and what raises it
  const float past = kSpPast / c2;
  double L = 0.0;
  auto step = [&](Tile &A, int64_t tile) __attribute__((always_inline)) {
    const int p0 = (int)tile * kKv4Tile;
    sf4 S[2];
#pragma unroll
    for (int t2 = 0; t2 < 2; t2++) {
      S[t2] = sf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NK; k++)
        S[t2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A.key(t2, k, ones), qb[k], S[t2], 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; e++) S[t2][e] = join_parts<Tile::kInf>(S[t2][e], low);
    }
    if (!(p0 + 31 <= p && (p0 >= first || p0 + 31 < lead))) {  // uniform: some position is not seen
      asm volatile("");  // a branch, not selects in every tile
      uint32_t hid = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int at = p0 + 16 * (j >> 2) + 4 * kq + (j & 3);
        const bool no = (at > p) | ((at >= lead) & (at < first));
        hid |= (uint32_t)no << j;
        S[j >> 2][j & 3] = no ? -INFINITY : S[j >> 2][j & 3];
      }
      A.hide(hid);
    }
    float mt = fmaxf(fmaxf(fmaxf(S[0][0], S[0][1]), fmaxf(S[0][2], S[0][3])),
                     fmaxf(fmaxf(S[1][0], S[1][1]), fmaxf(S[1][2], S[1][3])));
    if (__any(mt > top)) {
      mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
      mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
      const bool up = mt > top;
      const float al = up ? __builtin_amdgcn_exp2f((M - mt) * c2) : 1.f;
      L *= (double)al;
#pragma unroll
      for (int d = 0; d < ND; d++) O[d] *= al;
      M = up ? mt : M;
      top = M + past;
    }
    const float Mu = M == -INFINITY ? 0.f : M;  // no key of this row yet: every score is -inf
    uint32_t pb[4];
    float ts[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float P0 = __builtin_amdgcn_exp2f((S[j >> 1][2 * (j & 1)] - Mu) * c2);
      const float P1 = __builtin_amdgcn_exp2f((S[j >> 1][2 * (j & 1) + 1] - Mu) * c2);
      ts[0] += P0;
      ts[1] += P1;
      const float Q0 = P0 * kSpUp, Q1 = P1 * kSpUp;
      uint32_t hi = __builtin_bit_cast(uint32_t, fh2{(_Float16)Q0, (_Float16)Q1});
      asm("" : "+v"(hi));  // rounded once: the compiler made the halves again for the low parts
      const fh2 lo = {(_Float16)(Q0 - half_lo(hi)), (_Float16)(Q1 - half_hi(hi))};
      pb[j] = low ? __builtin_bit_cast(uint32_t, lo) : hi;
    }
    const fh8 pv = as_fh8(pb[0], pb[1], pb[2], pb[3]);
    L += (double)(ts[0] + ts[1]);
#pragma unroll
    for (int e = 0; e < E; e++) {
      O[4 * e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A.template val<0>(e, ones), pv, O[4 * e], 0, 0, 0);
      O[4 * e + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A.template val<1>(e, ones), pv, O[4 * e + 1], 0, 0, 0);
      O[4 * e + 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A.template val<2>(e, ones), pv, O[4 * e + 2], 0, 0, 0);
      O[4 * e + 3] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A.template val<3>(e, ones), pv, O[4 * e + 3], 0, 0, 0);
    }
  };
#pragma unroll 1
  while (i < i1) {
#pragma unroll
    for (int a = 0; a < NT; a++) {
      if (i + (NT - 1) * W < i1) T[(a + NT - 1) % NT].load(K, V, stride, tl.tile(i + (NT - 1) * W), p, lane);
      step(T[a], tl.tile(i));
      i += W;
      if (i >= i1) break;
    }
  }
  // the waves' sums under their largest maximum; of two neighbouring lanes one writes the even blocks, one the odd
  L += __shfl_xor(L, 16, 64);
  L += __shfl_xor(L, 32, 64);
#pragma unroll
  for (int d = 0; d < ND; d += 2) {
    sf4 o;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float a = join_parts<Tile::kInf>(O[d][e], low), b = join_parts<Tile::kInf>(O[d + 1][e], low);
      o[e] = low ? b : a;
    }
    so[wv][col >> 1][4 * (d + (int)low) + kq] = o;
  }
  if (!low && kq == 0) {
    sm[wv][col >> 1] = M;
    sl[wv][col >> 1] = L;
    sc2[col >> 1] = c2;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * HD; e += 64 * W) {
    const int gg = e / (HD / 4), four = e % (HD / 4), h = cb * 8 + gg;
    if (h >= G) break;
    float m = sm[0][gg];
#pragma unroll
    for (int w = 1; w < W; w++) m = fmaxf(m, sm[w][gg]);
    sf4 o = {0.f, 0.f, 0.f, 0.f};
    double l = 0.0;
#pragma unroll
    for (int w = 0; w < W; w++) {
      const float f = __builtin_amdgcn_exp2f((sm[w][gg] - m) * sc2[gg]);
      o += so[w][gg][four] * f;
      l += sl[w][gg] * (double)f;
    }
    const int64_t row = (int64_t)t * H + kvh * G + h;
    if (runs == 1) {
      const double r = (1.0 / kSpUp) / l;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = (float)((double)o[j] * r);
      span_store<HD>(out + row * HD, four, o);
    } else {
      float *rec = part + (row * U.most + mine) * (HD + 4);
      *reinterpret_cast<sf4 *>(rec + 4 * four) = o;
      if (four == 0) {
        rec[HD] = m;
        rec[HD + 1] = sc2[gg];
        *reinterpret_cast<double *>(rec + HD + 2) = l;
      }
    }
  }
}

// Rows of more than one run: the runs' sums under their largest maximum. A workgroup per (row, head): the
// runs' factors once, into LDS; then HD / 4 threads to a record, the records over the groups in turn, each group's
// sum in order and the groups' in order.
template <int HD>
__global__ __launch_bounds__(256) void span_join_kernel(const float *__restrict__ part, int H, SpanRuns U,
                                                        float *__restrict__ out) {
  constexpr int TH = HD / 4, NG = 256 / TH;
  __shared__ float f[kSpRuns], sm[4];
  __shared__ double sl[4];
  __shared__ sf4 so[NG][TH];
  const int h = blockIdx.x, t = blockIdx.y, tid = threadIdx.x;
  const int n = U.off[t + 1] - U.off[t];
  if (n == 1) return;
  const int64_t row = (int64_t)t * H + h;
  const float *rec = part + row * U.most * (HD + 4);
  static_assert(kSpRuns == 256, "a thread per run");
  const float *mine = rec + (tid < n ? tid : n - 1) * (HD + 4);
  const float m1 = mine[HD], c2 = mine[HD + 1];
  const double l1 = *reinterpret_cast<const double *>(mine + HD + 2);
  float m = wave_max_f(m1);
  if ((tid & 63) == 0) sm[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const float f1 = tid < n ? __builtin_amdgcn_exp2f((m1 - m) * c2) : 0.f;
  f[tid] = f1;
  const double l = wave_sum_d(tid < n ? l1 * (double)f1 : 0.0);
  if ((tid & 63) == 0) sl[tid >> 6] = l;
  __syncthreads();
  const int g = tid / TH, x = tid % TH;
  sf4 o = {0.f, 0.f, 0.f, 0.f};
  for (int i = g; i < n; i += 4 * NG) {
    sf4 v[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int r = i + k * NG < n ? i + k * NG : i;
      v[k] = *reinterpret_cast<const sf4 *>(rec + r * (HD + 4) + 4 * x);
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (i + k * NG < n) o += v[k] * f[i + k * NG];
  }
  so[g][x] = o;
  __syncthreads();
  if (tid < TH) {
    sf4 s = so[0][tid];
#pragma unroll
    for (int k = 1; k < NG; k++) s += so[k][tid];
    const double r = (1.0 / kSpUp) / ((sl[0] + sl[1]) + (sl[2] + sl[3]));
    sf4 w;
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = (float)((double)s[e] * r);
    span_store<HD>(out + row * HD, tid, w);
  }
}

// Tiles of each run of a row of n tiles (a rule on the row alone). Up to 16 tiles one run, and no second launch
// (32 heads of 64, 7 rows at 333: 6.0 us, two runs 9.2). More: two tiles a wave, where a lone row is short of waves, to
// four from 256 tiles on, where a run's fixed work (the query's parts, the sums through LDS, its record) weighs more
// (64 heads of 128: one row after 4,000 10.1 us, four tiles a wave 11.7; 32 rows of up to 9,001 62 us, two
// tiles 69, one 89). And no more runs than give every CU two workgroups.
static int span_per(int n, int units) {
  if (n <= 16) return n;
  int fill = (512 + units - 1) / units;
  fill = fill > kSpRuns ? kSpRuns : fill;
  int per = (n + 15) / 16;
  per = per < 2 * kSpWaves ? 2 * kSpWaves : per > 4 * kSpWaves ? 4 * kSpWaves : per;
  return per < (n + fill - 1) / fill ? (n + fill - 1) / fill : per;
}

static bool span_tiled(const KvCache &c) {
  return c.bits == 4 || ((c.HD == 64 || c.HD == 128) && ((uintptr_t)c.K & 15) == 0 && ((uintptr_t)c.V & 15) == 0);
}
static bool span_decodes(const KvCache &c, const KvRows &R) { return span_tiled(c) && (R.batch || R.n < 16); }

static SpanRuns span_plan(const KvCache &c, int H, const Span &s, const KvRows &R) {
  SpanRuns U = {};
  const int units = c.KH * ((H / c.KH + 7) / 8);
  for (int t = 0; t < R.n; t++) {
    const int n = SpanTiles(s, R.position(t)).n;
    U.per[t] = span_per(n, units);
    const int r = (n + U.per[t] - 1) / U.per[t];
    U.off[t + 1] = U.off[t] + r;
    U.most = r > U.most ? r : U.most;
  }
  return U;
}

template <int HD, class Tile>
static hipError_t span_decode_launch(const float *q, int H, const KvCache &c, const Span &s, const KvRows &R, float scale,
                                     float *part, float *out, hipStream_t st) {
  const SpanRuns U = span_plan(c, H, s, R);
  const int G = H / c.KH;
  hipLaunchKernelGGL((span_decode_kernel<HD, Tile>), dim3(c.KH, U.off[R.n], (G + 7) / 8), dim3(64 * kSpWaves), 0, st, q,
                     H, G, c, s, R, U, scale, part, out);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || U.most == 1) return e;
  hipLaunchKernelGGL(span_join_kernel<HD>, dim3(H, R.n), dim3(256), 0, st, part, H, U, out);
  return hipGetLastError();
}

static int64_t span_max_n(const Span &s, const KvRows &R) {
  int64_t m = 0;
  if (!R.batch) return s.seen(R.pos0 + R.n - 1);
  for (int i = 0; i < R.n; i++) m = s.seen(R.pos[i]) > m ? s.seen(R.pos[i]) : m;
  return m;
}

int64_t attention_span_scratch_floats(const KvCache &c, int H, const Span &s, const KvRows &R) {
  if (R.n <= 0) return 0;
  if (span_decodes(c, R)) {
    const SpanRuns U = span_plan(c, H, s, R);
    return U.most > 1 ? (int64_t)R.n * H * U.most * (c.HD + 4) : 0;
  }
  return (int64_t)R.n * H * span_max_n(s, R);
}

hipError_t attention_span_launch(const float *q, int H, const KvCache &c, const Span &s, const KvRows &R, float scale,
                                 float *scratch, float *out, hipStream_t st) {
  if (R.n <= 0) return hipSuccess;
  if (span_decodes(c, R)) {
    if (c.bits == 4)
      return c.HD == 64 ? span_decode_launch<64, TileKv4<64>>(q, H, c, s, R, scale, scratch, out, st)
                        : span_decode_launch<128, TileKv4<128>>(q, H, c, s, R, scale, scratch, out, st);
    return c.HD == 64 ? span_decode_launch<64, TileF16<64>>(q, H, c, s, R, scale, scratch, out, st)
                      : span_decode_launch<128, TileF16<128>>(q, H, c, s, R, scale, scratch, out, st);
  }
  hipLaunchKernelGGL(span_rows_kernel, dim3(H, R.n), dim3(256), 0, st, q, H, c, s, R, scale, scratch, span_max_n(s, R),
                     out);
  return hipGetLastError();
}

}  // namespace wl
