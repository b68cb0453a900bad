// wl_attention_span.hip - attention over 4-bit caches (wl_kv4.h), and over fp16 caches with a sliding
// window and first tokens that stay visible (Attention, src/Transformer.cs:351-393, over the
// positions Span names).
#include "wl_attention_span.h"

#include "wl_fmma_codec.h"

#include <type_traits>

#pragma clang fp contract(off)

namespace wl {

struct F16Rows {
  const uint16_t *K, *V;
  int64_t kv_dim;
  __device__ float key(int64_t j, int i) const { return (float)__builtin_bit_cast(_Float16, K[j * kv_dim + i]); }
  __device__ float val(int64_t j, int i) const { return (float)__builtin_bit_cast(_Float16, V[j * kv_dim + i]); }
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

// fp16 caches of other head dims than 64 and 128: one workgroup per (head, row): scores, their maximum,
// exponentials, sums.
__device__ void span_row(const F16Rows &c, const float *qp, int HD, int p, const Span &s, float scale, float *sp, float *op) {
  __shared__ double shd[4];
  __shared__ float shf[4];
  const int first = s.first(p), lead = s.lead(p), n = s.seen(p);
  float mx = -INFINITY;
  for (unsigned i = threadIdx.x; i < (unsigned)n; i += 256) {  // a step past the last position may pass 2^31
    const int64_t j = i < (unsigned)lead ? i : first + (i - lead);
    float d = 0.f;
    for (int e = 0; e < HD; e++) d += qp[e] * c.key(j, e);
    d *= scale;
    sp[i] = d;
    mx = fmaxf(mx, d);
  }
  mx = span_max(mx, shf);
  double sum = 0.0;
  for (unsigned i = threadIdx.x; i < (unsigned)n; i += 256) {
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
                                                        int t0, float scale, float *__restrict__ scores, int64_t max_n,
                                                        float *__restrict__ out) {
  const int h = blockIdx.x, t = t0 + blockIdx.y, kvh = h / (H / c.KH), HD = c.HD;
  const int64_t row = ((int64_t)t * H + h), off = (int64_t)R.slot_of(t) * c.slot_bytes;
  const float *qp = q + row * HD;
  const int64_t head = off + (int64_t)kvh * HD * 2;
  span_row(F16Rows{(const uint16_t *)(c.K + head), (const uint16_t *)(c.V + head), (int64_t)c.KH * HD}, qp, HD,
           R.position(t), s, scale,
           scores + ((int64_t)blockIdx.y * H + h) * max_n, out + row * HD);
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
//
// What bounds it: a 4-bit position of a head is 2.25 HD bytes for 4 HD G products. One row after 131,000 (8B, 151 MB) takes
// 32.2 us and the join 4.7, against 24.8 for reading the bytes: the loads wait 44% of the wave cycles and the unpacking
// keeps the VALU 57% busy. 32 rows of up to 9,001 (70B, 249 MB): 59.3 us, VALU 69%, matrix cores 9%; short contexts are
// two launches' latency (70B after 4,000: 6.3 and 3.8 us). Measured and not kept: the last workgroup of a row joining its
// runs (with fences 770 us for the 32 rows; with device-scope stores 66.9 against 61.6, and 41.7 against 35.5 for the long
// row), records loaded ahead in the join (62.5 -> 66), eight waves a workgroup.
typedef float sf4 __attribute__((ext_vector_type(4)));
// A running maximum is raised only by scores more than 2^6 past it, so nearly never after a wave's first tile: the
// exponentials reach 2^6, and 2^8 of them are fp16 parts (22 bits down to 2^-22 of the row's largest, 2^-33 of it below).
constexpr float kSpUp = 0x1p8f, kSpPast = 6.f;
// In the scores' units: finite where those are the smallest there are, so that a lane without a key yet keeps -inf as what
// raises its maximum.
__device__ __forceinline__ float past_of(float c2) { return fminf(kSpPast / c2, 3.4028235e38f); }
constexpr int kSpWaves = 4;
constexpr int kSpRuns = 256;      // runs of a row at most

// Units that hold n positions; n up to 2^31 - 1, which no rounding up may pass.
__host__ __device__ constexpr int units_of(int n, int unit) { return n / unit + (n % unit != 0); }

// The tiles a row at p reads, in order: those of the first tokens, then the window's.
struct SpanTiles {
  int lead, from, n;
  __host__ __device__ SpanTiles(const Span &s, int p) {
    lead = units_of(s.lead(p), kKv4Tile);
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

// Two probabilities, times kSpUp, as their fp16 parts.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t &hi, uint32_t &lo) {
  hi = __builtin_bit_cast(uint32_t, fh2{(_Float16)__builtin_fmaf(a, kSpUp, 0.f), (_Float16)__builtin_fmaf(b, kSpUp, 0.f)});
  asm("" : "+v"(hi));  // rounded once: the compiler made the halves again for the low parts
  lo = __builtin_bit_cast(uint32_t, fh2{(_Float16)__builtin_fmaf(a, kSpUp, -half_lo(hi)),
                                        (_Float16)__builtin_fmaf(b, kSpUp, -half_hi(hi))});  // exact but for their rounding
}

// Tiles of 4-bit caches. hide(m): bit j set where key j of the lane (keys 16 (j / 4) + 4 kq + j % 4) is not seen:
// its values become zeros.
template <int HD>
struct TileKv4 {
  static constexpr int E = HD / 64, NB = HD / 32;
  u32x4_t v[E], vs;
  uint32_t k[2][4 * E / 2], ks;
  // nontemporal: a step reads a cache once (8B after 131,000 positions 39.0 -> 35.9 us)
  __device__ __forceinline__ void load(const uint8_t *K, const uint8_t *V, int64_t, int64_t tile, int, int lane) {
    const uint8_t *kt = K + tile * (18 * HD), *vt = V + tile * (18 * HD);
    const int r = lane & 15, q = lane >> 4;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const uint8_t *kp = kt + (16 * t + r) * (HD / 2) + q * (HD / 8);
      if constexpr (E == 2) {
        const u32x4_t w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(kp));
        k[t][0] = w.x, k[t][1] = w.y, k[t][2] = w.z, k[t][3] = w.w;
      } else {
        const u32x2_t w = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t *>(kp));
        k[t][0] = w.x, k[t][1] = w.y;
      }
    }
    ks = reinterpret_cast<const uint32_t *>(kt + 16 * HD)[r * NB + (E == 2 ? q : q >> 1)];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(vt) + e * 64 + lane);
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

// What sums under the maximum M weigh under a larger one. Scores of -inf alone leave M at -inf and sums of zeros (or NaN, from
// a NaN score): a factor of zero, also where no other sums have a maximum, and 0 / 0 is such a row's output.
__device__ __forceinline__ float weight_of(float M, float m, float c2) {
  return M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((M - m) * c2);
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
  const float past = past_of(c2);
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
      uint32_t hi, lo;
      split_pair(P0, P1, hi, lo);
      pb[j] = low ? lo : hi;
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
      const float f = weight_of(sm[w][gg], m, sc2[gg]);
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
  const float f1 = tid < n ? weight_of(m1, m, c2) : 0.f;
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
// (32 heads of 64, 7 rows at 333: 6.0 us, two runs 9.2). Up to 160 tiles (5,120 positions) as many runs as give every CU a
// workgroup, of four tiles at least, a tile a wave (64 heads of 128 after 4,000: 9.7 us, 16 tiles a run 11.7; fp16, a
// window of 4,096: 11.4 us, eight tiles 13.0). More: four tiles a wave, where a run's fixed work (the query's parts, the
// sums through LDS, its record) weighs more than a lone row's waves (32 rows of up to 9,001 65 us, two tiles a wave
// 73, one 93; 8 rows of 8B 21.0, 22.3, 28.4), and no more runs than give every CU two workgroups. A lone row of 8 KV heads
// pays for it between 5,120 and 10,000 positions: 11.9 us at 5,200 and 12.1 at 8,000, two tiles a wave 10.1-10.8; at
// 12,000 and 16,000 12.2 and 12.4, two tiles 12.6 and 12.7.
static int span_per(int n, int units) {
  if (n <= 16) return n;
  const int64_t all = (int64_t)n * units;
  int64_t per = 4 * kSpWaves, one = (all + 255) / 256, two = (all + 511) / 512;
  if (n <= 160) per = one < kSpWaves ? kSpWaves : one < per ? one : per;
  per = per < two ? two : per;
  const int most = (n + kSpRuns - 1) / kSpRuns;
  return per < most ? most : (int)per;
}

// ------------------------------------------------------------------------------- prompts
// Rows of 16 tokens and more on v_mfma_f32_32x32x16_f16 (head dims 64 and 128), the products and parts of
// wl_attention.hip: S^T = K Q^T, a column per (token, query head of the KV head) in the order token * G + head,
// 32 columns a wave, 64 keys a step, staged in LDS for the workgroup's four waves as fp16 rows of keys and, transposed,
// rows of values in the order in which the scores' registers meet them. Two stages: a step's keys are unpacked while the
// step before is multiplied, with one barrier between steps. The exponential's argument is the score's difference from the
// running maximum, times the scale, as above: scores of any size keep their largest near 1.
//
// What bounds it: both products twice (two parts), 206 GFLOP for 2,048 tokens of the 8B model's 32 heads after 2,048, in
// 205-214 us on the cards measured: 960 to 1,005 TFLOP/s, where a library's product of 4,096 x 4,096 matrices reaches 1,100. The matrix cores are busy 40%
// of the cycles and the VALU 48%, with two waves a SIMD that seldom overlap them; 254 registers leave no room for a second
// tile of scores, and kernels that kept one (the scores of 32 keys beside the exponentials of the 32 before) spilled and
// took 297-308 us; the next step's unpacking among a chain's products, 225-245 us, for the same reason. Rows cut in two and more chunks where whole rows fill the CUs: 282 us; 2 and 4 chunks for a window of
// 1,500 rows, whose 376 workgroups are one and two a CU: 114 and 131 us against 102.
constexpr int kTlK = 64, kTlW = 4, kTlCols = 32 * kTlW;
typedef float sf16 __attribute__((ext_vector_type(16)));

// The steps of a workgroup whose rows are t0 .. t1 at pos0: those of the first tokens, then the windows'.
struct SpanSteps {
  int lead, from, n;
  __host__ __device__ SpanSteps(const Span &s, int first_row, int last_row) {
    lead = units_of(s.lead(last_row), kTlK);
    from = s.first(first_row) / kTlK;
    from = from < lead ? lead : from;
    n = last_row / kTlK >= from ? lead + last_row / kTlK - from + 1 : lead;
  }
  __host__ __device__ int at(int i) const { return (i < lead ? i : from + (i - lead)) * kTlK; }
};

struct TilesArgs {
  Span s;
  int T, pos0, G, KH, nz, chunks, steps;  // nz workgroups of columns a KV head, chunks of `steps` steps each
  __host__ __device__ int row0(int z) const { return pos0 + (int)((int64_t)z * kTlCols / G); }
  __host__ __device__ int row1(int z) const {
    const int64_t last = ((int64_t)z * kTlCols + kTlCols - 1) / G;
    return pos0 + (int)(last < T - 1 ? last : T - 1);
  }
};

// LDS place (halves) of value row `dim`: rows of 128 bytes, the 16-byte pieces of a row in an order of the row's own, so
// that reads of 32 rows and writes of every eighth row both meet all banks.
__device__ __forceinline__ int val_at(int dim, int slot) {
  return dim * kTlK + ((((slot >> 3) ^ dim ^ (dim >> 3)) & 7) << 3 | (slot & 7));
}
// Bits 15 and 31 set where a half of w is an infinity or NaN: its exponent's ones carry.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return (w & 0x7c007c00u) + 0x04000400u; }
constexpr uint32_t kNotFinite = 0x80008000u;
// Keeps a value from being computed ahead of a loop into a register of its own.
__device__ __forceinline__ int here(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// A step's keys and values of one KV head from 4-bit tiles, a block of 32 key values and one of 4 x 8 values a thread.
template <int HD>
struct StageKv4 {
  static constexpr int NB = HD / 32, E = HD / 64, UN = 64 * NB;  // units of 16 bytes of each
  static constexpr bool kInf = false, kPrio = false;
  u32x4_t k, v, vs;
  uint16_t ks;
  int kkey, kblk, vt, vl, ve, vblk;
  const uint8_t *K, *V;
  bool doK, doV;
  __device__ void init(const KvCache &c, int kvh, int tid) {
    const int64_t head = (int64_t)kvh * ((c.positions + 31) / 32) * (18 * HD);
    K = c.K + head;
    V = c.V + head;
    doK = HD == 128 || tid < UN;
    doV = HD == 128 || tid >= UN;
    const int ku = tid & (UN - 1);
    kkey = ku / NB;
    kblk = ku % NB;
    vt = ku / (UN / 2);  // tile of the step
    ve = ku / 64 % E;
    vl = ku % 64;
    vblk = (vl & 15) * E / 8;
  }
  __device__ __forceinline__ void fetch(int j0, int last) {
    const int lt = last / 32;
    if (doK) {
      const int tile = (j0 + kkey) / 32 < lt ? (j0 + kkey) / 32 : lt, r = kkey & 31;
      const uint8_t *t = K + (int64_t)tile * (18 * HD);
      k = *reinterpret_cast<const u32x4_t *>(t + r * (HD / 2) + 16 * kblk);
      ks = reinterpret_cast<const uint16_t *>(t + 16 * HD)[kv4_key_scale(r, kblk, HD)];
    }
    if (doV) {
      const int tile = j0 / 32 + vt < lt ? j0 / 32 + vt : lt;
      const uint8_t *t = V + (int64_t)tile * (18 * HD);
      v = reinterpret_cast<const u32x4_t *>(t)[ve * 64 + vl];
      vs = *reinterpret_cast<const u32x4_t *>(t + 16 * HD + ((vl >> 4) * NB + vblk) * 16);
    }
  }
  // Into LDS; true where a value of a position up to `last` is NaN (it becomes zero there).
  __device__ __forceinline__ bool stage(uint16_t *lk, uint16_t *lv, int j0, int last, uint32_t ones, bool &) {
    constexpr int KS = HD + 8;
    if (doK) {
      const _Float16 h = __builtin_bit_cast(_Float16, ks);
      const fh2 sc = {h, h}, s15 = scale15(sc);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t w = k[i];
        *reinterpret_cast<u32x4_t *>(lk + kkey * KS + 32 * kblk + 8 * i) =
            u32x4_t{kv4_pair<0>(w, sc, s15, ones), kv4_pair<1>(w, sc, s15, ones), kv4_pair<2>(w, sc, s15, ones),
                    kv4_pair<3>(w, sc, s15, ones)};
      }
    }
    bool bad = false;
    if (doV) {
      const int kq = vl >> 4, dim = 4 * E * (vl & 15) + 4 * ve, p0 = j0 + 32 * vt + 4 * kq;
      u32x4_t sc = vs;
      const uint32_t odd = not_finite(sc.x) | not_finite(sc.y) | not_finite(sc.z) | not_finite(sc.w);
      if (j0 + kTlK - 1 > last || __any(odd & kNotFinite)) {  // uniform over the wave, and rare
        asm volatile("");
#pragma unroll
        for (int j = 0; j < 4; j++) {  // a scale is finite or NaN; past `last` it may be anything
          const int at = p0 + 16 * (j >> 1) + 2 * (j & 1);
          sc[j] &= (at > last ? 0u : 0xffffu) | (at + 1 > last ? 0u : 0xffff0000u);
          const bool lo = (sc[j] & 0x7c00u) == 0x7c00u, hi = (sc[j] & 0x7c000000u) == 0x7c000000u;
          bad |= lo | hi;
          sc[j] = lo ? sc[j] & 0xffff0000u : sc[j];
          sc[j] = hi ? sc[j] & 0xffffu : sc[j];
        }
      }
      // val_at(dim + i, slot + 16 h): dim is a multiple of 4
      const int base = here(val_at(dim, 32 * vt + 8 * (kq & 1) + 4 * (kq >> 1)));
      fh2 s2[4], s15[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        s2[j] = as_fh2(sc[j]);
        s15[j] = scale15(s2[j]);
      }
      auto put = [&](auto I) __attribute__((always_inline)) {
        constexpr int i = decltype(I)::value;
#pragma unroll
        for (int h = 0; h < 2; h++)
          *reinterpret_cast<u32x2_t *>(lv + ((base + i * kTlK) ^ (i ^ 2 * h) << 3)) =
              u32x2_t{kv4_pair<i>(v[2 * h], s2[2 * h], s15[2 * h], ones),
                      kv4_pair<i>(v[2 * h + 1], s2[2 * h + 1], s15[2 * h + 1], ones)};
      };
      put(std::integral_constant<int, 0>());
      put(std::integral_constant<int, 1>());
      put(std::integral_constant<int, 2>());
      put(std::integral_constant<int, 3>());
    }
    return bad;
  }
  // NaN blocks of position p into the outputs of a lane that sees it (block d of its 32-value blocks).
  template <class O>
  __device__ void add_bad(int p, int, O &o) const {
    const uint16_t *sc = reinterpret_cast<const uint16_t *>(V + (int64_t)(p / 32) * (18 * HD) + 16 * HD);
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
      if ((sc[kv4_val_scale(p % 32, d, HD)] & 0x7c00u) == 0x7c00u) o[d] += __builtin_nanf("");
  }
};

// The same from fp16 rows.
template <int HD>
struct StageF16 {
  static constexpr int U = HD / 8, KI = 64 * U / 256;
  static constexpr bool kInf = true;
  // exponentials and the products after them before the other wave's work: a window of 1,500 rows 93.5 -> 88.8 us (with 4-bit
  // tiles, whose staging is the VALU's, 205 -> 211)
  static constexpr bool kPrio = true;
  u32x4_t k[KI], v[4];
  const uint16_t *K, *V;
  int64_t kv_dim;
  int tid, kg, dg;
  __device__ void init(const KvCache &c, int kvh, int t) {
    K = reinterpret_cast<const uint16_t *>(c.K) + kvh * HD;
    V = reinterpret_cast<const uint16_t *>(c.V) + kvh * HD;
    kv_dim = (int64_t)c.KH * HD;
    tid = t;
    dg = t % U;
    kg = t / U;
  }
  __device__ __forceinline__ void fetch(int j0, int last) {
#pragma unroll
    for (int i = 0; i < KI; i++) {
      const int e = tid + 256 * i, row = j0 + e / U < last ? j0 + e / U : last;  // past the end: the last row again, masked
      k[i] = *reinterpret_cast<const u32x4_t *>(K + (int64_t)row * kv_dim + 8 * (e % U));
    }
    if (kg < 16) {
#pragma unroll
      for (int b = 0; b < 4; b++) {
        const int row = j0 + 4 * kg + b < last ? j0 + 4 * kg + b : last;
        v[b] = *reinterpret_cast<const u32x4_t *>(V + (int64_t)row * kv_dim + 8 * dg);
      }
    }
  }
  __device__ static __forceinline__ uint32_t odd(u32x4_t w) {
    return not_finite(w.x) | not_finite(w.y) | not_finite(w.z) | not_finite(w.w);
  }
  __device__ __forceinline__ bool stage(uint16_t *lk, uint16_t *lv, int, int, uint32_t, bool &badk) {
    constexpr int KS = HD + 8;
    bool bad = false;
    uint32_t oddk = 0;
#pragma unroll
    for (int i = 0; i < KI; i++) {
      const int e = tid + 256 * i;
      oddk |= odd(k[i]);
      *reinterpret_cast<u32x4_t *>(lk + (e / U) * KS + 8 * (e % U)) = k[i];
    }
    badk = (oddk & kNotFinite) != 0;
    if (kg < 16) {
      uint32_t oddv = 0;
#pragma unroll
      for (int b = 0; b < 4; b++) oddv |= odd(v[b]);
      bad = (oddv & kNotFinite) != 0;
      if (bad) {
#pragma unroll
        for (int b = 0; b < 4; b++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            v[b][i] = (v[b][i] & 0x7c00u) == 0x7c00u ? v[b][i] & 0xffff0000u : v[b][i];
            v[b][i] = (v[b][i] & 0x7c000000u) == 0x7c000000u ? v[b][i] & 0xffffu : v[b][i];
          }
      }
      // val_at(8 dg + i, slot)
      const int base = here(val_at(8 * dg, 16 * (kg >> 2) + 8 * (kg & 1) + 4 * ((kg >> 1) & 1)));
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t a0 = __builtin_amdgcn_perm(v[1][i], v[0][i], 0x05040100u);
        const uint32_t a1 = __builtin_amdgcn_perm(v[3][i], v[2][i], 0x05040100u);
        const uint32_t b0 = __builtin_amdgcn_perm(v[1][i], v[0][i], 0x07060302u);
        const uint32_t b1 = __builtin_amdgcn_perm(v[3][i], v[2][i], 0x07060302u);
        *reinterpret_cast<u32x2_t *>(lv + ((base + 2 * i * kTlK) ^ 2 * i << 3)) = u32x2_t{a0, a1};
        *reinterpret_cast<u32x2_t *>(lv + ((base + (2 * i + 1) * kTlK) ^ (2 * i + 1) << 3)) = u32x2_t{b0, b1};
      }
    }
    return bad;
  }
  template <class O>
  __device__ void add_bad(int p, int hf, O &o) const {
    const uint16_t *vp = V + (int64_t)p * kv_dim;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const uint16_t w = vp[32 * d + 8 * (i >> 2) + 4 * hf + (i & 3)];
        if ((w & 0x7c00u) == 0x7c00u) o[d][i] += (float)__builtin_bit_cast(_Float16, w);
      }
  }
};

template <int HD, class Stage>
__global__ __launch_bounds__(256, 2) void span_tiles_kernel(const float *__restrict__ q, KvCache c, TilesArgs A,
                                                            float scale, float *__restrict__ part,
                                                            float *__restrict__ out) {
  constexpr int NK = HD / 16, ND = HD / 32, KS = HD + 8;
  __shared__ __attribute__((aligned(16))) uint16_t lk[2][kTlK * KS];
  __shared__ __attribute__((aligned(16))) uint16_t lv[2][HD * kTlK];
  __shared__ int bads[2][2][kTlW];
  const int kvh = blockIdx.x % A.KH, ch = blockIdx.x / A.KH % A.chunks, r = blockIdx.x / A.KH / A.chunks;
  // longest and shortest rows in turn: the workgroups that share a CU (the grid's halves) add up
  const int z = r < (A.nz + 1) / 2 ? A.nz - 1 - r : r - (A.nz + 1) / 2;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hf = lane >> 5, col = lane & 31, G = A.G, H = G * A.KH;
  const int last = A.row1(z);
  const SpanSteps st(A.s, A.row0(z), last);
  const int i0 = ch * A.steps, i1 = i0 + A.steps < st.n ? i0 + A.steps : st.n;
  if (i0 >= i1) return;  // uniform over the workgroup
  const int64_t NC = (int64_t)A.T * G, u = (int64_t)z * kTlCols + 32 * wv + col, uc = u < NC ? u : NC - 1;
  const int t = (int)(uc / G), h = kvh * G + (int)(uc % G);
  const int p = A.pos0 + t, first = A.s.first(p), lead = A.s.lead(p);
  // the wave's rows
  const int64_t w0 = (int64_t)z * kTlCols + 32 * wv;
  const bool idle = w0 >= NC;
  const int pa = A.pos0 + (int)((w0 < NC ? w0 : NC - 1) / G), pb = A.pos0 + (int)((w0 + 31 < NC ? w0 + 31 : NC - 1) / G);
  const int firsta = A.s.first(pa), firstb = A.s.first(pb), leada = A.s.lead(pa), leadb = A.s.lead(pb);

  Stage sg;
  sg.init(c, kvh, tid);
  sg.fetch(st.at(i0), last);
  // the query's parts, in operand order: k = 16 i + 8 hf + 0..7
  fh8 qh[NK], ql[NK];
  float c2;
  {
    const float *qp = q + ((int64_t)t * H + h) * HD + 8 * hf;
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < NK; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float a = fabsf(qp[16 * i + j]);
        m = a < INFINITY ? fmaxf(m, a) : m;
      }
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    float f, inv;
    unit_scale(m, f, inv);
    // scores in units of log2: c2 > 0 (a negative scale negates the query)
    c2 = fmaxf(fabsf(scale) * 1.4426950408889634f * inv, 1.1754944e-38f);
    f = scale < 0.f ? -f : f;
    if (scale != scale) c2 = scale;
#pragma unroll
    for (int i = 0; i < NK; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float X = qp[16 * i + j] * f;
        const _Float16 a = (_Float16)X;
        qh[i][j] = a;
        ql[i][j] = (_Float16)(__builtin_isinf(X) ? 0.f : X - (float)a);
      }
  }
  sf16 O[ND];
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int i = 0; i < 16; i++) O[d][i] = 0.f;
  float M = -INFINITY, top = -INFINITY;  // the running maximum, and what raises it
  const float past = past_of(c2);
  double L = 0.0;
  const uint32_t ones = fp16_ones();
  auto stage = [&](int b, int j0) __attribute__((always_inline)) {
    bool bk = false;
    const bool bv = sg.stage(lk[b], lv[b], j0, last, ones, bk);
    const bool ak = Stage::kInf && __any(bk), av = __any(bv);
    if (lane == 0) {
      bads[b][0][wv] = ak;
      bads[b][1][wv] = av;
    }
  };
  stage(0, st.at(i0));
  if (i0 + 1 < i1) sg.fetch(st.at(i0 + 1), last);
  __syncthreads();
#pragma unroll 1
  for (int i = i0; i < i1; i++) {
    const int b = (i - i0) & 1, j0 = st.at(i);
    const uint16_t *kb = lk[b], *vb = lv[b];
    const bool badk = Stage::kInf && (bads[b][0][0] | bads[b][0][1] | bads[b][0][2] | bads[b][0][3]) != 0;
    const bool badv = (bads[b][1][0] | bads[b][1][1] | bads[b][1][2] | bads[b][1][3]) != 0;
    // uniform over the wave: some row of it sees some key
    const bool on = !idle && j0 <= pb && (j0 + kTlK - 1 >= firsta || j0 < leadb);
    float ts[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 2; s++) {
      if (on) {
        const uint16_t *kp = kb + (32 * s + col) * KS + 8 * hf;
        sf16 S;
#pragma unroll
        for (int e = 0; e < 16; e++) S[e] = 0.f;
#pragma unroll
        for (int k = 0; k < NK; k++)
          S = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const fh8 *>(kp + 16 * k), ql[k], S, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < NK; k++)
          S = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const fh8 *>(kp + 16 * k), qh[k], S, 0, 0, 0);
        if (badk) {  // past an infinity the low parts' product means nothing: there the high parts' alone
          sf16 A;
#pragma unroll
          for (int e = 0; e < 16; e++) A[e] = 0.f;
#pragma unroll
          for (int k = 0; k < NK; k++)
            A = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const fh8 *>(kp + 16 * k), qh[k], A, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 16; e++) S[e] = __builtin_isfinite(A[e]) ? S[e] : A[e];
        }
        const int js = j0 + 32 * s;
        if (!(js + 31 <= pa && (js >= firstb || js + 31 < leada))) {  // uniform: some row does not see every key
          asm volatile("");
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const int at = js + 8 * (e >> 2) + 4 * hf + (e & 3);
            S[e] = (at > p) | ((at >= lead) & (at < first)) ? -INFINITY : S[e];
          }
        }
        if constexpr (Stage::kPrio) __builtin_amdgcn_s_setprio(1);
        float mt = S[0];
#pragma unroll
        for (int e = 1; e < 16; e++) mt = fmaxf(mt, S[e]);
        if (__any(mt > top)) {
          mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
          const bool up = mt > top;
          const float al = up ? __builtin_amdgcn_exp2f((M - mt) * c2) : 1.f;
          L *= (double)al;
#pragma unroll
          for (int e = 0; e < 4; e++) ts[e] *= al;
#pragma unroll
          for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) O[d][e] *= al;
          M = up ? mt : M;
          top = M + past;
        }
        const float Mu = M == -INFINITY ? 0.f : M;  // no key of this row yet: every score is -inf
        const int va = here(val_at(col, 8 * hf));
#pragma unroll
        for (int k = 0; k < 2; k++) {
          uint32_t ph[4], pl[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float P0 = __builtin_amdgcn_exp2f((S[8 * k + 2 * e] - Mu) * c2);
            const float P1 = __builtin_amdgcn_exp2f((S[8 * k + 2 * e + 1] - Mu) * c2);
            ts[2 * (e & 1)] += P0;
            ts[2 * (e & 1) + 1] += P1;
            split_pair(P0, P1, ph[e], pl[e]);
          }
          const fh8 vh = as_fh8(ph[0], ph[1], ph[2], ph[3]), vl = as_fh8(pl[0], pl[1], pl[2], pl[3]);
          fh8 a[ND];  // an output's two parts apart from each other: 214 -> 213 us, the window 97.4 -> 96.0
#pragma unroll
          for (int d = 0; d < ND; d++) {
            // val_at(32 d + col, 32 s + 16 k + 8 hf)
            a[d] = *reinterpret_cast<const fh8 *>(vb + 32 * d * kTlK + (va ^ ((4 * d ^ 4 * s ^ 2 * k) & 7) << 3));
            O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[d], vh, O[d], 0, 0, 0);
          }
#pragma unroll
          for (int d = 0; d < ND; d++) O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[d], vl, O[d], 0, 0, 0);
        }
      }
      if constexpr (Stage::kPrio) __builtin_amdgcn_s_setprio(0);
      if (s == 0 && i + 1 < i1) {
        stage(b ^ 1, st.at(i + 1));
        if (i + 2 < i1) sg.fetch(st.at(i + 2), last);
      }
    }
    if (on) {
      L += (double)((ts[0] + ts[1]) + (ts[2] + ts[3]));
      if (badv) {
        for (int k = 0; k < kTlK && j0 + k <= last; k++)
          if (j0 + k <= p && (j0 + k < lead || j0 + k >= first)) sg.add_bad(j0 + k, hf, O);
      }
    }
    __syncthreads();  // the next step is staged, and this one read
  }
  L += __shfl_xor(L, 32, 64);
  if (u >= NC) return;
  const int64_t row = (int64_t)t * H + h;
  const bool whole = A.chunks == 1;
  float *op = whole ? out + row * HD : part + (row * A.chunks + ch) * (HD + 4);
  const double f = whole ? 1.0 / L / kSpUp : 1.0;
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      sf4 o;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = (float)((double)O[d][4 * e + j] * f);
      *reinterpret_cast<f4a4 *>(op + 32 * d + 8 * e + 4 * hf) = o;
    }
  if (!whole && hf == 0) {
    op[HD] = M;
    op[HD + 1] = c2;
    *reinterpret_cast<double *>(op + HD + 2) = L;
  }
}

// Rows of more than one chunk: the chunks' sums under their largest maximum, in chunk order. One wave per (row, head).
template <int HD>
__global__ __launch_bounds__(256) void span_tiles_join_kernel(const float *__restrict__ part, TilesArgs A,
                                                              float *__restrict__ out) {
  const int H = A.G * A.KH;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (id >= (int64_t)A.T * H) return;
  const int lane = threadIdx.x & 63, t = (int)(id / H), h = (int)(id % H);
  const int z = (int)(((int64_t)t * A.G + h % A.G) / kTlCols);
  const int n = (SpanSteps(A.s, A.row0(z), A.row1(z)).n + A.steps - 1) / A.steps;
  const float *rec = part + id * A.chunks * (HD + 4);
  float m = -INFINITY;
  for (int i = 0; i < n; i++) m = fmaxf(m, rec[i * (HD + 4) + HD]);
  double L = 0.0;
  float o[HD / 64] = {};
  for (int i = 0; i < n; i++) {
    const float *rc = rec + i * (HD + 4);
    const float w = __builtin_amdgcn_exp2f((rc[HD] - m) * rc[HD + 1]);
    L += *reinterpret_cast<const double *>(rc + HD + 2) * (double)w;
#pragma unroll
    for (int e = 0; e < HD / 64; e++) o[e] = __builtin_fmaf(rc[lane + 64 * e], w, o[e]);
  }
  const double f = 1.0 / L / kSpUp;
#pragma unroll
  for (int e = 0; e < HD / 64; e++) out[id * HD + lane + 64 * e] = (float)((double)o[e] * f);
}

static TilesArgs tiles_plan(const KvCache &c, int H, const Span &s, const KvRows &R) {
  TilesArgs A;
  A.s = s;
  A.T = R.n;
  A.pos0 = R.pos0;
  A.KH = c.KH;
  A.G = H / c.KH;
  A.nz = (int)(((int64_t)R.n * A.G + kTlCols - 1) / kTlCols);
  int most = 0;
  for (int z = 0; z < A.nz; z++) {
    const int n = SpanSteps(s, A.row0(z), A.row1(z)).n;
    most = n > most ? n : most;
  }
  // Whole rows where the workgroups of columns alone give every CU one; fewer are cut so that they give two (8B after 2,000:
  // 500 rows 66 us, whole 104; a window of 1,024 49, whole 66; but 1,500 rows, whole, 175, cut 199). Just below the border
  // cutting costs more than it gives: 992 rows 140 us, whole 124, the window's 87, whole 68.
  const int64_t wgs = (int64_t)c.KH * A.nz;
  int64_t S = wgs >= 256 ? 1 : (512 + wgs - 1) / wgs;
  S = S > most ? most : S;
  A.steps = (int)((most + S - 1) / S);
  A.chunks = (most + A.steps - 1) / A.steps;
  return A;
}

template <int HD, class Stage>
static hipError_t span_tiles_launch(const float *q, int H, const KvCache &c, const Span &s, const KvRows &R, float scale,
                                    float *part, float *out, hipStream_t st) {
  const TilesArgs A = tiles_plan(c, H, s, R);
  // one grid dimension: the others hold 65,535 workgroups
  hipLaunchKernelGGL((span_tiles_kernel<HD, Stage>), dim3((unsigned)((int64_t)c.KH * A.chunks * A.nz)), dim3(256), 0, st, q,
                     c, A, scale, part, out);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || A.chunks == 1) return e;
  hipLaunchKernelGGL(span_tiles_join_kernel<HD>, dim3((unsigned)(((int64_t)R.n * H + 3) / 4)), dim3(256), 0, st, part, A,
                     out);
  return hipGetLastError();
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

// Rows of the plain kernel's launches: their scores take at most 256 MB, where one row's do.
static int span_rows_step(int H, const Span &s, const KvRows &R) {
  const int64_t one = (int64_t)H * span_max_n(s, R), fit = ((int64_t)64 << 20) / one;
  return (int)(fit < 1 ? 1 : fit > 32768 ? 32768 : fit < R.n ? fit : R.n);
}

int64_t attention_span_scratch_floats(const KvCache &c, int H, const Span &s, const KvRows &R) {
  if (R.n <= 0) return 0;
  if (span_decodes(c, R)) {
    const SpanRuns U = span_plan(c, H, s, R);
    return U.most > 1 ? (int64_t)R.n * H * U.most * (c.HD + 4) : 0;
  }
  if (span_tiled(c)) {
    const TilesArgs A = tiles_plan(c, H, s, R);
    return A.chunks > 1 ? (int64_t)R.n * H * A.chunks * (c.HD + 4) : 0;
  }
  return (int64_t)span_rows_step(H, s, R) * H * span_max_n(s, R);
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
  if (span_tiled(c)) {
    if (c.bits == 4)
      return c.HD == 64 ? span_tiles_launch<64, StageKv4<64>>(q, H, c, s, R, scale, scratch, out, st)
                        : span_tiles_launch<128, StageKv4<128>>(q, H, c, s, R, scale, scratch, out, st);
    return c.HD == 64 ? span_tiles_launch<64, StageF16<64>>(q, H, c, s, R, scale, scratch, out, st)
                      : span_tiles_launch<128, StageF16<128>>(q, H, c, s, R, scale, scratch, out, st);
  }
  const int step = span_rows_step(H, s, R);
  for (int t0 = 0; t0 < R.n; t0 += step) {
    const int n = R.n - t0 < step ? R.n - t0 : step;
    hipLaunchKernelGGL(span_rows_kernel, dim3(H, n), dim3(256), 0, st, q, H, c, s, R, t0, scale, scratch, span_max_n(s, R),
                       out);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace wl
