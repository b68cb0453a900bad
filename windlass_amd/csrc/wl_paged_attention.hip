// wl_paged_attention.hip - attention over KV caches in pages (wl_paged.h): over all positions of a row's sequence, over a prefix
// that the rows of many sequences share, and over chosen pages.
//
// A column is a (row, query head of the KV head) pair, row * G + head within its entry, its query as two fp16 parts (22 bits of
// its largest value). S^T = K Q^T and O^T = V^T P^T, the probabilities in two parts as well; a page holds both operands as the
// matrix cores take them, so that keys and values go from memory (or LDS) to the products as they lie. Rows of few columns take
// paged_few_kernel (16 columns, the waves one tile of 32 positions in turn), others paged_many_kernel (32 columns a wave, the
// positions staged in LDS). Both cut long rows in runs, whose outputs, maxima and sums paged_join_kernel adds; a shared prefix is
// one such launch over the rows of all entries, without a mask, and its runs are added beside those of each entry's own.
#include "wl_paged.h"

#include "wl_attention_parts.h"
#include "wl_paged_device.h"

#include <algorithm>
#include <math.h>

#pragma clang fp contract(off)

namespace wl {

typedef float sf16 __attribute__((ext_vector_type(16)));

constexpr int kFewCols = 16, kFewWaves = 4;
constexpr int kManyWaves = 4, kManyCols = 32 * kManyWaves, kManyUnits = 4;  // units of a step
constexpr int kPgRuns = 256;  // of a row at most
constexpr uint32_t kNowhere = 0xfffffff0u;  // the position of a unit that no row sees

// A launch's items go entry by entry, column block by column block, run by run of `per` tiles or steps each. An entry's records,
// a run after the other for each (row, head), begin H * rec records into `part`; alone: a row of one run is the output itself. Of
// the items flat0 .. flat1 - 1, a prefix', all rows see what the entry's position does.
struct PagedPlan {
  PageItems it;
  int flat0, flat1;
  int base;          // units before base are not read (but by a prefix' items)
  int alone;
};
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// What a column needs of its query: the factor of its parts, and of its scores in units of log2.
__device__ __forceinline__ void query_scale(float m, float scale, float &f, float &c2) {
  float inv;
  unit_scale(m, f, inv);
  // c2 > 0: a negative scale negates the query
  c2 = fmaxf(fabsf(scale) * 1.4426950408889634f * inv, 1.1754944e-38f);
  f = scale < 0.f ? -f : f;
  if (scale != scale) c2 = scale;
}
__device__ __forceinline__ void query_parts(float x, float f, _Float16 &hi, _Float16 &lo) {
  const float X = x * f;
  hi = (_Float16)X;
  lo = (_Float16)(__builtin_isinf(X) ? 0.f : X - (float)hi);  // an infinity is all in its high part
}

// Weights are exp2 of a score's difference from the column's maximum M, times 2^8: all that follows is by their sum. M is one of
// the scores seen, and is raised only where a step's weights would pass 2^15 (fp16 parts end at 2^16) or a column has none yet, so
// that no step looks for its maximum. The largest weighs 2^8 at least; two parts, the high one cut, are 22 bits of a weight down to
// 2^-3, and off by 2^-25 at most below (half a step of the least fp16 numbers), 2^-33 of the largest.
constexpr float kUp = 8.f, kFull = 0x1p15f;
__device__ __forceinline__ float weight(float s, float M, float c2) { return __builtin_amdgcn_exp2f(__builtin_fmaf(s - M, c2, kUp)); }
// Two weights as their fp16 parts: the high ones cut, the low ones what is left, rounded.
__device__ __forceinline__ void weight_parts(float a, float b, uint32_t &hi, uint32_t &lo) {
  hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
  asm("" : "+v"(hi));
  lo = __builtin_bit_cast(uint32_t, fh2{(_Float16)__builtin_fmaf(a, 1.f, -half_lo(hi)), (_Float16)__builtin_fmaf(b, 1.f, -half_hi(hi))});
}

// Bits 15 and 31 set where a half of w is an infinity or NaN: its exponent's ones carry.
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }

// Of a lane's eight values of a channel, positions at .. at + 7: those that no column sees (past pb) become zeros, and of those
// that some do not see (past pa) the infinite and NaN ones; true where one of these was seen by some.
__device__ __forceinline__ bool clear_unseen(u32x4_t &w, uint32_t at, uint32_t pa, uint32_t pb) {
  uint32_t bad = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t a = at + 2 * j, b = a + 1;
    const uint32_t odd = odd_halves(w[j]);
    const uint32_t all = (a <= pa ? 0xffffu : 0u) | (b <= pa ? 0xffff0000u : 0u);
    const uint32_t some = (a <= pb ? 0xffffu : 0u) | (b <= pb ? 0xffff0000u : 0u);
    const uint32_t drop = ((odd >> 15) * 0xffffu & ~all) | ~some;
    bad |= (odd >> 15) * 0xffffu & ~all & some;
    w[j] &= ~drop;
  }
  return bad != 0;
}

// ------------------------------------------------------------------------------- few columns

// The keys of a tile are loaded again once its scores are made, and its values once they are multiplied: half a tile is in flight
// all the time, and a SIMD holds three waves.
template <int HD>
struct FewTile {
  static constexpr int NK = HD / 32, ND = HD / 16;
  u32x4_t k[2][NK], v[ND];
  uint32_t up[2];  // the positions of the units' first values
  // a, b: halves before the tile's two units
  __device__ __forceinline__ void keys(const PagePool &P, int64_t a, int64_t b, int lane) {
    const int m = lane & 15, kq = lane >> 4;
    const uint16_t *kp = P.K + (m < 8 ? a : b) + kq * 64 + (m & 7) * 8;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int i = 0; i < NK; i++)
        k[t][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(kp + t * 8 * HD + i * 256));
  }
  __device__ __forceinline__ void values(const PagePool &P, int64_t a, int64_t b, int lane) {
    const int m = lane & 15, kq = lane >> 4;
    const uint16_t *vp = P.V + (kq < 2 ? a : b) + (kq & 1) * 8 * HD + m * 8;
#pragma unroll
    for (int d = 0; d < ND; d++) v[d] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(vp + d * 128));
  }
};

// 16 columns and a run of tiles a workgroup: S^T = K Q^T of 32 positions by two products of 16 keys each per 32 channels and part of
// q, the weights, O^T += V^T P^T by one product per 16 channels and part of the weights. A product of 16 columns is half empty with
// the eight heads of 70B and no matter: keys and values pass once and memory bounds it (48 rows up to 9,001 of 70B 224-230 us, 5.8 TB/s
// of the 7.1 that a read can reach here; matrix cores 7% busy, VALU 18%). So nothing is staged: a wave's loads are its operands, whole lines of
// pieces of 16 bytes, and its tiles go to no other wave. Small calls are a wave's tiles one after the other, about 1 us each.
template <int HD, bool CHOSEN>
__global__ __launch_bounds__(64 * kFewWaves, HD == 64 ? 4 : 3) void paged_few_kernel(PagePool P, PagedPlan U,
                                                                                    const float *__restrict__ q, int G,
                                                                                    const int32_t *__restrict__ blocks,
                                                                                    int nblocks, float scale,
                                                                                    float *__restrict__ part,
                                                                                    float *__restrict__ out) {
  constexpr int NK = HD / 32, ND = HD / 16, W = kFewWaves;
  __shared__ sf4 so[W][kFewCols][HD / 4 + 1];
  __shared__ float sm[W][kFewCols], sc2[kFewCols];
  __shared__ double sl[W][kFewCols];
  __shared__ fh8 qs[2][NK][64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kq = lane >> 4, KH = P.KH, H = G * KH, us = P.shift - 4;
  const int kvh = blockIdx.x % KH, item = blockIdx.x / KH;
  const PageEntry E = entry_of(U.it, item);
  const bool flat = item >= U.flat0 && item < U.flat1;
  const int inc = flat ? 0 : 1, base = flat ? 0 : U.base;
  const int runs = E.runs, per = E.per, run = uniform((item - E.off) % runs);
  int cb = uniform((item - E.off) / runs), t0 = 0, T = E.rows;  // the block's rows: T from the entry's t0
  if constexpr (CHOSEN) {
    const int nb = (G + kFewCols - 1) / kFewCols;
    t0 = uniform(cb / nb);
    cb = uniform(cb % nb);
    T = 1;
  }
  const int row0 = E.row0 + t0, pos = E.pos + t0;
  const int NC = T * G, c0 = cb * kFewCols, c = c0 + col < NC ? c0 + col : NC - 1;
  const int t = c / G, h = kvh * G + c % G;
  const int p = pos + t * inc, pa = uniform(pos + c0 / G * inc);
  const int pb = uniform(pos + (c0 + kFewCols - 1 < NC ? c0 + kFewCols - 1 : NC - 1) / G * inc);
  int nu;  // units
  if constexpr (CHOSEN) nu = ((pos >> P.shift) + 1 < nblocks ? (pos >> P.shift) + 1 : nblocks) << us;
  else nu = (pb >> 4) - base + 1;
  const int nt = (nu + 1) / 2, i0 = run * per, i1 = i0 + per < nt ? i0 + per : nt;

  // The wave's units, 64 (32 tiles) at a time: lane 2 k + x has unit x of its k-th tile.
  int64_t off;
  uint32_t up;
  auto units = [&](int first) __attribute__((always_inline)) {
    const int tile = first + W * (lane >> 1), j = 2 * tile + (lane & 1);
    off = 0;
    up = kNowhere;
    if (tile >= i1 || j >= nu) return;
    int b, u;
    if constexpr (CHOSEN) {
      b = blocks[((int64_t)row0 * KH + kvh) * nblocks + (j >> us)];
      if (b < 0) return;
      u = (b << us) + (j & ((1 << us) - 1));
    } else {
      u = base + j;
      b = u >> us;
    }
    const int id = P.id(E.seq, b);
    if (id < 0) return;
    off = P.at(id, kvh) + (int64_t)(u & ((1 << us) - 1)) * 16 * HD;
    up = 16u * (uint32_t)u;
  };
  auto lane64 = [](int64_t v, int l) __attribute__((always_inline)) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)v, l));
  };
  FewTile<HD> a;
  int64_t oa, ob;  // the next tile's units
  uint32_t ua, ub;
  auto next_tile = [&](int k) __attribute__((always_inline)) {
    oa = lane64(off, 2 * k);
    ob = lane64(off, 2 * k + 1);
    ua = (uint32_t)__builtin_amdgcn_readlane((int)up, 2 * k);
    ub = (uint32_t)__builtin_amdgcn_readlane((int)up, 2 * k + 1);
  };
  int tile = i0 + wv, k = 0;
  units(tile);
  if (tile < i1) {
    next_tile(0);
    a.keys(P, oa, ob, lane);
    a.values(P, oa, ob, lane);
  }

  // the columns' parts: a wave makes those of the steps wv, wv + W, ..; all read them from LDS
  float c2;
  {
    const float *qp = q + ((int64_t)(row0 + t) * H + h) * HD + kq * 8;
    sf4 x[2 * NK];
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 2 * NK; e++) x[e] = *reinterpret_cast<const f4a4 *>(qp + e / 2 * 32 + e % 2 * 4);
#pragma unroll
    for (int e = 0; e < 2 * NK; e++)
#pragma unroll
      for (int j = 0; j < 4; j++) m = fabsf(x[e][j]) < INFINITY ? fmaxf(m, fabsf(x[e][j])) : m;
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    float f;
    query_scale(m, scale, f, c2);
#pragma unroll
    for (int s = 0; s < NK; s++) {
      if (s % W != wv) continue;  // uniform
      fh8 a, b;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        _Float16 hi, lo;
        query_parts(x[2 * s + e / 4][e % 4], f, hi, lo);
        a[e] = hi;
        b[e] = lo;
      }
      qs[0][s][lane] = a;
      qs[1][s][lane] = b;
    }
  }
  __syncthreads();
  sf4 O[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) O[d] = sf4{0.f, 0.f, 0.f, 0.f};
  float M = -INFINITY;
  double L = 0.0;
#pragma unroll 1
  for (; tile < i1; tile += W) {
    a.up[0] = ua;
    a.up[1] = ub;
    const bool more = tile + W < i1;  // uniform
    if (more) {
      if (++k == 32) {
        k = 0;
        units(tile + W);
      }
      next_tile(k);
    }
    fh8 qh[NK], ql[NK];  // read again for each tile: in registers they were spilled
#pragma unroll
    for (int s = 0; s < NK; s++) {
      ql[s] = qs[1][s][lane];
      qh[s] = qs[0][s][lane];
    }
    sf4 S[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      S[x] = sf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < NK; s++) {
        S[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fh8, a.k[x][s]), ql[s], S[x], 0, 0, 0);
        S[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fh8, a.k[x][s]), qh[s], S[x], 0, 0, 0);
      }
    }
    const uint32_t at = (kq >> 1 ? a.up[1] : a.up[0]) + 8 * (kq & 1);  // of the lane's eight positions
    bool bad = false;
    if (a.up[0] + 15 > (uint32_t)pa || a.up[1] + 15 > (uint32_t)pa) {  // uniform: some column does not see every position
      asm volatile("");  // a branch, not selects in every tile
#pragma unroll
      for (int j = 0; j < 8; j++) S[j >> 2][j & 3] = at + j > (uint32_t)p ? -INFINITY : S[j >> 2][j & 3];
#pragma unroll
      for (int d = 0; d < ND; d++) bad |= clear_unseen(a.v[d], at, pa, pb);
      bad = __any(bad);
    }
    float e[8], ts;
    auto weigh = [&]() __attribute__((always_inline)) {
      const float Mu = M == -INFINITY ? 0.f : M;  // no score of this column yet: all are -inf
#pragma unroll
      for (int j = 0; j < 8; j++) e[j] = weight(S[j >> 2][j & 3], Mu, c2);
      ts = ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
    };
    weigh();
    if (__any(!(ts < kFull) || M == -INFINITY)) {
      asm volatile("");
      bool odd = false;
#pragma unroll
      for (int j = 0; j < 8; j++) odd |= S[j >> 2][j & 3] != S[j >> 2][j & 3];
      if (__any(odd)) {  // past an infinity the low parts' product means nothing: a score of -inf may be NaN here
#pragma unroll
        for (int x = 0; x < 2; x++) {
          sf4 A1 = sf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < NK; s++)
            A1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fh8, a.k[x][s]), qh[s], A1, 0, 0, 0);
#pragma unroll
          for (int j = 0; j < 4; j++) S[x][j] = A1[j] == -INFINITY && S[x][j] != S[x][j] ? -INFINITY : S[x][j];
        }
      }
      float mt = fmaxf(fmaxf(fmaxf(S[0][0], S[0][1]), fmaxf(S[0][2], S[0][3])),
                       fmaxf(fmaxf(S[1][0], S[1][1]), fmaxf(S[1][2], S[1][3])));
      mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
      mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
      const bool raise = mt > M;
      const float al = raise ? __builtin_amdgcn_exp2f((M - mt) * c2) : 1.f;
      L *= (double)al;
#pragma unroll
      for (int d = 0; d < ND; d++) O[d] *= al;
      M = raise ? mt : M;
      weigh();
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) a.keys(P, oa, ob, lane);
    __builtin_amdgcn_sched_barrier(0);
    L += (double)ts;
    uint32_t ph[4], pl[4];
#pragma unroll
    for (int j = 0; j < 4; j++) weight_parts(e[2 * j], e[2 * j + 1], ph[j], pl[j]);
    const fh8 eh = as_fh8(ph[0], ph[1], ph[2], ph[3]), el = as_fh8(pl[0], pl[1], pl[2], pl[3]);
#pragma unroll
    for (int d = 0; d < ND; d++) O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fh8, a.v[d]), el, O[d], 0, 0, 0);
#pragma unroll
    for (int d = 0; d < ND; d++) O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fh8, a.v[d]), eh, O[d], 0, 0, 0);
    if (bad) {  // infinite and NaN values into the columns that see them
      for (int x = 0; x < 32; x++) {
        const uint32_t w = (x >> 4 ? a.up[1] : a.up[0]) + (x & 15);
        if (w <= (uint32_t)pa || w > (uint32_t)pb) continue;  // uniform
        const uint16_t *vp = P.V + P.at(P.id(E.seq, (int)(w >> P.shift)), kvh);
        const int o = (int)(w & (P.page - 1));
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const uint16_t y = vp[pg_val(o, 16 * d + 4 * kq + j, HD)];
            if ((y & 0x7c00u) == 0x7c00u && w <= (uint32_t)p) O[d][j] += (float)__builtin_bit_cast(_Float16, y);
            __builtin_amdgcn_sched_barrier(0);  // one value at a time: this is rare, and its registers all the loop's
          }
      }
    }
    if (more) a.values(P, oa, ob, lane);
  }
  // the waves' sums under their largest maximum
  L += __shfl_xor(L, 16, 64);
  L += __shfl_xor(L, 32, 64);
#pragma unroll
  for (int d = 0; d < ND; d++) so[wv][col][4 * d + kq] = O[d];
  if (kq == 0) {
    sm[wv][col] = M;
    sl[wv][col] = L;
    sc2[col] = c2;
  }
  __syncthreads();
  const bool whole = U.alone && !flat && runs == 1;
  for (int e = threadIdx.x; e < kFewCols * HD / 4; e += 64 * W) {
    const int g = e / (HD / 4), four = e % (HD / 4), cc = c0 + g;
    if (cc >= NC) break;
    float m = sm[0][g];
#pragma unroll
    for (int w = 1; w < W; w++) m = fmaxf(m, sm[w][g]);
    sf4 o = {0.f, 0.f, 0.f, 0.f};
    double l = 0.0;
#pragma unroll
    for (int w = 0; w < W; w++) {
      const float f = weight_of(sm[w][g], m, sc2[g]);
      o += so[w][g][four] * f;
      l += sl[w][g] * (double)f;
    }
    const int64_t at = (int64_t)(t0 + cc / G) * H + kvh * G + cc % G, row = (int64_t)E.row0 * H + at;
    if (whole) {
      const double r = 1.0 / l;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = l == 0.0 ? 0.f : (float)((double)o[j] * r);
      *reinterpret_cast<f4a4 *>(out + row * HD + 4 * four) = o;
    } else {
      float *rec = part + ((int64_t)E.rec * H + at * runs + run) * (HD + 4);
      *reinterpret_cast<sf4 *>(rec + 4 * four) = o;
      if (four == 0) {
        rec[HD] = m;
        rec[HD + 1] = sc2[g];
        *reinterpret_cast<double *>(rec + HD + 2) = l;
      }
    }
  }
}

// ------------------------------------------------------------------------------- many columns

// 16 bytes a lane from memory to LDS, lane after lane from `to` on; complete after landed(). The compiler's own form made
// every read of LDS after it wait for it, also reads of the buffer before. It writes m0, and says so: the compiler, which gives that
// register to no value of its own, may set it for an instruction and use it again, and warns of the name in a list.
typedef __attribute__((address_space(3))) uint16_t lds_u16;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void to_lds(const uint16_t *from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// 128 columns and a run of steps a workgroup, 32 columns a wave: the products of 32 keys (64 positions a step) with both parts of q
// from registers, and of 32 channels with both parts of the weights. The four waves share keys and values in LDS, where they lie
// as in the page (a wave's 16-byte reads are whole lines: no bank conflicts), brought by direct loads a step ahead. Two workgroups
// fit a CU (64 KB, 256 registers a lane), so that one wave's weights run beside the other's products (64 rows of 70B on a prefix of
// 8,192 are but one a CU: matrix cores 24% busy). The SIMDs' issue bounds it: prompts of 2,001, 2,001 and 667 rows (8B) take 436-447
// us, 530 TFLOP/s of 4 HD flops a score and column (twice that in two parts), matrix cores 41% and VALU 36% busy, waits 25% of the
// wave cycles.
template <int HD>
__global__ __launch_bounds__(64 * kManyWaves, 2) void paged_many_kernel(PagePool P, PagedPlan U, const float *__restrict__ q,
                                                                        int G, float scale, float *__restrict__ part,
                                                                        float *__restrict__ out) {
  constexpr int NK = HD / 16, ND = HD / 32, UN = 16 * HD;  // halves of a unit
  __shared__ __attribute__((aligned(1024))) uint16_t lk[2][kManyUnits * UN], lv[2][kManyUnits * UN];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hf = lane >> 5, col = lane & 31, KH = P.KH, H = G * KH, us = P.shift - 4;
  const int kvh = blockIdx.x % KH, item = blockIdx.x / KH;
  const PageEntry E = entry_of(U.it, item);
  const bool flat = item >= U.flat0 && item < U.flat1;
  const int inc = flat ? 0 : 1, base = flat ? 0 : U.base;
  const int row0 = E.row0, T = E.rows, pos = E.pos, per = E.per, runs = E.runs;
  const int64_t NC = (int64_t)T * G;
  const int nz = (int)((NC + kManyCols - 1) / kManyCols), run = uniform((item - E.off) % runs), r = uniform((item - E.off) / runs);
  // longest and shortest rows in turn: the workgroups that share a CU (the grid's halves) add up
  const int z = r < (nz + 1) / 2 ? nz - 1 - r : r - (nz + 1) / 2;
  const int64_t z0 = (int64_t)z * kManyCols, w0 = z0 + 32 * wv, u = w0 + col, uc = u < NC ? u : NC - 1;
  auto position = [&](int64_t c) __attribute__((always_inline)) { return pos + (int)((c < NC ? c : NC - 1) / G) * inc; };
  const int t = (int)(uc / G), h = kvh * G + (int)(uc % G), p = pos + t * inc;
  const int pa = uniform(position(w0)), pb = uniform(position(w0 + 31)), last = uniform(position(z0 + kManyCols - 1));
  const bool idle = w0 >= NC;
  const int nu = (last >> 4) - base + 1, ns = (nu + kManyUnits - 1) / kManyUnits;
  const int i0 = run * per, i1 = i0 + per < ns ? i0 + per : ns;

  // The pages of 16 steps: lane l has unit l of theirs; those of the 16 after them are loaded ahead.
  auto page_of = [&](int first) __attribute__((always_inline)) {
    const int j = kManyUnits * first + lane;
    return j < nu && first < i1 ? P.id(E.seq, (base + j) >> us) : -1;
  };
  int ids = page_of(i0), ahead = page_of(i0 + 16);
  uint64_t there = __ballot(ids >= 0);
  // step s into buffer b, a unit a wave; returns which units are there
  auto stage = [&](int b, int s) __attribute__((always_inline)) {
    const int x = s - i0;
    if (x && (x & 15) == 0) {  // uniform
      ids = ahead;
      ahead = page_of(s + 16);
      there = __ballot(ids >= 0);
    }
    const int l = (x & 15) * kManyUnits, id = __builtin_amdgcn_readlane(ids, l + wv);
    const int unit = base + kManyUnits * s + wv;
    const int64_t off = P.at(id < 0 ? 0 : id, kvh) + (int64_t)(unit & ((1 << us) - 1)) * UN;
    // keys lie in LDS as [HD / 8][16 rows of the products][8]
    const uint16_t *kp = P.K + off + (lane >> 3 & 1) * 8 * HD + (lane >> 4) * 64 + (lane & 7) * 8;
    const uint16_t *vp = P.V + off + lane * 8;
    const uint32_t ko = (uint32_t)(uintptr_t)(lds_u16 *)(lk[b] + wv * UN);
    const uint32_t vo = (uint32_t)(uintptr_t)(lds_u16 *)(lv[b] + wv * UN);
#pragma unroll
    for (int c = 0; c < UN / 512; c++) {
      to_lds(kp + c * 256, ko + c * 1024);
      to_lds(vp + c * 512, vo + c * 1024);
    }
    return (int)(there >> l) & 15;
  };
  int have = i0 < i1 ? stage(0, i0) : 0;
  // the columns' parts, in operand order: k = 16 i + 8 hf + 0..7
  fh8 qh[NK], ql[NK];
  float c2;
  {
    const float *qp = q + ((int64_t)(row0 + t) * H + h) * HD + 8 * hf;
    float m = 0.f;
#pragma unroll
    for (int s = 0; s < NK; s++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float a = fabsf(qp[16 * s + j]);
        m = a < INFINITY ? fmaxf(m, a) : m;
      }
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    float f;
    query_scale(m, scale, f, c2);
#pragma unroll
    for (int s = 0; s < NK; s++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        _Float16 hi, lo;
        query_parts(qp[16 * s + j], f, hi, lo);
        qh[s][j] = hi;
        ql[s][j] = lo;
      }
  }
  sf16 O[ND];
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int e = 0; e < 16; e++) O[d][e] = 0.f;
  float M = -INFINITY;
  double L = 0.0;
  landed();
  __syncthreads();
#pragma unroll 1
  for (int s = i0; s < i1; s++) {
    const int b = (s - i0) & 1, here = have;
    if (s + 1 < i1) have = stage(b ^ 1, s + 1);
    const uint32_t s0 = 16u * (uint32_t)(base + kManyUnits * s);  // the step's first position
    const bool on = !idle && s0 <= (uint32_t)pb;
    if (on) {
      float ts = 0.f;
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const uint16_t *kb = lk[b] + (2 * x + (col >> 4)) * UN + hf * 128 + (col & 15) * 8;
        sf16 S;
#pragma unroll
        for (int e = 0; e < 16; e++) S[e] = 0.f;
#pragma unroll
        for (int k = 0; k < NK; k++) {
          const fh8 a = *reinterpret_cast<const fh8 *>(kb + 256 * k);
          S = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[k], S, 0, 0, 0);
          S = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[k], S, 0, 0, 0);
        }
        const uint32_t p0 = s0 + 32 * x;
        const bool cut = p0 + 31 > (uint32_t)pa || (here >> (2 * x) & 3) != 3;  // uniform: some column does not see all
        uint32_t up[2];
#pragma unroll
        for (int k = 0; k < 2; k++) up[k] = here >> (2 * x + k) & 1 ? p0 + 16 * k : kNowhere;
        if (cut) {
          asm volatile("");
#pragma unroll
          for (int e = 0; e < 16; e++) S[e] = up[e >> 3] + 8 * hf + (e & 7) > (uint32_t)p ? -INFINITY : S[e];
        }
        // weights before the other wave's work: 191.7 -> 188.3 us for 80 rows of a prefix of 60,000
        __builtin_amdgcn_s_setprio(1);
        float w[16], tt;
        auto weigh = [&]() __attribute__((always_inline)) {
          const float Mu = M == -INFINITY ? 0.f : M;  // no score of this column yet: all are -inf
          float tx[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 16; e++) {
            w[e] = weight(S[e], Mu, c2);
            tx[e & 3] += w[e];
          }
          tt = (tx[0] + tx[1]) + (tx[2] + tx[3]);
        };
        weigh();
        if (__any(!(tt < kFull) || M == -INFINITY)) {
          asm volatile("");
          bool odd = false;
#pragma unroll
          for (int e = 0; e < 16; e++) odd |= S[e] != S[e];
          if (__any(odd)) {  // past an infinity the low parts' product means nothing: a score of -inf may be NaN here
            sf16 A;
#pragma unroll
            for (int e = 0; e < 16; e++) A[e] = 0.f;
#pragma unroll
            for (int k = 0; k < NK; k++)
              A = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const fh8 *>(kb + 256 * k), qh[k], A, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 16; e++) S[e] = A[e] == -INFINITY && S[e] != S[e] ? -INFINITY : S[e];
          }
          float mt = S[0];
#pragma unroll
          for (int e = 1; e < 16; e++) mt = fmaxf(mt, S[e]);
          mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
          const bool raise = mt > M;
          const float al = raise ? __builtin_amdgcn_exp2f((M - mt) * c2) : 1.f;
          L *= (double)al;
          ts *= al;
#pragma unroll
          for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) O[d][e] *= al;
          M = raise ? mt : M;
          weigh();
        }
        ts += tt;
        bool bad = false;
#pragma unroll
        for (int k = 0; k < 2; k++) {
          uint32_t ph[4], pl[4];
#pragma unroll
          for (int e = 0; e < 4; e++) weight_parts(w[8 * k + 2 * e], w[8 * k + 2 * e + 1], ph[e], pl[e]);
          const fh8 eh = as_fh8(ph[0], ph[1], ph[2], ph[3]), el = as_fh8(pl[0], pl[1], pl[2], pl[3]);
          const uint16_t *vb = lv[b] + (2 * x + k) * UN + hf * 8 * HD + col * 8;
          u32x4_t a[ND];
#pragma unroll
          for (int d = 0; d < ND; d++) a[d] = *reinterpret_cast<const u32x4_t *>(vb + 256 * d);
          if (cut) {
            asm volatile("");
#pragma unroll
            for (int d = 0; d < ND; d++) bad |= clear_unseen(a[d], up[k] + 8 * hf, pa, pb);
          }
#pragma unroll
          for (int d = 0; d < ND; d++) O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(fh8, a[d]), eh, O[d], 0, 0, 0);
#pragma unroll
          for (int d = 0; d < ND; d++) O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(fh8, a[d]), el, O[d], 0, 0, 0);
        }
        __builtin_amdgcn_s_setprio(0);
        if (__any(bad)) {  // infinite and NaN values into the columns that see them
          for (int y = 0; y < 32; y++) {
            const uint32_t w = (y >> 4 ? up[1] : up[0]) + (y & 15);
            if (w <= (uint32_t)pa || w > (uint32_t)pb) continue;  // uniform
            const uint16_t *vp = lv[b] + (2 * x + (y >> 4)) * UN;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
              for (int e = 0; e < 16; e++) {
                const uint16_t o = vp[pg_val(y & 15, 32 * d + 8 * (e >> 2) + 4 * hf + (e & 3), HD)];
                if ((o & 0x7c00u) == 0x7c00u && w <= (uint32_t)p) O[d][e] += (float)__builtin_bit_cast(_Float16, o);
                __builtin_amdgcn_sched_barrier(0);
              }
          }
        }
      }
      L += (double)ts;
    }
    landed();
    __syncthreads();  // the next step is there, and this one read
  }
  L += __shfl_xor(L, 32, 64);
  if (u >= NC) return;
  const int64_t at = (int64_t)t * H + h;
  const bool whole = U.alone && !flat && runs == 1;
  float *op = whole ? out + ((int64_t)row0 * H + at) * HD : part + ((int64_t)E.rec * H + at * runs + run) * (HD + 4);
  const double f = whole ? 1.0 / L : 1.0;
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      sf4 o;
#pragma unroll
      for (int j = 0; j < 4; j++) o[j] = whole && L == 0.0 ? 0.f : (float)((double)O[d][4 * e + j] * f);
      *reinterpret_cast<f4a4 *>(op + 32 * d + 8 * e + 4 * hf) = o;
    }
  if (!whole && hf == 0) {
    op[HD] = M;
    op[HD + 1] = c2;
    *reinterpret_cast<double *>(op + HD + 2) = L;
  }
}

// ------------------------------------------------------------------------------- runs

// The entries whose rows have records, a row an item, and the prefix' runs of every row.
struct PagedRuns {
  PageItems it;
  int pre, pre_rec;
};

// The records of a row's runs under their largest maximum. A workgroup per (row, head): the runs' factors once, into LDS; then
// HD / 4 threads to a record, the records over the groups in turn, each group's sum in order and the groups' in order. Two dependent
// reads and a launch bound it: a row of 64 heads of up to 9,000 positions 14.8 us with its attention, 15.6 by the kernel below.
template <int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(const float *__restrict__ part, int H, PagedRuns U,
                                                         float *__restrict__ out) {
  constexpr int TH = HD / 4, NG = 256 / TH;
  __shared__ float f[kPgRuns], sm[4];
  __shared__ double sl[4];
  __shared__ sf4 so[NG][TH];
  const PageEntry E = entry_of(U.it, blockIdx.x / H);
  const int64_t at = (int64_t)blockIdx.x - (int64_t)E.off * H, row = (int64_t)E.row0 * H + at;  // (row, head) pairs
  const int tid = threadIdx.x, n = U.pre + E.runs;
  const float *pre = part + ((int64_t)U.pre_rec * H + row * U.pre) * (HD + 4);
  const float *ours = part + ((int64_t)E.rec * H + at * E.runs) * (HD + 4);
  auto record = [&](int k) { return k < U.pre ? pre + k * (HD + 4) : ours + (k - U.pre) * (HD + 4); };
  static_assert(kPgRuns == 256, "a thread per run");
  const float *mine = record(tid < n ? tid : n - 1);
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
  for (int j = g; j < n; j += 4 * NG) {
    sf4 v[4];
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = *reinterpret_cast<const sf4 *>(record(j + k * NG < n ? j + k * NG : j) + 4 * x);
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (j + k * NG < n) o += v[k] * f[j + k * NG];
  }
  so[g][x] = o;
  __syncthreads();
  if (tid < TH) {
    sf4 s = so[0][tid];
#pragma unroll
    for (int k = 1; k < NG; k++) s += so[k][tid];
    const double all = (sl[0] + sl[1]) + (sl[2] + sl[3]), r = 1.0 / all;
#pragma unroll
    for (int e = 0; e < 4; e++) s[e] = all == 0.0 ? 0.f : (float)((double)s[e] * r);
    *reinterpret_cast<f4a4 *>(out + row * HD + 4 * tid) = s;
  }
}

// The same sums in the same order, for rows of up to 64 runs where there are many of them: a wave per (row, head), which has the
// groups' sums in the lanes of its two or four records at once.
template <int HD>
__global__ __launch_bounds__(256) void paged_join_rows_kernel(const float *__restrict__ part, int H, PagedRuns U,
                                                              float *__restrict__ out) {
  constexpr int TH = HD / 4, NG = 256 / TH, AT = 64 / TH, PG = NG / AT;  // records at once, groups a lane
  const int64_t pair = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const bool there = pair < (int64_t)U.it.items * H;
  const int lane = threadIdx.x & 63;
  const PageEntry E = entry_of(U.it, (int)((there ? pair : 0) / H));
  if (!there) return;
  const int64_t at = pair - (int64_t)E.off * H, row = (int64_t)E.row0 * H + at;
  const int n = U.pre + E.runs;
  const float *pre = part + ((int64_t)U.pre_rec * H + row * U.pre) * (HD + 4);
  const float *ours = part + ((int64_t)E.rec * H + at * E.runs) * (HD + 4);
  auto record = [&](int k) { return k < U.pre ? pre + k * (HD + 4) : ours + (k - U.pre) * (HD + 4); };
  const float *mine = record(lane < n ? lane : n - 1);
  const float m1 = mine[HD], c2 = mine[HD + 1];
  const double l1 = *reinterpret_cast<const double *>(mine + HD + 2);
  const int g = lane / TH, x = lane % TH;
  sf4 v[PG], o[PG];
#pragma unroll
  for (int k = 0; k < PG; k++) {  // the first record of each of the lane's groups k * AT + g
    o[k] = sf4{0.f, 0.f, 0.f, 0.f};
    v[k] = *reinterpret_cast<const sf4 *>(record(k * AT + g < n ? k * AT + g : n - 1) + 4 * x);
  }
  const float m = wave_max_f(m1), f1 = lane < n ? weight_of(m1, m, c2) : 0.f;
  const double all = wave_sum_d(lane < n ? l1 * (double)f1 : 0.0);
  for (int j = 0; j < n; j += NG) {
#pragma unroll
    for (int k = 0; k < PG; k++) {
      const int r = j + k * AT + g;
      const float f = __shfl(f1, r < n ? r : 0, 64);
      if (r < n) o[k] += v[k] * f;
    }
    if (j + NG < n) {
#pragma unroll
      for (int k = 0; k < PG; k++) {
        const int r = j + NG + k * AT + g;
        v[k] = *reinterpret_cast<const sf4 *>(record(r < n ? r : n - 1) + 4 * x);
      }
    }
  }
  sf4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < PG; k++)
#pragma unroll
    for (int a = 0; a < AT; a++) {
      sf4 w;
#pragma unroll
      for (int e = 0; e < 4; e++) w[e] = __shfl(o[k][e], a * TH + x, 64);
      s = k + a ? s + w : w;
    }
  const double r = 1.0 / all;
#pragma unroll
  for (int e = 0; e < 4; e++) s[e] = all == 0.0 ? 0.f : (float)((double)s[e] * r);
  if (g == 0) *reinterpret_cast<f4a4 *>(out + row * HD + 4 * x) = s;
}

// ------------------------------------------------------------------------------- plans

static int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Whether paged_few_kernel takes an entry: one that its keys and values pass once anyway, or one of so few products (columns times
// the positions that they see on average, in all KV heads) that the other's 128 columns a workgroup leave CUs idle. At the border, in
// us, few and many: 8B, 700 rows from 0 25.6 and 43.5, 300 up to 1,000 20.3 and 31.3, 4 up to 60,000 44.1 and 49.2, 60 up to 4,000 29.5
// and 29.0; past it, 16 up to 20,000 40.0 and 32.4, 8 up to 60,000 77.1 and 49.5; 70B, 700 from 0 48.6 and 38.7, but 300 up to 1,000
// 32.1 and 44.2; 16 rows on a prefix of 5,000 21.1 and 34.4.
static bool is_few(int64_t columns, int first, int last, int KH) {
  return columns <= kFewCols || (double)columns * (0.5 * ((double)first + last) + 1.0) * KH <= 0x1p23;
}

// Tiles of each run of an entry of n tiles, of `units` workgroups a run: a rule on the entry alone, so that its bits do not depend
// on the others. Up to `whole` tiles one run, and no second launch; then runs of `least` tiles (four waves of two or four), for what a
// run costs beside its tiles (the query's parts, the waves' sums, its record) weighs in a batch: 64 rows of up to 1,000 (70B) 33.5
// us whole and 52.4 with a tile a wave, 32 rows of up to 3,000 54.6 and 67.3; a lone row of 1,000 or 2,000 pays 1.9-2.1 us for it
// (11.2 and 9.3, 11.8 and 9.8), of 4,000 1.2. Long rows take no more runs than give every CU two workgroups.
static int few_per(int n, int units, int whole, int least) {
  if (n <= whole) return n;
  const int two = (int)(((int64_t)n * units + 511) / 512), most = ceil_div(n, kPgRuns / 2);
  return std::max({least, two, most});
}
constexpr int kFewWhole = 32, kFewLeast = 16;
// Chosen pages: 16 rows of 32 pages of 64 (70B) 53.5 us with two tiles a wave, 49.8 with four and 58.6 with one; a lone row of 64
// pages 25.6, 26.8 and 24.8. Whole up to 32 tiles as above, 64 rows of 32 pages of 32 (70B) would take 71 us, not 83, but 8 rows of 8B
// 26.4, not 23.5, and rows of long contexts come in small batches.
constexpr int kChosenWhole = 16, kChosenLeast = 8;

// Steps of each run of an entry in wgs workgroups of columns, whose shortest columns take n0 steps and whose longest n. A CU takes
// two workgroups at once, in 1.2 times the time of two halves' sum alone, and a run costs five steps beside its own; the runs go
// round by round over the CUs. In us, with as many runs as 512 workgroups make and with the rule's: 8B, 700 rows up to 20,000 478 and
// 455, 1,300 863 and 758, 2,500 1,579 and 1,403; 600 up to 3,000 94 and 79; 1B, 700 up to 9,000 164 and 136. Where most positions are
// the rows' own, the workgroups, longest and shortest in turn, even out by themselves (1,300 from 0 59 us; in two runs 80).
static int many_per(int n0, int n, int64_t wgs) {
  if (2 * n0 < n) {
    const int64_t S = wgs >= 256 ? 1 : 512 / wgs;
    return ceil_div(n, std::min({S, (int64_t)n, (int64_t)kPgRuns / 2}));
  }
  constexpr double kRunSteps = 5, kAlone = 1.2;
  const double work = 0.5 * ((double)n0 + n) * wgs;
  int best = n;
  double least = INFINITY;
  for (int S = 1; S <= n && S <= kPgRuns / 2 && (S == 1 || S * wgs < 8 * 256); S++) {
    const int per = ceil_div(n, S);
    if (ceil_div(n, per) != S) continue;
    const double runs = S == 1 ? wgs : 0.5 * wgs * (ceil_div(n0, per) + S);
    const int64_t rounds = (int64_t)ceil(runs / 256);
    const double t = (work / runs + kRunSteps) * (rounds == 1 ? kAlone : rounds & 1 ? rounds + 0.5 * (kAlone - 1) : rounds);
    if (t < least) {
      least = t;
      best = per;
    }
  }
  return best;
}

// Whether a prefix is read once for all rows: where what its entries would read of it, a pass for each 16 of their columns, is more
// than 2^18 positions of keys and values (in all KV heads); else the join that it needs costs more, and each entry reads it for
// itself, from the caches after the first (7 rows of 8B on 2,048: 72 MB asked of the L2, 17 MB not there, what all entries' pages
// hold together). At the border, in us, read once and by each entry: 8B, 16 rows on 2,048 19.2 and 16.9, on
// 4,096 20.8 and 28.1; 2 on 8,192 19.0 and 16.6, on 16,384 22.2 and 27.2; 64 on 512 24.4 and 19.7, on 1,024 26.4 and 33.0, but 110 on
// 512 38.4 and 34.7, so 1,024 at least. Entries that fill the workgroups by themselves (four of 300 rows on 4,096: 243 and 204;
// of 100 83 and 104) gain nothing.
static bool prefix_pays(const PagePool &p, const PageRows &r, int G, int prefix) {
  int64_t passes = 0;
  for (int i = 0; i < r.n; i++) passes += ceil_div((int64_t)r.rows(i) * G, kFewCols);
  return prefix >= 1024 && (double)passes * prefix * p.KH > 0x1p18 && (int64_t)r.row0[r.n] * G <= (int64_t)1024 * r.n;
}

// The launches of a call.
struct PagedLaunches {
  PagedPlan few, many;
  PagedRuns runs;
  int records = 0, most_runs = 0;  // records of a head, runs of a row that has some
};

// most: the pages that a row may take (0: all positions).
static void paged_launches(const PagePool &p, const PageRows &r, int H, int prefix, int most, PagedLaunches &L) {
  const int G = H / p.KH, rows = r.row0[r.n], upp = p.page / kPgUnit;
  if (prefix && !prefix_pays(p, r, G, prefix)) prefix = 0;
  L.few.alone = L.many.alone = !prefix;
  L.few.base = L.many.base = prefix / kPgUnit;
  L.few.flat0 = L.few.flat1 = L.many.flat0 = L.many.flat1 = 0;
  L.runs.pre = L.runs.pre_rec = 0;
  if (prefix) {
    PageRows all;  // the rows of all entries, without a mask
    all.n = 1;
    all.seq[0] = r.seq[0];
    all.pos[0] = prefix - 1;
    all.row0[0] = 0;
    all.row0[1] = rows;
    const bool f = is_few((int64_t)rows * G, prefix, prefix, p.KH);
    PagedPlan &U = f ? L.few : L.many;
    const int blocks = ceil_div((int64_t)rows * G, f ? kFewCols : kManyCols), n = ceil_div(prefix / kPgUnit, f ? 2 : kManyUnits);
    const int per = f ? few_per(n, p.KH * blocks, kFewWaves, kFewWaves) : many_per(n, n, (int64_t)p.KH * blocks);
    L.runs.pre = ceil_div(n, per);
    U.it.add(all, 0, L.runs.pre * blocks, per, 0, L.runs.pre);
    U.flat1 = U.it.items;
    L.records = rows * L.runs.pre;
  }
  struct {
    bool few;
    int items, per, runs;
  } e[kPgRows];
  int order[kPgRows], n = 0, many = 0;
  for (int i = 0; i < r.n; i++) {
    const int T = r.rows(i), last = r.pos[i] + T - 1;
    if (!T) continue;
    const int64_t NC = (int64_t)T * G;
    const bool f = most || is_few(NC, r.pos[i] - prefix, last - prefix, p.KH);
    int blocks, per, runs;
    if (most) {  // rows one by one, cut by a rule on the choice alone
      const int took = std::min((last >> p.shift) + 1, most);
      blocks = T * ceil_div(G, kFewCols);
      per = few_per(ceil_div((int64_t)most * upp, 2), p.KH * ceil_div(G, kFewCols), kChosenWhole, kChosenLeast);
      runs = ceil_div(ceil_div((int64_t)took * upp, 2), per);
    } else {
      const int units = (last >> 4) - prefix / kPgUnit + 1, n = ceil_div(units, f ? 2 : kManyUnits);
      const int n0 = ceil_div((r.pos[i] >> 4) - prefix / kPgUnit + 1, kManyUnits);
      blocks = ceil_div(NC, f ? kFewCols : kManyCols);
      per = f ? few_per(n, p.KH * blocks, kFewWhole, kFewLeast) : many_per(n0, n, (int64_t)p.KH * blocks);
      runs = ceil_div(n, per);
    }
    e[i] = {f, runs * blocks, per, runs};
    order[n++] = i;
    many += !f;
  }
  // the longest runs first, so that the short ones fill the end (prompts of 2,001, 667 and 50 rows 505 -> 492 us)
  if (many > 1) std::stable_sort(order, order + n, [&](int a, int b) { return e[a].per > e[b].per; });
  for (int k = 0; k < n; k++) {
    const int i = order[k], T = r.rows(i);
    (e[i].few ? L.few : L.many).it.add(r, i, e[i].items, e[i].per, L.records, e[i].runs);
    if (e[i].runs == 1 && !prefix) continue;
    L.runs.it.add(r, i, T, 0, L.records, e[i].runs);
    L.records += T * e[i].runs;
    L.most_runs = std::max(L.most_runs, L.runs.pre + e[i].runs);
  }
}

int64_t paged_attention_scratch_floats(const PagePool &p, const PageRows &r, int H, int prefix, int most) {
  if (r.row0[r.n] <= 0) return 0;
  PagedLaunches L;
  paged_launches(p, r, H, prefix, most, L);
  return (int64_t)L.records * H * (p.HD + 4);
}

template <int HD>
static hipError_t paged_attend(const PagePool &p, const PageRows &r, const float *q, int H, int prefix, const int32_t *blocks,
                               int most, float scale, float *part, float *out, hipStream_t st) {
  PagedLaunches L;
  paged_launches(p, r, H, prefix, most, L);
  const int G = H / p.KH;
  hipError_t e = hipSuccess;
  if (L.many.it.n) {
    hipLaunchKernelGGL(paged_many_kernel<HD>, dim3((unsigned)L.many.it.items * p.KH), dim3(64 * kManyWaves), 0, st, p, L.many, q,
                       G, scale, part, out);
    e = hipGetLastError();
  }
  if (e == hipSuccess && L.few.it.n) {
    const dim3 grid((unsigned)L.few.it.items * p.KH), block(64 * kFewWaves);
    if (blocks)
      hipLaunchKernelGGL((paged_few_kernel<HD, true>), grid, block, 0, st, p, L.few, q, G, blocks, most, scale, part, out);
    else
      hipLaunchKernelGGL((paged_few_kernel<HD, false>), grid, block, 0, st, p, L.few, q, G, nullptr, 0, scale, part, out);
    e = hipGetLastError();
  }
  if (e != hipSuccess || !L.records) return e;
  // many rows of few runs: a workgroup each would be idle for the most part (667 rows of
  // 32 heads and 3 runs among others 34.0 -> 16.2 us)
  const int64_t pairs = (int64_t)L.runs.it.items * H;
  if (L.most_runs <= 64 && (L.most_runs <= 8 || pairs >= 1024))
    hipLaunchKernelGGL(paged_join_rows_kernel<HD>, dim3((unsigned)((pairs + 3) / 4)), dim3(256), 0, st, part, H, L.runs, out);
  else
    hipLaunchKernelGGL(paged_join_kernel<HD>, dim3((unsigned)pairs), dim3(256), 0, st, part, H, L.runs, out);
  return hipGetLastError();
}

hipError_t paged_attention_launch(const PagePool &p, const PageRows &r, const float *q, int H, int prefix,
                                  const int32_t *blocks, int most, float scale, float *scratch, float *out, hipStream_t st) {
  if (r.row0[r.n] <= 0) return hipSuccess;
  return p.HD == 64 ? paged_attend<64>(p, r, q, H, prefix, blocks, most, scale, scratch, out, st)
                    : paged_attend<128>(p, r, q, H, prefix, blocks, most, scale, scratch, out, st);
}

}  // namespace wl
