// wl_paged.hip - rows rotated into the pages of a KV cache, and back (wl_paged.h).
#include "wl_paged.h"

#include "wl_paged_device.h"
#include "wl_rope.h"

#include <math.h>

#pragma clang fp contract(off)

namespace wl {

// Values (of q and k) up to which a call's rows go by themselves, past which by units: 8B in us 20.2 and 23.1 at 1,536 rows, 24.8 and
// 24.6 at 2,048; 70B 20.8 and 22.5 at 1,024, 28.2 and 30.5 at 1,536 of 64 sequences, 26.6 and 25.3 at 1,500 of one; 1B 13.3 and 20.1
// at 2,000.
constexpr int64_t kPgRowValues = (int64_t)10 << 20;
// Query heads of a row that share a wave and its angles: one row of 8B takes 5.2 us as with two each, 110 rows of 70B 8.5 (12.5).
constexpr int kPgRowHeads = 8;

struct StoreArgs {
  PagePool p;
  PageRope e;
  const float *q, *k, *v;
  float *qr;
  int H, parts, each;  // parts of a row or unit, query heads of a unit's each
};

__device__ __forceinline__ uint16_t half_of(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
__device__ __forceinline__ uint32_t halves_of(float x, float y) { return half_of(x) | (uint32_t)half_of(y) << 16; }

// The two values of a head that lane pair x turns: (2 x, 2 x + 1), or (x, x + n / 2) among a NeoX head's first n; what is not
// rotated goes in twos.
struct Pair {
  int a, b;
  bool turns;
  __device__ Pair(const PageRope &e, int x) : turns(x < e.n / 2) {
    a = e.neox && turns ? x : 2 * x;
    b = e.neox && turns ? x + e.n / 2 : 2 * x + 1;
  }
  __device__ __forceinline__ float2 load(const float *h) const { return make_float2(h[a], h[b]); }
  __device__ __forceinline__ float2 turn(float2 v, float c, float s) const {
    return turns ? make_float2(v.x * c - v.y * s, v.x * s + v.y * c) : v;
  }
};

// The smaller or larger of each; a NaN stays.
__device__ __forceinline__ fh8 least(fh8 a, fh8 b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ fh8 most(fh8 a, fh8 b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ fh8 lane_swap(fh8 v, int m) {
  u32x4_t w = __builtin_bit_cast(u32x4_t, v);
#pragma unroll
  for (int e = 0; e < 4; e++) w[e] = __shfl_xor(w[e], m, 64);
  return __builtin_bit_cast(fh8, w);
}

// Few rows: a wave per part of a row, kPgRowHeads query heads or the keys and values of one KV head (two of 64), a lane per pair, so
// that the heads of a part share its angles. With one row of each sequence the waves of the keys also make their page's bounds.
// Latency bounds it: one row of 32 + 8 heads of 128 5.2 us, of which a launch takes 4.9; 64 rows of 64 + 8 with bounds
// 6.3, whose pages' keys are loaded beside the row (after it 7.9).
template <int HD, bool BOUNDS>
__global__ __launch_bounds__(64) void paged_rows_kernel(StoreArgs A, PageItems U) {
  constexpr int NP = HD / 2, HS = 64 / NP, N = kPgRowHeads / HS;  // pairs, heads at once, and of a part one after the other
  __shared__ double theta[NP];
  __shared__ __attribute__((aligned(16))) uint16_t fresh[HS][HD];
  const int lane = threadIdx.x, x = lane % NP, sub = lane / NP, KH = A.p.KH;
  const int row = blockIdx.x / A.parts, part = blockIdx.x % A.parts, half = A.e.n / 2;
  const PageEntry E = entry_of(U, row);
  const int p = E.pos + row - E.row0, off = p & (A.p.page - 1);
  const Pair pr(A.e, x);
  const int q_parts = A.parts - (KH + HS - 1) / HS;
  const bool isq = part < q_parts;
  const int h0 = isq ? part * kPgRowHeads : (part - q_parts) * HS;
  const float freq = A.e.freqs && x < half ? A.e.freqs[x] : 1.f;
  // loads first, then the angles
  float2 v[N], w = make_float2(0.f, 0.f);
  int id = -1;
  // the page's keys, 16 bytes a lane: eight channels lane / 8 (+ 8 for every other piece of a head of 128) of position slot (+ 4)
  constexpr int SETS = HD / 64, AHEAD = 4;  // units loaded before the angles are made
  const int slot = (lane >> 2 & 1) * 8 + (lane & 3);
  fh8 ahead[HS][AHEAD][2 * SETS];
  if (isq) {
#pragma unroll
    for (int e = 0; e < N; e++) {
      const int h = h0 + e * HS + sub;
      if (h < A.H) v[e] = pr.load(A.q + ((int64_t)row * A.H + h) * HD);
    }
  } else {
    id = A.p.id(E.seq, p >> A.p.shift);
    const int64_t r = ((int64_t)row * KH + (h0 + sub < KH ? h0 + sub : KH - 1)) * HD;
    v[0] = pr.load(A.k + r);
    w = make_float2(A.v[r + 2 * x], A.v[r + 2 * x + 1]);
    if (BOUNDS && id >= 0) {
#pragma unroll
      for (int g = 0; g < HS; g++) {
        const uint16_t *K = A.p.K + A.p.at(id, h0 + g < KH ? h0 + g : KH - 1) + lane * 8;
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
#pragma unroll
          for (int e = 0; e < 2 * SETS; e++)
            if (16 * u + slot + 4 * (e / SETS) < off) ahead[g][u][e] = *reinterpret_cast<const fh8 *>(K + u * 16 * HD + e * 512);
      }
    }
  }
  float c = 1.f, s = 0.f;
  if (half) {
    if (lane == 0) rope_chain<1>(theta, 0, p, half, A.e.theta_scale, A.e.freq_scale);
    __syncthreads();
    rope_cs_of(theta[x < half ? x : 0], freq, A.e.freqs != nullptr, c, s);
  }
  if (isq) {
#pragma unroll
    for (int e = 0; e < N; e++) {
      const int h = h0 + e * HS + sub;
      if (h < A.H) {
        const float2 y = pr.turn(v[e], c, s);
        float *o = A.qr + ((int64_t)row * A.H + h) * HD;
        o[pr.a] = y.x;
        o[pr.b] = y.y;
      }
    }
    return;
  }
  if (id < 0) return;  // uniform
  const float2 y = pr.turn(v[0], c, s);
  fresh[sub][pr.a] = half_of(y.x);
  fresh[sub][pr.b] = half_of(y.y);
  if (h0 + sub < KH) {
    const int64_t at = A.p.at(id, h0 + sub);
    A.p.K[at + pg_key(off, pr.a, HD)] = half_of(y.x);
    A.p.K[at + pg_key(off, pr.b, HD)] = half_of(y.y);
    A.p.V[at + pg_val(off, 2 * x, HD)] = half_of(w.x);
    A.p.V[at + pg_val(off, 2 * x + 1, HD)] = half_of(w.y);
  }
  if constexpr (!BOUNDS) return;
  __syncthreads();
#pragma unroll
  for (int g = 0; g < HS; g++) {
    if (h0 + g >= KH) break;
    const uint16_t *K = A.p.K + A.p.at(id, h0 + g) + lane * 8;
    fh8 lo[SETS], hi[SETS];
#pragma unroll
    for (int e = 0; e < SETS; e++) lo[e] = hi[e] = *reinterpret_cast<const fh8 *>(&fresh[g][64 * e + lane / 8 * 8]);
    auto take = [&](fh8 k, int e) __attribute__((always_inline)) {
      lo[e % SETS] = least(lo[e % SETS], k);
      hi[e % SETS] = most(hi[e % SETS], k);
    };
#pragma unroll
    for (int u = 0; u < AHEAD; u++)
#pragma unroll
      for (int e = 0; e < 2 * SETS; e++)
        if (16 * u + slot + 4 * (e / SETS) < off) take(ahead[g][u][e], e);
    for (int u = AHEAD; 16 * u < off; u++)
#pragma unroll
      for (int e = 0; e < 2 * SETS; e++)
        if (16 * u + slot + 4 * (e / SETS) < off) take(*reinterpret_cast<const fh8 *>(K + u * 16 * HD + e * 512), e);
#pragma unroll
    for (int e = 0; e < SETS; e++) {
#pragma unroll
      for (int m = 1; m <= 4; m <<= 1) {
        lo[e] = least(lo[e], lane_swap(lo[e], m));
        hi[e] = most(hi[e], lane_swap(hi[e], m));
      }
      uint16_t *b = A.p.bounds + ((int64_t)id * KH + h0 + g) * 2 * HD + 64 * e + lane / 8 * 8;
      if ((lane & 7) == 0) *reinterpret_cast<fh8 *>(b) = lo[e];
      if ((lane & 7) == 1) *reinterpret_cast<fh8 *>(b + HD) = hi[e];
    }
  }
}

// Prompts: a workgroup per part of a unit of 16 positions, a wave per position. The products of the angles once (a lane per
// position), the heads' rows by their waves; keys and values of two KV heads at a time go through LDS and leave as whole pieces of the
// page, a value's eight positions together. HBM bounds it: 4,248 rows of 32 + 8 heads of 128 32.4 us, 5.9 TB/s in and out.
template <int HD>
__global__ __launch_bounds__(1024) void paged_units_kernel(StoreArgs A, PageItems U) {
  constexpr int NP = HD / 2, HS = 64 / NP, LD = HD + 8, PIECES = 2 * HD;  // 16-byte pieces of a unit's keys
  __shared__ double theta[64 * 16];
  __shared__ __attribute__((aligned(16))) uint16_t ks[2][16 * LD], vs[2][16 * LD];
  const int tid = threadIdx.x, lane = tid & 63, r = __builtin_amdgcn_readfirstlane(tid >> 6), x = lane % NP, sub = lane / NP;
  const int KH = A.p.KH, half = A.e.n / 2;
  const int item = blockIdx.x / A.parts, part = blockIdx.x % A.parts;
  const PageEntry E = entry_of(U, item);
  const int u = (E.pos >> 4) + item - E.off, p = 16 * u + r;
  const bool on = p >= E.pos && p < E.pos + E.rows;
  const int64_t row = (int64_t)E.row0 + (on ? p - E.pos : 0);
  const int id = A.p.id(E.seq, 16 * u >> A.p.shift);
  const Pair pr(A.e, x);
  const float freq = A.e.freqs && x < half ? A.e.freqs[x] : 1.f;
  float c = 1.f, s = 0.f;
  if (half) {
    if (tid < 16) rope_chain<16>(theta, tid, 16 * u + tid, half, A.e.theta_scale, A.e.freq_scale);
    __syncthreads();
    rope_cs_of(theta[(x < half ? x : 0) * 16 + r], freq, A.e.freqs != nullptr, c, s);
  }
  if (on) {
    const int h1 = (part + 1) * A.each < A.H ? (part + 1) * A.each : A.H;
    for (int h = part * A.each + sub; h < h1; h += 4 * HS) {
      float2 v[4];
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (h + e * HS < h1) v[e] = pr.load(A.q + (row * A.H + h + e * HS) * HD);
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (h + e * HS < h1) {
          const float2 y = pr.turn(v[e], c, s);
          float *o = A.qr + (row * A.H + h + e * HS) * HD;
          o[pr.a] = y.x;
          o[pr.b] = y.y;
        }
    }
  }
  if (id < 0) return;  // uniform over the workgroup
  const int k1 = (int)((int64_t)(part + 1) * KH / A.parts);
  for (int h0 = (int)((int64_t)part * KH / A.parts); h0 < k1; h0 += 2) {
    __syncthreads();  // the heads before are written
    if (on)
      for (int g = sub; g < 2; g += HS)
        if (h0 + g < k1) {
          const int64_t at = (row * KH + h0 + g) * HD;
          const float2 y = pr.turn(pr.load(A.k + at), c, s);
          ks[g][r * LD + pr.a] = half_of(y.x);
          ks[g][r * LD + pr.b] = half_of(y.y);
          *reinterpret_cast<uint32_t *>(&vs[g][r * LD + 2 * x]) = halves_of(A.v[at + 2 * x], A.v[at + 2 * x + 1]);
        }
    __syncthreads();
    // pieces of the first head's keys, its values, and so the second's
    for (int e = tid; e < 4 * PIECES; e += 1024) {
      const int g = e / (2 * PIECES), c8 = e % PIECES;
      if (h0 + g >= k1) break;
      const int64_t to = A.p.at(id, h0 + g) + (int64_t)(u & ((A.p.page >> 4) - 1)) * 16 * HD + c8 * 8;
      if (e / PIECES % 2 == 0) {
        const int off = (c8 >> 2 & 1) * 8 + c8 / HD * 4 + (c8 & 3), oct = c8 / 8 % (HD / 8), at = 16 * u + off;
        if (at >= E.pos && at < E.pos + E.rows)
          *reinterpret_cast<u32x4_t *>(A.p.K + to) = *reinterpret_cast<const u32x4_t *>(&ks[g][off * LD + oct * 8]);
      } else {
        const int o8 = c8 / HD * 8, d = c8 % HD, at = 16 * u + o8;
        uint16_t w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = vs[g][(o8 + j) * LD + d];
        if (at >= E.pos && at <= E.pos + E.rows - 8) {
          u32x4_t y;
#pragma unroll
          for (int j = 0; j < 4; j++) y[j] = w[2 * j] | (uint32_t)w[2 * j + 1] << 16;
          *reinterpret_cast<u32x4_t *>(A.p.V + to) = y;
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (at + j >= E.pos && at + j < E.pos + E.rows) A.p.V[to + j] = w[j];
        }
      }
    }
  }
}

// The bounds of the pages written to: a workgroup per page and KV head, 16 bytes of keys a thread and step, from the caches that
// the rows were just written to (4,248 rows of 8 heads in pages of 16: 6.1 us).
__global__ __launch_bounds__(256) void paged_bounds_kernel(PagePool P, PageItems U) {
  __shared__ fh8 lo[4][16], hi[4][16];
  const int kvh = blockIdx.x % P.KH, item = blockIdx.x / P.KH, tid = threadIdx.x, HD = P.HD, oct = tid / 8 % (HD / 8);
  const PageEntry E = entry_of(U, item);
  const int j = (E.pos >> P.shift) + item - E.off;
  const int id = P.id(E.seq, j);
  if (id < 0) return;  // uniform
  const int last = E.pos + E.rows - 1 - (j << P.shift);  // of the page; past it where the page is full
  const uint16_t *K = P.K + P.at(id, kvh);
  const _Float16 inf = (_Float16)INFINITY;
  fh8 l, h;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    l[e] = inf;
    h[e] = -inf;
  }
  for (int c = tid; c < P.page * HD / 8; c += 256) {
    const int u = c / (2 * HD), t = c / HD & 1, s = c & 7;
    if (16 * u + 8 * (s >> 2) + 4 * t + (s & 3) > last) continue;
    const fh8 x = *reinterpret_cast<const fh8 *>(K + 8 * c);
    l = least(l, x);
    h = most(h, x);
  }
  // the eight positions of a piece, then the threads that hold the same channels (2 or 4 of each)
#pragma unroll
  for (int m = 1; m <= 4; m <<= 1) {
    l = least(l, lane_swap(l, m));
    h = most(h, lane_swap(h, m));
  }
  if ((tid & 7) == 0) {
    lo[tid / HD][oct] = l;
    hi[tid / HD][oct] = h;
  }
  __syncthreads();
  if (tid >= HD / 4) return;
  const int o = tid % (HD / 8);
  const bool up = tid >= HD / 8;
  fh8 m = up ? hi[0][o] : lo[0][o];
  for (int e = 1; e < 256 / HD; e++) m = up ? most(m, hi[e][o]) : least(m, lo[e][o]);
  *reinterpret_cast<fh8 *>(P.bounds + (((int64_t)id * P.KH + kvh) * 2 + up) * HD + 8 * o) = m;
}

// Rows as they were, a value a thread: for tests and for moving a sequence elsewhere, nothing that a step waits for.
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
  PageItems each, units, pages;
  int T = 0;
  for (int i = 0; i < r.n; i++) {
    const int t = r.rows(i), last = r.pos[i] + t - 1;
    T = T > t ? T : t;
    each.add(r, i, t);
    units.add(r, i, t ? (last >> 4) - (r.pos[i] >> 4) + 1 : 0);
    pages.add(r, i, t ? (last >> p.shift) - (r.pos[i] >> p.shift) + 1 : 0);
  }
  StoreArgs A{p, rope, q, k, v, qr, H, 0, 0};
  if (T == 1 || (int64_t)rows * (H + p.KH) * p.HD <= kPgRowValues) {
    const int hs = 128 / p.HD;  // heads of a wave at once
    A.parts = (H + kPgRowHeads - 1) / kPgRowHeads + (p.KH + hs - 1) / hs;
    const dim3 grid((unsigned)((int64_t)rows * A.parts));
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64), 0, st, A, each); };
    const bool bounds = p.bounds && T == 1;  // rows of a page, by several waves, cannot
    if (p.HD == 64) bounds ? run(paged_rows_kernel<64, true>) : run(paged_rows_kernel<64, false>);
    else bounds ? run(paged_rows_kernel<128, true>) : run(paged_rows_kernel<128, false>);
  } else {
    // Parts of a unit, of a KV head or a query head at least: as many as give every CU six workgroups (4,248 rows of 32 + 8 heads
    // of 128 39.5 us, 4.8 TB/s; two 52.2, eight 41.9, sixteen, whose angles are made as often, 59.6).
    const int most = p.KH > H ? p.KH : H;
    A.parts = 1536 / units.items;
    A.parts = A.parts < 1 ? 1 : A.parts > most ? most : A.parts;
    A.each = (H + A.parts - 1) / A.parts;
    const dim3 grid((unsigned)((int64_t)units.items * A.parts));
    if (p.HD == 64) hipLaunchKernelGGL(paged_units_kernel<64>, grid, dim3(1024), 0, st, A, units);
    else hipLaunchKernelGGL(paged_units_kernel<128>, grid, dim3(1024), 0, st, A, units);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.bounds || T == 1) return e;
  hipLaunchKernelGGL(paged_bounds_kernel, dim3(pages.items * p.KH), dim3(256), 0, st, p, pages);
  return hipGetLastError();
}

hipError_t paged_read_launch(const PagePool &p, int seq, int pos0, int T, float *k, float *v, hipStream_t st) {
  const int64_t n = (int64_t)T * p.KH * p.HD;
  if (n <= 0) return hipSuccess;
  hipLaunchKernelGGL(paged_read_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p, seq, pos0, T, k, v);
  return hipGetLastError();
}

}  // namespace wl
