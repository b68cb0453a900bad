// wl_paged_select.hip - the pages that a row and KV head attends to, by a bound of their scores (wl_paged.h).
//
// The score of a page is the largest, over the heads g of the group, of sum_d max(q_gd, 0) hi_d + min(q_gd, 0) lo_d: a product
// of the heads' [2 HD] halves with the pages', in 64 bits on v_mfma_f64_4x4x4_f64 (four heads to 16 pages), since which page is
// taken must not hang on a rounding (a product of a 24-bit query and an 11-bit bound is exact, a sum of 256 of them off by 2^-45
// of its terms). Scores are kept as whole numbers of the same order, and the pages taken are those from a border (score, page) on, found by
// histograms of a narrowing range.
#include "wl_paged.h"

#include "wl_paged_device.h"

#include <algorithm>

#pragma clang fp contract(off)

namespace wl {

constexpr int kScorePages = 64;  // of a workgroup, 16 a wave

// Pages from .. to - 1 are open to choice for a row whose own page is cur.
struct OpenPages {
  int from, to;
  __host__ __device__ OpenPages(const PageSelect &s, int cur) {
    from = s.first < cur + 1 ? s.first : cur + 1;
    to = s.recent > cur + 1 - from ? from : cur + 1 - s.recent;
  }
};

// A whole number in the order of x, a score that is not finite as +inf; 0 is no page.
__device__ __forceinline__ uint64_t score_key(double x) {
  x = __builtin_isfinite(x) ? x : INFINITY;
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  return b >> 63 ? ~b : b | 1ull << 63;
}

// A wave makes the scores of 16 pages: column l % 16 is a page, row l % 4 of four a head (past the group's last the last again),
// and lane l has the channels l / 16 * HD / 4 on of both, so that its loads are whole. The rows come out in lanes l / 16; the
// largest of a column is the page's score. The heads' halves lie in LDS in 64 bits: converting them in each wave took as long
// as the products. 16 rows of 70B on up to 500 pages of 64 take 12.9 us: 33 MB of bounds, and 6.6 us of products after them.
// Three waves a SIMD are named where the loops that follow a sum that is not finite would leave two.
template <int HD, int NB>
__global__ __launch_bounds__(256, HD == 64 ? 1 : NB == 2 ? 3 : 1) void paged_score_kernel(PagePool P, PageItems U, PageSelect S,
                                                          const float *__restrict__ q, int G, uint64_t *__restrict__ keys,
                                                          int64_t width) {
  constexpr int N = HD / 4;
  __shared__ double2 qs[NB * N * 16];  // [four heads][channel of a quarter][quarter][head]: (larger than 0, smaller)
  const int lane = threadIdx.x & 63, x = lane & 15, k = lane >> 4;
  const int kvh = blockIdx.x % P.KH, item = blockIdx.x / P.KH, H = G * P.KH;
  const PageEntry E = entry_of(U, item);  // per workgroups for each of its rows
  const int t = (item - E.off) / E.per, row = E.row0 + t;
  const OpenPages o(S, (E.pos + t) >> P.shift);
  const int j = o.from + (item - E.off) % E.per * kScorePages + (threadIdx.x >> 6) * 16 + x;
  const int id = j < o.to ? P.id(E.seq, j) : -1;
  const uint16_t *b = P.bounds + ((int64_t)(id < 0 ? 0 : id) * P.KH + kvh) * 2 * HD + k * N;
  fh8 lo[N / 8], hi[N / 8];
#pragma unroll
  for (int e = 0; e < N / 8; e++) {
    lo[e] = *reinterpret_cast<const fh8 *>(b + 8 * e);
    hi[e] = *reinterpret_cast<const fh8 *>(b + HD + 8 * e);
  }
  double best = -INFINITY;
  bool odd = false;
  for (int g0 = 0; g0 < G; g0 += 4 * NB) {
    if (g0) __syncthreads();
#pragma unroll
    for (int e = threadIdx.x; e < 4 * NB * HD; e += 256) {
      const int g = e / HD, d = e % HD;
      const float v = q[((int64_t)row * H + kvh * G + (g0 + g < G ? g0 + g : G - 1)) * HD + d];
      // a NaN goes with both
      qs[(g / 4 * N + d % N) * 16 + d / N * 4 + g % 4] = make_double2((double)(v < 0.f ? 0.f : v), (double)(v > 0.f ? 0.f : v));
    }
    __syncthreads();
    double up[NB], down[NB];
#pragma unroll
    for (int h = 0; h < NB; h++) up[h] = down[h] = 0.0;
#pragma unroll
    for (int e = 0; e < N; e++) {
      const double bh = (double)(float)hi[e / 8][e % 8], bl = (double)(float)lo[e / 8][e % 8];
#pragma unroll
      for (int h = 0; h < NB; h++) {
        const double2 a = qs[(h * N + e) * 16 + k * 4 + (lane & 3)];
        up[h] = __builtin_amdgcn_mfma_f64_4x4x4f64(a.x, bh, up[h], 0, 0, 0);
        down[h] = __builtin_amdgcn_mfma_f64_4x4x4f64(a.y, bl, down[h], 0, 0, 0);
      }
    }
#pragma unroll
    for (int h = 0; h < NB; h++) {
      const double s = up[h] + down[h];
      odd |= !__builtin_isfinite(s);
      best = fmax(best, __builtin_isfinite(s) ? s : INFINITY);
    }
  }
  if (__any(odd && id >= 0)) {
    // A bound or query is infinite or NaN, and the zero that stands for a query of the other sign makes NaN also of the infinite bound
    // that max(q lo, q hi) does not take. So by that itself, head by head, a quarter of the channels a lane: rare, and its loops
    // are small ones, since the products again would take twice the registers of all that is above.
    best = -INFINITY;
#pragma unroll 1
    for (int g = 0; g < G; g++) {
      const float *qp = q + ((int64_t)row * H + kvh * G + g) * HD + k * N;
      double s = 0.0;
#pragma unroll 1
      for (int c = 0; c < N; c += 8) {
        const fh8 l8 = *reinterpret_cast<const fh8 *>(b + c), h8 = *reinterpret_cast<const fh8 *>(b + HD + c);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const double x = (double)qp[c + e], low = x * (double)(float)l8[e], high = x * (double)(float)h8[e];
          s += low != low || low > high ? low : high;  // a NaN of either
        }
      }
      s += __shfl_xor(s, 16, 64);
      s += __shfl_xor(s, 32, 64);
      best = fmax(best, __builtin_isfinite(s) ? s : INFINITY);
    }
  }
  best = fmax(best, __shfl_xor(best, 16, 64));
  best = fmax(best, __shfl_xor(best, 32, 64));
  if (k == 0 && j < o.to) keys[((int64_t)row * P.KH + kvh) * width + j - o.from] = id < 0 ? 0 : score_key(best);
}

template <int HD>
static void score_launch(dim3 grid, const PagePool &p, const PageItems &U, const PageSelect &s, const float *q, int G,
                         uint64_t *keys, int64_t width, hipStream_t st) {
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p, U, s, q, G, keys, width); };
  if (G <= 4) run(paged_score_kernel<HD, 1>);
  else if (G <= 8) run(paged_score_kernel<HD, 2>);
  else run(paged_score_kernel<HD, 4>);
}

// Sum over the workgroup's threads up to and with this one, and of all.
template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int *sh, int &all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  // within rows of 16 lanes by shifts, then each row's last into the rows after it
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31), r2 = __builtin_amdgcn_readlane(v, 47);
  v += (lane >= 16 ? r0 : 0) + (lane >= 32 ? r1 : 0) + (lane >= 48 ? r2 : 0);
  __syncthreads();
  if (lane == 63) sh[w] = v;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; i++) {
    const int s = sh[i];
    v += i < w ? s : 0;
    all += s;
  }
  return v;
}

__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
  auto up = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  v = up(v, dpp32<0xB1>(v));
  v = up(v, dpp32<0x4E>(v));
  v = up(v, dpp32<0x124>(v));
  v = up(v, dpp32<0x128>(v));
  auto at = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
  return up(up(at(0), at(16)), up(at(32), at(48)));
}

// A workgroup per row and KV head. Thread t has pages t * m .. of the m = ceil(n / THREADS) each has, in registers up to kOwn of
// them. Its time is its passes' latency, so each thread has few: the whole call of a row with 8 KV heads takes 23.6 us on 4,096 pages
// and 31.9 on 8,190 by 1,024 threads of 8 pages each, 25.9 by 256 of 16, 26.0 and 38.1 where 1,024 read them again each pass; up to
// 1,024 pages 256 threads do as well (20.5 us on 940; 21.5 by 1,024).
template <int THREADS, int kOwn>
__global__ __launch_bounds__(THREADS) void paged_take_kernel(PagePool P, PageItems U, PageSelect S,
                                                             const uint64_t *__restrict__ keys, int64_t width,
                                                             int32_t *__restrict__ blocks) {
  constexpr int BINS = 1024;
  __shared__ int bins[BINS], sh[THREADS / 64], pick[3];
  __shared__ uint32_t ends[2][THREADS / 64];
  const int kvh = blockIdx.x % P.KH, row = blockIdx.x / P.KH, tid = threadIdx.x;
  const PageEntry E = entry_of(U, row);
  const int cur = (E.pos + row - E.row0) >> P.shift;
  const OpenPages o(S, cur);
  const int n = o.to - o.from, m = (n + THREADS - 1) / THREADS;
  const uint64_t *kp = keys + ((int64_t)row * P.KH + kvh) * width;
  int32_t *out = blocks + ((int64_t)row * P.KH + kvh) * S.most();
  uint64_t mine[kOwn > 0 ? kOwn : 1];
  if constexpr (kOwn > 0) {
#pragma unroll
    for (int e = 0; e < kOwn; e++) mine[e] = e < m && tid * m + e < n ? kp[tid * m + e] : 0;
  }
  // f(key, page) over the thread's pages that are there
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (kOwn > 0) {
#pragma unroll
      for (int e = 0; e < kOwn; e++)
        if (mine[e]) f(mine[e], tid * m + e);
    } else {
      for (int e = 0; e < m && (int64_t)tid * m + e < n; e++)
        if (const uint64_t v = kp[tid * m + e]) f(v, tid * m + e);
    }
  };
  int all = 0;
  uint32_t least = ~0u, most = 0;  // of the keys' high words
  each([&](uint64_t v, int) {
    all++;
    least = (uint32_t)(v >> 32) < least ? (uint32_t)(v >> 32) : least;
    most = (uint32_t)(v >> 32) > most ? (uint32_t)(v >> 32) : most;
  });
  least = ~wave_max_u(~least);
  most = wave_max_u(most);
  if ((tid & 63) == 0) {
    ends[0][tid >> 6] = least;
    ends[1][tid >> 6] = most;
  }
  (void)block_scan<THREADS>(all, sh, all);  // its barriers also order the ends
  for (int w = 0; w < THREADS / 64; w++) {
    least = ends[0][w] < least ? ends[0][w] : least;
    most = ends[1][w] > most ? ends[1][w] : most;
  }
  uint64_t lo = (uint64_t)least << 32, hi = (uint64_t)most << 32 | 0xffffffffu;
  // The border: pages of a key above `key`, and those of that key up to page `upto`. `need` of the pages in lo .. hi (by key, then,
  // among equal keys, by page from the last) are taken, and all above hi.
  uint64_t key = 0;
  int upto = -1, need = S.top;
  if (need >= all) {
    key = 0;
  } else if (need == 0) {
    key = ~0ull;
  } else {
    bool ties = false;
    for (;;) {
      const uint64_t span = hi - lo;
      const int shift = span >> 10 ? 54 - __builtin_clzll(span) : 0;  // span >> shift is below 1024
      for (int e = tid; e < BINS; e += THREADS) bins[e] = 0;
      __syncthreads();
      each([&](uint64_t v, int page) {
        const uint64_t w = ties ? ~(uint32_t)page : v;
        if ((!ties || v == key) && w >= lo && w <= hi) atomicAdd(&bins[(w - lo) >> shift], 1);
      });
      __syncthreads();
      // from the top: a thread has EACH bins
      constexpr int EACH = BINS / THREADS;
      int c[EACH], sum = 0, total;
#pragma unroll
      for (int e = 0; e < EACH; e++) sum += c[e] = bins[BINS - 1 - EACH * tid - e];
      int before = block_scan<THREADS>(sum, sh, total) - sum;
      if (before < need && before + sum >= need) {  // one thread
        int e = 0;
        while (before + c[e] < need) before += c[e++];
        pick[0] = BINS - 1 - EACH * tid - e;
        pick[1] = before;
        pick[2] = c[e];
      }
      __syncthreads();
      need -= pick[1];
      const int in = pick[2];
      lo += (uint64_t)pick[0] << shift;
      const uint64_t bin = (1ull << shift) - 1;
      hi = hi - lo < bin ? hi : lo + bin;
      if (in == need) {  // the whole bin
        if (ties) upto = (int)~(uint32_t)lo;
        else key = lo - 1;
        break;
      }
      if (shift == 0) {  // equal keys: by page, which ends with one page a bin
        ties = true;
        key = lo;
        lo = ~(uint32_t)(n - 1);
        hi = 0xffffffffu;
      }
    }
  }
  auto taken = [&](uint64_t v, int page) { return v > key || (v == key && page <= upto); };
  int count = 0, total;
  each([&](uint64_t v, int page) { count += taken(v, page); });
  int at = o.from + block_scan<THREADS>(count, sh, total) - count;
  each([&](uint64_t v, int page) {
    if (taken(v, page)) out[at++] = o.from + page;
  });
  for (int e = tid; e < o.from; e += THREADS) out[e] = e;
  const int rest = o.from + total, last = rest + cur + 1 - o.to;
  for (int e = rest + tid; e < S.most(); e += THREADS) out[e] = e < last ? o.to + e - rest : -1;
}

// Pages open to choice of any row of a call.
static int64_t open_width(const PagePool &p, const PageRows &r, const PageSelect &s) {
  int64_t w = 1;
  for (int i = 0; i < r.n; i++)
    if (r.rows(i)) {
      const OpenPages o(s, (r.pos[i] + r.rows(i) - 1) >> p.shift);
      w = std::max(w, (int64_t)o.to - o.from);
    }
  return w;
}

int64_t paged_select_scratch_bytes(const PagePool &p, const PageRows &r, const PageSelect &s) {
  return (int64_t)r.row0[r.n] * p.KH * open_width(p, r, s) * 8;
}

hipError_t paged_select_launch(const PagePool &p, const PageRows &r, const float *q, int H, const PageSelect &s,
                               void *scratch, int32_t *blocks, hipStream_t st) {
  const int rows = r.row0[r.n], G = H / p.KH;
  if (rows <= 0) return hipSuccess;
  const int64_t width = open_width(p, r, s);
  uint64_t *keys = (uint64_t *)scratch;
  PageItems U, each;
  for (int i = 0; i < r.n; i++) {
    const int T = r.rows(i);
    const OpenPages o(s, T ? (r.pos[i] + T - 1) >> p.shift : 0);
    const int per = (o.to - o.from + kScorePages - 1) / kScorePages;
    U.add(r, i, T * per, per);
    each.add(r, i, T);
  }
  if (U.n) {
    const dim3 grid((unsigned)((int64_t)U.items * p.KH));
    if (p.HD == 64) score_launch<64>(grid, p, U, s, q, G, keys, width, st);
    else score_launch<128>(grid, p, U, s, q, G, keys, width, st);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  const dim3 grid((unsigned)(rows * p.KH));
  auto take = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, st, p, each, s, keys, width, blocks);
  };
  if (width <= 256 * 4) take(paged_take_kernel<256, 4>, 256);
  else if (width <= 1024 * 8) take(paged_take_kernel<1024, 8>, 1024);
  else take(paged_take_kernel<1024, 0>, 1024);
  return hipGetLastError();
}

}  // namespace wl
