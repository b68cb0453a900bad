// wl_sample.hip - the next token of each row of logits by temperature, top-k, top-p, min-p and a given
// number u (Sampler.Sample, src/Engine.cs:353-382, the draw).
//
// Definition. Tokens in order: larger logit first, of equals the lower id. w = exp((l - max) / t).
// Kept is the longest prefix with at most top_k tokens, whose tokens before the last weigh less than
// top_p of the top_k tokens' weight, and w >= min_p; drawn is the first token at which the weight
// summed in that order passes u of the kept weight. Every step is a question about a prefix of that
// order, so nothing is sorted but the few tokens around a prefix's end.
//
// Arithmetic: weights in double (a polynomial for 2^f), cut to whole numbers of 2^-shift (2^-45 at 128,000
// tokens), so that sums are exact and do not depend on the order in which workgroups and atomics add them.
//
// Three launches. (1) Each part of 4,096 tokens of a row: its largest and least finite logit. (2) Each part: the count
// and weight of its tokens in 256 bins of equal width below the row's maximum (64 t wide at most, weights below e^-64
// in the last bin), its tokens' places by bin, and what has w >= min_p. (3) One workgroup a row adds the parts'
// bins and answers the questions: a prefix's end lies in one bin, whose tokens it gathers and narrows down by their
// bits; with top_k of few tokens it gathers the whole prefix and puts that in order.
//
// What bounds it: a row of 128,256 is read from HBM in launch 1 and from the caches after (64 rows, 33 MB: 6.4 us), then
// 64 rows' bins take 25.4 us (LDS atomics, the double polynomial and their latency) and their questions 20 (a workgroup a
// row, each question a few dependent loads). One row is three dependent launches: 2.5, 6.5 and 10.4 us.
#include "wl_sample.h"

#include "wl_device.h"

#include <math.h>

#pragma clang fp contract(off)

namespace wl {

constexpr int kSmBins = 256, kSmPart = 4096, kSmList = 4096, kSmFew = 64, kSmPrefix = 256, kSmGroup = 64;
typedef unsigned long long u64;

// A part's record.
struct SmPart {
  float top, low;       // largest logit (-inf: none), least finite one (+inf: none)
  unsigned minp_count;  // tokens with w >= min_p, and their weight
  u64 minp_mass;
};

// What the launches leave each other, by row and part.
struct SmScratch {
  SmPart *rec;
  u64 *mass;      // [bins] weights
  uint16_t *end;  // [bins] tokens in the bins up to each
  uint16_t *id;   // [kSmPart] the tokens' places in the part, by bin
};

// Order-preserving bits of a logit; -0 as 0.
__device__ __forceinline__ uint32_t sm_key(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sm_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// ln(2)^i / i!. Held in scalar registers past the compiler's sight: as plain constants they were moved to vector
// registers, two instructions before each of the polynomial's.
struct SmSeries {
  double c[12];
  __device__ __forceinline__ SmSeries()
      : c{1.0, 0.6931471805599453, 0.2402265069591007, 0.055504108664821576,
          0.009618129107628477, 0.0013333558146428441, 0.00015403530393381606, 1.5252733804059838e-05,
          1.3215486790144305e-06, 1.0178086009239696e-07, 7.054911620801121e-09, 4.44553827187081e-10} {
#pragma unroll
    for (int i = 0; i < 12; i++) asm("" : "+s"(c[i]));
  }
};

// What every launch after the first derives from the parts' records: the row's maximum and its bins.
struct SmRow {
  float m, R, c;  // the maximum (of infinity: the largest finite value), the bins' reach and scale
  double per;     // log2(e) / t; for t = 0 so large that only the maximum weighs anything
  int shift;
  __device__ void set(float top, float low, float t, int sh) {
    m = cap(top);
    shift = sh;
    per = t > 0.f ? fmin(1.4426950408889634 / (double)t, 1e300) : 1e300;
    R = fminf(fminf(m - low, 64.f * t), 3.4028235e38f);
    if (!(R > 1e-30f)) R = 0.f;  // the bins' scale stays finite; what lies lower is the last bin's
    c = R > 0.f ? (float)(kSmBins - 2) / R : 0.f;
  }
  __device__ static float cap(float l) { return fminf(l, 3.4028235e38f); }
  __device__ int bin(float l) const {
    const float d = m - cap(l);
    return d > R ? kSmBins - 1 : min((int)(d * c), kSmBins - 2);
  }
  // w in units of 2^-shift: 2^x for x = (l - m) log2(e) / t, as 2^k times 2^f, f in [-1/2, 1/2], by its series to the 11th
  // power (the rest is below 2^-47 of it), its significand shifted.
  __device__ __forceinline__ u64 mass(float l, const SmSeries &C) const {
    double x = ((double)cap(l) - (double)m) * per;
    x = fmax(x, -80.0);  // nothing is left there
    const double k = rint(x), f = x - k;
    double p = C.c[11];
#pragma unroll
    for (int i = 10; i >= 0; i--) p = __builtin_fma(p, f, C.c[i]);
    const u64 bits = __builtin_bit_cast(u64, p);
    const u64 sig = (bits & (((u64)1 << 52) - 1)) | (u64)1 << 52;
    const int down = 52 - shift - (int)k - ((int)(bits >> 52) - 1023);  // from 0 (shift <= 52)
    return sig >> (down < 63 ? down : 63);
  }
};

__device__ __forceinline__ void sm_row_of(const SmPart *__restrict__ part, int parts, float t, int shift, SmRow &r,
                                          float *sh) {
  // every thread of the workgroup; sh holds 2 floats
  if (threadIdx.x < 64) {
    float top = -INFINITY, low = INFINITY;
    for (int i = threadIdx.x; i < parts; i += 64) {
      top = fmaxf(top, part[i].top);
      low = fminf(low, part[i].low);
    }
    top = wave_max_f(top);
    low = -wave_max_f(-low);
    if (threadIdx.x == 0) {
      sh[0] = top;
      sh[1] = low;
    }
  }
  __syncthreads();
  r.set(sh[0], sh[1], t, shift);
}

// Running sums over the bins of 256 threads (all of the workgroup call it; sh holds 4 of each).
__device__ __forceinline__ void sm_scan(unsigned &c, u64 &m, unsigned *sc, u64 *sm) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const unsigned a = __shfl_up(c, s, 64);
    const u64 b = __shfl_up(m, s, 64);
    c += lane >= s ? a : 0;
    m += lane >= s ? b : 0;
  }
  if (lane == 63 && wv < 4) {
    sc[wv] = c;
    sm[wv] = m;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 3; w++) {
    c += w < wv ? sc[w] : 0;
    m += w < wv ? sm[w] : 0;
  }
}

__global__ __launch_bounds__(256) void sample_range_kernel(const float *__restrict__ logits, int64_t n, SmScratch X) {
  __shared__ float st[4], sl[4];
  const float *l = logits + (int64_t)blockIdx.y * n;
  const int64_t lo = (int64_t)blockIdx.x * kSmPart, hi = lo + kSmPart < n ? lo + kSmPart : n;
  float top = -INFINITY, low = INFINITY;
  float v[kSmPart / 256];
#pragma unroll
  for (int j = 0; j < kSmPart / 256; j++) {
    const int64_t i = lo + threadIdx.x + 256 * j;
    v[j] = l[i < hi ? i : hi - 1];
  }
#pragma unroll
  for (int j = 0; j < kSmPart / 256; j++) {
    top = v[j] > top ? v[j] : top;  // a NaN never compares greater
    low = __builtin_isfinite(v[j]) ? fminf(low, v[j]) : low;
  }
  top = wave_max_f(top);
  low = -wave_max_f(-low);
  if ((threadIdx.x & 63) == 0) {
    st[threadIdx.x >> 6] = top;
    sl[threadIdx.x >> 6] = low;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    SmPart &p = X.rec[(int64_t)blockIdx.y * gridDim.x + blockIdx.x];
    p.top = fmaxf(fmaxf(st[0], st[1]), fmaxf(st[2], st[3]));
    p.low = fminf(fminf(sl[0], sl[1]), fminf(sl[2], sl[3]));
  }
}

template <int WIDE>
__global__ __launch_bounds__(WIDE) void sample_bins_kernel(const float *__restrict__ logits, int64_t n, SampleSets sets,
                                                          int shift, SmScratch X) {
  constexpr int N = kSmPart / WIDE;
  __shared__ unsigned cn[kSmBins];
  __shared__ u64 ms[kSmBins];
  __shared__ __attribute__((aligned(16))) uint16_t ids[kSmPart];
  __shared__ float sh[2];
  __shared__ unsigned mc, sc[4];
  __shared__ u64 mm, sm[4];
  const int row = blockIdx.y, parts = gridDim.x, tid = threadIdx.x;
  const SampleSet set = sets.row[row];
  const float *l = logits + (int64_t)row * n;
  const int64_t lo = (int64_t)blockIdx.x * kSmPart, hi = lo + kSmPart < n ? lo + kSmPart : n;
  float v[N];
#pragma unroll
  for (int j = 0; j < N; j++) {
    const int64_t i = lo + tid + WIDE * j;
    v[j] = i < hi ? l[i] : __builtin_nanf("");
  }
  if (tid < kSmBins) {
    cn[tid] = 0;
    ms[tid] = 0;
  }
  if (tid == 0) {
    mc = 0;
    mm = 0;
  }
  SmRow r;
  sm_row_of(X.rec + (int64_t)row * parts, parts, set.temperature, shift, r, sh);
  const SmSeries C;
  const u64 least = (u64)ceil(ldexp((double)set.min_p, shift));
  unsigned at[N];  // the token's bin and its place there
  unsigned c = 0;
  u64 m = 0;
#pragma unroll
  for (int j = 0; j < N; j++) {
    at[j] = ~0u;
    const u64 M = r.mass(v[j], C);
    if (v[j] != v[j]) continue;
    const int b = r.bin(v[j]);
    at[j] = (unsigned)b << 16 | atomicAdd(&cn[b], 1u);
    if (M) atomicAdd(&ms[b], M);
    c += M >= least;
    m += M >= least ? M : 0;
  }
  if (set.min_p > 0.f) {  // uniform
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) {
      c += __shfl_xor(c, s, 64);
      m += __shfl_xor(m, s, 64);
    }
    if ((tid & 63) == 0) {
      atomicAdd(&mc, c);
      atomicAdd(&mm, m);
    }
  }
  __syncthreads();
  const int64_t part = (int64_t)row * parts + blockIdx.x;
  unsigned end = tid < kSmBins ? cn[tid] : 0;
  u64 none = 0;
  const unsigned mine = end;
  sm_scan(end, none, sc, sm);
  if (tid < kSmBins) {
    cn[tid] = end - mine;
    X.mass[part * kSmBins + tid] = ms[tid];
    X.end[part * kSmBins + tid] = (uint16_t)end;
  }
  if (tid == 0) {
    X.rec[part].minp_count = mc;
    X.rec[part].minp_mass = mm;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < N; j++)
    if (at[j] != ~0u) ids[cn[at[j] >> 16] + (at[j] & 0xffffu)] = (uint16_t)(tid + WIDE * j);
  __syncthreads();
  // places past the part's tokens hold nothing that is read
#pragma unroll
  for (int j = 0; j < (kSmPart / 8 + WIDE - 1) / WIDE; j++)
    if (tid + WIDE * j < kSmPart / 8)
      reinterpret_cast<uint4 *>(X.id + part * kSmPart)[tid + WIDE * j] = reinterpret_cast<const uint4 *>(ids)[tid + WIDE * j];
}

// A question: the shortest prefix with at least `count` tokens, or of at least `mass`, or of more.
enum SmAsk { SM_COUNT, SM_MASS, SM_OVER };
struct SmPrefix {
  unsigned count;
  u64 mass;
  int token;  // its last token
};

struct SmShared {
  unsigned cn[kSmBins];  // summed over the bins before and with this one
  u64 ms[kSmBins];
  unsigned sub_n[kSmBins];
  u64 sub_m[kSmBins];
  u64 list[kSmList];  // ~key, id of gathered tokens
  u64 few[kSmPrefix], weight[kSmPrefix];
  unsigned from[kSmGroup + 1];  // of a group of parts: where each part's gathered tokens begin
  uint16_t off[kSmGroup];       // and the first in the part's order
  unsigned used;
  int pick;
  uint32_t lo, hi;
  unsigned wave[16], sc[4];
  u64 sm[4];
  SmPrefix got;
  float f2[2];
};

__device__ __forceinline__ bool sm_yes(SmAsk a, u64 target, unsigned c, u64 m) {
  return a == SM_COUNT ? c >= target : a == SM_MASS ? m >= target : m > target;
}

struct SmView {
  const float *l;
  int64_t n;
  int parts;
  const uint16_t *end, *id;  // the row's
};

// f(key, id) for every token of the bins b0 .. b1, over the workgroup's threads (all of them call it). Parts in groups of
// 64: one wave lines up what each holds, then a thread takes every blockDim.x-th token of the group.
template <class F>
__device__ __forceinline__ void sm_each(SmShared &S, const SmView &V, int b0, int b1, const F &f) {
  const int tid = threadIdx.x, nt = blockDim.x;
  for (int g = 0; g < V.parts; g += kSmGroup) {
    if (tid < 64) {
      const int p = g + tid;
      unsigned first = 0, last = 0;
      if (p < V.parts) {
        first = b0 ? V.end[(int64_t)p * kSmBins + b0 - 1] : 0;
        last = V.end[(int64_t)p * kSmBins + b1];
      }
      unsigned sum = last - first;
#pragma unroll
      for (int s = 1; s < 64; s <<= 1) {
        const unsigned a = __shfl_up(sum, s, 64);
        sum += tid >= s ? a : 0;
      }
      S.off[tid] = (uint16_t)first;
      S.from[tid + 1] = sum;
      if (tid == 0) S.from[0] = 0;
    }
    __syncthreads();
    const unsigned all = S.from[kSmGroup];
    for (unsigned i = tid; i < all; i += nt) {
      int p = 0;  // the last part that begins at or before i
#pragma unroll
      for (int s = kSmGroup / 2; s >= 1; s >>= 1)
        if (S.from[p + s] <= i) p += s;
      const unsigned at = S.off[p] + (i - S.from[p]);
      const int64_t id = (int64_t)(g + p) * kSmPart + V.id[(int64_t)(g + p) * kSmPart + at];
      f(sm_key(V.l[id]), (uint32_t)id);
    }
    __syncthreads();
  }
}

// Few tokens (at most 64) of S.few in a wave's lanes: each one's place among them and the weight up to it.
__device__ __forceinline__ void sm_few(SmShared &S, SmAsk a, u64 target, unsigned in, unsigned c0, u64 m0,
                                       const SmRow &r) {
  const int tid = threadIdx.x;
  if (tid < 64) {
    const bool on = tid < (int)in;
    const u64 me = on ? S.few[tid] : ~(u64)0;
    const u64 w = on ? r.mass(sm_value(~(uint32_t)(me >> 32)), SmSeries()) : 0;
    unsigned place = 1;
    u64 sum = w;
    for (int i = 0; i < (int)in; i++) {
      const u64 o = S.few[i];
      const u64 ow = __shfl(w, i, 64);
      place += o < me ? 1u : 0u;
      sum += o < me ? ow : 0;
    }
    const bool y = on && sm_yes(a, target, c0 + place, m0 + sum);
    if (y && !sm_yes(a, target, c0 + place - 1, m0 + sum - w)) S.got = SmPrefix{c0 + place, m0 + sum, (int)(uint32_t)me};
  }
  __syncthreads();
}

// The prefix that answers (a, target): every thread of the workgroup calls it and gets the answer.
__device__ SmPrefix sm_answer(SmShared &S, SmAsk a, u64 target, const SmView &V, const SmRow &r, bool token) {
  const int tid = threadIdx.x, nt = blockDim.x;
  __syncthreads();
  if (tid < kSmBins) {
    const bool y = sm_yes(a, target, S.cn[tid], S.ms[tid]);
    if (y && (tid == 0 || !sm_yes(a, target, S.cn[tid - 1], S.ms[tid - 1]))) S.pick = tid;
  }
  if (tid == 0) {
    S.lo = 0xffffffffu;
    S.hi = 0;
    S.used = 0;
  }
  __syncthreads();
  const int bin = S.pick;
  unsigned c0 = bin ? S.cn[bin - 1] : 0, in = S.cn[bin] - c0;
  u64 m0 = bin ? S.ms[bin - 1] : 0;
  // a whole bin's prefix needs no token of it
  if (a == SM_COUNT && !token && c0 + in == target) return SmPrefix{c0 + in, S.ms[bin], 0};
  if (in <= kSmFew) {
    sm_each(S, V, bin, bin, [&](uint32_t key, uint32_t id) { S.few[atomicAdd(&S.used, 1u)] = (u64)~key << 32 | id; });
    sm_few(S, a, target, in, c0, m0, r);
    return S.got;
  }
  const bool listed = in <= kSmList;
  {
    uint32_t lo = 0xffffffffu, hi = 0;
    sm_each(S, V, bin, bin, [&](uint32_t key, uint32_t id) {
      if (listed) S.list[atomicAdd(&S.used, 1u)] = (u64)~key << 32 | id;
      lo = min(lo, key);
      hi = max(hi, key);
    });
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) {
      lo = min(lo, (uint32_t)__shfl_xor((int)lo, s, 64));
      hi = max(hi, (uint32_t)__shfl_xor((int)hi, s, 64));
    }
    if ((tid & 63) == 0) {
      atomicMin(&S.lo, lo);
      atomicMax(&S.hi, hi);
    }
  }
  __syncthreads();
  uint32_t lo = S.lo, hi = S.hi;
  const unsigned have = in;
  // every token of the bin whose key lies in [lo, hi]
  auto inside = [&](auto f) {
    if (listed) {
      for (unsigned i = tid; i < have; i += nt) {
        const uint32_t key = ~(uint32_t)(S.list[i] >> 32);
        if (key >= lo && key <= hi) f(key, (uint32_t)S.list[i]);
      }
    } else {
      sm_each(S, V, bin, bin, [&](uint32_t key, uint32_t id) {
        if (key >= lo && key <= hi) f(key, id);
      });
    }
  };
  while (in > kSmFew && lo < hi) {
    __syncthreads();
    if (tid < kSmBins) {
      S.sub_n[tid] = 0;
      S.sub_m[tid] = 0;
    }
    __syncthreads();
    const uint32_t width = (hi - lo) / kSmBins + 1;
    inside([&](uint32_t key, uint32_t) {
      const uint32_t b = (hi - key) / width;
      atomicAdd(&S.sub_n[b], 1u);
      atomicAdd(&S.sub_m[b], r.mass(sm_value(key), SmSeries()));
    });
    __syncthreads();
    unsigned c = tid < kSmBins ? S.sub_n[tid] : 0;
    u64 m = tid < kSmBins ? S.sub_m[tid] : 0;
    sm_scan(c, m, S.sc, S.sm);
    __syncthreads();
    if (tid < kSmBins) {
      S.sub_n[tid] = c;
      S.sub_m[tid] = m;
    }
    __syncthreads();
    if (tid < kSmBins) {
      const bool y = sm_yes(a, target, c0 + c, m0 + m);
      if (y && (tid == 0 || !sm_yes(a, target, c0 + S.sub_n[tid - 1], m0 + S.sub_m[tid - 1]))) S.pick = tid;
    }
    __syncthreads();
    const int b = S.pick;
    const unsigned cb = b ? S.sub_n[b - 1] : 0;
    in = S.sub_n[b] - cb;
    c0 += cb;
    m0 += b ? S.sub_m[b - 1] : 0;
    hi -= (uint32_t)b * width;
    lo = hi - lo >= width ? hi - width + 1 : lo;
  }
  __syncthreads();
  if (in <= kSmFew) {
    if (tid == 0) S.used = 0;
    __syncthreads();
    inside([&](uint32_t key, uint32_t id) { S.few[atomicAdd(&S.used, 1u)] = (u64)~key << 32 | id; });
    __syncthreads();
    sm_few(S, a, target, in, c0, m0, r);
    return S.got;
  }
  // equal logits: the prefix takes the first `need` of them by id
  const u64 w = r.mass(sm_value(lo), SmSeries());
  const u64 need64 = a == SM_COUNT ? target - c0
                     : w == 0      ? 1
                     : a == SM_MASS ? (target - m0 + w - 1) / w
                                    : (target - m0) / w + 1;
  const unsigned need = need64 < 1 ? 1 : need64 > in ? in : (unsigned)need64;
  SmPrefix g{c0 + need, m0 + need * w, 0};
  if (token) {
    unsigned before = 0;
    for (int64_t i0 = 0; i0 < V.n && before < need; i0 += nt) {
      const int64_t i = i0 + tid;
      const float v = i < V.n ? V.l[i] : 0.f;
      const bool y = i < V.n && v == v && sm_key(v) == lo;
      const u64 vote = __ballot(y);
      if ((tid & 63) == 0) S.wave[tid >> 6] = (unsigned)__popcll(vote);
      __syncthreads();
      unsigned at = before, all = 0;
      for (int k = 0; k < nt / 64; k++) {
        if (k < (tid >> 6)) at += S.wave[k];
        all += S.wave[k];
      }
      at += (unsigned)__popcll(vote & ((1ull << (tid & 63)) - 1));
      if (y && at + 1 == need) S.got.token = (int)i;
      before += all;
      __syncthreads();
    }
    __syncthreads();
    g.token = S.got.token;
  }
  return g;
}

// The weight that top_p of `mass` asks for, and the one that u of it passes.
__device__ __forceinline__ u64 sm_top_p(float p, u64 mass) {
  const u64 x = (u64)ceil((double)p * (double)mass);
  return x < 1 ? 1 : x > mass ? mass : x;
}
__device__ __forceinline__ u64 sm_draw(float u, u64 mass) {
  const double y = u > 0.f ? (double)u * (double)mass : 0.0;  // a NaN draws the first
  const u64 x = y < (double)mass ? (u64)y : mass;
  return x < mass ? x : mass - 1;
}

__global__ __launch_bounds__(1024) void sample_pick_kernel(const float *__restrict__ logits, int64_t n, int parts,
                                                           SampleSets sets, int shift, SmScratch X,
                                                           const float *__restrict__ us, int *__restrict__ out) {
  __shared__ SmShared S;
  const int row = blockIdx.x, tid = threadIdx.x;
  const SampleSet set = sets.row[row];
  const bool greedy = set.temperature == 0.f;
  const float u = us[row];
  SmView V;
  V.l = logits + (int64_t)row * n;
  V.n = n;
  V.parts = parts;
  const SmPart *rec = X.rec + (int64_t)row * parts;
  V.end = X.end + (int64_t)row * parts * kSmBins;
  V.id = X.id + (int64_t)row * parts * kSmPart;
  const u64 *masses = X.mass + (int64_t)row * parts * kSmBins;
  const float l0 = V.l[0];
  if (tid < kSmBins) {
    S.cn[tid] = 0;
    S.ms[tid] = 0;
  }
  // four threads a bin, each a quarter of the parts; the counts come as running sums
  unsigned c = 0;
  u64 m = 0;
  const int b = tid & (kSmBins - 1);
#pragma unroll 8
  for (int p = tid / kSmBins; p < parts; p += 4) {
    c += V.end[(int64_t)p * kSmBins + b];
    m += masses[(int64_t)p * kSmBins + b];
  }
  unsigned mpc = 0;
  u64 mpm = 0;
  if (set.min_p > 0.f)
    for (int p = 0; p < parts; p++) {
      mpc += rec[p].minp_count;
      mpm += rec[p].minp_mass;
    }
  SmRow r;
  sm_row_of(rec, parts, set.temperature, shift, r, S.f2);
  if (r.m == -INFINITY || (greedy && l0 != l0)) {  // as the greedy pick
    if (tid == 0) out[row] = 0;
    return;
  }
  {
    atomicAdd(&S.cn[b], c);
    atomicAdd(&S.ms[b], m);
    __syncthreads();
    m = tid < kSmBins ? S.ms[tid] : 0;
    c = 0;
    sm_scan(c, m, S.sc, S.sm);
    if (tid < kSmBins) S.ms[tid] = m;
    __syncthreads();
  }
  const unsigned all = S.cn[kSmBins - 1];
  SmPrefix kept{all, S.ms[kSmBins - 1], 0};
  const bool top_k = !greedy && set.top_k > 0 && (unsigned)set.top_k < all;
  if (top_k) {
    // the bins up to the one where top_k ends, put in order where they hold few tokens
    if (tid < kSmBins && S.cn[tid] >= (unsigned)set.top_k && (tid == 0 || S.cn[tid - 1] < (unsigned)set.top_k)) S.pick = tid;
    if (tid == 0) S.used = 0;
    __syncthreads();
    const int bin = S.pick;
    const unsigned in = S.cn[bin];
    if (in <= kSmPrefix) {
      sm_each(S, V, 0, bin, [&](uint32_t key, uint32_t id) { S.list[atomicAdd(&S.used, 1u)] = (u64)~key << 32 | id; });
      if (tid < (int)in) {  // to its place, by counting those before it
        const u64 me = S.list[tid];
        unsigned place = 0;
        for (unsigned i = 0; i < in; i++) place += S.list[i] < me ? 1u : 0u;
        S.few[place] = me;
      }
      __syncthreads();
      unsigned c = 0;
      u64 m = tid < (int)in ? r.mass(sm_value(~(uint32_t)(S.few[tid] >> 32)), SmSeries()) : 0;
      sm_scan(c, m, S.sc, S.sm);
      if (tid < (int)in) S.weight[tid] = m;  // up to and with the token
      __syncthreads();
      unsigned count = (unsigned)set.top_k;
      if (set.top_p < 1.f) {
        const u64 x = sm_top_p(set.top_p, S.weight[count - 1]);
        if (tid < (int)count && S.weight[tid] >= x && (tid == 0 || S.weight[tid - 1] < x)) S.pick = tid + 1;
        __syncthreads();
        count = (unsigned)S.pick;
      }
      if (set.min_p > 0.f && mpc < count) count = mpc;
      const u64 x = sm_draw(u, S.weight[count - 1]);
      if (tid < (int)count && S.weight[tid] > x && (tid == 0 || S.weight[tid - 1] <= x))
        out[row] = (int)(uint32_t)S.few[tid];
      return;
    }
    kept = sm_answer(S, SM_COUNT, (u64)set.top_k, V, r, false);
  }
  u64 x = 0;
  if (!greedy) {
    if (set.top_p < 1.f) {
      const SmPrefix p = sm_answer(S, SM_MASS, sm_top_p(set.top_p, kept.mass), V, r, false);
      if (p.count < kept.count) kept = p;
    }
    if (set.min_p > 0.f && mpc < kept.count) kept = SmPrefix{mpc, mpm, 0};
    x = sm_draw(u, kept.mass);
  }
  const SmPrefix d = sm_answer(S, SM_OVER, x, V, r, true);
  if (tid == 0) out[row] = d.token;
}

static int sample_parts(int64_t n) { return (int)((n + kSmPart - 1) / kSmPart); }

int64_t sample_scratch_bytes(int rows, int64_t n) {
  return (int64_t)rows * sample_parts(n) *
         (int64_t)(sizeof(SmPart) + kSmBins * (sizeof(u64) + sizeof(uint16_t)) + kSmPart * sizeof(uint16_t));
}

hipError_t sample_launch(const float *logits, int rows, int64_t n, const SampleSets &sets, const float *u, int *out,
                         void *scratch, hipStream_t st) {
  if (rows <= 0) return hipSuccess;
  const int parts = sample_parts(n);
  int bits = 1;
  while ((int64_t)1 << bits < n) bits++;
  const int shift = bits > 10 ? 62 - bits : 52;  // n weights of at most 1 stay below 2^63
  const int64_t all = (int64_t)rows * parts;
  SmScratch X;  // each array a multiple of 16 bytes from the one before
  X.mass = (u64 *)scratch;
  X.id = (uint16_t *)(X.mass + all * kSmBins);
  X.end = X.id + all * kSmPart;
  X.rec = (SmPart *)(X.end + all * kSmBins);
  hipLaunchKernelGGL(sample_range_kernel, dim3(parts, rows), dim3(256), 0, st, logits, n, X);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // eight tokens a thread while there is at most a part for each CU (one row of 128,256: 6.8 us, 16 a thread 8.4), 16 where
  // CUs take several (64 rows: 25.9 us, eight a thread 29.3)
  if (all <= 256)
    hipLaunchKernelGGL(sample_bins_kernel<512>, dim3(parts, rows), dim3(512), 0, st, logits, n, sets, shift, X);
  else
    hipLaunchKernelGGL(sample_bins_kernel<256>, dim3(parts, rows), dim3(256), 0, st, logits, n, sets, shift, X);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  hipLaunchKernelGGL(sample_pick_kernel, dim3(rows), dim3(1024), 0, st, logits, n, parts, sets, shift, X, u, out);
  return hipGetLastError();
}

}  // namespace wl
