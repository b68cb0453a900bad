// wl_sample.hip - the next token of each row of logits by temperature, top-k, top-p, min-p and a given
// number u (Sampler.Sample, src/Engine.cs:353-382, the draw).
//
// Definition. Tokens in order: larger logit first, of equals the lower id. w = exp((l - max) / t).
// Kept is the longest prefix with at most top_k tokens, whose tokens before the last weigh less than
// top_p of the top_k tokens' weight, and w >= min_p; drawn is the first token at which the weight
// summed in that order passes u of the kept weight. Every step is a question about a prefix of that
// order, so nothing is sorted but the few tokens around a prefix's end.
//
// Arithmetic: weights in double (a polynomial for 2^f), cut to whole numbers of 2^-shift, so that sums are exact and do not
// depend on the order in which workgroups and atomics add them. Up to 2^18 tokens a unit that leaves the sum of n weights of 1
// at 2^63 at most: what is cut off is below n 2^(bits of n - 63), 2^-29 of the weight at 128,000 tokens. Longer rows bound their
// weight first, each part's tokens at the part's largest, at most 4,096 times the weight: n 2^-49 of it is cut off at most,
// 2^-25 at 2^24 (with the unit of n weights of 1, one logit 20 above 2^24 others of deviation 2 lost them more than half of
// what they weigh together). Bounding every row took one row of 128,256 from 15.0 to 15.2 us, 64 rows from 46.8 to 47.9.
//
// Three launches. (1) Each part of 4,096 tokens of a row: its largest and least finite logit. (2) Each part: the count
// and weight of its tokens in 256 bins of equal width below the row's maximum (64 t wide at most, weights below e^-64
// in the last bin), its tokens' places by bin, and what has w >= min_p. (3) One workgroup a row adds the parts'
// bins and answers the questions: a prefix's end lies in one bin, whose tokens it gathers and narrows down by their
// bits, and equal ones by their ids; with top_k of few tokens it gathers the whole prefix and puts that in order.
//
// What bounds it: a row of 128,256 is read from HBM in launch 1 and from the caches after (64 rows, 33 MB: 6.6 us), then
// 64 rows' bins take 23.0 us (50 VALU instructions a token, and LDS atomics that meet: two or four copies of the bins, votes
// for the last bin and no min_p sums where none is asked each gained less than a microsecond or lost) and their questions
// 17.1 (a workgroup a row: chains of LDS and cache latencies, 2.5 to 6 us a question). One row is three dependent launches:
// 2.6, 6.8 and 6.3 us.
#include "wl_sample.h"

#include "wl_device.h"

#include <math.h>

#pragma clang fp contract(off)

namespace wl {

constexpr int kSmBins = 256, kSmPart = 4096, kSmList = 4096, kSmFew = 256, kSmGroup = 64;
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
  __device__ void set(float top, float low, float t) {
    m = cap(top);
    per = t > 0.f ? fmin(1.4426950408889634 / (double)t, 1e300) : 1e300;
    R = fminf(fminf(m - low, 64.f * t), 3.4028235e38f);
    if (!(R > 1e-30f)) R = 0.f;  // the bins' scale stays finite; what lies lower is the last bin's
    c = R > 0.f ? (float)(kSmBins - 2) / R : 0.f;
  }
  __device__ static float cap(float l) { return fminf(l, 3.4028235e38f); }
  // The weight of a part's largest logit. In 32 bits: off by 2^-16 of it at most, and nothing below 2^-126.
  __device__ float largest(float part_top) const {
    return __builtin_amdgcn_exp2f((float)fmax(((double)cap(part_top) - (double)m) * per, -200.0));
  }
  // At most 2^63 units: n weights of 1, or kSmPart times the parts' largest weights, which add up to `sum`, and 1% for its rounding.
  __device__ void unit(int64_t n, bool bounded, float sum) {
    int e = 32 - __clz((int)n - 1);
    if (bounded) frexpf(1.01f * sum * (float)kSmPart, &e);
    shift = e > 11 ? 63 - e : 52;
  }
  __device__ int bin(float l) const {
    const float d = m - cap(l);
    return d > R ? kSmBins - 1 : min((int)(d * c), kSmBins - 2);
  }
  // Bounds of the keys of a bin's logits: its edges, past what bin() rounds.
  __device__ void keys(int b, uint32_t &lo, uint32_t &hi) const {
    const double step = (double)R * (1.0 / (kSmBins - 2));  // 1 / c, but for c's rounding
    const double up = (double)min(b, kSmBins - 2) * step * (1.0 - 0x1p-20), down = (double)(b + 1) * step * (1.0 + 0x1p-20);
    hi = b ? sm_key((float)((double)m - up)) + 1 : m < 3.4028235e38f ? sm_key(m) : sm_key(INFINITY);
    lo = sm_key(-INFINITY);
    if (b < kSmBins - 1) lo = sm_key(fmaxf((float)((double)m - down), -3.4028235e38f)) - 1;
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

// The sum over a wave, the same in every lane.
__device__ __forceinline__ float wave_sum_f(float v) {
  v += __builtin_bit_cast(float, dpp32<0xB1>(__builtin_bit_cast(uint32_t, v)));  // as wave_max_f
  v += __builtin_bit_cast(float, dpp32<0x4E>(__builtin_bit_cast(uint32_t, v)));
  v += __builtin_bit_cast(float, dpp32<0x124>(__builtin_bit_cast(uint32_t, v)));
  v += __builtin_bit_cast(float, dpp32<0x128>(__builtin_bit_cast(uint32_t, v)));
  return (lane_f(v, 0) + lane_f(v, 16)) + (lane_f(v, 32) + lane_f(v, 48));
}

__device__ __forceinline__ void sm_row_of(const SmPart *__restrict__ part, int parts, int64_t n, float t, SmRow &r,
                                          float *sh) {
  // every thread of the workgroup; sh holds 3 floats
  const bool bounded = parts > 64;
  if (threadIdx.x < 64) {
    float top = -INFINITY, low = INFINITY, sum = 0.f;
    for (int i = threadIdx.x; i < parts; i += 64) {
      top = fmaxf(top, part[i].top);
      low = fminf(low, part[i].low);
    }
    top = wave_max_f(top);
    low = -wave_max_f(-low);
    if (bounded) {
      r.set(top, low, t);
      for (int i = threadIdx.x; i < parts; i += 64) sum += r.largest(part[i].top);
      sum = wave_sum_f(sum);
    }
    if (threadIdx.x == 0) {
      sh[0] = top;
      sh[1] = low;
      sh[2] = sum;
    }
  }
  __syncthreads();
  r.set(sh[0], sh[1], t);
  r.unit(n, bounded, sh[2]);
}

// Running sums over a wave's lanes (all of them active): within rows of 16 by lane shifts, then the rows' sums. A general
// shuffle goes through LDS, and each of its six steps costs that latency (one row's draw 15.7 us, with these 15.1).
template <int CTRL>
__device__ __forceinline__ unsigned sm_dpp(unsigned v) {
  return dpp32<CTRL>(v);
}
template <int CTRL>
__device__ __forceinline__ u64 sm_dpp(u64 v) {
  return (u64)dpp32<CTRL>((uint32_t)(v >> 32)) << 32 | dpp32<CTRL>((uint32_t)v);
}
__device__ __forceinline__ unsigned sm_lane(unsigned v, int l) { return (unsigned)__builtin_amdgcn_readlane((int)v, l); }
__device__ __forceinline__ u64 sm_lane(u64 v, int l) {
  return (u64)sm_lane((unsigned)(v >> 32), l) << 32 | sm_lane((unsigned)v, l);
}
template <class T>
__device__ __forceinline__ T sm_running(T v) {
  v += sm_dpp<0x111>(v);  // row_shr 1, 2, 4, 8: zeros from before the row
  v += sm_dpp<0x112>(v);
  v += sm_dpp<0x114>(v);
  v += sm_dpp<0x118>(v);
  const T a = sm_lane(v, 15), b = a + sm_lane(v, 31), c = b + sm_lane(v, 47);
  const int row = (threadIdx.x & 63) >> 4;
  return v + (row == 0 ? T(0) : row == 1 ? a : row == 2 ? b : c);
}
// The sum over 4 (by = 2) or 16 (by = 4) neighbouring lanes, in each of them.
template <class T>
__device__ __forceinline__ T sm_sum(T v, int by) {
  v += sm_dpp<0xB1>(v);  // quad_perm 1,0,3,2
  v += sm_dpp<0x4E>(v);  // quad_perm 2,3,0,1
  if (by == 4) {
    v += sm_dpp<0x124>(v);  // row_ror 4, 8
    v += sm_dpp<0x128>(v);
  }
  return v;
}

// Running sums over the bins of 256 threads (all of the workgroup call it; sh holds 4 of each).
__device__ __forceinline__ void sm_scan(unsigned &c, u64 &m, unsigned *sc, u64 *sm) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  if (wv < 4) {
    c = sm_running(c);
    m = sm_running(m);
    if (lane == 63) {
      sc[wv] = c;
      sm[wv] = m;
    }
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
                                                          SmScratch X) {
  constexpr int N = kSmPart / WIDE;
  __shared__ unsigned cn[kSmBins];
  __shared__ u64 ms[kSmBins];
  __shared__ __attribute__((aligned(16))) uint16_t ids[kSmPart];
  __shared__ float sh[3];
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
  sm_row_of(X.rec + (int64_t)row * parts, parts, n, set.temperature, r, sh);
  const SmSeries C;
  const u64 least = (u64)ceil(ldexp((double)set.min_p, r.shift));
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
  u64 few[kSmFew], weight[kSmFew];
  unsigned minp_count;  // the row's tokens with w >= min_p, and their weight
  u64 minp_mass;
  unsigned from[kSmGroup + 1];  // of a group of parts: where each part's gathered tokens begin
  uint16_t off[kSmGroup];       // and the first in the part's order
  unsigned used;
  int pick;
  unsigned sc[4];
  u64 sm[4];
  SmPrefix got;
  float f3[3];
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
      const unsigned sum = sm_running(last - first);
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

// The answer among few tokens (at most 256, in S.few, after c0 tokens of weight m0): 16 or 4 threads a token count those up
// to it and add their weights.
__device__ __forceinline__ void sm_few(SmShared &S, SmAsk a, u64 target, unsigned in, unsigned c0, u64 m0,
                                       const SmRow &r) {
  const int tid = threadIdx.x, by = in <= 64 ? 4 : 2;  // log2 of them
  if (tid < (int)in) S.weight[tid] = r.mass(sm_value(~(uint32_t)(S.few[tid] >> 32)), SmSeries());
  __syncthreads();
  const unsigned i = tid >> by, k0 = tid & ((1 << by) - 1);
  if (i < in) {
    const u64 me = S.few[i];
    unsigned place = 0;
    u64 sum = 0;
#pragma unroll 4
    for (unsigned k = k0; k < in; k += 1 << by) {
      const bool up = S.few[k] <= me;
      place += up ? 1u : 0u;
      sum += up ? S.weight[k] : 0;
    }
    place = sm_sum(place, by);
    sum = sm_sum(sum, by);
    if (k0 == 0 && sm_yes(a, target, c0 + place, m0 + sum) && !sm_yes(a, target, c0 + place - 1, m0 + sum - S.weight[i]))
      S.got = SmPrefix{c0 + place, m0 + sum, (int)(uint32_t)me};
  }
  __syncthreads();
}

// The prefix that answers (a, target): every thread of the workgroup calls it and gets the answer.
__device__ __forceinline__ SmPrefix sm_answer(SmShared &S, SmAsk a, u64 target, const SmView &V, const SmRow &r) {
  const int tid = threadIdx.x, nt = blockDim.x;
  __syncthreads();
  if (tid < kSmBins) {
    const bool y = sm_yes(a, target, S.cn[tid], S.ms[tid]);
    if (y && (tid == 0 || !sm_yes(a, target, S.cn[tid - 1], S.ms[tid - 1]))) S.pick = tid;
  }
  if (tid == 0) S.used = 0;
  __syncthreads();
  const int bin = S.pick;
  unsigned c0 = bin ? S.cn[bin - 1] : 0, in = S.cn[bin] - c0;
  u64 m0 = bin ? S.ms[bin - 1] : 0;
  // a whole bin's prefix needs no token of it
  if (a == SM_COUNT && c0 + in == target) return SmPrefix{c0 + in, S.ms[bin], 0};
  // narrowed down to few by the keys, 256 steps at a time, and equal logits by their ids
  uint32_t lo, hi, id0 = 0, id1 = 0xffffffffu;
  r.keys(bin, lo, hi);
  const uint32_t floor = sm_key(S.f3[1]);  // the least finite logit
  bool listed = false;
  unsigned have = 0;
  auto inside = [&](uint32_t key, uint32_t id) { return key >= lo && key <= hi && id >= id0 && id <= id1; };
  for (;;) {
    if (!listed && in <= kSmList) {
      sm_each(S, V, bin, bin, [&](uint32_t key, uint32_t id) {
        if (inside(key, id)) S.list[atomicAdd(&S.used, 1u)] = (u64)~key << 32 | id;
      });
      listed = true;
      have = in;
    }
    if (in <= kSmFew) break;
    const bool keys = lo < hi;
    if (!keys && id1 >= V.n) id1 = (uint32_t)V.n - 1;
    // -inf, which would spread the steps, is the last step's
    const uint32_t range = keys ? hi - (floor > lo && floor <= hi ? floor : lo) : id1 - id0;
    const int wide = range >> 8 ? 24 - __clz((int)range) : 0;  // log2 of a step
    if (tid < kSmBins) {
      S.sub_n[tid] = 0;
      S.sub_m[tid] = 0;
    }
    __syncthreads();
    auto count = [&](uint32_t key, uint32_t id) {
      if (!inside(key, id)) return;
      const uint32_t b = min((keys ? hi - key : id - id0) >> wide, (uint32_t)kSmBins - 1);
      atomicAdd(&S.sub_n[b], 1u);
      atomicAdd(&S.sub_m[b], r.mass(sm_value(key), SmSeries()));
    };
    if (listed)
      for (unsigned i = tid; i < have; i += nt) count(~(uint32_t)(S.list[i] >> 32), (uint32_t)S.list[i]);
    else
      sm_each(S, V, bin, bin, count);
    __syncthreads();
    unsigned c = tid < kSmBins ? S.sub_n[tid] : 0;
    u64 m = tid < kSmBins ? S.sub_m[tid] : 0;
    sm_scan(c, m, S.sc, S.sm);
    if (tid < kSmBins) {  // each thread its own; the ones before it below
      S.sub_n[tid] = c;
      S.sub_m[tid] = m;
    }
    __syncthreads();
    if (tid < kSmBins) {
      const bool y = sm_yes(a, target, c0 + c, m0 + m);
      if (y && (tid == 0 || !sm_yes(a, target, c0 + S.sub_n[tid - 1], m0 + S.sub_m[tid - 1]))) S.pick = tid;
    }
    __syncthreads();
    const uint32_t b = (uint32_t)S.pick, step = (uint32_t)1 << wide;
    const unsigned cb = b ? S.sub_n[b - 1] : 0;
    in = S.sub_n[b] - cb;
    c0 += cb;
    m0 += b ? S.sub_m[b - 1] : 0;
    const bool end = b == kSmBins - 1;
    if (keys) {
      hi -= b << wide;
      lo = !end && hi - lo >= step ? hi - step + 1 : lo;
    } else {
      id0 += b << wide;
      id1 = !end && id1 - id0 >= step ? id0 + step - 1 : id1;
    }
    __syncthreads();
  }
  if (tid == 0) S.used = 0;
  __syncthreads();
  for (unsigned i = tid; i < have; i += nt) {
    const u64 t = S.list[i];
    if (inside(~(uint32_t)(t >> 32), (uint32_t)t)) S.few[atomicAdd(&S.used, 1u)] = t;
  }
  __syncthreads();
  sm_few(S, a, target, in, c0, m0, r);
  return S.got;
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
                                                           SampleSets sets, SmScratch X,
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
  if (set.min_p > 0.f && tid >= 64 && tid < 128) {  // beside the first wave's reading of the range
    unsigned n_ = 0;
    u64 m_ = 0;
    for (int p = tid - 64; p < parts; p += 64) {
      n_ += rec[p].minp_count;
      m_ += rec[p].minp_mass;
    }
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) {
      n_ += __shfl_xor(n_, x, 64);
      m_ += __shfl_xor(m_, x, 64);
    }
    if (tid == 64) {
      S.minp_count = n_;
      S.minp_mass = m_;
    }
  }
  SmRow r;
  sm_row_of(rec, parts, n, set.temperature, r, S.f3);
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
    if (in <= kSmFew) {
      // each bin's tokens together, then each token to its place among its bin's, four threads a token
      if (tid <= bin) S.sub_n[tid] = tid ? S.cn[tid - 1] : 0;
      sm_each(S, V, 0, bin, [&](uint32_t key, uint32_t id) {
        S.list[atomicAdd(&S.sub_n[r.bin(sm_value(key))], 1u)] = (u64)~key << 32 | id;
      });
      if (tid >> 2 < (int)in) {
        const u64 me = S.list[tid >> 2];
        const int b = r.bin(sm_value(~(uint32_t)(me >> 32)));
        const unsigned from = b ? S.cn[b - 1] : 0, to = S.cn[b];
        unsigned place = 0;
        for (unsigned i = from + (tid & 3); i < to; i += 4) place += S.list[i] < me ? 1u : 0u;
        place = sm_sum(place, 2);
        if ((tid & 3) == 0) S.few[from + place] = me;
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
      if (set.min_p > 0.f && S.minp_count < count) count = S.minp_count;
      const u64 x = sm_draw(u, S.weight[count - 1]);
      if (tid < (int)count && S.weight[tid] > x && (tid == 0 || S.weight[tid - 1] <= x))
        out[row] = (int)(uint32_t)S.few[tid];
      return;
    }
  }
  // the questions in turn, in one copy of the code (a launch runs it once or twice: most of its time is the fetching)
#pragma unroll 1
  for (int q = 0; q < 3; q++) {
    SmAsk a = SM_OVER;
    u64 x = 0;
    if (q == 0) {
      if (!top_k) continue;
      a = SM_COUNT;
      x = (u64)set.top_k;
    } else if (q == 1) {
      if (greedy || !(set.top_p < 1.f)) continue;
      a = SM_MASS;
      x = sm_top_p(set.top_p, kept.mass);
    } else if (!greedy) {
      if (set.min_p > 0.f && S.minp_count < kept.count) kept = SmPrefix{S.minp_count, S.minp_mass, 0};
      x = sm_draw(u, kept.mass);
    }
    const SmPrefix p = sm_answer(S, a, x, V, r);
    if (q == 2 && tid == 0) out[row] = p.token;
    if (p.count < kept.count) kept = p;
  }
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
    hipLaunchKernelGGL(sample_bins_kernel<512>, dim3(parts, rows), dim3(512), 0, st, logits, n, sets, X);
  else
    hipLaunchKernelGGL(sample_bins_kernel<256>, dim3(parts, rows), dim3(256), 0, st, logits, n, sets, X);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  hipLaunchKernelGGL(sample_pick_kernel, dim3(rows), dim3(1024), 0, st, logits, n, parts, sets, X, u, out);
  return hipGetLastError();
}

}  // namespace wl
