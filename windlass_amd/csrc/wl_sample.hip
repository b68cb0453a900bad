// wl_sample.hip - the next token of each row of logits by temperature, top-k, top-p, min-p and a given
// number u (Sampler.Sample, src/Engine.cs:353-382, the draw).
//
// Definition. Tokens in order: larger logit first, of equals the lower id. w = exp((l - max) / t).
// Kept is the longest prefix with at most top_k tokens, whose tokens before the last weigh less than
// top_p of the top_k tokens' weight, and w >= min_p; drawn is the first token at which the weight
// summed in that order passes u of the kept weight. Every step is a question about a prefix of that
// order, so nothing is sorted but the few tokens around a prefix's end.
//
// Arithmetic: weights in double, then as whole numbers of 2^-shift (about 2^-45 at 128,000 tokens), so
// that sums are exact and do not depend on the order in which workgroups and atomics add them.
//
// Three launches. (1) Each part of a row: its largest and least finite logit. (2) Each part: count and
// weight of its tokens in 256 bins of equal width below the row's maximum (64 t wide at most, weights
// below e^-64 in the last bin), and of those with w >= min_p. (3) One workgroup a row adds the parts' bins
// and answers the questions: a prefix's end lies in one bin, whose tokens it gathers from the
// parts that have any and narrows down by their bits.
#include "wl_sample.h"

#include "wl_device.h"

#include <math.h>

#pragma clang fp contract(off)

namespace wl {

constexpr int kSmBins = 256, kSmPart = 4096, kSmList = 4096, kSmFew = 64;
typedef unsigned long long u64;

// A part's record, and after the records of all parts their bins: counts, then weights.
struct SmPart {
  float top, low;       // largest logit (-inf: none), least finite one (+inf: none)
  unsigned minp_count;  // tokens with w >= min_p, and their weight
  u64 minp_mass;
};

// Order-preserving bits of a logit; -0 as 0.
__device__ __forceinline__ uint32_t sm_key(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// What every launch after the first derives from the parts' records: the row's maximum and its bins.
struct SmRow {
  float m, R, c, t;
  int shift;
  __device__ void set(float top, float low, float temperature, int sh) {
    m = top;
    t = temperature;
    shift = sh;
    R = fminf(fminf(top - low, 64.f * t), 3.4028235e38f);
    if (!(R > 1e-30f)) R = 0.f;  // the bins' scale stays finite; what lies lower is the last bin's
    c = R > 0.f ? (float)(kSmBins - 2) / R : 0.f;
  }
  __device__ float below(float l) const { return l == m ? 0.f : m - l; }
  __device__ int bin(float l) const {
    const float d = below(l);
    return d > R ? kSmBins - 1 : min((int)(d * c), kSmBins - 2);
  }
  __device__ double weight(float l) const {
    if (l == m) return 1.0;
    return t > 0.f ? exp(((double)l - (double)m) / (double)t) : 0.0;
  }
  __device__ u64 mass(double w) const { return (u64)rint(ldexp(w, shift)); }
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

__global__ __launch_bounds__(256) void sample_range_kernel(const float *__restrict__ logits, int64_t n,
                                                           SmPart *__restrict__ rec) {
  __shared__ float st[4], sl[4];
  const float *l = logits + (int64_t)blockIdx.y * n;
  const int64_t lo = (int64_t)blockIdx.x * kSmPart, hi = lo + kSmPart < n ? lo + kSmPart : n;
  float top = -INFINITY, low = INFINITY;
  for (int64_t i = lo + threadIdx.x; i < hi; i += 256) {
    const float v = l[i];
    if (v > top) top = v;  // a NaN never compares greater
    if (__builtin_isfinite(v)) low = fminf(low, v);
  }
  top = wave_max_f(top);
  low = -wave_max_f(-low);
  if ((threadIdx.x & 63) == 0) {
    st[threadIdx.x >> 6] = top;
    sl[threadIdx.x >> 6] = low;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    SmPart &p = rec[(int64_t)blockIdx.y * gridDim.x + blockIdx.x];
    p.top = fmaxf(fmaxf(st[0], st[1]), fmaxf(st[2], st[3]));
    p.low = fminf(fminf(sl[0], sl[1]), fminf(sl[2], sl[3]));
  }
}

__global__ __launch_bounds__(256) void sample_bins_kernel(const float *__restrict__ logits, int64_t n, SampleSets sets,
                                                          int shift, SmPart *__restrict__ rec,
                                                          unsigned *__restrict__ counts, u64 *__restrict__ masses) {
  __shared__ unsigned cn[kSmBins];
  __shared__ u64 ms[kSmBins];
  __shared__ float sh[2];
  __shared__ unsigned mc;
  __shared__ u64 mm;
  const int row = blockIdx.y, parts = gridDim.x, tid = threadIdx.x;
  const SampleSet set = sets.row[row];
  cn[tid] = 0;
  ms[tid] = 0;
  if (tid == 0) {
    mc = 0;
    mm = 0;
  }
  SmRow r;
  sm_row_of(rec + (int64_t)row * parts, parts, set.temperature, shift, r, sh);
  const float *l = logits + (int64_t)row * n;
  const int64_t lo = (int64_t)blockIdx.x * kSmPart, hi = lo + kSmPart < n ? lo + kSmPart : n;
  for (int64_t i = lo + tid; i < hi; i += 256) {
    const float v = l[i];
    if (v != v) continue;
    const double w = r.weight(v);
    const u64 M = r.mass(w);
    const int b = r.bin(v);
    atomicAdd(&cn[b], 1u);
    atomicAdd(&ms[b], M);
    if (set.min_p > 0.f && w >= (double)set.min_p) {
      atomicAdd(&mc, 1u);
      atomicAdd(&mm, M);
    }
  }
  __syncthreads();
  const int64_t at = (int64_t)row * parts + blockIdx.x;
  counts[at * kSmBins + tid] = cn[tid];
  masses[at * kSmBins + tid] = ms[tid];
  if (tid == 0) {
    rec[at].minp_count = mc;
    rec[at].minp_mass = mm;
  }
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
  u64 list[kSmList];     // ~key, id of gathered tokens
  u64 few[kSmFew];
  unsigned used;
  int pick;
  uint32_t lo, hi;
  unsigned wave[16];
  SmPrefix got;
  float f2[2];
};

__device__ __forceinline__ bool sm_yes(SmAsk a, u64 target, unsigned c, u64 m) {
  return a == SM_COUNT ? c >= target : a == SM_MASS ? m >= target : m > target;
}

// Sums c[0..255], m[0..255] into running sums (threads 0..255 of the workgroup take part; all call it).
__device__ void sm_scan(unsigned *c, u64 *m) {
  for (int s = 1; s < kSmBins; s <<= 1) {
    unsigned a = 0;
    u64 b = 0;
    const int i = threadIdx.x;
    if (i < kSmBins && i >= s) {
      a = c[i - s];
      b = m[i - s];
    }
    __syncthreads();
    if (i < kSmBins) {
      c[i] += a;
      m[i] += b;
    }
    __syncthreads();
  }
}

// The prefix that answers (a, target): every thread of the workgroup calls it and gets the answer.
__device__ SmPrefix sm_answer(SmShared &S, SmAsk a, u64 target, const float *__restrict__ l, int64_t n, int parts,
                              const unsigned *__restrict__ counts, const SmRow &r, bool token) {
  const int tid = threadIdx.x, nt = blockDim.x;
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
  // every token of the bin: f(key, id)
  auto each = [&](auto f) {
    for (int p = 0; p < parts; p++) {
      if (!counts[(int64_t)p * kSmBins + bin]) continue;  // uniform
      const int64_t lo = (int64_t)p * kSmPart, hi = lo + kSmPart < n ? lo + kSmPart : n;
      for (int64_t i = lo + tid; i < hi; i += nt) {
        const float v = l[i];
        if (v == v && r.bin(v) == bin) f(sm_key(v), (uint32_t)i, v);
      }
    }
  };
  auto value = [](uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); };
  bool listed = in <= kSmList;
  if (listed) {
    each([&](uint32_t key, uint32_t id, float) {
      const unsigned at = atomicAdd(&S.used, 1u);
      S.list[at] = (u64)~key << 32 | id;
      atomicMin(&S.lo, key);
      atomicMax(&S.hi, key);
    });
  } else {
    each([&](uint32_t key, uint32_t, float) {
      atomicMin(&S.lo, key);
      atomicMax(&S.hi, key);
    });
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
      each([&](uint32_t key, uint32_t id, float) {
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
      atomicAdd(&S.sub_m[b], r.mass(r.weight(value(key))));
    });
    __syncthreads();
    sm_scan(S.sub_n, S.sub_m);
    if (tid < kSmBins) {
      const bool y = sm_yes(a, target, c0 + S.sub_n[tid], m0 + S.sub_m[tid]);
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
    if (tid < 64) {  // each token's place among them, and the weight up to it
      const bool on = tid < (int)in;
      const u64 me = on ? S.few[tid] : ~(u64)0;
      const u64 w = on ? r.mass(r.weight(value(~(uint32_t)(me >> 32)))) : 0;
      unsigned place = 1;
      u64 sum = w;
      for (int i = 0; i < (int)in; i++) {
        const u64 o = S.few[i];
        const u64 ow = __shfl(w, i, 64);
        if (o < me) {
          place++;
          sum += ow;
        }
      }
      const bool y = on && sm_yes(a, target, c0 + place, m0 + sum);
      if (y && !sm_yes(a, target, c0 + place - 1, m0 + sum - w))
        S.got = SmPrefix{c0 + place, m0 + sum, (int)(uint32_t)me};
    }
    __syncthreads();
    return S.got;
  }
  // equal logits: the prefix takes the first `need` of them by id
  const u64 w = r.mass(r.weight(value(lo)));
  const u64 need64 = a == SM_COUNT ? target - c0
                     : w == 0      ? 1
                     : a == SM_MASS ? (target - m0 + w - 1) / w
                                    : (target - m0) / w + 1;
  const unsigned need = need64 < 1 ? 1 : need64 > in ? in : (unsigned)need64;
  SmPrefix g{c0 + need, m0 + need * w, 0};
  if (token) {
    unsigned before = 0;
    for (int p = 0; p < parts && before < need; p++) {
      if (!counts[(int64_t)p * kSmBins + bin]) continue;
      for (int64_t i0 = (int64_t)p * kSmPart; i0 < (int64_t)(p + 1) * kSmPart && i0 < n && before < need; i0 += nt) {
        const int64_t i = i0 + tid;
        const float v = i < n ? l[i] : 0.f;
        const bool y = i < n && v == v && sm_key(v) == lo;
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
    }
    __syncthreads();
    g.token = S.got.token;
  }
  return g;
}

__global__ __launch_bounds__(1024) void sample_pick_kernel(const float *__restrict__ logits, int64_t n, int parts,
                                                           SampleSets sets, int shift, const SmPart *__restrict__ rec,
                                                           const unsigned *__restrict__ counts,
                                                           const u64 *__restrict__ masses, const float *__restrict__ us,
                                                           int *__restrict__ out) {
  __shared__ SmShared S;
  const int row = blockIdx.x, tid = threadIdx.x;
  const SampleSet set = sets.row[row];
  const float *l = logits + (int64_t)row * n;
  rec += (int64_t)row * parts;
  counts += (int64_t)row * parts * kSmBins;
  masses += (int64_t)row * parts * kSmBins;
  SmRow r;
  sm_row_of(rec, parts, set.temperature, shift, r, S.f2);
  const float l0 = l[0];
  if (r.m == -INFINITY || (set.temperature == 0.f && l0 != l0)) {  // as the greedy pick
    if (tid == 0) out[row] = 0;
    return;
  }
  {
    // four threads a bin, each a quarter of the parts
    unsigned c = 0;
    u64 m = 0;
    const int b = tid & (kSmBins - 1);
    for (int p = tid / kSmBins; p < parts; p += 4) {
      c += counts[(int64_t)p * kSmBins + b];
      m += masses[(int64_t)p * kSmBins + b];
    }
    if (tid < kSmBins) {
      S.cn[tid] = 0;
      S.ms[tid] = 0;
    }
    __syncthreads();
    atomicAdd(&S.cn[b], c);
    atomicAdd(&S.ms[b], m);
    __syncthreads();
    sm_scan(S.cn, S.ms);
  }
  const unsigned all = S.cn[kSmBins - 1];
  SmPrefix kept{all, S.ms[kSmBins - 1], 0};
  if (set.temperature > 0.f) {
    if (set.top_k > 0 && (unsigned)set.top_k < all)
      kept = sm_answer(S, SM_COUNT, (u64)set.top_k, l, n, parts, counts, r, false);
    if (set.top_p < 1.f) {
      const double want = ceil((double)set.top_p * (double)kept.mass);
      u64 x = (u64)want;
      x = x < 1 ? 1 : x > kept.mass ? kept.mass : x;
      __syncthreads();
      const SmPrefix p = sm_answer(S, SM_MASS, x, l, n, parts, counts, r, false);
      if (p.count < kept.count) kept = p;
    }
    if (set.min_p > 0.f) {
      unsigned c = 0;
      u64 m = 0;
      for (int p = 0; p < parts; p++) {
        c += rec[p].minp_count;
        m += rec[p].minp_mass;
      }
      if (c < kept.count) kept = SmPrefix{c, m, 0};
    }
  }
  u64 x = 0;
  if (set.temperature > 0.f) {
    const double u = (double)us[row];
    const double y = u > 0.0 ? u * (double)kept.mass : 0.0;  // a NaN draws the first
    x = y < (double)kept.mass ? (u64)y : kept.mass;
    x = x < kept.mass ? x : kept.mass - 1;
  }
  __syncthreads();
  const SmPrefix d = sm_answer(S, SM_OVER, x, l, n, parts, counts, r, true);
  if (tid == 0) out[row] = d.token;
}

static int sample_parts(int64_t n) { return (int)((n + kSmPart - 1) / kSmPart); }

int64_t sample_scratch_bytes(int rows, int64_t n) {
  return (int64_t)rows * sample_parts(n) * (int64_t)(sizeof(SmPart) + kSmBins * (sizeof(unsigned) + sizeof(u64)));
}

hipError_t sample_launch(const float *logits, int rows, int64_t n, const SampleSets &sets, const float *u, int *out,
                         void *scratch, hipStream_t st) {
  if (rows <= 0) return hipSuccess;
  const int parts = sample_parts(n);
  int bits = 1;
  while ((int64_t)1 << bits < n) bits++;
  const int shift = 62 - bits;  // n weights of at most 1 stay below 2^63
  SmPart *rec = (SmPart *)scratch;
  u64 *masses = (u64 *)(rec + (int64_t)rows * parts);
  unsigned *counts = (unsigned *)(masses + (int64_t)rows * parts * kSmBins);
  hipLaunchKernelGGL(sample_range_kernel, dim3(parts, rows), dim3(256), 0, st, logits, n, rec);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(sample_bins_kernel, dim3(parts, rows), dim3(256), 0, st, logits, n, sets, shift, rec, counts,
                     masses);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  hipLaunchKernelGGL(sample_pick_kernel, dim3(rows), dim3(1024), 0, st, logits, n, parts, sets, shift, rec, counts,
                     masses, u, out);
  return hipGetLastError();
}

}  // namespace wl
