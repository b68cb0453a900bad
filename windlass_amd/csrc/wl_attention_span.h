// wl_attention_span.h - host interface of wl_attention_span.hip: attention over 4-bit caches, and over
// fp16 caches with a window.
#pragma once
#include "wl_kv4.h"

namespace wl {

// What a row at position p sees: positions j <= p with j < sinks or j > p - window; all of them with
// window 0.
struct Span {
  int window = 0, sinks = 0;
  // the first position of the window of a row at p, and the first tokens before it
  __host__ __device__ int first(int p) const { return window > 0 && p >= window ? p - window + 1 : 0; }
  __host__ __device__ int lead(int p) const { return sinks < first(p) ? sinks : first(p); }
  __host__ __device__ int seen(int p) const { return p + 1 - first(p) + lead(p); }
};

// Caches of fp16 rows [positions][KH * HD] (bits 16), or of wl_kv4.h's tiles (bits 4); `positions` of
// each slot, slot_bytes apart.
struct KvCache {
  const uint8_t *K = nullptr, *V = nullptr;
  int bits = 16, KH = 0, HD = 0;
  int64_t positions = 0, slot_bytes = 0;
};

int64_t attention_span_scratch_floats(const KvCache &c, int H, const Span &s, const KvRows &rows);
// q, out [rows][H * HD]
hipError_t attention_span_launch(const float *q, int H, const KvCache &c, const Span &s, const KvRows &rows,
                                 float scale, float *scratch, float *out, hipStream_t st);

}  // namespace wl
