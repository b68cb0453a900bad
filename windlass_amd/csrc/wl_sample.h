// wl_sample.h - host interface of wl_sample.hip: the draw of the next token.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace wl {

struct SampleSet {
  float temperature;
  int top_k;
  float top_p, min_p;
};
constexpr int kSampleRows = 64;  // rows that one launch takes
struct SampleSets {
  SampleSet row[kSampleRows];
};

// Bytes of scratch for `rows` (at most kSampleRows) rows of n logits.
int64_t sample_scratch_bytes(int rows, int64_t n);
hipError_t sample_launch(const float *logits, int rows, int64_t n, const SampleSets &sets, const float *u, int *out,
                         void *scratch, hipStream_t st);

}  // namespace wl
