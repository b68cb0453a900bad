// wl_rope.h - RoPE's angles, the same bits for the layer's and the pages' stores.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace wl {

// The angle of rotated pair i at a position: RopeTable's running product in double
// (src/Transformer.cs:396-414) taken to step i, divided by the pair's frequency factor when the
// model has them (rope_freqs.weight, `half` of them). The product is the same sequence for every
// pair, so a wave runs it once for all its lanes (the trip count `half` is uniform) and each lane
// keeps the value after its own i steps: every lane gets the bits the sequential table has
// without a divergent loop of up to 63 dependent multiplies per lane.
__device__ __forceinline__ void rope_cs(int p, int i, int half, double theta_scale, double freq_scale,
                                        const float *__restrict__ freqs, float &c, float &s) {
#pragma clang fp contract(off)
  double theta = (double)p * freq_scale, mine = theta;
  for (int k = 1; k < half; k++) {
    theta *= theta_scale;
    if (k == i) mine = theta;
  }
  const double a = freqs && i < half ? mine / (double)freqs[i] : mine;
  c = (float)cos(a);
  s = (float)sin(a);
}

// The same in two steps, for many positions at once. Lane r of a wave makes the products of position p, theta[i][r] after i steps
// (ROWS positions a step, i below half); the cosine and sine of a pair from its product.
template <int ROWS>
__device__ __forceinline__ void rope_chain(double *theta, int r, int p, int half, double theta_scale, double freq_scale) {
#pragma clang fp contract(off)
  double t = (double)p * freq_scale;
  for (int i = 0; i < half; i++) {
    theta[i * ROWS + r] = t;
    t *= theta_scale;
  }
}
__device__ __forceinline__ void rope_cs_of(double theta, float freq, bool has, float &c, float &s) {
#pragma clang fp contract(off)
  const double a = has ? theta / (double)freq : theta;
  c = (float)cos(a);
  s = (float)sin(a);
}

}  // namespace wl
