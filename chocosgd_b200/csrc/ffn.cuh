// What the kernels of the gated feed-forward block share: its activations, and the entry for few tokens.
#pragma once
#include "vec.cuh"

#define ACT_SILU 0
#define ACT_GELU 1
#define ACT_RELU 2
#define ACT_SIGMOID 3

// activation and (wanted) its derivative.  The reciprocal is the approximate one (1 unit of the last place); FAST: so is the
// exponential (relative error |z| 2^-23), which suits 16-bit results.
template <int ACT, bool GRAD, bool FAST>
__device__ __forceinline__ float ff_act(float z, float& slope) {
  if (ACT == ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    if (GRAD) {
      const float e = -0.5f * z * z;
      slope = fmaf(z * 0.39894228040143268f, FAST ? __expf(e) : expf(e), cdf);
    }
    return z * cdf;
  }
  if (ACT == ACT_RELU) {
    if (GRAD) slope = z > 0.f ? 1.f : 0.f;
    return z < 0.f ? 0.f : z;
  }
  float sg;
  asm("rcp.approx.f32 %0, %1;" : "=f"(sg) : "f"(1.f + (FAST ? __expf(-z) : expf(-z))));
  if (ACT == ACT_SILU) {
    const float a = z * sg;
    if (GRAD) slope = fmaf(a, 1.f - sg, sg);
    return a;
  }
  if (GRAD) slope = fmaf(-sg, sg, sg);
  return sg;
}

// gated_ffn_few.cu: most tokens that the form for few tokens takes, and the form itself (h: m x pad16(f) fp32)
int ffn_few_tokens(int dt);
int ffn_few_forward(const void* x, long long ldx, const void* w_in, long long ld_in, const void* w_out, long long ld_out, float* h,
                    void* y, int m, int d, int f, int n, int act, int dt, cudaStream_t st);
