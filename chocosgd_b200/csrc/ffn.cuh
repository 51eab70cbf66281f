// What the kernels of the gated feed-forward block share: its activations, the split of fp32 operands, and the entry for few tokens.
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

__device__ __forceinline__ uint32_t pack2(float a, float b, int fp16) {
  if (fp16) {
    const __half2 q = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&q);
  }
  const __nv_bfloat162 q = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&q);
}

// two fp32 numbers as three pairs of bf16 numbers, each the rounded remainder of the ones before.  The first is limited to
// the largest bf16 number, so that fp32 numbers above it keep a finite split; non-finite numbers stay non-finite.
__device__ __forceinline__ void split3(float x, float y, uint32_t (&q)[3]) {
  const float big = __uint_as_float(0x7F7F0000u);
#pragma unroll
  for (int s = 0; s < 3; ++s) {
    q[s] = s == 0 ? pack2(fminf(fmaxf(x, -big), big), fminf(fmaxf(y, -big), big), 0) : pack2(x, y, 0);
    x -= __uint_as_float(q[s] << 16);
    y -= __uint_as_float(q[s] & 0xFFFF0000u);
  }
}

// gated_ffn_few.cu: whether the form for few tokens takes these sizes, and the form itself (h: m x pad16(f) fp32)
bool ffn_few_fits(int m, int d, int f, int n, int dt);
int ffn_few_forward(const void* x, long long ldx, const void* w_in, long long ld_in, const void* w_out, long long ld_out, float* h,
                    void* y, int m, int d, int f, int n, int act, int dt, cudaStream_t st);
