// activations.cuh — the activation functions of the GEMM epilogues.
#pragma once
#include "ptx_sm100.cuh"

namespace b2g {

// tanh-form GELU, the formula of the reference's gelu_val (kernels.cu:266-269).
// Evaluated through the identity 0.5 v (1 + tanh(u)) = v * sigmoid(2u) = v / (1 + e^(-2u)),
// with e^(-2u) = 2^(-2u log2(e)) from the hardware base-2 exponential (ex2.approx, relative
// error ~2^-22) and a fast division: a few instructions instead of an accurate tanhf, and
// within a few fp32 ulps of the formula.  For large negative v the limit is -0.  kFar: it is reached,
// the exponential being infinite there, at any v.  Otherwise the exponent is capped at 2^126, which
// leaves v * 2^-126: 0 to fp32 precision for the sums of 16-bit operands, but -1.2 at v = -1e38, which 8-bit
// layers can meet, as a token's scale takes any size.
template <bool kFar = false>
__device__ __forceinline__ float gelu_tanh(float v) {
  const float u = 0.7978845608f * (v + 0.044715f * v * v * v);
  const float x = -2.8853900817779268f * u;
  const float e = fast_exp2(kFar ? x : fminf(x, 126.0f));
  return __fdividef(v, 1.0f + e);
}

// SiLU, the formula of the reference's silu_val (kernels.cu): v / (1 + e^-v), with e^-v from
// the hardware base-2 exponential and a fast division; kFar as above.
template <bool kFar = false>
__device__ __forceinline__ float silu_fast(float v) {
  const float x = -1.4426950408889634f * v;
  return __fdividef(v, 1.0f + fast_exp2(kFar ? x : fminf(x, 126.0f)));
}

}  // namespace b2g
