// activations.cuh — the activation functions of the GEMM epilogues.
#pragma once
#include "ptx_sm100.cuh"

namespace b2g {

// tanh-form GELU, the formula of the reference's gelu_val (kernels.cu:266-269).
// Evaluated through the identity 0.5 v (1 + tanh(u)) = v * sigmoid(2u) = v / (1 + e^(-2u)),
// with e^(-2u) = 2^(-2u log2(e)) from the hardware base-2 exponential (ex2.approx, relative
// error ~2^-22) and a fast division: a few instructions instead of an accurate tanhf, and
// within a few fp32 ulps of the formula.  The exponent is capped at 2^126 (the quotient is
// then -0 to fp32 precision, GELU's limit for large negative v).
__device__ __forceinline__ float gelu_tanh(float v) {
  const float u = 0.7978845608f * (v + 0.044715f * v * v * v);
  const float e = fast_exp2(fminf(-2.8853900817779268f * u, 126.0f));
  return __fdividef(v, 1.0f + e);
}

// SiLU, the formula of the reference's silu_val (kernels.cu): v / (1 + e^-v), with e^-v from
// the hardware base-2 exponential (capped at 2^126, where the quotient is -0 to fp32
// precision) and a fast division.
__device__ __forceinline__ float silu_fast(float v) {
  return __fdividef(v, 1.0f + fast_exp2(fminf(-1.4426950408889634f * v, 126.0f)));
}

}  // namespace b2g
