// Epilogue of the linear layer: y = act(x W^T + bias) + residual, on fp32 accumulators, rounded once to bf16.
#pragma once
#include "rl_ptx.cuh"

namespace rl {

// values of RL_ACT_* in include/rmsnorm_linear.h
enum Activation : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4 };

// z / (1 + e^t).  The fast exponential and division are good to about 2^-18 relative over the range where the result
// is not negligible, against the 2^-9 of the bf16 rounding that follows; an IEEE division per output would be the
// longest part of the epilogue.  e^t beyond fp32 gives z / inf = 0, the limit.
__device__ __forceinline__ float div_one_plus_exp(float z, float t) { return __fdividef(z, 1.0f + __expf(t)); }

// `act` is the same for the whole grid: one branch around the loops, not one per value.
template <int NV>
__device__ __forceinline__ void apply_activation(float (&z)[NV], int act) {
  if (act == ACT_NONE) return;
  if (act == ACT_RELU) {
#pragma unroll
    for (int i = 0; i < NV; ++i) z[i] = (z[i] < 0.f) ? 0.f : z[i];  // (NaN stays NaN)
  } else if (act == ACT_GELU) {
    // z * Phi(z) = z * erfc(-z / sqrt 2) / 2: the complementary function keeps its relative accuracy for negative z,
    // where 1 + erf(z / sqrt 2) would cancel
#pragma unroll
    for (int i = 0; i < NV; ++i) z[i] = 0.5f * z[i] * erfcf(-0.70710678118654752f * z[i]);
  } else if (act == ACT_GELU_TANH) {
    // (1 + tanh u) / 2 = 1 / (1 + e^-2u), u = sqrt(2 / pi) (z + 0.044715 z^3)
#pragma unroll
    for (int i = 0; i < NV; ++i)
      z[i] = div_one_plus_exp(z[i], -1.5957691216057308f * fmaf(0.044715f * z[i] * z[i], z[i], z[i]));
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) z[i] = div_one_plus_exp(z[i], -z[i]);
  }
}

// 16 consecutive bf16 of a row as 8 packed words, zeros from `n` = N on.  `vec`: the address is 16-byte aligned.
// Plain loads, not the read-only path: a residual may be the output itself (each element is read before the thread
// block that owns it stores it).
__device__ __forceinline__ void load16_bf16(const __nv_bfloat16* src, int n, int N, bool vec, uint32_t (&w)[8]) {
  if (vec && n + 16 <= N) {
    const uint4 a = reinterpret_cast<const uint4*>(src)[0], b = reinterpret_cast<const uint4*>(src)[1];
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    return;
  }
  const unsigned short* s = reinterpret_cast<const unsigned short*>(src);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t lo = (n + 2 * i < N) ? s[2 * i] : 0u, hi = (n + 2 * i + 1 < N) ? s[2 * i + 1] : 0u;
    w[i] = lo | (hi << 16);
  }
}

// 16 accumulator columns -> 8 packed bf16 words: + bias, activation, + residual
__device__ __forceinline__ void epilogue16(float (&z)[16], const uint32_t (&bias)[8], const uint32_t (&res)[8], int act,
                                           uint32_t* o) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    z[2 * i] += bf16lo(bias[i]);
    z[2 * i + 1] += bf16hi(bias[i]);
  }
  apply_activation(z, act);
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = pack_bf16x2(z[2 * i] + bf16lo(res[i]), z[2 * i + 1] + bf16hi(res[i]));
}

}  // namespace rl
