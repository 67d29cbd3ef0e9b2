// Epilogue of the linear layer: y = act(x W^T + bias) + residual, on fp32 accumulators, rounded once to bf16.
#pragma once
#include "rl_ptx.cuh"

namespace rl {

// values of RL_ACT_* in include/rmsnorm_linear.h
enum Activation : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4 };

// The arithmetic runs on packed pairs (f32x2): the epilogue warps share the SM with a main loop that waits for them, and a
// value costs about 8 instructions this way, about 20 one by one.
//
// 2^x and 1/x are the approximate instructions: relative errors of 2^-22 and, through the argument, |x| 2^-24, so better
// than 2^-14 wherever the result is not negligible, against the 2^-9 of the bf16 rounding that follows.
__device__ __forceinline__ float ex2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// z / (1 + 2^t); 2^t beyond fp32 gives z * 0, the limit
__device__ __forceinline__ uint64_t div_one_plus_ex2(uint64_t z, uint64_t t) {
  const float2 tv = unpack2(t);
  const float2 d = unpack2(add2(pack2(ex2_approx(tv.x), ex2_approx(tv.y)), pack2(1.0f, 1.0f)));
  return mul2(z, pack2(rcp_approx(d.x), rcp_approx(d.y)));
}

// z Phi(z) = max(z, 0) - |z| Phi(-|z|), which has no cancellation for negative z, with Phi(-a) = e^(-a^2 / 2) S(a).
// S(a) = erfcx(a / sqrt 2) / 2 as t P(t), t = 1 / (1 + 0.36 a): the degree-6 P with the smallest largest relative error
// on a <= 14 (Lawson's iteration on a Chebyshev grid), 2^-20; beyond 14 the product is zero in fp32.  erfcf in its place
// cost 600 us against 340 without an activation on 4096 x 14336 x 4096.
__device__ __forceinline__ uint64_t gelu_erf(uint64_t z) {
  const float2 zv = unpack2(z);
  const float ax = fminf(fabsf(zv.x), 14.0f), ay = fminf(fabsf(zv.y), 14.0f);
  const uint64_t a = pack2(ax, ay);
  const float2 d = unpack2(fma2(pack2(0.36f, 0.36f), a, pack2(1.0f, 1.0f)));
  const uint64_t t = pack2(rcp_approx(d.x), rcp_approx(d.y));
  uint64_t q = fma2(pack2(4.705606680e-02f, 4.705606680e-02f), t, pack2(-1.797639464e-01f, -1.797639464e-01f));
  q = fma2(q, t, pack2(1.809530295e-01f, 1.809530295e-01f));
  q = fma2(q, t, pack2(2.654996838e-02f, 2.654996838e-02f));
  q = fma2(q, t, pack2(1.397190467e-01f, 1.397190467e-01f));
  q = fma2(q, t, pack2(1.417724895e-01f, 1.417724895e-01f));
  q = fma2(q, t, pack2(1.437130432e-01f, 1.437130432e-01f));
  const float2 e = unpack2(mul2(mul2(a, a), pack2(-0.72134752044f, -0.72134752044f)));  // -a^2 / 2 in powers of two
  const uint64_t h = mul2(mul2(q, t), pack2(ex2_approx(e.x), ex2_approx(e.y)));
  const uint64_t top = pack2((zv.x < 0.f) ? 0.f : zv.x, (zv.y < 0.f) ? 0.f : zv.y);  // (NaN stays NaN)
  return fma2(mul2(a, h), pack2(-1.0f, -1.0f), top);
}

// NV pairs.  `act` is the same for the whole grid: one branch around the loops, not one per value.
template <int NV>
__device__ __forceinline__ void apply_activation(uint64_t (&z)[NV], int act) {
  if (act == ACT_NONE) return;
  if (act == ACT_RELU) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float2 v = unpack2(z[i]);
      z[i] = pack2((v.x < 0.f) ? 0.f : v.x, (v.y < 0.f) ? 0.f : v.y);  // (NaN stays NaN)
    }
  } else if (act == ACT_GELU) {
#pragma unroll
    for (int i = 0; i < NV; ++i) z[i] = gelu_erf(z[i]);
  } else if (act == ACT_GELU_TANH) {
    // (1 + tanh u) / 2 = 1 / (1 + e^-2u), u = sqrt(2 / pi) (z + 0.044715 z^3); -2 u log2 e = z (c1 + c3 z^2)
    const uint64_t c1 = pack2(-2.3022081985f, -2.3022081985f), c3 = pack2(-0.10294323960f, -0.10294323960f);
#pragma unroll
    for (int i = 0; i < NV; ++i) z[i] = div_one_plus_ex2(z[i], mul2(z[i], fma2(mul2(z[i], z[i]), c3, c1)));
  } else {
    const uint64_t c1 = pack2(-1.4426950409f, -1.4426950409f);
#pragma unroll
    for (int i = 0; i < NV; ++i) z[i] = div_one_plus_ex2(z[i], mul2(z[i], c1));
  }
}

// Four consecutive bf16 of a row from column n; zeros from N on.  `vec`: the address is 8-byte aligned.
// Plain loads, not the read-only path: a residual may be the output itself (each element is read before the thread
// block that owns it stores it).
__device__ __forceinline__ uint2 load4_bf16(const __nv_bfloat16* src, int n, int N, bool vec) {
  if (vec && n + 4 <= N) return *reinterpret_cast<const uint2*>(src);
  const unsigned short* s = reinterpret_cast<const unsigned short*>(src);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (n + i < N) ? s[i] : 0u;
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// NV pairs of accumulators -> NV packed bf16 words: + bias, activation, + residual
template <int NV>
__device__ __forceinline__ void linear_epilogue(uint64_t (&z)[NV], const uint32_t (&bias)[NV], const uint32_t (&res)[NV],
                                                int act, uint32_t (&o)[NV]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) z[i] = add2(z[i], widen2(bias[i]));
  apply_activation(z, act);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float2 v = unpack2(add2(z[i], widen2(res[i])));
    o[i] = pack_bf16x2(v.x, v.y);
  }
}

}  // namespace rl
