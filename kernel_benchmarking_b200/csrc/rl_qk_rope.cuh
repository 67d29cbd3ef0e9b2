// RMSNorm of every query and key head and the rotation by position, in one pass over the QKV projection's output.
//
//   n = x * gamma / sqrt(mean_d x^2 + eps)                       (over the D channels of one head)
//   (y_i, y_j) = (n_i cos - n_j sin, n_j cos + n_i sin)          for the rot / 2 pairs (i, j) of the rotated channels,
//   y = n                                                        for the channels from rot on
//
// pairs: j = i + rot / 2 (halves), or (2 i, 2 i + 1) (interleaved).  cos and sin come from a table [positions, rot], cos
// first, in fp32.  Everything between the load and the one rounding of y to bf16 is fp32.
//
// Memory bound: 4 D bytes per row for about 60 D / 8 instructions.
#pragma once
#include "rl_rows.cuh"

namespace rl {

struct QkRopeParams {
  const __nv_bfloat16 *q, *k, *q_gamma, *k_gamma;  // gammas [D] or nullptr (ones)
  __nv_bfloat16 *q_out, *k_out;
  const float* table;     // [n_pos, rot], leading dimension ld_table
  const void* positions;  // [T] int32 or int64
  int pos64, n_pos;
  int T, Hq, Hk, D, rot;
  int parts;  // warps per token
  int steps;  // row groups per warp
  long long ld_table;
  long long q_t, q_h, k_t, k_h, qo_t, qo_h, ko_t, ko_h;  // strides in elements: token, head
  float eps;
};

template <int G, bool INTER>
__global__ void __launch_bounds__(128) qk_rope_kernel(const QkRopeParams p) {
  constexpr int R = 32 / G;  // rows per step
  launch_dependents();
  grid_dependency_wait();
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int c = lane & (G - 1);  // chunk of 8 channels
  const int t = (int)(w / p.parts), part = (int)(w - (long long)t * p.parts);
  if (t >= p.T) return;
  const long long pos = load_index(p.positions, t, p.pos64);
  if (pos < 0 || pos >= p.n_pos) {
    if (lane == 0 && part == 0) record_bad_index(BAD_POSITION, t, pos);
    return;
  }
  const bool have = c * 8 < p.D;
  const float inv_d = 1.0f / (float)p.D;
  // this lane's cos and sin (INTER: of its four pairs; halves: of its eight channels' pairs), and its partner's chunk
  const int half = p.rot >> 1, hc = half >> 3;
  const float* tab = p.table + (size_t)pos * p.ld_table;
  float cs[8], sn[8];
  bool turns;
  int mate = c;
  if (INTER) {
    turns = c * 8 < p.rot;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cs[i] = turns ? tab[c * 4 + i] : 1.f;
      sn[i] = turns ? tab[half + c * 4 + i] : 0.f;
    }
  } else {
    turns = c < 2 * hc;
    const bool second = c >= hc;
    if (turns) mate = second ? c - hc : c + hc;
    const int at = (second ? c - hc : c) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      cs[i] = turns ? tab[at + i] : 1.f;
      const float s = turns ? tab[half + at + i] : 0.f;
      sn[i] = second ? s : -s;  // y = n cos + n_mate (+-) sin
    }
  }
  const int H = p.Hq + p.Hk;
  for (int s = 0; s < p.steps; ++s) {
    const int h = (part * p.steps + s) * R + lane / G;
    const bool is_q = h < p.Hq;
    const int hh = is_q ? h : h - p.Hq;
    const bool row = h < H;
    const __nv_bfloat16* gamma = is_q ? p.q_gamma : p.k_gamma;
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (row && have)
      u = *reinterpret_cast<const uint4*>((is_q ? p.q + (size_t)t * p.q_t + (size_t)hh * p.q_h
                                                : p.k + (size_t)t * p.k_t + (size_t)hh * p.k_h) + c * 8);
    const uint32_t xs[4] = {u.x, u.y, u.z, u.w};
    float x[8], ss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16lo(xs[i]);
      x[2 * i + 1] = bf16hi(xs[i]);
      ss = fmaf(x[2 * i], x[2 * i], ss);
      ss = fmaf(x[2 * i + 1], x[2 * i + 1], ss);
    }
    ss = row_sum<G>(ss);
    const float r = 1.0f / sqrtf(fmaf(ss, inv_d, p.eps));
    uint4 g = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);  // bf16 ones
    if (gamma != nullptr && have) g = *reinterpret_cast<const uint4*>(gamma + c * 8);
    const uint32_t gs[4] = {g.x, g.y, g.z, g.w};
    float n[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      n[2 * i] = x[2 * i] * r * bf16lo(gs[i]);
      n[2 * i + 1] = x[2 * i + 1] * r * bf16hi(gs[i]);
    }
    uint32_t o[4];
    if (INTER) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = pack_bf16x2(n[2 * i] * cs[i] - n[2 * i + 1] * sn[i], n[2 * i + 1] * cs[i] + n[2 * i] * sn[i]);
    } else {
      float m[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) m[i] = __shfl_sync(0xffffffffu, n[i], mate, G);
      if (turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) n[i] = n[i] * cs[i] + m[i] * sn[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(n[2 * i], n[2 * i + 1]);
    }
    if (row && have)
      *reinterpret_cast<uint4*>((is_q ? p.q_out + (size_t)t * p.qo_t + (size_t)hh * p.qo_h
                                      : p.k_out + (size_t)t * p.ko_t + (size_t)hh * p.ko_h) + c * 8) =
          make_uint4(o[0], o[1], o[2], o[3]);
  }
}

}  // namespace rl
