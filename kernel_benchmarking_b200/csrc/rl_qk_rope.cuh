// RMSNorm of every query and key head and the rotation by position, in one pass over the QKV projection's output.
//
//   n = x * gamma / sqrt(mean_d x^2 + eps)                       (over the D channels of one head)
//   (y_i, y_j) = (n_i cos - n_j sin, n_j cos + n_i sin)          for the rot / 2 pairs (i, j) of the rotated channels,
//   y = n                                                        for the channels from rot on
//
// pairs: j = i + rot / 2 (halves), or (2 i, 2 i + 1) (interleaved).  cos and sin come from a table [positions, rot], cos
// first, in fp32.  Everything between the load and the one rounding of y to bf16 is fp32.
//
// gamma and the table's values are the same for all query heads of a token, and for all its key heads: with
// A_i = gamma_i cos and B_i = +- gamma_mate(i) sin, made once per warp and kind of heads, a channel is
// y_i = r (x_i A_i + x_mate(i) B_i).  A warp takes `steps` groups of 32 / G rows of one token, query heads' groups first.
// 16384 tokens of 32 + 8 heads of 128 (344 MB) in 60.5 us: 5690 GB/s, 87 % of the copy bandwidth; the rest is the chain of
// reduction, root and products, which needs the 24 warps an SM holds (20 warps: 68 us, 16: 86) and two groups interleaved.
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
  int parts, steps;       // warps per token, row groups per warp
  long long ld_table;
  long long q_t, q_h, k_t, k_h, qo_t, qo_h, ko_t, ko_h;  // strides in elements: token, head
  float eps;
};

// where the channel that turns with this one sits: its neighbour; the same place of the lane's other chunk (halves of
// rot = 16 G channels: whole heads of 64, 128 or 256); or any lane's chunk
enum Mate : int { MATE_NEIGHBOUR = 0, MATE_OTHER_CHUNK = 1, MATE_ANY = 2 };

// Warps per block.  Several groups per warp: one, so that a token that is done makes room for the next at once (16384 tokens
// of 32 + 8 heads: 60.9 us, 68.3 with four).  One group: four, which an SM takes in faster (1021 tokens of 6 + 3 heads of
// 80: 2.8 us, 3.9 with one).
__host__ __device__ constexpr int qk_rope_warps(int U) { return U == 1 ? 4 : 1; }

// U: groups whose loads are in flight, and whose arithmetic is interleaved
template <int G, int MATE, int U>
__global__ void __launch_bounds__(qk_rope_warps(U) * 32, 24 / qk_rope_warps(U)) qk_rope_kernel(const QkRopeParams p) {
  constexpr int R = 32 / G;  // rows per group
  launch_dependents();
  grid_dependency_wait();
  const long long w = (long long)blockIdx.x * qk_rope_warps(U) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int c = lane & (G - 1);
  const int t = (int)(w / p.parts), part = (int)(w - (long long)t * p.parts);
  if (t >= p.T) return;
  const long long pos = load_index(p.positions, t, p.pos64);
  const int q_groups = (p.Hq + R - 1) / R, groups = q_groups + (p.Hk + R - 1) / R;
  const int g0 = part * p.steps, g1 = min(g0 + p.steps, groups);
  uint32_t x[U][2][4];
  // U groups from g, all of one kind (below `end`)
  auto load_rows = [&](int g, int end) {
    const bool is_q = g < q_groups;
    const int H = is_q ? p.Hq : p.Hk;
    const __nv_bfloat16* src = is_q ? p.q + (size_t)t * p.q_t : p.k + (size_t)t * p.k_t;
    const long long src_h = is_q ? p.q_h : p.k_h;
    const int h0 = (is_q ? g : g - q_groups) * R + lane / G;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * R;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (g + u < end && h < H && (c + j * G) * 8 < p.D) v = *reinterpret_cast<const uint4*>(src + h * src_h + (c + j * G) * 8);
        x[u][j][0] = v.x; x[u][j][1] = v.y; x[u][j][2] = v.z; x[u][j][3] = v.w;
      }
    }
  };
  // the first rows are on their way while the position, and then its row of the table, are looked up
  load_rows(g0, g0 < q_groups ? min(g1, q_groups) : g1);
  if (pos < 0 || pos >= p.n_pos) {
    if (lane == 0 && part == 0) record_bad_index(BAD_POSITION, t, pos);
    return;
  }
  const float* tab = p.table + (size_t)pos * p.ld_table;
  const int half = p.rot >> 1, hc = half >> 3;
  const float inv_d = 1.0f / (float)p.D;
#pragma unroll 1
  for (int first = g0; first < g1;) {
    // ---- the query heads, then the key heads, of this warp's groups: coefficients
    const bool is_q = first < q_groups;
    const int end = is_q ? min(g1, q_groups) : g1;
    const __nv_bfloat16* gamma = is_q ? p.q_gamma : p.k_gamma;
    bool have[2];
    int mate[2];  // MATE_ANY: the chunk this one turns with (itself where nothing turns)
    uint64_t A[2][4], B[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int ch = c + j * G;
      have[j] = ch * 8 < p.D;
      const bool turns = ch * 8 < p.rot;
      const bool second = MATE != MATE_NEIGHBOUR && ch >= hc;
      mate[j] = (MATE == MATE_NEIGHBOUR || !turns) ? ch : (second ? ch - hc : ch + hc);
      uint4 g = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u), gm = g;  // bf16 ones
      if (gamma != nullptr && have[j]) {
        g = *reinterpret_cast<const uint4*>(gamma + ch * 8);
        gm = (MATE == MATE_NEIGHBOUR) ? g : *reinterpret_cast<const uint4*>(gamma + mate[j] * 8);
      }
      const uint32_t gs[4] = {g.x, g.y, g.z, g.w}, ms[4] = {gm.x, gm.y, gm.z, gm.w};
      if (MATE == MATE_NEIGHBOUR) {
        float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
        if (turns) {
          cs = *reinterpret_cast<const float4*>(tab + ch * 4);
          sn = *reinterpret_cast<const float4*>(tab + half + ch * 4);
        }
        const float cv[4] = {cs.x, cs.y, cs.z, cs.w}, sv[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          A[j][i] = pack2(bf16lo(gs[i]) * cv[i], bf16hi(gs[i]) * cv[i]);
          B[j][i] = pack2(-bf16hi(gs[i]) * sv[i], bf16lo(gs[i]) * sv[i]);
        }
      } else {
        float cv[8], sv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) { cv[i] = 1.f; sv[i] = 0.f; }
        if (turns) {
          const float4* cp = reinterpret_cast<const float4*>(tab + (second ? ch - hc : ch) * 8);
          const float4* sp = reinterpret_cast<const float4*>(tab + half + (second ? ch - hc : ch) * 8);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float4 a = cp[i], b = sp[i];
            cv[4 * i] = a.x; cv[4 * i + 1] = a.y; cv[4 * i + 2] = a.z; cv[4 * i + 3] = a.w;
            sv[4 * i] = b.x; sv[4 * i + 1] = b.y; sv[4 * i + 2] = b.z; sv[4 * i + 3] = b.w;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          A[j][i] = pack2(bf16lo(gs[i]) * cv[2 * i], bf16hi(gs[i]) * cv[2 * i + 1]);
          const float s0 = second ? sv[2 * i] : -sv[2 * i], s1 = second ? sv[2 * i + 1] : -sv[2 * i + 1];
          B[j][i] = pack2(bf16lo(ms[i]) * s0, bf16hi(ms[i]) * s1);
        }
      }
    }
    const int H = is_q ? p.Hq : p.Hk;
    __nv_bfloat16* dst = is_q ? p.q_out + (size_t)t * p.qo_t : p.k_out + (size_t)t * p.ko_t;
    const long long dst_h = is_q ? p.qo_h : p.ko_h;
    const int h_first = (is_q ? first : first - q_groups) * R + lane / G;
#pragma unroll 1
    for (int g = first; g < end; g += U) {
      if (g > g0) load_rows(g, end);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h_first + (g - first + u) * R;
        float2 ss2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) ffma2_sq(ss2, bf16lo(x[u][j][i]), bf16hi(x[u][j][i]));
        float ss = ss2.x + ss2.y;
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        // (the approximate reciprocal root is good to 2^-22)
        const float r = rsqrtf(fmaf(ss, inv_d, p.eps));
        const uint64_t r2 = pack2(r, r);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t m[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (MATE == MATE_NEIGHBOUR) {
              m[i] = __byte_perm(x[u][j][i], 0u, 0x1032);  // the two channels change places
            } else if (MATE == MATE_OTHER_CHUNK) {
              m[i] = x[u][1 - j][i];
            } else {
              const uint32_t a = __shfl_sync(0xffffffffu, x[u][0][i], mate[j] & (G - 1), G);
              const uint32_t b = __shfl_sync(0xffffffffu, x[u][1][i], mate[j] & (G - 1), G);
              m[i] = mate[j] >= G ? b : a;
            }
          }
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 y = unpack2(mul2(r2, fma2(widen2(x[u][j][i]), A[j][i], mul2(widen2(m[i]), B[j][i]))));
            o[i] = pack_bf16x2(y.x, y.y);
          }
          if (g + u < end && h < H && have[j])
            *reinterpret_cast<uint4*>(dst + h * dst_h + (c + j * G) * 8) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
      if (U == 1) return;  // one group per warp
    }
    first = end;
  }
}

}  // namespace rl
