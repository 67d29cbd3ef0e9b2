// Keys and values written into a paged e4m3 cache, and the pages of each sequence read back as bf16.
//
// One fp32 scale per (token, head), so a row needs nothing of any other row and a token can be written alone:
//   a = max(max_d |x_d|, 2^-100),  scale = a / 448,  code_d = e4m3(448 x_d / a),  read back: bf16(code_d * scale)
// The floor gives rows of zeros (and of values that small) a scale whose reciprocal fp32 can hold.  A NaN is stored as
// NaN and does not count for a; a row with an infinity reads back as NaN throughout.
//
// Both kernels move bytes: 3 D + 4 per row, read and written together.  131072 tokens of 8 heads of 128 are read back in 126
// us (6460 GB/s, 99 % of the copy bandwidth); 16384 are written in 20.3 us (5010 GB/s), of which 2 are the launch: the
// reduction, the two divisions and the exact rounding keep the SMs issuing for two thirds of the time.
#pragma once
#include <cuda_fp8.h>

#include "rl_rows.cuh"

namespace rl {

constexpr int KV_WARPS = 4;  // per block

struct KvCache {           // codes [pages, page_size, H, D], scales [pages, page_size, H]; values laid out like keys
  uint8_t *k_codes, *v_codes;
  float *k_scale, *v_scale;
  long long c_page, c_off, c_head;  // strides of the codes in bytes
  long long s_page, s_off, s_head;  // strides of the scales in elements
  int num_pages, page_size, H, D;
};

struct KvWriteParams {
  KvCache c;
  const __nv_bfloat16 *k, *v;
  long long k_t, k_h, v_t, v_h;  // strides in elements: token, head
  const void* slots;             // [T] int32 or int64: page * page_size + place in the page; negative: left out
  int slots64, T, parts, steps;
};

// e4m3 codes of eight bf16 (packed) times inv = 448 / a.
// The code is the exact quotient's, ties to even: x and a have 8 significant bits each and a midpoint between codes 5, so
// a quotient that is no midpoint is at least 2^-13 of itself away from one, while x * inv is off by at most 2^-23.
// Rounding the product to 18 bits first puts the midpoints back in their place and moves nothing across one.
__device__ __forceinline__ uint2 e4m3_codes(const uint32_t (&xs)[4], float inv) {
  const uint64_t inv2 = pack2(inv, inv), split = pack2(65.0f, 65.0f), minus = pack2(-1.0f, -1.0f);
  uint32_t code[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t q = mul2(widen2(xs[i]), inv2);
    const uint64_t t = mul2(q, split);                       // Veltkamp's splitting, 24 - 6 bits: t - (t - q), each
    const float2 v = unpack2(fma2(fma2(q, minus, t), minus, t));  // difference rounded once
    code[i] = __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(code[0] | (code[1] << 16), code[2] | (code[3] << 16));
}

// U: groups whose loads are in flight together
template <int G, int U>
__global__ void __launch_bounds__(32 * KV_WARPS) kv_write_kernel(const KvWriteParams p) {
  constexpr int R = 32 / G;
  launch_dependents();
  grid_dependency_wait();
  const long long w = (long long)blockIdx.x * KV_WARPS + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, c = lane & (G - 1);
  const int t = (int)(w / p.parts), part = (int)(w - (long long)t * p.parts);
  if (t >= p.T) return;
  const int k_groups = (p.c.H + R - 1) / R;  // the key heads' groups, then as many of the value heads
  const int g0 = part * p.steps, g1 = min(g0 + p.steps, 2 * k_groups);
  uint32_t x[U][2][4];
  // U groups from g, all of one kind (below `end`)
  auto load_rows = [&](int g, int end) {
    const bool is_k = g < k_groups;
    const __nv_bfloat16* src = (is_k ? p.k + (size_t)t * p.k_t : p.v + (size_t)t * p.v_t) + c * 8;
    const long long src_h = is_k ? p.k_h : p.v_h;
    const int h0 = (is_k ? g : g - k_groups) * R + lane / G;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * R;
      const bool row = g + u < end && h < p.c.H;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row && (c + j * G) * 8 < p.c.D) v = *reinterpret_cast<const uint4*>(src + h * src_h + j * G * 8);
        x[u][j][0] = v.x; x[u][j][1] = v.y; x[u][j][2] = v.z; x[u][j][3] = v.w;
      }
    }
  };
  load_rows(g0, g0 < k_groups ? min(g1, k_groups) : g1);  // on their way while the slot is looked up
  const long long slot = load_index(p.slots, t, p.slots64);
  if (slot < 0) return;
  const long long page = slot / p.c.page_size;
  const int off = (int)(slot - page * p.c.page_size);
  if (page >= p.c.num_pages) {
    if (lane == 0 && part == 0) record_bad_index(BAD_SLOT, t, slot);
    return;
  }
  const long long code_at = page * p.c.c_page + off * p.c.c_off + c * 8, scale_at = page * p.c.s_page + off * p.c.s_off;
#pragma unroll 1
  for (int g = g0; g < g1;) {
    const bool is_k = g < k_groups;
    const int end = is_k ? min(g1, k_groups) : g1;
    if (g > g0) load_rows(g, end);
    uint8_t* codes = (is_k ? p.c.k_codes : p.c.v_codes) + code_at;
    float* scales = (is_k ? p.c.k_scale : p.c.v_scale) + scale_at;
    const int h0 = (is_k ? g : g - k_groups) * R + lane / G;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * R;
      // largest |x| of the row, NaN left out
      __nv_bfloat162 m = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&x[u][j][i])));
      uint32_t mu = *reinterpret_cast<uint32_t*>(&m);
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, mu, o);
        m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&mu), *reinterpret_cast<const __nv_bfloat162*>(&other));
        mu = *reinterpret_cast<uint32_t*>(&m);
      }
      const float a = fmaxf(fmaxf(bf16lo(mu), bf16hi(mu)), 0x1p-100f);
      const float inv = 448.0f / a;
      if (g + u < end && h < p.c.H) {
        uint8_t* dst = codes + h * p.c.c_head;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if ((c + j * G) * 8 < p.c.D) *reinterpret_cast<uint2*>(dst + j * G * 8) = e4m3_codes(x[u][j], inv);
        if (c == 0) scales[h * p.c.s_head] = a / 448.0f;
      }
    }
    g = (g + U < end) ? g + U : end;
  }
}

struct KvReadParams {
  KvCache c;
  const int* pages;  // [B, max_pages], leading dimension ld_pages
  long long ld_pages;
  const int* cu;     // [B + 1]: sequence b's tokens are rows cu[b] .. cu[b+1] - 1 of the output
  int B, max_pages, T, zero_tail, parts, steps;  // T: rows of the output
  __nv_bfloat16 *k_out, *v_out;
  long long ko_t, ko_h, vo_t, vo_h;
};

// The last b in [0, B) with cu[b] <= i, by the 32 lanes of a warp (empty sequences: the one that holds row i).
__device__ __forceinline__ int find_sequence(const int* cu, int B, int i, int lane) {
  int lo = 0, n = B;
  while (n > 1) {
    const int step = (n + 31) >> 5;
    const int at = lo + lane * step;
    const bool below = at < lo + n && cu[at] <= i;
    const unsigned hits = __ballot_sync(0xffffffffu, below);
    const int last = hits ? 31 - __clz(hits) : 0;
    n = min(step, n - last * step);
    lo += last * step;
  }
  return lo;
}

__device__ __forceinline__ uint32_t dequant2(uint32_t codes, float scale) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return pack_bf16x2(f.x * scale, f.y * scale);
}

template <int G>
__global__ void __launch_bounds__(32 * KV_WARPS) kv_read_kernel(const KvReadParams p) {
  constexpr int R = 32 / G;
  constexpr int U = 4;  // groups whose loads are in flight together
  launch_dependents();
  grid_dependency_wait();
  const long long w = (long long)blockIdx.x * KV_WARPS + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, c = lane & (G - 1);
  const int i = (int)(w / p.parts), part = (int)(w - (long long)i * p.parts);
  if (i >= p.T) return;
  bool held = p.B > 0 && i < p.cu[p.B];
  long long code_at = 0, scale_at = 0;
  if (!held) {
    if (!p.zero_tail) return;
  } else {
    const int b = find_sequence(p.cu, p.B, i, lane);
    const int pos = i - p.cu[b];
    const int col = pos / p.c.page_size;
    const int page = (pos >= 0 && col < p.max_pages) ? p.pages[b * p.ld_pages + col] : -1;
    if (page < 0 || page >= p.c.num_pages) {
      if (lane == 0 && part == 0) record_bad_index(BAD_PAGE, i, page);
      if (!p.zero_tail) return;
      held = false;  // (a fresh output: the row becomes zero)
    } else {
      const int off = pos - col * p.c.page_size;
      code_at = page * p.c.c_page + off * p.c.c_off;
      scale_at = page * p.c.s_page + off * p.c.s_off;
    }
  }
  const int k_groups = (p.c.H + R - 1) / R;
  const int g0 = part * p.steps, g1 = min(g0 + p.steps, 2 * k_groups);
#pragma unroll 1
  for (int g = g0; g < g1; g += U) {
    uint2 code[U][2];
    float scale[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool is_k = g + u < k_groups;
      const int h = (is_k ? g + u : g + u - k_groups) * R + lane / G;
      const bool row = held && g + u < g1 && h < p.c.H;
      scale[u] = row ? (is_k ? p.c.k_scale : p.c.v_scale)[scale_at + h * p.c.s_head] : 0.f;
      const uint8_t* src = (is_k ? p.c.k_codes : p.c.v_codes) + code_at + h * p.c.c_head;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int ch = c + j * G;
        code[u][j] = (row && ch * 8 < p.c.D) ? *reinterpret_cast<const uint2*>(src + ch * 8) : make_uint2(0u, 0u);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool is_k = g + u < k_groups;
      const int h = (is_k ? g + u : g + u - k_groups) * R + lane / G;
      if (g + u >= g1 || h >= p.c.H) continue;
      __nv_bfloat16* dst = is_k ? p.k_out + (size_t)i * p.ko_t + h * p.ko_h : p.v_out + (size_t)i * p.vo_t + h * p.vo_h;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int ch = c + j * G;
        const uint2 q = code[u][j];
        if (ch * 8 < p.c.D)
          *reinterpret_cast<uint4*>(dst + ch * 8) =
              make_uint4(dequant2(q.x & 0xffffu, scale[u]), dequant2(q.x >> 16, scale[u]), dequant2(q.y & 0xffffu, scale[u]),
                         dequant2(q.y >> 16, scale[u]));
      }
    }
  }
}

}  // namespace rl
