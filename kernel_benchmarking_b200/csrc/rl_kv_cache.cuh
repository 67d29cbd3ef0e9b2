// Keys and values written into a paged e4m3 cache, and the pages of each sequence read back as bf16.
//
// One fp32 scale per (token, head), so a row needs nothing of any other row and a token can be written alone:
//   a = max(max_d |x_d|, 2^-100),  scale = a / 448,  code_d = e4m3(448 x_d / a),  read back: bf16(code_d * scale)
// The floor gives rows of zeros (and of values that small) a scale whose reciprocal fp32 can hold.  A NaN is stored as
// NaN and does not count for a; a row with an infinity reads back as NaN throughout.
//
// Both kernels move bytes: 3 D + 4 per row, read and written together.
#pragma once
#include <cuda_fp8.h>

#include "rl_rows.cuh"

namespace rl {

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
  uint32_t code[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float q[2] = {bf16lo(xs[i]) * inv, bf16hi(xs[i]) * inv};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float t = __fmul_rn(q[j], 65.0f);  // Veltkamp's splitting: 24 - 6 bits
      q[j] = __fsub_rn(t, __fsub_rn(t, q[j]));
    }
    code[i] = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(code[0] | (code[1] << 16), code[2] | (code[3] << 16));
}

// largest |x| of eight packed bf16 over the lanes of a row, NaN left out
template <int G>
__device__ __forceinline__ float row_amax(const uint32_t (&xs)[4]) {
  __nv_bfloat162 m = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&xs[i])));
  uint32_t u = *reinterpret_cast<uint32_t*>(&m);
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    const uint32_t v = __shfl_xor_sync(0xffffffffu, u, o);
    m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&v));
    u = *reinterpret_cast<uint32_t*>(&m);
  }
  return fmaxf(bf16lo(u), bf16hi(u));
}

template <int G>
__global__ void __launch_bounds__(128) kv_write_kernel(const KvWriteParams p) {
  constexpr int R = 32 / G;
  launch_dependents();
  grid_dependency_wait();
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, c = lane & (G - 1);
  const int t = (int)(w / p.parts), part = (int)(w - (long long)t * p.parts);
  if (t >= p.T) return;
  const long long slot = load_index(p.slots, t, p.slots64);
  if (slot < 0) return;
  const long long page = slot / p.c.page_size;
  const int off = (int)(slot - page * p.c.page_size);
  if (page >= p.c.num_pages) {
    if (lane == 0 && part == 0) record_bad_index(BAD_SLOT, t, slot);
    return;
  }
  const long long code_at = page * p.c.c_page + off * p.c.c_off, scale_at = page * p.c.s_page + off * p.c.s_off;
  const bool have = c * 8 < p.c.D;
  for (int s = 0; s < p.steps; ++s) {
    const int h = (part * p.steps + s) * R + lane / G;  // key heads, then value heads
    const bool is_k = h < p.c.H, row = h < 2 * p.c.H;
    const int hh = is_k ? h : h - p.c.H;
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (row && have)
      u = *reinterpret_cast<const uint4*>((is_k ? p.k + (size_t)t * p.k_t + (size_t)hh * p.k_h
                                                : p.v + (size_t)t * p.v_t + (size_t)hh * p.v_h) + c * 8);
    const uint32_t xs[4] = {u.x, u.y, u.z, u.w};
    const float a = fmaxf(row_amax<G>(xs), 0x1p-100f);
    const uint2 codes = e4m3_codes(xs, 448.0f / a);
    if (row && have)
      *reinterpret_cast<uint2*>((is_k ? p.c.k_codes : p.c.v_codes) + code_at + (long long)hh * p.c.c_head + c * 8) = codes;
    if (row && c == 0) (is_k ? p.c.k_scale : p.c.v_scale)[scale_at + (long long)hh * p.c.s_head] = a / 448.0f;
  }
}

struct KvReadParams {
  KvCache c;
  const int* pages;  // [B, max_pages], leading dimension ld_pages
  long long ld_pages;
  const int* cu;     // [B + 1]: sequence b's tokens are rows cu[b] .. cu[b+1] - 1 of the output
  int B, max_pages, total, zero_tail, parts, steps;
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
__global__ void __launch_bounds__(128) kv_read_kernel(const KvReadParams p) {
  constexpr int R = 32 / G;
  launch_dependents();
  grid_dependency_wait();
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, c = lane & (G - 1);
  const int i = (int)(w / p.parts), part = (int)(w - (long long)i * p.parts);
  if (i >= p.total) return;
  const bool held = p.B > 0 && i < p.cu[p.B];
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
      return;
    }
    const int off = pos - col * p.c.page_size;
    code_at = page * p.c.c_page + off * p.c.c_off;
    scale_at = page * p.c.s_page + off * p.c.s_off;
  }
  const bool have = c * 8 < p.c.D;
  for (int s = 0; s < p.steps; ++s) {
    const int h = (part * p.steps + s) * R + lane / G;
    const bool is_k = h < p.c.H;
    const int hh = is_k ? h : h - p.c.H;
    if (h >= 2 * p.c.H || !have) continue;
    uint32_t o[4] = {0u, 0u, 0u, 0u};
    if (held) {
      const float scale = (is_k ? p.c.k_scale : p.c.v_scale)[scale_at + (long long)hh * p.c.s_head];
      const uint2 u =
          *reinterpret_cast<const uint2*>((is_k ? p.c.k_codes : p.c.v_codes) + code_at + (long long)hh * p.c.c_head + c * 8);
      o[0] = dequant2(u.x & 0xffffu, scale);
      o[1] = dequant2(u.x >> 16, scale);
      o[2] = dequant2(u.y & 0xffffu, scale);
      o[3] = dequant2(u.y >> 16, scale);
    }
    *reinterpret_cast<uint4*>((is_k ? p.k_out + (size_t)i * p.ko_t + (size_t)hh * p.ko_h
                                    : p.v_out + (size_t)i * p.vo_t + (size_t)hh * p.vo_h) + c * 8) =
        make_uint4(o[0], o[1], o[2], o[3]);
  }
}

}  // namespace rl
