// What the per-head row kernels (rl_qk_rope.cuh, rl_kv_cache.cuh) share: the record of a bad index, and how a warp
// lays the rows of one token over its lanes.
//
// A row is the D channels of one head of one token (D a multiple of 8, at most 256), in chunks of eight channels (16
// bytes of bf16).  G lanes hold it, G the power of two from D / 16 up: lane c has chunks c and c + G, so that a row's
// loads and stores are contiguous over the lanes, and a warp takes 32 / G rows of the same token at a time.  (One chunk
// per lane spends twice the reductions, roots and divisions per row; these kernels issue nearly as long as they load.)
#pragma once
#include "rl_ptx.cuh"

namespace rl {

// First position, slot or page that a kernel found outside its table since the status was last taken:
// [0] IndexKind (0 = none), [1] row of the call, [2], [3] the index (low and high word).  The kernel leaves out the
// access.  It lives in the library's device image (one per GPU), so it needs no workspace and captured graphs, which
// keep no pointer of the caller's alive for it, report through it as well.
enum IndexKind : int { BAD_POSITION = 1, BAD_SLOT = 2, BAD_PAGE = 3 };
static __device__ int g_index_status[4];

__device__ __noinline__ void record_bad_index(int kind, int row, long long index) {
  if (atomicCAS(g_index_status, 0, kind) == 0) {
    g_index_status[1] = row;
    g_index_status[2] = (int)(index & 0xffffffffll);
    g_index_status[3] = (int)(index >> 32);
  }
}

__device__ __forceinline__ long long load_index(const void* p, int i, int is64) {
  return is64 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}

}  // namespace rl
