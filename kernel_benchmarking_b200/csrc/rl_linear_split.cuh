// The linear layer for few tokens or few tiles: y = act(x W^T + bias) + residual with the k-loop of every tile shared by the
// CTAs of a cluster.
//
// Operands are swapped so that the 128-wide UMMA M dimension runs over output channels: A = W tile [128 x 64], B = x tile
// [NT tokens x 64], D[channel, token] in tensor memory.  The `split` CTAs of a cluster (1, 2, 4 or 8) take one contiguous
// part of the tile's k-blocks each.  Each then finishes a share of the tokens: once all have read their operands (a cluster
// barrier that the read of tensor memory overlaps), every CTA stores its fp32 accumulators where the finishing ranks' operands
// were, and after a second barrier each rank adds its tokens' parts in rank order out of its own shared memory.  Results do
// not depend on timing, and nothing is exchanged through global memory: no workspace, no counters, and no CTA waits for one
// outside its cluster, which the hardware schedules together.  (Parts left in place and read by the finishing ranks took
// 3.4 us from the last MMA to the kernel's end on 333 x 1000 x 1144: the loads' round trips, and a barrier behind them.)
//
// Bound by W from HBM: 28672 x 4096 with 16 tokens in 39.9 us is 5920 GB/s, 90 % of the copy bandwidth; 4096 x 4096 (33 MB) in
// 9.0 us is launch, first load and exchange as much as stream.  Ring depths and CTAs per SM: about 100 KB per CTA, two CTAs on
// an SM, so that one's start and exchange run under the other's stream; where every SM has one at most, 64- and 128-token
// tiles take 190 KB (128 x 4096 x 4096 in 128 CTAs 12.1 us, 13.3 with 100 KB; 700 x 1536 x 6144 18.2, 22.7).
//
// Warps: 0 TMA producer, 1 UMMA issuer, then the epilogue's.
#pragma once
#include "rl_epilogue.cuh"
#include "rl_ptx.cuh"

namespace rl {

struct SplitParams {
  int M, N, K;
  int token_tiles, split, act;
  const __nv_bfloat16* bias;      // [N] or nullptr
  const __nv_bfloat16* residual;  // [M, N] with leading dimension ld_res, or nullptr; may be y itself
  __nv_bfloat16* y;
  long long ld_res, ldy;
  int res_vec, y_vec;             // rows start on 8-byte boundaries
};

template <int NT_, int STAGES_>
struct SplitCfg {
  static constexpr int NT = NT_, STAGES = STAGES_;
  // epilogue warps: eight halve the time of the wide tiles' epilogues, four cost the short ones less to launch (0.5 us)
  static constexpr int EPI_WARPS = NT >= 64 ? 8 : 4, THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int W_BYTES = 128 * 64 * 2, X_BYTES = NT * 64 * 2;
  static constexpr int OFF_W = 0, OFF_X = STAGES * W_BYTES;
  static constexpr int RING_BYTES = STAGES * (W_BYTES + X_BYTES);
  static constexpr int OFF_BAR = RING_BYTES;
  static constexpr int OFF_MISC = OFF_BAR + (2 * STAGES + 1) * 8;
  static constexpr int SMEM_BYTES = OFF_MISC + 64 + 1024;
  static constexpr int TMEM_COLS = NT < 32 ? 32 : NT;
  static_assert(NT == 16 || NT == 32 || NT == 64 || NT == 128, "tokens per tile");
  static_assert(NT * 128 * 4 <= RING_BYTES, "the accumulator fits where the operands were");
};

// where a wait that ran out is recorded (layout of the status block); part of the device image like g_index_status
static __device__ int g_wait_status[RL_STATUS_INTS];

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
// the two halves of cluster_sync_all
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// the h-th 16 tokens of a channel to the ranks that finish them, 2^per_log2 >= P tokens each: one address per P of them
// (one per token: 0.1 to 0.3 us more on 64 and 128 tokens a tile)
template <int P>
__device__ __forceinline__ void push16(uint32_t to, const uint32_t (&v)[16], int h, int per_log2) {
#pragma unroll
  for (int j = 0; j < 16; j += P) {
    const int tk = h * 16 + j, r = tk >> per_log2;
    const uint32_t at = mapa_shared(to + (uint32_t)(tk - (r << per_log2)) * 512u, (uint32_t)r);
#pragma unroll
    for (int i = 0; i < P; ++i) st_cluster_f32(at + i * 512u, __uint_as_float(v[j + i]));
  }
}

// residual of tokens first and first + EW (zeros where there is none)
template <int EW>
__device__ __forceinline__ void split_residual(const SplitParams& p, int m0, int n, int first, int last, uint2 (&res)[2]) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int tk = first + EW * u;
    res[u] = make_uint2(0u, 0u);
    if (tk < last && p.residual != nullptr && n < p.N)
      res[u] = load4_bf16(p.residual + (size_t)(m0 + tk) * p.ld_res + n, n, p.N, p.res_vec != 0);
  }
}

// The tokens first, first + EW, .. below `last` of a tile (EW epilogue warps), four channels per lane: parts in rank order,
// bias, activation, residual.  `part` is this lane's place in the rank's [S][per][128] parts, whose tokens count from a
// multiple of per.  Two tokens at a time; `res` comes in with the first two's residual, and the next two's is on its way
// while these are finished.
template <int S, int EW>
__device__ __forceinline__ void split_finish(const SplitParams& p, const float4* part, int per, int m0, int n, int first,
                                             int last, const uint32_t (&bias)[2], uint2 (&res)[2]) {
  for (int t0 = first; t0 < last; t0 += 2 * EW) {
    float4 v[2][S];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < S; ++r)
        if (t0 + EW * u < last) v[u][r] = part[(r * per + ((t0 + EW * u) & (per - 1))) * 32];
    uint2 next[2];
    split_residual<EW>(p, m0, n, t0 + 2 * EW, last, next);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int tk = t0 + EW * u;
      if (tk >= last || n >= p.N) continue;
      uint64_t z[2] = {pack2(v[u][0].x, v[u][0].y), pack2(v[u][0].z, v[u][0].w)};
#pragma unroll
      for (int r = 1; r < S; ++r) {
        z[0] = add2(z[0], pack2(v[u][r].x, v[u][r].y));
        z[1] = add2(z[1], pack2(v[u][r].z, v[u][r].w));
      }
      const uint32_t rw[2] = {res[u].x, res[u].y};
      uint32_t o[2];
      linear_epilogue(z, bias, rw, p.act, o);
      __nv_bfloat16* dst = p.y + (size_t)(m0 + tk) * p.ldy + n;
      if (p.y_vec && n + 4 <= p.N) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
      } else {
        unsigned short* d = reinterpret_cast<unsigned short*>(dst);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < p.N) d[i] = (unsigned short)(o[i >> 1] >> ((i & 1) * 16));
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) res[u] = next[u];
  }
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 2)
linear_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const SplitParams p) {
  constexpr int NT = Cfg::NT, STAGES = Cfg::STAGES, EW = Cfg::EPI_WARPS;
  extern __shared__ uint8_t smem_raw[];
  // (every CTA of the kernel has the same shared-memory layout, so the aligned base is the same in the whole cluster)
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + Cfg::OFF_BAR;
  auto bar_full = [&](int s) { return bar0 + 8u * s; };
  auto bar_empty = [&](int s) { return bar0 + 8u * (STAGES + s); };
  const uint32_t bar_acc = bar0 + 8u * (2 * STAGES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_MISC);
  CtaCtl* ctl = reinterpret_cast<CtaCtl*>(smem + Cfg::OFF_MISC + 16);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = p.split;
  const int rank = (int)(blockIdx.x % S), tile = (int)(blockIdx.x / S);
  const int tt = tile % p.token_tiles, ct = tile / p.token_tiles;
  const int KB = (p.K + 63) >> 6;
  const int kb0 = (int)((long long)rank * KB / S), kb1 = (int)((long long)(rank + 1) * KB / S);  // never empty: S <= KB
  const int m0 = tt * NT, n0 = ct * 128;
  const int tokens = min(NT, p.M - m0);
  const int n_pre = min(STAGES, kb1 - kb0);  // k-blocks whose loads go out before the CTA-wide sync

  // W is read once where one tile holds all tokens; x, and W otherwise, by several clusters
  const bool w_once = p.token_tiles == 1;
  auto issue = [&](int s, int kb, uint64_t pol_w, uint64_t pol_x) {
    mbar_expect_tx(bar_full(s), Cfg::W_BYTES + Cfg::X_BYTES);
    if (w_once) tma_load_2d_hint(sbase + Cfg::OFF_W + s * Cfg::W_BYTES, &tm_w, bar_full(s), kb * 64, n0, pol_w);
    else tma_load_2d(sbase + Cfg::OFF_W + s * Cfg::W_BYTES, &tm_w, bar_full(s), kb * 64, n0);
    tma_load_2d_hint(sbase + Cfg::OFF_X + s * Cfg::X_BYTES, &tm_x, bar_full(s), kb * 64, m0, pol_x);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    mbar_init(bar_acc, 1);
    ctl->abort = 0;
    ctl->status = g_wait_status;
    ctl->limit_ns = 0;
    fence_mbar_init();
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
    grid_dependency_wait();
    // fill the ring right away: the first loads need neither tensor memory nor the other warps
    const uint64_t pol_w = l2_policy_evict_first(), pol_x = l2_policy_evict_last();
    for (int i = 0; i < n_pre; ++i) issue(i, kb0 + i, pol_w, pol_x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // only now may the next kernel's CTAs come in beside this one: its tensor memory is taken already
  launch_dependents();
  grid_dependency_wait();

  // the tokens this warp will finish (rank's share, from `first` in steps of EW), and what that needs early: the bias of the
  // lane's four channels and the first tokens' residual
  const int per = NT / S;
  const int first = rank * per + (warp - 2), last = min(tokens, (rank + 1) * per);
  uint2 res[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
  if (warp >= 2) split_residual<EW>(p, m0, n0 + lane * 4, first, last, res);
  uint32_t bias[2] = {0u, 0u};
  if (warp >= 2 && p.bias != nullptr && n0 + lane * 4 < p.N) {
    const uint2 w = load4_bf16(p.bias + n0 + lane * 4, n0 + lane * 4, p.N, true);
    bias[0] = w.x;
    bias[1] = w.y;
  }
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    const uint64_t pol_w = l2_policy_evict_first(), pol_x = l2_policy_evict_last();
    int s = 0;
    uint32_t ph = 1;  // (the first turn of the ring is on its way already)
    for (int kb = kb0 + STAGES; kb < kb1; ++kb) {
      if (!mbar_wait_warp(bar_empty(s), ph ^ 1, ctl, 0, STAGES + s, kb)) break;
      if (elect_one()) issue(s, kb, pol_w, pol_x);
      __syncwarp();
      if (++s == STAGES) { s = 0; ph ^= 1; }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ UMMA issuer
    constexpr uint32_t idesc = make_idesc(128, NT, 1, 1);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(bar_full(s), ph, ctl, 1, s, kb)) { ok = false; break; }
      tc_fence_after();
      const uint64_t adesc = make_sw128_kmajor_desc(sbase + Cfg::OFF_W + s * Cfg::W_BYTES);
      const uint64_t bdesc = make_sw128_kmajor_desc(sbase + Cfg::OFF_X + s * Cfg::X_BYTES);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_ss(tmem_base, adesc + 2 * k, bdesc + 2 * k, idesc, (kb != kb0) || (k != 0));
        umma_commit(bar_empty(s));
      }
      __syncwarp();
      if (++s == STAGES) { s = 0; ph ^= 1; }
    }
    if (ok && elect_one()) umma_commit(bar_acc);
    __syncwarp();
  } else {
    mbar_wait_warp(bar_acc, 0, ctl, 2, 2 * STAGES, kb0);
  }
  // ------------------------------------------------------------ accumulators -> the finishing ranks, [S][per][128 channels]
  // This CTA's MMAs are done (or a wait of it ran out, which it has recorded; the barriers are reached all the same).
  if (S > 1) cluster_arrive();
  tc_fence_after();
  const int q = warp & 3, half = (warp - 2) >> 2;
  constexpr int HALVES = EW / 4;  // a quarter's two warps share the tokens
  uint32_t v[16];
  auto load16 = [&](int h) {
    tmem_ld16(tmem_base + ((uint32_t)(q * 32) << 16) + h * 16, v);
    tmem_wait_ld();
  };
  const bool mine = warp >= 2 && half * 16 < tokens;
  if (mine) load16(half);
  if (S > 1) cluster_wait();  // every rank's operands have been read: their place may be written
  else __syncthreads();
  if (mine) {
    const int per_log2 = 31 - __clz(per);  // NT and S are powers of two
    const uint32_t to = sbase + (uint32_t)(rank * per * 128 + q * 32 + lane) * 4u;
#pragma unroll
    for (int hh = 0; hh < NT / 16 / HALVES; ++hh) {
      const int h = hh * HALVES + half;
      if (h * 16 >= tokens) break;
      if (hh > 0) load16(h);
      if (h * 16 + 16 <= tokens) {
        if (per >= 16) push16<16>(to, v, h, per_log2);
        else if (per == 8) push16<8>(to, v, h, 3);
        else if (per == 4) push16<4>(to, v, h, 2);
        else push16<2>(to, v, h, 1);
        continue;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int tk = h * 16 + j, r = tk >> per_log2;
        if (tk < tokens) st_cluster_f32(mapa_shared(to + (uint32_t)(tk - r * per) * 512u, (uint32_t)r), __uint_as_float(v[j]));
      }
    }
    tc_fence_before();
  }
  if (S > 1) cluster_sync_all();
  else __syncthreads();
  const int my_abort = ctl->abort;
  if (warp >= 2 && !my_abort) {
    // ------------------------------------------------------------ this rank's tokens
    const float4* part = reinterpret_cast<const float4*>(smem) + lane;
    if (S == 1) split_finish<1, EW>(p, part, per, m0, n0 + lane * 4, first, last, bias, res);
    else if (S == 2) split_finish<2, EW>(p, part, per, m0, n0 + lane * 4, first, last, bias, res);
    else if (S == 4) split_finish<4, EW>(p, part, per, m0, n0 + lane * 4, first, last, bias, res);
    else split_finish<8, EW>(p, part, per, m0, n0 + lane * 4, first, last, bias, res);
  }
  // ------------------------------------------------------------ teardown
  if (my_abort) {  // copies still in flight must land before the shared memory is given up
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  // (nobody touches a neighbour's shared memory after the second barrier)
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace rl
