// Attention within packed samples on the tensor cores: backward pass, bf16, head sizes up to 128 (multiples of 8).
//
//   P = exp(scale S - lse),  dP = dO V^T,  dS = P * (dP - delta),  delta = sum_c dO * O
//   dQ = scale dS K,  dV = P^T dO,  dK = scale dS^T Q (summed over the query heads that share the key head)
//
// Two kernels, each with its result in tensor memory until the end, so nothing is added with atomics and every gradient is stored
// once: k_attention_dq has 128 queries and walks over the keys they see, k_attention_dkv has 128 keys and walks over the
// queries (of all heads) that see them. S and dP are made in both: seven products of which five would do, against fp32 additions of
// every dQ tile through the L2 and a pass that converts them.
// In the second kernel the products are transposed, S^T = K Q^T: a key is then a lane of tensor memory, and P^T and dS^T, written
// back to it as bf16, are A operands as they stand. P and dS are rounded to bf16 as the tensor cores ask, an error of the size of the
// gradients' own rounding; statistics and sums are fp32.
//
// A step is 128 rows of the other side at head sizes above 64, and eight warps do the arithmetic between the products, each thread with
// 64 columns of one row. Up to 64 a step is 64 rows and four warps: half the tensor memory, so that two blocks share an SM and one's
// arithmetic runs beside the other's products and waits (8192 rows x 16 heads of 64 1155 us, with 128-row steps and one
// block 1333; 1264 now, with clocks of a longer run and waits that are votes). 16 heads of 128: 1790 us, 768 TFLOP/s by the five products
// of the formula, causal 892 us; the tensor pipe is active 43 and 50 % of the two kernels' time, the rest is the chain from a product
// over the arithmetic to the next. P and dS of the second kernel take the places of S and dP, which are made anew once they have been
// used.
// One warp makes the bulk copies (and fetches the queries' statistics), one issues the products.
// Where the key tiles alone would leave the GPU waiting for the longest sample's first ones, the query heads that share a key head
// are dealt out to the blocks of a cluster, whose sums of dK and dV are added up through shared memory in the order of the blocks.
#include "rmn_attention_tc.cuh"

#include <math_constants.h>

#include <algorithm>

namespace rmn {
namespace tc {
namespace {

constexpr uint32_t kTailBytes = 2560;  // of BwdTail

template <int DP>
struct BwdShape {
  static constexpr int ATOMS = DP / 64;
  static constexpr int STEP = DP == 64 ? 64 : 128;               // rows of a step
  static constexpr int WORK = STEP / 16, HALVES = WORK / 4;      // warps of the arithmetic; groups of four with 64 columns each
  static constexpr int THREADS = (WORK + 2) * 32;
  static constexpr int BLOCKS = DP == 64 ? 2 : 1;                // an SM
  static constexpr uint32_t COLUMNS = DP == 64 ? 256 : 512;      // tensor memory
  static constexpr uint32_t HELD = ATOMS * kAtomBytes;           // a resident tile
  static constexpr uint32_t TILE = ATOMS * STEP * 128;           // a tile of a step
  static constexpr int SLOTS = DP == 64 ? 8 : 5;
  static constexpr uint32_t RING = 2 * HELD, TAIL = RING + SLOTS * TILE;  // two resident tiles, the ring, the rest
  static constexpr size_t SMEM = TAIL + kTailBytes;
};
constexpr int kStats = 2;  // steps whose queries' statistics are in shared memory

struct BwdTail {
  uint64_t full[8], empty[8], held;     // ring slots; the resident tiles
  uint64_t s_full, s_free, dp_full, p_full, ds_full, dv_done, dk_done, st_full[kStats], st_empty[kStats];
  FoundTile found;
  int32_t warp_sums[10];
  uint32_t tmem_slot;
  alignas(16) float lse[kStats][128];   // negative, times log2 e
  alignas(16) float delta[kStats][128]; // negative
};
static_assert(sizeof(BwdTail) <= kTailBytes, "tail");

__device__ __forceinline__ void tc_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  tc_ld32_at<0>(taddr, r);
  tc_ld32_at<32>(taddr + 32, r);
}

// 32 columns of tensor memory times `by` as bf16 to row[c ... c + 31], those below dim; zeros where there are no steps
__device__ __forceinline__ void store32(uint32_t taddr, float by, __nv_bfloat16* row, int c, int dim, bool mine, bool zero) {
  uint32_t o[32];
  if (!zero) {
    tc_ld32(taddr, o);
    tc_wait_ld();
  }
#pragma unroll
  for (int k = 0; k < 32; k += 8) {
    if (!mine || c + k >= dim) continue;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = zero || by == 0.f ? 0u : pack_bf16(__uint_as_float(o[k + 2 * e]) * by, __uint_as_float(o[k + 2 * e + 1]) * by);
    *reinterpret_cast<uint4*>(row + c + k) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// the barriers, the same in both kernels
template <int DP>
__device__ __forceinline__ void init_barriers(BwdTail* tail) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < 8; ++s) {
      mbar_init(&tail->full[s], 1);
      mbar_init(&tail->empty[s], 1);
    }
    uint64_t* ones[] = {&tail->held, &tail->s_full, &tail->dp_full, &tail->dv_done, &tail->dk_done};
    for (uint64_t* b : ones) mbar_init(b, 1);
    uint64_t* all[] = {&tail->s_free, &tail->p_full, &tail->ds_full};
    for (uint64_t* b : all) mbar_init(b, BwdShape<DP>::WORK * 32);
    for (int i = 0; i < kStats; ++i) {
      mbar_init(&tail->st_full[i], 32);
      mbar_init(&tail->st_empty[i], BwdShape<DP>::WORK * 32);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
}

// map_q and map_g (the output's gradient) in boxes of 128 rows, map_k and map_v of a step's
template <int DP>
__global__ void __launch_bounds__(BwdShape<DP>::THREADS, BwdShape<DP>::BLOCKS)
    k_attention_dq(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_g,
                   const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttnArgs a) {
  using C = BwdShape<DP>;
  constexpr int SLOTS = C::SLOTS, STEP = C::STEP;
  constexpr uint32_t T_S = 0, T_DP = STEP, T_DS = 2 * STEP, T_DQ = DP == 64 ? 192 : 320;
  extern __shared__ __align__(1024) uint8_t smem[];
  BwdTail* tail = reinterpret_cast<BwdTail*>(smem + C::TAIL);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  init_barriers<DP>(tail);
  if (tid == C::WORK * 32) {
    tma_prefetch_map(&map_q);
    tma_prefetch_map(&map_k);
    tma_prefetch_map(&map_v);
    tma_prefetch_map(&map_g);
  }
  if (warp == C::WORK + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tail->tmem_slot)),
                 "r"(C::COLUMNS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  after_previous_kernel();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tail->tmem_slot);
  const uint32_t smem_base = smem_u32(smem), ring = smem_base + C::RING;
  bool timed_out = false;

  const int head = blockIdx.x % a.heads;
  const bool exists = find_tile<C::THREADS, TilesOf::kQueries>(a, blockIdx.x / a.heads, 128, &tail->found, tail->warp_sums);
  const Segment g = tail->found.g;
  const int first = (tail->found.tiles - 1 - tail->found.tile) * 128;  // the tiles that see the most keys first
  const int rows = min(128, g.n_q - first);
  const int steps = exists ? (visible_keys(g, first + rows - 1, a.causal) + STEP - 1) / STEP : 0;

  auto lane_wait = [&](uint64_t* bar, uint32_t parity) {
    if (!timed_out && !mbar_wait(bar, parity)) timed_out = true;
    return !timed_out;
  };
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // of a whole warp
    if (!timed_out && !warp_wait(bar, parity)) timed_out = true;
    return !timed_out;
  };
  if (!exists) {
    // nothing to do
  } else if (warp == C::WORK) {
    // ------------------------------ bulk copies: K 0, V 0, K 1, V 1, ... ---------------------
    if (lane == 0 && steps > 0) {
      const int kv = head / (a.heads / a.kv_heads);
      mbar_arrive_expect_tx(&tail->held, 2 * C::HELD);
#pragma unroll
      for (int c = 0; c < C::ATOMS; ++c) {
        tma_load_3d(smem_base + c * kAtomBytes, &map_q, &tail->held, c * 64, head, g.q0 + first);
        tma_load_3d(smem_base + C::HELD + c * kAtomBytes, &map_g, &tail->held, c * 64, head, g.q0 + first);
      }
      uint32_t i = 0;
      for (; i < 2u * (uint32_t)steps; ++i) {
        const uint32_t s = i % SLOTS;
        if (!lane_wait(&tail->empty[s], ((i / SLOTS) & 1u) ^ 1u)) break;
        mbar_arrive_expect_tx(&tail->full[s], C::TILE);
        const CUtensorMap* map = (i & 1u) ? &map_v : &map_k;
#pragma unroll
        for (int c = 0; c < C::ATOMS; ++c)
          tma_load_3d(ring + s * C::TILE + c * (STEP * 128), map, &tail->full[s], c * 64, kv, g.k0 + (int)(i >> 1) * STEP);
      }
      if (timed_out) {  // no copy may be in flight when the block ends
        for (uint32_t k = i > SLOTS ? i - SLOTS : 0; k < i; ++k) mbar_wait(&tail->full[k % SLOTS], (k / SLOTS) & 1u);
        mbar_wait(&tail->held, 0);
      }
    }
  } else if (warp == C::WORK + 1) {
    // ------------------------------ products -------------------------------------------
    const int ksteps = (a.dim + 15) / 16;
    const uint32_t idesc_s = instr_desc(128, STEP, false);
    const uint32_t idesc_o = instr_desc(128, 0, true) | ((uint32_t)(ksteps * 2) << 17);
    auto slot = [&](uint32_t i) { return ring + i % SLOTS * C::TILE; };
    auto ready = [&](uint32_t i) { return wait(&tail->full[i % SLOTS], (i / SLOTS) & 1u); };
    // S and dP of step j
    auto first_products = [&](int j) {
      if (!ready(2u * j)) return;
      if (g.n_k - j * STEP < STEP) zero_rows<STEP>(slot(2u * j), g.n_k - j * STEP, C::ATOMS);  // dS is zero there, K has to be finite
      if (j > 0 && !wait(&tail->s_free, (uint32_t)(j - 1) & 1u)) return;
      tc_fence_after();
      mma_rows<STEP>(tmem + T_S, smem_base, slot(2u * j), idesc_s, ksteps);
      tc_commit_elect(&tail->s_full);
      if (!ready(2u * j + 1u)) return;
      tc_fence_after();
      mma_rows<STEP>(tmem + T_DP, smem_base + C::HELD, slot(2u * j + 1u), idesc_s, ksteps);
      tc_commit_elect(&tail->dp_full);
      tc_commit_elect(&tail->empty[(2u * j + 1u) % SLOTS]);
    };
    if (steps > 0 && wait(&tail->held, 0)) first_products(0);
    for (int j = 0; j < steps && !timed_out; ++j) {
      if (j + 1 < steps) first_products(j + 1);
      if (!wait(&tail->ds_full, (uint32_t)j & 1u)) break;
      tc_fence_after();
      mma_columns<STEP>(tmem + T_DQ, tmem + T_DS, slot(2u * j), idesc_o, j > 0);
      tc_commit_elect(&tail->dk_done);
      tc_commit_elect(&tail->empty[2u * j % SLOTS]);
    }
  } else {
    // ------------------------------ arithmetic -----------------------------------------
    const int half = warp >> 2;
    const uint32_t lanes = ((uint32_t)(warp & 3) * 32u) << 16;
    const int r = (warp & 3) * 32 + lane, row = first + r;
    const bool mine = row < g.n_q;
    const int see = mine ? visible_keys(g, row, a.causal) : 0;
    float lse = 0.f, delta = 0.f;
    const size_t at = ((size_t)(g.q0 + row) * a.heads + head) * a.dim;
    if (mine) {
      // (two halves of the warps take every second eight channels)
      const __nv_bfloat16* grad = static_cast<const __nv_bfloat16*>(a.grad) + (int64_t)(g.q0 + row) * a.grad_row +
                                  (int64_t)head * a.grad_head;
      const __nv_bfloat16* out = static_cast<const __nv_bfloat16*>(a.fwd_out) + at;
      const __nv_bfloat16* low = static_cast<const __nv_bfloat16*>(a.low);
#pragma unroll 4
      for (int c = half * 8; c < a.dim; c += 8 * C::HALVES) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(grad + c)), y = __ldg(reinterpret_cast<const uint4*>(out + c));
        const uint4 z = low ? __ldg(reinterpret_cast<const uint4*>(low + at + c)) : make_uint4(0, 0, 0, 0);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w}, zs[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          delta = fmaf(__uint_as_float(xs[e] << 16), __uint_as_float(ys[e] << 16) + __uint_as_float(zs[e] << 16), delta);
          delta = fmaf(__uint_as_float(xs[e] & 0xffff0000u),
                       __uint_as_float(ys[e] & 0xffff0000u) + __uint_as_float(zs[e] & 0xffff0000u), delta);
        }
      }
      lse = __ldg(a.lse + (size_t)head * a.rows_q + g.q0 + row) * kLog2e;
    }
    if constexpr (C::HALVES == 2) {
      tail->delta[half][r] = delta;
      asm volatile("bar.sync 1, %0;" ::"n"(C::WORK * 32) : "memory");
      delta = tail->delta[0][r] + tail->delta[1][r];
    }
    if (mine && half == 0) a.delta[(size_t)head * a.rows_q + g.q0 + row] = delta;
    const Pair scale = make_pair(a.scale * kLog2e, a.scale * kLog2e), minus_lse = make_pair(-lse, -lse),
               minus_delta = make_pair(-delta, -delta);
    for (int j = 0; j < steps; ++j) {
      const uint32_t ph = (uint32_t)j & 1u;
      uint32_t s[64], dp[64];
      if (!wait(&tail->s_full, ph)) break;
      tc_fence_after();
      tc_ld64(tmem + lanes + T_S + half * 64, s);
      if (!wait(&tail->dp_full, ph)) break;
      tc_fence_after();
      tc_ld64(tmem + lanes + T_DP + half * 64, dp);
      tc_wait_ld();
      tc_fence_before();
      mbar_arrive(&tail->s_free);
      uint32_t w[32];
      const int left = see - j * STEP - half * 64;  // columns that this row sees
#pragma unroll
      for (int c = 0; c < 64; c += 2) {
        float x, y;
        parts(fma(pair_of(s[c], s[c + 1]), scale, minus_lse), x, y);
        const Pair p = make_pair(exp2_approx(x), exp2_approx(y));
        parts(mul(p, add(pair_of(dp[c], dp[c + 1]), minus_delta)), x, y);
        w[c / 2] = pack_bf16(x, y);
      }
      if (left < 64) {
#pragma unroll
        for (int c = 0; c < 32; ++c) w[c] = 2 * c >= left ? 0u : 2 * c + 1 >= left ? w[c] & 0xffffu : w[c];
      }
      if (j > 0 && !wait(&tail->dk_done, ph ^ 1u)) break;  // dS of the step before has been used
      tc_fence_after();
      tc_st32<0>(tmem + lanes + T_DS + half * 32, w);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&tail->ds_full);
    }
    if (steps > 0) wait(&tail->dk_done, (uint32_t)(steps - 1) & 1u);
    tc_fence_after();
    if (!timed_out) {
      __nv_bfloat16* dq = static_cast<__nv_bfloat16*>(a.dq) + at;
      constexpr int PART = DP / C::HALVES;
#pragma unroll
      for (int c = 0; c < PART; c += 32)
        store32(tmem + lanes + T_DQ + half * PART + c, a.scale, dq, half * PART + c, a.dim, mine, steps == 0);
    }
  }

  if (timed_out) atomicExch(a.status, (uint32_t)RMN_ERR_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == C::WORK + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLUMNS) : "memory");
  }
}

// map_k and map_v in boxes of 128 rows, map_q and map_g of a step's
template <int DP>
__global__ void __launch_bounds__(BwdShape<DP>::THREADS, BwdShape<DP>::BLOCKS)
    k_attention_dkv(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_g, const AttnArgs a) {
  using C = BwdShape<DP>;
  constexpr int SLOTS = C::SLOTS, STEP = C::STEP;
  constexpr uint32_t T_S = 0, T_DP = STEP, T_DV = 2 * STEP, T_DK = T_DV + DP;  // P and dS: in the first halves of 64 columns of S, dP
  extern __shared__ __align__(1024) uint8_t smem[];
  BwdTail* tail = reinterpret_cast<BwdTail*>(smem + C::TAIL);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  init_barriers<DP>(tail);
  if (tid == C::WORK * 32) {
    tma_prefetch_map(&map_q);
    tma_prefetch_map(&map_k);
    tma_prefetch_map(&map_v);
    tma_prefetch_map(&map_g);
  }
  if (warp == C::WORK + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tail->tmem_slot)),
                 "r"(C::COLUMNS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  after_previous_kernel();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tail->tmem_slot);
  const uint32_t smem_base = smem_u32(smem), ring = smem_base + C::RING;
  bool timed_out = false;

  const int blocks = (int)cluster_size(), rank = (int)cluster_rank(), group = a.heads / a.kv_heads / blocks;  // heads of this block
  const int kv = blockIdx.x / blocks % a.kv_heads, head0 = (kv * blocks + rank) * group;
  const bool exists =
      find_tile<C::THREADS, TilesOf::kSlots>(a, blockIdx.x / blocks / a.kv_heads, 128, &tail->found, tail->warp_sums);
  const Segment g = tail->found.g;
  const int first = tail->found.tile * 128;  // the first keys are seen by the most queries
  // steps of each head that see any of these keys
  const int from = first_query(g, first, a.causal) / STEP;
  const int tiles = exists && first < g.n_k ? max(0, (g.n_q + STEP - 1) / STEP - from) : 0;
  const int steps = tiles * group;

  auto lane_wait = [&](uint64_t* bar, uint32_t parity) {
    if (!timed_out && !mbar_wait(bar, parity)) timed_out = true;
    return !timed_out;
  };
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // of a whole warp
    if (!timed_out && !warp_wait(bar, parity)) timed_out = true;
    return !timed_out;
  };
  if (!exists) {
    // nothing to do
  } else if (warp == C::WORK) {
    // ------------------------------ bulk copies (Q 0, dO 0, Q 1, dO 1, ...) and statistics -----
    if (lane == 0 && steps > 0) {
      mbar_arrive_expect_tx(&tail->held, 2 * C::HELD);
#pragma unroll
      for (int c = 0; c < C::ATOMS; ++c) {
        tma_load_3d(smem_base + c * kAtomBytes, &map_k, &tail->held, c * 64, kv, g.k0 + first);
        tma_load_3d(smem_base + C::HELD + c * kAtomBytes, &map_v, &tail->held, c * 64, kv, g.k0 + first);
      }
    }
    uint32_t i = 0;  // tiles asked for
    int h = head0, q0 = from * STEP;
    for (int step = 0; step < steps; ++step) {
      // the statistics first: their loads run while the slots are waited for
      constexpr int N = STEP / 32;
      const size_t at = (size_t)h * a.rows_q + g.q0;
      float x[N], y[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int q = q0 + k * 32 + lane;
        x[k] = q < g.n_q ? __ldg(a.lse + at + q) * -kLog2e : 0.f;
        y[k] = q < g.n_q ? -__ldg(a.delta + at + q) : 0.f;
      }
      if (lane == 0) {
        for (int which = 0; which < 2; ++which, ++i) {
          const uint32_t s = i % SLOTS;
          if (!lane_wait(&tail->empty[s], ((i / SLOTS) & 1u) ^ 1u)) break;
          mbar_arrive_expect_tx(&tail->full[s], C::TILE);
#pragma unroll
          for (int c = 0; c < C::ATOMS; ++c)
            tma_load_3d(ring + s * C::TILE + c * (STEP * 128), which ? &map_g : &map_q, &tail->full[s], c * 64, h, g.q0 + q0);
        }
      }
      const int b = step % kStats;
      lane_wait(&tail->st_empty[b], (((uint32_t)step / kStats) & 1u) ^ 1u);
      if (__any_sync(0xffffffffu, timed_out)) {  // the warp leaves together
        timed_out = true;
        break;
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        tail->lse[b][k * 32 + lane] = x[k];
        tail->delta[b][k * 32 + lane] = y[k];
      }
      mbar_arrive(&tail->st_full[b]);
      q0 += STEP;
      if (q0 >= g.n_q) {
        q0 = from * STEP;
        ++h;
      }
    }
    if (lane == 0 && steps > 0 && timed_out) {  // no copy may be in flight when the block ends
      for (uint32_t k = i > SLOTS ? i - SLOTS : 0; k < i; ++k) mbar_wait(&tail->full[k % SLOTS], (k / SLOTS) & 1u);
      mbar_wait(&tail->held, 0);
    }
  } else if (warp == C::WORK + 1) {
    // ------------------------------ products -------------------------------------------
    const int ksteps = (a.dim + 15) / 16;
    const uint32_t idesc_s = instr_desc(128, STEP, false);
    const uint32_t idesc_o = instr_desc(128, 0, true) | ((uint32_t)(ksteps * 2) << 17);
    auto slot = [&](uint32_t i) { return ring + i % SLOTS * C::TILE; };
    // tile i of the ring has arrived; rows behind the sample's last query become zeros, as P and dS are there
    auto ready = [&](uint32_t i) {
      if (!wait(&tail->full[i % SLOTS], (i / SLOTS) & 1u)) return false;
      const int q = (from + (int)(i >> 1) % tiles) * STEP;
      if (g.n_q - q < STEP) zero_rows<STEP>(slot(i), g.n_q - q, C::ATOMS);
      tc_fence_after();
      return true;
    };
    auto make_s = [&](int i) {
      if (!ready(2u * i)) return;
      mma_rows<STEP>(tmem + T_S, smem_base, slot(2u * i), idesc_s, ksteps);
      tc_commit_elect(&tail->s_full);
    };
    auto make_dp = [&](int i) {
      if (!ready(2u * i + 1u)) return;
      mma_rows<STEP>(tmem + T_DP, smem_base + C::HELD, slot(2u * i + 1u), idesc_s, ksteps);
      tc_commit_elect(&tail->dp_full);
    };
    if (steps > 0 && wait(&tail->held, 0)) {
      make_s(0);
      if (!timed_out) make_dp(0);
    }
    for (int i = 0; i < steps && !timed_out; ++i) {
      const uint32_t ph = (uint32_t)i & 1u;
      const bool more = i + 1 < steps;
      if (!wait(&tail->p_full, ph)) break;
      tc_fence_after();
      mma_columns<STEP, 64>(tmem + T_DV, tmem + T_S, slot(2u * i + 1u), idesc_o, i > 0);
      tc_commit_elect(&tail->dv_done);
      tc_commit_elect(&tail->empty[(2u * i + 1u) % SLOTS]);
      if (more && wait(&tail->dv_done, ph)) make_s(i + 1);  // P has been used
      if (!wait(&tail->ds_full, ph)) break;
      tc_fence_after();
      mma_columns<STEP, 64>(tmem + T_DK, tmem + T_DP, slot(2u * i), idesc_o, i > 0);
      tc_commit_elect(&tail->dk_done);
      tc_commit_elect(&tail->empty[2u * i % SLOTS]);
      if (more && wait(&tail->dk_done, ph)) make_dp(i + 1);  // dS has been used
    }
  } else {
    // ------------------------------ arithmetic -----------------------------------------
    const int half = warp >> 2;
    const uint32_t lanes = ((uint32_t)(warp & 3) * 32u) << 16;
    const int row = first + (warp & 3) * 32 + lane;  // key
    const int sees = first_query(g, row, a.causal);  // its first query
    const Pair scale = make_pair(a.scale * kLog2e, a.scale * kLog2e);
    int q0 = from * STEP;
    for (int i = 0; i < steps; ++i) {
      const uint32_t ph = (uint32_t)i & 1u;
      const int b = i % kStats;
      const int lo = sees - q0 - half * 64, hi = g.n_q - q0 - half * 64;  // columns of the queries that see this key
      q0 = q0 + STEP >= g.n_q ? from * STEP : q0 + STEP;
      const ulonglong2* lse = reinterpret_cast<const ulonglong2*>(&tail->lse[b][half * 64]);
      const ulonglong2* delta = reinterpret_cast<const ulonglong2*>(&tail->delta[b][half * 64]);
      uint32_t s[64], w[32];
      if (!wait(&tail->st_full[b], ((uint32_t)i / kStats) & 1u) || !wait(&tail->s_full, ph)) break;
      tc_fence_after();
      tc_ld64(tmem + lanes + T_S + half * 64, s);
      tc_wait_ld();
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        const ulonglong2 l = lse[c / 4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x, y;
          parts(fma(pair_of(s[c + 2 * e], s[c + 2 * e + 1]), scale, Pair{e ? l.y : l.x}), x, y);
          s[c + 2 * e] = __float_as_uint(exp2_approx(x));
          s[c + 2 * e + 1] = __float_as_uint(exp2_approx(y));
        }
      }
      if (lo > 0 || hi < 64) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c < lo || c >= hi) s[c] = 0u;
      }
#pragma unroll
      for (int c = 0; c < 32; ++c) w[c] = pack_bf16(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1]));
      tc_st32<0>(tmem + lanes + T_S + half * 64, w);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&tail->p_full);
      uint32_t dp[64];
      if (!wait(&tail->dp_full, ph)) break;
      tc_fence_after();
      tc_ld64(tmem + lanes + T_DP + half * 64, dp);
      tc_wait_ld();
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        const ulonglong2 d = delta[c / 4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int k = c + 2 * e;
          float x, y;
          parts(mul(pair_of(s[k], s[k + 1]), add(pair_of(dp[k], dp[k + 1]), Pair{e ? d.y : d.x})), x, y);
          w[k / 2] = pack_bf16(x, y);
        }
      }
      mbar_arrive(&tail->st_empty[b]);
      if (lo > 0 || hi < 64) {  // (zero times what is not finite)
#pragma unroll
        for (int c = 0; c < 32; ++c)
          w[c] &= (2 * c < lo || 2 * c >= hi ? 0u : 0xffffu) | (2 * c + 1 < lo || 2 * c + 1 >= hi ? 0u : 0xffff0000u);
      }
      tc_st32<0>(tmem + lanes + T_DP + half * 64, w);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&tail->ds_full);
    }
    if (steps > 0 && wait(&tail->dv_done, (uint32_t)(steps - 1) & 1u)) wait(&tail->dk_done, (uint32_t)(steps - 1) & 1u);
    tc_fence_after();
    if (!timed_out) {
      const size_t at = ((size_t)(g.k0 + row) * a.kv_heads + kv) * a.dim;
      const bool mine = row < g.k_slot;
#pragma unroll
      for (int which = 0; which < 2; ++which) {  // dv, dk; where there are two halves of the warps, one each
        if (C::HALVES == 2 && which != half) continue;
        const uint32_t from_t = tmem + lanes + (which ? T_DK : T_DV);
        if (blocks == 1) {
          __nv_bfloat16* to = static_cast<__nv_bfloat16*>(which ? a.dk : a.dv) + at;
          const float by = row >= g.n_k ? 0.f : which ? a.scale : 1.f;
#pragma unroll
          for (int c = 0; c < DP; c += 32) store32(from_t + c, by, to, c, a.dim, mine, steps == 0);
        } else {
          // this block's part, for all of the cluster: [which][channel / 4][key], in the place of the tiles
#pragma unroll
          for (int c = 0; c < DP; c += 32) {
            uint32_t o[32];
            if (steps > 0) {
              tc_ld32(from_t + c, o);
              tc_wait_ld();
            }
            float4* to = reinterpret_cast<float4*>(smem) + (which * DP + c) / 4 * 128 + (row - first);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              to[k * 128] = steps == 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                                       : make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                                     __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
          }
        }
      }
    }
  }
  if (blocks > 1) {
    static_assert(2 * DP * 128 * sizeof(float) <= C::TAIL, "parts in the place of the tiles");
    cluster_sync();
    if (exists && tid < 128) {
      // every block sums its share of the eights of channels, over the blocks in their order
      const int row = first + tid;
      const size_t at = ((size_t)(g.k0 + row) * a.kv_heads + kv) * a.dim;
      for (int e = rank; e < 2 * DP / 8; e += blocks) {
        const int which = e / (DP / 8), c = e % (DP / 8) * 8;
        if (c >= a.dim) continue;
        const uint32_t addr = smem_base + (uint32_t)(e * 2 * 128 + tid) * 16u;
        float4 x = load_of_block(addr, 0), y = load_of_block(addr + 128 * 16, 0);
        for (int r = 1; r < blocks; ++r) {
          const float4 u = load_of_block(addr, (uint32_t)r), v = load_of_block(addr + 128 * 16, (uint32_t)r);
          x.x += u.x; x.y += u.y; x.z += u.z; x.w += u.w;
          y.x += v.x; y.y += v.y; y.z += v.z; y.w += v.w;
        }
        if (row >= g.k_slot) continue;
        const float by = which ? a.scale : 1.f;
        __nv_bfloat16* to = static_cast<__nv_bfloat16*>(which ? a.dk : a.dv) + at + c;
        *reinterpret_cast<uint4*>(to) =
            row >= g.n_k ? make_uint4(0u, 0u, 0u, 0u)
                         : make_uint4(pack_bf16(x.x * by, x.y * by), pack_bf16(x.z * by, x.w * by), pack_bf16(y.x * by, y.y * by),
                                      pack_bf16(y.z * by, y.w * by));
      }
    }
    cluster_sync();  // no block leaves while another reads its part
  }

  if (timed_out) atomicExch(a.status, (uint32_t)RMN_ERR_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == C::WORK + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLUMNS) : "memory");
  }
}

template <int DP>
int launch_bwd(const AttnArgs& a, cudaStream_t stream) {
  using C = BwdShape<DP>;
  static SmemOptIn opt_q, opt_kv;
  // [0]: boxes of 128 rows, [1]: of a step's
  CUtensorMap q[2], k[2], v[2], g[2];
  for (int i = 0; i < (C::STEP == 128 ? 1 : 2); ++i) {
    const int rows = i ? C::STEP : 128;
    if (!make_head_map(&q[i], a.q, a.rows_q, a.heads, a.dim, a.q_row, a.q_head, rows) ||
        !make_head_map(&k[i], a.k, a.rows_k, a.kv_heads, a.dim, a.k_row, a.k_head, rows) ||
        !make_head_map(&v[i], a.v, a.rows_k, a.kv_heads, a.dim, a.v_row, a.v_head, rows) ||
        !make_head_map(&g[i], a.grad, a.rows_q, a.heads, a.dim, a.grad_row, a.grad_head, rows))
      return RMN_ERR_UNSUPPORTED;
  }
  constexpr int STEPS = C::STEP == 128 ? 0 : 1;
  const uint64_t q_blocks = most_tiles(a.rows_q, a.sequences, 128) * a.heads;
  const uint64_t k_blocks = most_tiles(a.rows_k, a.sequences, 128) * a.kv_heads;
  // With fewer than two tiles of keys for each block that fits the GPU (a sample has a tile at least): clusters of as many blocks, up to
  // eight (the portable size), as the query heads of a key head divide into. Backward of 8 samples of 151 ... 5003 rows, 8 / 2 heads of
  // 64, 238 tiles for 296 places: 560 us without, 340 with; of two samples of 3989 and 4600 rows, 16 / 8 heads of 128, 536 tiles for 148
  // places: 548 and 604; of 4096 samples of 4 rows, 8 / 1 heads of 64: 990 and 2121.
  const int group = a.heads / a.kv_heads;
  int cluster = 1;
  const uint64_t samples = std::max<uint64_t>(1, std::min(a.sequences, a.rows_k));  // (that can have a row)
  const uint64_t tiles = samples * ((a.rows_k / samples + 127) / 128);
  if (tiles * a.kv_heads < 2 * 148 * C::BLOCKS) {
    for (int n = 2; n <= 8; ++n)
      if (group % n == 0) cluster = n;
  }
  if (k_blocks * cluster > 0x7fffffffull) return RMN_ERR_UNSUPPORTED;
  if (q_blocks > 0x7fffffffull || k_blocks > 0x7fffffffull) return RMN_ERR_UNSUPPORTED;
  RMN_CUDA_TRY(opt_q.apply(reinterpret_cast<const void*>(k_attention_dq<DP>), C::SMEM));
  RMN_CUDA_TRY(opt_kv.apply(reinterpret_cast<const void*>(k_attention_dkv<DP>), C::SMEM));
  RMN_CUDA_TRY(launch_overlapped(k_attention_dq<DP>, dim3((uint32_t)q_blocks), dim3(C::THREADS), C::SMEM, stream, q[0], g[0],
                                 k[STEPS], v[STEPS], a));
  RMN_LAUNCH_CHECK();
  count_tc_launch();
  RMN_CUDA_TRY(launch_overlapped_clusters(k_attention_dkv<DP>, (uint32_t)cluster, dim3((uint32_t)(k_blocks * cluster)),
                                          dim3(C::THREADS), C::SMEM, stream, k[0], v[0], q[STEPS], g[STEPS], a));
  RMN_LAUNCH_CHECK();
  count_tc_launch();
  return RMN_OK;
}

}  // namespace
}  // namespace tc

int attention_tc_backward(const AttnArgs& a, cudaStream_t stream) {
  using namespace tc;
  if (a.dim > 128 || !(a.scale > 0.f)) return RMN_ERR_UNSUPPORTED;
  for (const void* p : {a.fwd_out, (const void*)a.low, (const void*)a.dq, (const void*)a.dk, (const void*)a.dv})
    if ((uintptr_t)p & 15) return RMN_ERR_UNSUPPORTED;
  return a.dim <= 64 ? launch_bwd<64>(a, stream) : launch_bwd<128>(a, stream);
}

}  // namespace rmn
