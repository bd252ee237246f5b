// Attention within packed samples on the tensor cores: backward pass, bf16, head sizes up to 128 (multiples of 8).
//
//   P = exp(scale S - lse),  dP = dO V^T,  dS = P * (dP - delta),  delta = sum_c dO * O
//   dQ = scale dS K,  dV = P^T dO,  dK = scale dS^T Q (summed over the query heads that share the key head)
//
// Two kernels, each with its result in tensor memory until the end, so nothing is added with atomics and every gradient is stored
// once: k_attention_dq has 128 queries and walks over the keys they see, k_attention_dkv has 128 keys and walks over the
// queries (of all heads) that see them. S and dP are made in both: seven products of which five would do, 4/7 of the tensor
// cores' time at most, against fp32 additions of every dQ tile through the L2 and a pass that converts them.
// In the second kernel the products are transposed, S^T = K Q^T: a key is then a lane of tensor memory, and P^T and dS^T, written
// back to it as bf16, are A operands as they stand. P and dS are rounded to bf16 as the tensor cores ask, an error of the size of the
// gradients' own rounding; statistics and sums are fp32.
//
// Warps: eight for the arithmetic between the products (a thread has 64 columns of one row: warps 0 - 3 the left half, 4 - 7 the
// right), one for the bulk copies, one that issues the products, one for the rows' statistics. The four products of a step take
// 16 * head size clocks on the tensor cores in the second kernel, the exponentials 1024 (16 a clock): at 128 channels the
// first bounds, at 64 and below the exponentials and the passage through registers.
#include "rmn_attention_tc.cuh"

#include <math_constants.h>

namespace rmn {
namespace tc {
namespace {

constexpr int kBwdThreads = 384;

template <int DP>
struct BwdShape {
  static constexpr int ATOMS = DP / 64;
  static constexpr uint32_t TILE = ATOMS * kAtomBytes;
  static constexpr int SLOTS = DP == 128 ? 5 : 6;
  static constexpr uint32_t RING = 2 * TILE, TAIL = RING + SLOTS * TILE;  // two resident tiles, the ring, the rest
  static constexpr size_t SMEM = TAIL + 2560;
};

struct BwdTail {
  uint64_t full[6], empty[6], held;     // ring slots; the resident tiles
  uint64_t s_full, s_free, dp_full, dp_free, p_full, ds_full, dv_done, dk_done, st_full[2], st_empty[2];
  FoundTile found;
  int32_t warp_sums[kBwdThreads / 32];
  uint32_t tmem_slot;
  alignas(16) float lse[2][128];
  alignas(16) float delta[2][128];
};
static_assert(sizeof(BwdTail) <= 2560, "tail");

__device__ __forceinline__ void tc_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  tc_ld32_at<0>(taddr, r);
  tc_ld32_at<32>(taddr + 32, r);
}

// 32 columns of tensor memory times `by` as bf16 to row[c ... c + 31], those below dim
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
      w[e] = zero ? 0u : pack_bf16(__uint_as_float(o[k + 2 * e]) * by, __uint_as_float(o[k + 2 * e + 1]) * by);
    *reinterpret_cast<uint4*>(row + c + k) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// the barriers, the same in both kernels
__device__ __forceinline__ void init_barriers(BwdTail* tail) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < 6; ++s) {
      mbar_init(&tail->full[s], 1);
      mbar_init(&tail->empty[s], 1);
    }
    uint64_t* ones[] = {&tail->held, &tail->s_full, &tail->dp_full, &tail->dv_done, &tail->dk_done};
    for (uint64_t* b : ones) mbar_init(b, 1);
    uint64_t* all[] = {&tail->s_free, &tail->dp_free, &tail->p_full, &tail->ds_full, &tail->st_empty[0], &tail->st_empty[1]};
    for (uint64_t* b : all) mbar_init(b, 256);
    mbar_init(&tail->st_full[0], 32);
    mbar_init(&tail->st_full[1], 32);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
}

template <int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
    k_attention_dq(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g, const AttnArgs a) {
  using C = BwdShape<DP>;
  constexpr int SLOTS = C::SLOTS;
  constexpr uint32_t T_S = 0, T_DP = 128, T_DS = 256, T_DQ = 320;
  extern __shared__ __align__(1024) uint8_t smem[];
  BwdTail* tail = reinterpret_cast<BwdTail*>(smem + C::TAIL);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  init_barriers(tail);
  if (tid == 8 * 32) {
    tma_prefetch_map(&map_q);
    tma_prefetch_map(&map_k);
    tma_prefetch_map(&map_v);
    tma_prefetch_map(&map_g);
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tail->tmem_slot)) : "memory");
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
  const bool exists = find_tile<kBwdThreads, TilesOf::kQueries>(a, blockIdx.x / a.heads, 128, &tail->found, tail->warp_sums);
  const Segment g = tail->found.g;
  const int first = (tail->found.tiles - 1 - tail->found.tile) * 128;  // the tiles that see the most keys first
  const int rows = min(128, g.n_q - first);
  const int steps = exists ? (visible_keys(g, first + rows - 1, a.causal) + 127) / 128 : 0;

  if (!exists) {
    // nothing to do
  } else if (warp == 8) {
    // ------------------------------ bulk copies: K 0, V 0, K 1, V 1, ... ---------------------
    if (lane == 0 && steps > 0) {
      const int kv = head / (a.heads / a.kv_heads);
      mbar_arrive_expect_tx(&tail->held, 2 * C::TILE);
#pragma unroll
      for (int c = 0; c < C::ATOMS; ++c) {
        tma_load_3d(smem_base + c * kAtomBytes, &map_q, &tail->held, c * 64, head, g.q0 + first);
        tma_load_3d(smem_base + C::TILE + c * kAtomBytes, &map_g, &tail->held, c * 64, head, g.q0 + first);
      }
      uint32_t i = 0;
      for (; i < 2u * (uint32_t)steps; ++i) {
        const uint32_t s = i % SLOTS;
        if (!mbar_wait(&tail->empty[s], ((i / SLOTS) & 1u) ^ 1u)) { timed_out = true; break; }
        mbar_arrive_expect_tx(&tail->full[s], C::TILE);
        const CUtensorMap* map = (i & 1u) ? &map_v : &map_k;
#pragma unroll
        for (int c = 0; c < C::ATOMS; ++c)
          tma_load_3d(ring + s * C::TILE + c * kAtomBytes, map, &tail->full[s], c * 64, kv, g.k0 + (int)(i >> 1) * 128);
      }
      if (timed_out) {  // no copy may be in flight when the block ends
        for (uint32_t k = i > SLOTS ? i - SLOTS : 0; k < i; ++k) mbar_wait(&tail->full[k % SLOTS], (k / SLOTS) & 1u);
        mbar_wait(&tail->held, 0);
      }
    }
  } else if (warp == 9) {
    // ------------------------------ products -------------------------------------------
    const int ksteps = (a.dim + 15) / 16;
    const uint32_t idesc_s = instr_desc(128, 128, false);
    const uint32_t idesc_o = instr_desc(128, 0, true) | ((uint32_t)(ksteps * 2) << 17);
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (!timed_out && !mbar_wait(bar, parity)) timed_out = true;
      return !timed_out;
    };
    auto slot = [&](uint32_t i) { return ring + i % SLOTS * C::TILE; };
    auto ready = [&](uint32_t i) { return wait(&tail->full[i % SLOTS], (i / SLOTS) & 1u); };
    // S and dP of step j
    auto first_products = [&](int j) {
      if (!ready(2u * j)) return;
      if (g.n_k - j * 128 < 128) zero_rows(slot(2u * j), g.n_k - j * 128, C::ATOMS);  // dS is zero there, K has to be finite
      if (j > 0 && !wait(&tail->s_free, (uint32_t)(j - 1) & 1u)) return;
      tc_fence_after();
      mma_rows(tmem + T_S, smem_base, slot(2u * j), idesc_s, ksteps);
      tc_commit_elect(&tail->s_full);
      if (!ready(2u * j + 1u)) return;
      tc_fence_after();
      mma_rows(tmem + T_DP, smem_base + C::TILE, slot(2u * j + 1u), idesc_s, ksteps);
      tc_commit_elect(&tail->dp_full);
      tc_commit_elect(&tail->empty[(2u * j + 1u) % SLOTS]);
    };
    if (steps > 0 && wait(&tail->held, 0)) first_products(0);
    for (int j = 0; j < steps && !timed_out; ++j) {
      if (j + 1 < steps) first_products(j + 1);
      if (!wait(&tail->ds_full, (uint32_t)j & 1u)) break;
      tc_fence_after();
      mma_columns(tmem + T_DQ, tmem + T_DS, slot(2u * j), idesc_o, j > 0);
      tc_commit_elect(&tail->dk_done);
      tc_commit_elect(&tail->empty[2u * j % SLOTS]);
    }
  } else if (warp < 8) {
    // ------------------------------ arithmetic -----------------------------------------
    const int half = warp >> 2;
    const uint32_t lanes = ((uint32_t)(warp & 3) * 32u) << 16;
    const int r = (warp & 3) * 32 + lane, row = first + r;
    const bool mine = row < g.n_q;
    const int see = mine ? visible_keys(g, row, a.causal) : 0;
    const float scale = a.scale * kLog2e;
    float lse = 0.f;
    const size_t at = ((size_t)(g.q0 + row) * a.heads + head) * a.dim;
    {
      // delta: the two halves of the warps take the two halves of the channels
      float d = 0.f;
      if (mine) {
        const __nv_bfloat16* grad = static_cast<const __nv_bfloat16*>(a.grad) + (int64_t)(g.q0 + row) * a.grad_row +
                                    (int64_t)head * a.grad_head;
        const __nv_bfloat16* out = static_cast<const __nv_bfloat16*>(a.fwd_out) + at;
        const __nv_bfloat16* low = static_cast<const __nv_bfloat16*>(a.low);
#pragma unroll 4
        for (int c = half * 8; c < a.dim; c += 16) {
          const uint4 x = __ldg(reinterpret_cast<const uint4*>(grad + c)), y = __ldg(reinterpret_cast<const uint4*>(out + c));
          const uint4 z = low ? __ldg(reinterpret_cast<const uint4*>(low + at + c)) : make_uint4(0, 0, 0, 0);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w}, zs[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d = fmaf(__uint_as_float(xs[e] << 16), __uint_as_float(ys[e] << 16) + __uint_as_float(zs[e] << 16), d);
            d = fmaf(__uint_as_float(xs[e] & 0xffff0000u),
                     __uint_as_float(ys[e] & 0xffff0000u) + __uint_as_float(zs[e] & 0xffff0000u), d);
          }
        }
        lse = __ldg(a.lse + (size_t)head * a.rows_q + g.q0 + row) * kLog2e;
      }
      tail->delta[half][r] = d;
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");  // the eight warps
    const float delta = tail->delta[0][r] + tail->delta[1][r];
    if (mine && half == 0) a.delta[(size_t)head * a.rows_q + g.q0 + row] = delta;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (!timed_out && !mbar_wait(bar, parity)) timed_out = true;
      return !timed_out;
    };
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
      const int left = see - j * 128 - half * 64;  // columns that this row sees
#pragma unroll
      for (int c = 0; c < 64; c += 2) {
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp2_approx(fmaf(__uint_as_float(s[c + e]), scale, -lse));
          x[e] = p * (__uint_as_float(dp[c + e]) - delta);
        }
        if (left < 64) {
          if (c >= left) x[0] = 0.f;
          if (c + 1 >= left) x[1] = 0.f;
        }
        w[c / 2] = pack_bf16(x[0], x[1]);
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
#pragma unroll
      for (int c = 0; c < DP / 2; c += 32)
        store32(tmem + lanes + T_DQ + half * (DP / 2) + c, a.scale, dq, half * (DP / 2) + c, a.dim, mine, steps == 0);
    }
  }

  if (timed_out) atomicExch(a.status, (uint32_t)RMN_ERR_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
    k_attention_dkv(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g, const AttnArgs a) {
  using C = BwdShape<DP>;
  constexpr int SLOTS = C::SLOTS;
  // Up to 64 channels P and dS have columns of their own, and the next S and dP are made while these are worked on; above, they
  // take the places of S and dP (each half of the warps within its own columns).
  constexpr bool kAlias = DP == 128;
  constexpr int kHalf = kAlias ? 64 : 32;
  constexpr uint32_t T_S = 0, T_DP = 128, T_P = kAlias ? T_S : 256, T_DS = kAlias ? T_DP : 320, T_DV = kAlias ? 256 : 384,
                     T_DK = T_DV + DP;
  extern __shared__ __align__(1024) uint8_t smem[];
  BwdTail* tail = reinterpret_cast<BwdTail*>(smem + C::TAIL);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  init_barriers(tail);
  if (tid == 8 * 32) {
    tma_prefetch_map(&map_q);
    tma_prefetch_map(&map_k);
    tma_prefetch_map(&map_v);
    tma_prefetch_map(&map_g);
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tail->tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  after_previous_kernel();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tail->tmem_slot);
  const uint32_t smem_base = smem_u32(smem), ring = smem_base + C::RING;
  bool timed_out = false;

  const int kv = blockIdx.x % a.kv_heads, group = a.heads / a.kv_heads;
  const bool exists = find_tile<kBwdThreads, TilesOf::kSlots>(a, blockIdx.x / a.kv_heads, 128, &tail->found, tail->warp_sums);
  const Segment g = tail->found.g;
  const int first = tail->found.tile * 128;  // the first keys are seen by the most queries
  // query tiles of each head that see any of these keys
  const int from = first_query(g, first, a.causal) / 128;
  const int tiles = exists && first < g.n_k ? max(0, (g.n_q + 127) / 128 - from) : 0;
  const int steps = tiles * group;

  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!timed_out && !mbar_wait(bar, parity)) timed_out = true;
    return !timed_out;
  };
  if (!exists) {
    // nothing to do
  } else if (warp == 8) {
    // ------------------------------ bulk copies: Q 0, dO 0, Q 1, dO 1, ... ---------------------
    if (lane == 0 && steps > 0) {
      mbar_arrive_expect_tx(&tail->held, 2 * C::TILE);
#pragma unroll
      for (int c = 0; c < C::ATOMS; ++c) {
        tma_load_3d(smem_base + c * kAtomBytes, &map_k, &tail->held, c * 64, kv, g.k0 + first);
        tma_load_3d(smem_base + C::TILE + c * kAtomBytes, &map_v, &tail->held, c * 64, kv, g.k0 + first);
      }
      uint32_t i = 0;
      for (; i < 2u * (uint32_t)steps; ++i) {
        const uint32_t s = i % SLOTS;
        if (!wait(&tail->empty[s], ((i / SLOTS) & 1u) ^ 1u)) break;
        mbar_arrive_expect_tx(&tail->full[s], C::TILE);
        const CUtensorMap* map = (i & 1u) ? &map_g : &map_q;
        const int step = (int)(i >> 1), h = kv * group + step / tiles, q = g.q0 + (from + step % tiles) * 128;
#pragma unroll
        for (int c = 0; c < C::ATOMS; ++c) tma_load_3d(ring + s * C::TILE + c * kAtomBytes, map, &tail->full[s], c * 64, h, q);
      }
      if (timed_out) {  // no copy may be in flight when the block ends
        for (uint32_t k = i > SLOTS ? i - SLOTS : 0; k < i; ++k) mbar_wait(&tail->full[k % SLOTS], (k / SLOTS) & 1u);
        mbar_wait(&tail->held, 0);
      }
    }
  } else if (warp == 9) {
    // ------------------------------ products -------------------------------------------
    const int ksteps = (a.dim + 15) / 16;
    const uint32_t idesc_s = instr_desc(128, 128, false);
    const uint32_t idesc_o = instr_desc(128, 0, true) | ((uint32_t)(ksteps * 2) << 17);
    auto slot = [&](uint32_t i) { return ring + i % SLOTS * C::TILE; };
    // tile i of the ring has arrived; rows behind the sample's last query become zeros, as P and dS are there
    auto ready = [&](uint32_t i) {
      if (!wait(&tail->full[i % SLOTS], (i / SLOTS) & 1u)) return false;
      const int q = (from + (int)(i >> 1) % tiles) * 128;
      if (g.n_q - q < 128) zero_rows(slot(i), g.n_q - q, C::ATOMS);
      tc_fence_after();
      return true;
    };
    auto make_s = [&](int i) {
      if (!ready(2u * i)) return;
      mma_rows(tmem + T_S, smem_base, slot(2u * i), idesc_s, ksteps);
      tc_commit_elect(&tail->s_full);
    };
    auto make_dp = [&](int i) {
      if (!ready(2u * i + 1u)) return;
      mma_rows(tmem + T_DP, smem_base + C::TILE, slot(2u * i + 1u), idesc_s, ksteps);
      tc_commit_elect(&tail->dp_full);
    };
    auto add_dv = [&](int i) {
      if (!wait(&tail->p_full, (uint32_t)i & 1u)) return;
      tc_fence_after();
      mma_columns<kHalf>(tmem + T_DV, tmem + T_P, slot(2u * i + 1u), idesc_o, i > 0);
      tc_commit_elect(&tail->dv_done);
      tc_commit_elect(&tail->empty[(2u * i + 1u) % SLOTS]);
    };
    auto add_dk = [&](int i) {
      if (!wait(&tail->ds_full, (uint32_t)i & 1u)) return;
      tc_fence_after();
      mma_columns<kHalf>(tmem + T_DK, tmem + T_DS, slot(2u * i), idesc_o, i > 0);
      tc_commit_elect(&tail->dk_done);
      tc_commit_elect(&tail->empty[2u * i % SLOTS]);
    };
    if (steps > 0 && wait(&tail->held, 0)) {
      make_s(0);
      if (!timed_out) make_dp(0);
    }
    for (int i = 0; i < steps && !timed_out; ++i) {
      const uint32_t ph = (uint32_t)i & 1u;
      const bool more = i + 1 < steps;
      if constexpr (kAlias) {
        add_dv(i);
        if (more && wait(&tail->dv_done, ph)) make_s(i + 1);
        if (!timed_out) add_dk(i);
        if (more && wait(&tail->dk_done, ph)) make_dp(i + 1);
      } else {
        if (more && wait(&tail->s_free, ph)) make_s(i + 1);
        if (!timed_out) add_dv(i);
        if (more && wait(&tail->dp_free, ph)) make_dp(i + 1);
        if (!timed_out) add_dk(i);
      }
    }
  } else if (warp == 10) {
    // ------------------------------ statistics of the queries --------------------------
    for (int i = 0; i < steps; ++i) {
      const int h = kv * group + i / tiles, q0 = (from + i % tiles) * 128, b = i & 1;
      const size_t at = (size_t)h * a.rows_q + g.q0;
      float x[4], y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int q = q0 + k * 32 + lane;
        x[k] = q < g.n_q ? __ldg(a.lse + at + q) * kLog2e : 0.f;
        y[k] = q < g.n_q ? __ldg(a.delta + at + q) : 0.f;
      }
      if (!wait(&tail->st_empty[b], (((uint32_t)i >> 1) & 1u) ^ 1u)) break;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        tail->lse[b][k * 32 + lane] = x[k];
        tail->delta[b][k * 32 + lane] = y[k];
      }
      mbar_arrive(&tail->st_full[b]);
    }
  } else if (warp < 8) {
    // ------------------------------ arithmetic -----------------------------------------
    const int half = warp >> 2;
    const uint32_t lanes = ((uint32_t)(warp & 3) * 32u) << 16;
    const int row = first + (warp & 3) * 32 + lane;  // key
    const int sees = first_query(g, row, a.causal);  // its first query
    const float scale = a.scale * kLog2e;
    for (int i = 0; i < steps; ++i) {
      const uint32_t ph = (uint32_t)i & 1u;
      const int b = i & 1, q0 = (from + i % tiles) * 128 + half * 64;
      const int lo = sees - q0, hi = g.n_q - q0;  // columns of the queries that see this key
      const float4* lse = reinterpret_cast<const float4*>(&tail->lse[b][half * 64]);
      const float4* delta = reinterpret_cast<const float4*>(&tail->delta[b][half * 64]);
      uint32_t s[64], w[32];
      if (!wait(&tail->st_full[b], ((uint32_t)i >> 1) & 1u) || !wait(&tail->s_full, ph)) break;
      tc_fence_after();
      tc_ld64(tmem + lanes + T_S + half * 64, s);
      tc_wait_ld();
      if constexpr (!kAlias) {
        tc_fence_before();
        mbar_arrive(&tail->s_free);
      }
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        const float4 l = lse[c / 4];
        const float ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float p = exp2_approx(fmaf(__uint_as_float(s[c + e]), scale, -ls[e]));
          s[c + e] = __float_as_uint(p);
        }
      }
      if (lo > 0 || hi < 64) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c < lo || c >= hi) s[c] = 0u;
      }
#pragma unroll
      for (int c = 0; c < 32; ++c) w[c] = pack_bf16(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1]));
      if constexpr (!kAlias) {
        if (i > 0 && !wait(&tail->dv_done, ph ^ 1u)) break;  // P of the step before has been used
        tc_fence_after();
      }
      tc_st32<0>(tmem + lanes + T_P + half * kHalf, w);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&tail->p_full);
      uint32_t dp[64];
      if (!wait(&tail->dp_full, ph)) break;
      tc_fence_after();
      tc_ld64(tmem + lanes + T_DP + half * 64, dp);
      tc_wait_ld();
      if constexpr (!kAlias) {
        tc_fence_before();
        mbar_arrive(&tail->dp_free);
      }
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        const float4 d = delta[c / 4];
        const float ds[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          dp[c + e] = __float_as_uint(__uint_as_float(s[c + e]) * (__uint_as_float(dp[c + e]) - ds[e]));
      }
      mbar_arrive(&tail->st_empty[b]);
      if (lo > 0 || hi < 64) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c < lo || c >= hi) dp[c] = 0u;
      }
#pragma unroll
      for (int c = 0; c < 32; ++c) w[c] = pack_bf16(__uint_as_float(dp[2 * c]), __uint_as_float(dp[2 * c + 1]));
      if constexpr (!kAlias) {
        if (i > 0 && !wait(&tail->dk_done, ph ^ 1u)) break;
        tc_fence_after();
      }
      tc_st32<0>(tmem + lanes + T_DS + half * kHalf, w);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&tail->ds_full);
    }
    // the left half of the warps stores dv, the right half dk
    if (steps > 0) wait(half == 0 ? &tail->dv_done : &tail->dk_done, (uint32_t)(steps - 1) & 1u);
    tc_fence_after();
    if (!timed_out) {
      __nv_bfloat16* to = static_cast<__nv_bfloat16*>(half == 0 ? a.dv : a.dk) +
                          ((size_t)(g.k0 + row) * a.kv_heads + kv) * a.dim;
      const bool mine = row < g.k_slot;
      const float by = row >= g.n_k ? 0.f : half == 0 ? 1.f : a.scale;
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32];
        if (steps > 0) {
          tc_ld32(tmem + lanes + (half == 0 ? T_DV : T_DK) + c, o);
          tc_wait_ld();
        }
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          if (!mine || c + k >= a.dim) continue;
          uint32_t v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = by == 0.f || steps == 0 ? 0u
                                           : pack_bf16(__uint_as_float(o[k + 2 * e]) * by, __uint_as_float(o[k + 2 * e + 1]) * by);
          *reinterpret_cast<uint4*>(to + c + k) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
    }
  }

  if (timed_out) atomicExch(a.status, (uint32_t)RMN_ERR_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <int DP>
int launch_bwd(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& g, const AttnArgs& a,
               cudaStream_t stream) {
  using C = BwdShape<DP>;
  static SmemOptIn opt_q, opt_kv;
  const uint64_t q_blocks = most_tiles(a.rows_q, a.sequences, 128) * a.heads;
  const uint64_t k_blocks = most_tiles(a.rows_k, a.sequences, 128) * a.kv_heads;
  if (q_blocks > 0x7fffffffull || k_blocks > 0x7fffffffull) return RMN_ERR_UNSUPPORTED;
  RMN_CUDA_TRY(opt_q.apply(reinterpret_cast<const void*>(k_attention_dq<DP>), C::SMEM));
  RMN_CUDA_TRY(opt_kv.apply(reinterpret_cast<const void*>(k_attention_dkv<DP>), C::SMEM));
  RMN_CUDA_TRY(launch_overlapped(k_attention_dq<DP>, dim3((uint32_t)q_blocks), dim3(kBwdThreads), C::SMEM, stream, q, k, v, g, a));
  RMN_LAUNCH_CHECK();
  count_tc_launch();
  RMN_CUDA_TRY(launch_overlapped(k_attention_dkv<DP>, dim3((uint32_t)k_blocks), dim3(kBwdThreads), C::SMEM, stream, q, k, v, g, a));
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
  CUtensorMap q, k, v, g;
  if (!make_head_map(&q, a.q, a.rows_q, a.heads, a.dim, a.q_row, a.q_head) ||
      !make_head_map(&k, a.k, a.rows_k, a.kv_heads, a.dim, a.k_row, a.k_head) ||
      !make_head_map(&v, a.v, a.rows_k, a.kv_heads, a.dim, a.v_row, a.v_head) ||
      !make_head_map(&g, a.grad, a.rows_q, a.heads, a.dim, a.grad_row, a.grad_head))
    return RMN_ERR_UNSUPPORTED;
  return a.dim <= 64 ? launch_bwd<64>(q, k, v, g, a, stream) : launch_bwd<128>(q, k, v, g, a, stream);
}

}  // namespace rmn
