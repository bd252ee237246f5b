// Attention within packed samples on the tensor cores: forward pass, bf16, head sizes up to 128 (multiples of 8).
//
// A block takes NQ tiles of 128 query rows of one head and walks over the keys they see, 128 at a time:
//   S = Q K^T (tcgen05.mma, 128 x 128 fp32 in tensor memory),  m' = max(m, scale * max_j S),  P = exp(scale S - m'),
//   l += sum_j P,  O += P V (P rounded to bf16, in tensor memory as the A operand),  out = O / l at the end.
// The sum l is taken of the unrounded P in fp32; rounding P to bf16 is what the tensor cores ask for and adds an error of the
// size of the output's own rounding. A thread owns a row: its 128 scores come out of tensor memory at once. O is scaled to a new
// maximum only when that exceeds the one in use by more than 2^8 (P then stays below 2^8, far inside fp32 and bf16).
//
// Warps: NQ groups of four for the softmax of one query tile each, one for the bulk copies, one that issues the products.
// Keys and values arrive as 128-row tiles in a ring of shared-memory slots. Bound by the exponentials: 16 a clock and SM, 1024
// clocks a 128 x 128 tile, against 8 * head size clocks of both products on the tensor cores.
// Head sizes up to 64: one query tile and two blocks an SM, P has columns of its own, and the next scores are made while the
// exponentials of these run (8192 rows, 16 heads of 64: 414 us; two tiles and one block 433: their softmax groups fall into step).
// Above, tensor memory has no room for it: P takes the place of S, and the next scores wait until P has been used (a softmax
// thread waits about half of the time then, while the other tile's works: 8192 rows, 16 heads of 128: 522 us, 1053 TFLOP/s).
#include "rmn_attention_tc.cuh"

#include <math_constants.h>

#include <atomic>

namespace rmn {
namespace tc {
namespace {

template <int DP, int NQ>
struct FwdShape {
  static constexpr int ATOMS = DP / 64;
  static constexpr uint32_t TILE = ATOMS * kAtomBytes;
  static constexpr bool kAlias = DP == 128;  // P in the columns of S
  static constexpr int SLOTS = DP == 128 ? (NQ == 2 ? 5 : 2) : 4;
  static constexpr int THREADS = NQ * 128 + 128;
  // registers of a softmax thread and of the others: what the block is launched with, dealt out anew
  static constexpr int SOFTMAX_REGS = NQ == 2 ? 216 : 200, OTHER_REGS = NQ == 2 ? 64 : 56;
  static constexpr int ALL_REGS = NQ * 128 * SOFTMAX_REGS + 128 * OTHER_REGS;
  static constexpr uint32_t COLUMNS = NQ * 256;
  static constexpr uint32_t S0 = 0, P0 = kAlias ? 0 : NQ * 128, O0 = kAlias ? NQ * 128 : NQ * 192;
  static constexpr uint32_t P_STEP = kAlias ? 128 : 64;
  static constexpr uint32_t BARS = NQ * TILE + SLOTS * TILE;  // offset of the barriers
  static constexpr size_t SMEM = BARS + 256 + 1024;           // (1024: the tiles start on a swizzle's period)
};

constexpr float kRescale = 8.f;  // log2 of how far a row's maximum may rise before O is scaled
constexpr int kOneTile = 4;      // softmax warps
constexpr int kTwoTiles = 8;

template <int DP, int NQ>
__global__ void __launch_bounds__(FwdShape<DP, NQ>::THREADS, NQ == 2 ? 1 : 2)
    k_attention_fwd(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const AttnArgs a) {
  using C = FwdShape<DP, NQ>;
  constexpr int SLOTS = C::SLOTS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ FoundTile found;
  __shared__ int32_t warp_sums[C::THREADS / 32];
  __shared__ uint32_t tmem_slot;
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BARS);  // [SLOTS]
  uint64_t* empty = full + SLOTS;                                // [SLOTS]
  uint64_t* q_full = empty + SLOTS;                              // [NQ]
  uint64_t* s_full = q_full + NQ;                                // scores made
  uint64_t* s_free = s_full + NQ;                                // scores in registers (own columns for P)
  uint64_t* p_full = s_free + NQ;                                // P written, O at the right scale
  uint64_t* o_done = p_full + NQ;                                // P used, O summed

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kCopyWarp = NQ * 4, kMmaWarp = NQ * 4 + 1;

  if (tid == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int t = 0; t < NQ; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&s_free[t], 128);
      mbar_init(&p_full[t], 128);
      mbar_init(&o_done[t], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(C::COLUMNS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == kCopyWarp && lane == 0) {
    tma_prefetch_map(&map_q);
    tma_prefetch_map(&map_k);
    tma_prefetch_map(&map_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  after_previous_kernel();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot);
  const uint32_t smem_base = smem_u32(smem), slots = smem_base + NQ * C::TILE;
  bool timed_out = false;

  const int head = blockIdx.x % a.heads;
  const bool exists = find_tile<C::THREADS, TilesOf::kQueries>(a, blockIdx.x / a.heads, 128 * NQ, &found, warp_sums);
  const Segment g = found.g;
  const int first = (found.tiles - 1 - found.tile) * 128 * NQ;  // the tiles that see the most keys first
  // key tiles of each query tile
  int key_tiles[NQ], most = 0;
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    const int rows = min(128, g.n_q - first - t * 128);
    key_tiles[t] = exists && rows > 0 ? (visible_keys(g, first + t * 128 + rows - 1, a.causal) + 127) / 128 : 0;
    most = max(most, key_tiles[t]);
  }

  auto softmax = [&] {
    // ------------------------------ softmax --------------------------------------------
    const int t = warp >> 2;
    const uint32_t lanes = ((uint32_t)(warp & 3) * 32u) << 16;
    const uint32_t s_t = tmem + lanes + C::S0 + t * 128, p_t = tmem + lanes + C::P0 + t * C::P_STEP,
                   o_t = tmem + lanes + C::O0 + t * DP;
    const int row = first + t * 128 + (warp & 3) * 32 + lane;
    const bool mine = row < g.n_q;
    const int see = visible_keys(g, row, a.causal);
    const float scale = a.scale * kLog2e;  // (> 0)
    float m = -CUDART_INF_F, l = 0.f;      // maximum in use (times scale, log 2), sum
    const int n_tiles = NQ == 1 ? key_tiles[0] : (t == 0 ? key_tiles[0] : key_tiles[NQ - 1]);
    for (int j = 0; j < n_tiles; ++j) {
      const uint32_t ph = (uint32_t)j & 1u;
      if (!warp_wait(&s_full[t], ph)) { timed_out = true; break; }
      tc_fence_after();
      uint32_t r[128];
      tc_ld32_at<0>(s_t, r);
      tc_ld32_at<32>(s_t + 32, r);
      tc_ld32_at<64>(s_t + 64, r);
      tc_ld32_at<96>(s_t + 96, r);
      tc_wait_ld();
      if constexpr (!C::kAlias) {
        tc_fence_before();
        mbar_arrive(&s_free[t]);
      }
      const int left = see - j * 128;  // columns that this row sees
      if (left < 128) {
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (c >= left) r[c] = 0xff800000u;
      }
      float top[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
      for (int c = 0; c < 128; c += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k) top[k] = max3(top[k], __uint_as_float(r[c + 2 * k]), __uint_as_float(r[c + 2 * k + 1]));
      const float m_new = fmaxf(m, fmaxf(max3(top[0], top[1], top[2]), top[3]) * scale);
      const bool rise = m_new > m + kRescale;  // (from -infinity: always, unless nothing is seen yet)
      float shrink = 1.f;
      if (rise) {
        shrink = exp2_approx(m - m_new);
        l *= shrink;
        m = m_new;
      }
      const float base = m == -CUDART_INF_F ? 0.f : m;
      const Pair by = make_pair(scale, scale), minus = make_pair(-base, -base);
      Pair sum[2] = {make_pair(0.f, 0.f), make_pair(0.f, 0.f)};
      uint32_t p[64];
#pragma unroll
      for (int c = 0; c < 128; c += 2) {
        float x, y;
        parts(fma(pair_of(r[c], r[c + 1]), by, minus), x, y);
        x = exp2_approx(x);
        y = exp2_approx(y);
        sum[(c >> 1) & 1] = add(sum[(c >> 1) & 1], make_pair(x, y));
        p[c / 2] = pack_bf16(x, y);
      }
      l += total(add(sum[0], sum[1]));
      if (j > 0) {
        // P and O of the tile before are free (kAlias: these scores were made behind that)
        if constexpr (!C::kAlias) {
          if (!warp_wait(&o_done[t], ph ^ 1u)) { timed_out = true; break; }
          tc_fence_after();
        }
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
          for (int c = 0; c < DP; c += 32) {
            uint32_t o[32];
            tc_ld32(o_t + c, o);
            tc_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * shrink);
            tc_st32<0>(o_t + c, o);
          }
        }
      }
      tc_st32<0>(p_t, p);
      tc_st32<32>(p_t + 32, p);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[t]);
    }
    // ------------------------------ output ---------------------------------------------
    if (!timed_out && n_tiles > 0) {
      if (!warp_wait(&o_done[t], (uint32_t)(n_tiles - 1) & 1u)) timed_out = true;
      tc_fence_after();
    }
    if (!timed_out) {
      const float by = l == 0.f ? 0.f : 1.f / l;
      const size_t at = ((size_t)(g.q0 + row) * a.heads + head) * a.dim;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + at;
      __nv_bfloat16* low = a.low ? static_cast<__nv_bfloat16*>(a.low) + at : nullptr;
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32];
        if (n_tiles > 0) {
          tc_ld32(o_t + c, o);
          tc_wait_ld();
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(o[k]) * by);
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          if (!mine || c + k >= a.dim) continue;
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = __uint_as_float(o[k + 2 * e]), y = __uint_as_float(o[k + 2 * e + 1]);
            hi[e] = pack_bf16(x, y);
            lo[e] = pack_bf16(x - __uint_as_float(hi[e] << 16), y - __uint_as_float(hi[e] & 0xffff0000u));
          }
          *reinterpret_cast<uint4*>(out + c + k) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          if (low) *reinterpret_cast<uint4*>(low + c + k) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
      if (mine && a.lse)
        a.lse[(size_t)head * a.rows_q + g.q0 + row] = l == 0.f ? -CUDART_INF_F : (m + log2f(l)) * kLn2;
    }
  };
  auto others = [&] {
    if (warp == kCopyWarp) {
      // ------------------------------ bulk copies ----------------------------------------
      if (lane == 0) {
        const int kv = head / (a.heads / a.kv_heads);
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
          if (key_tiles[t] == 0) continue;
          mbar_arrive_expect_tx(&q_full[t], C::TILE);
#pragma unroll
          for (int c = 0; c < C::ATOMS; ++c)
            tma_load_3d(smem_base + t * C::TILE + c * kAtomBytes, &map_q, &q_full[t], c * 64, head, g.q0 + first + t * 128);
        }
        const uint32_t loads = 2u * (uint32_t)most;
        uint32_t i = 0;
        for (; i < loads; ++i) {  // K 0, V 0, K 1, V 1, ...
          const uint32_t s = i % SLOTS;
          if (!mbar_wait(&empty[s], ((i / SLOTS) & 1u) ^ 1u)) { timed_out = true; break; }
          mbar_arrive_expect_tx(&full[s], C::TILE);
          const CUtensorMap* map = (i & 1u) ? &map_v : &map_k;
#pragma unroll
          for (int c = 0; c < C::ATOMS; ++c)
            tma_load_3d(slots + s * C::TILE + c * kAtomBytes, map, &full[s], c * 64, kv, g.k0 + (int)(i >> 1) * 128);
        }
        if (timed_out) {  // no copy may be in flight when the block ends
          for (uint32_t k = i > SLOTS ? i - SLOTS : 0; k < i; ++k) mbar_wait(&full[k % SLOTS], (k / SLOTS) & 1u);
          for (int t = 0; t < NQ; ++t)
            if (key_tiles[t]) mbar_wait(&q_full[t], 0);
        }
      }
    } else if (warp == kMmaWarp) {
      // ------------------------------ products -------------------------------------------
      const int steps = (a.dim + 15) / 16;
      const uint32_t idesc_s = instr_desc(128, 128, false);
      const uint32_t idesc_o = instr_desc(128, 0, true) | ((uint32_t)(steps * 2) << 17);
      auto ready = [&](uint32_t i) {  // load i has arrived
        if (!warp_wait(&full[i % SLOTS], (i / SLOTS) & 1u)) timed_out = true;
        return !timed_out;
      };
      auto scores = [&](int t, int j) {
        tc_fence_after();
        mma_rows(tmem + C::S0 + t * 128, smem_base + t * C::TILE, slots + (2u * j) % SLOTS * C::TILE, idesc_s, steps);
        tc_commit_elect(&s_full[t]);
      };
      if (most > 0 && ready(0)) {
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
          if (key_tiles[t] == 0 || timed_out) continue;
          if (!warp_wait(&q_full[t], 0)) { timed_out = true; break; }
          scores(t, 0);
        }
        if (!timed_out) tc_commit_elect(&empty[0]);
      }
      for (int j = 0; j < most && !timed_out; ++j) {
        const uint32_t ph = (uint32_t)j & 1u;
        const uint32_t v_s = slots + (2u * j + 1u) % SLOTS * C::TILE;
        bool v_here = false;
        // O of tile t += P V
        auto output = [&](int t) {
          if (!v_here) {
            if (!ready(2u * j + 1u)) return;
            v_here = true;
            if (g.n_k - j * 128 < 128) zero_rows(v_s, g.n_k - j * 128, C::ATOMS);
          }
          if (!warp_wait(&p_full[t], ph)) { timed_out = true; return; }
          tc_fence_after();
          mma_columns(tmem + C::O0 + t * DP, tmem + C::P0 + t * C::P_STEP, v_s, idesc_o, j > 0);
          tc_commit_elect(&o_done[t]);
        };
        if (j + 1 < most && !ready(2u * j + 2u)) break;
        if constexpr (C::kAlias) {
#pragma unroll
          for (int t = 0; t < NQ; ++t) {
            if (j >= key_tiles[t] || timed_out) continue;
            output(t);
            if (timed_out || j + 1 >= key_tiles[t]) continue;
            if (!warp_wait(&o_done[t], ph)) { timed_out = true; break; }  // P has been read
            scores(t, j + 1);
          }
        } else {
#pragma unroll
          for (int t = 0; t < NQ; ++t) {
            if (j + 1 >= key_tiles[t] || timed_out) continue;
            if (!warp_wait(&s_free[t], ph)) { timed_out = true; break; }
            scores(t, j + 1);
          }
#pragma unroll
          for (int t = 0; t < NQ; ++t)
            if (j < key_tiles[t] && !timed_out) output(t);
        }
        if (timed_out) break;
        tc_commit_elect(&empty[(2u * j + 1u) % SLOTS]);
        if (j + 1 < most) tc_commit_elect(&empty[(2u * j + 2u) % SLOTS]);
      }
    }
  };
  if (exists) {
    if constexpr (NQ == 2) {
      if (warp < kTwoTiles) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
        softmax();
      } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::OTHER_REGS));
        others();
      }
    } else {
      if (warp < kOneTile) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
        softmax();
      } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::OTHER_REGS));
        others();
      }
    }
  }

  if (timed_out) atomicExch(a.status, (uint32_t)RMN_ERR_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLUMNS) : "memory");
  }
}

template <int DP, int NQ>
int launch_fwd(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const AttnArgs& a, cudaStream_t stream) {
  using C = FwdShape<DP, NQ>;
  static SmemOptIn opt_in;
  auto kern = k_attention_fwd<DP, NQ>;
  const uint64_t blocks = most_tiles(a.rows_q, a.sequences, 128 * NQ) * a.heads;
  if (blocks > 0x7fffffffull) return RMN_ERR_UNSUPPORTED;
  // the registers dealt out have to be there: asked for once
  static std::atomic<int> enough{0};
  if (!enough.load(std::memory_order_relaxed)) {
    cudaFuncAttributes attr;
    RMN_CUDA_TRY(cudaFuncGetAttributes(&attr, reinterpret_cast<const void*>(kern)));
    enough.store(attr.numRegs * C::THREADS >= C::ALL_REGS ? 1 : 2, std::memory_order_relaxed);
  }
  if (enough.load(std::memory_order_relaxed) != 1) return RMN_ERR_UNSUPPORTED;
  RMN_CUDA_TRY(opt_in.apply(reinterpret_cast<const void*>(kern), C::SMEM));
  RMN_CUDA_TRY(launch_overlapped(kern, dim3((uint32_t)blocks), dim3(C::THREADS), C::SMEM, stream, q, k, v, a));
  RMN_LAUNCH_CHECK();
  count_tc_launch();
  return RMN_OK;
}

}  // namespace
}  // namespace tc

int attention_tc_forward(const AttnArgs& a, cudaStream_t stream) {
  using namespace tc;
  if (a.dim > 128 || !(a.scale > 0.f) || a.rows_k == 0 || ((uintptr_t)a.out & 15) || ((uintptr_t)a.low & 15))
    return RMN_ERR_UNSUPPORTED;
  CUtensorMap q, k, v;
  if (!make_head_map(&q, a.q, a.rows_q, a.heads, a.dim, a.q_row, a.q_head) ||
      !make_head_map(&k, a.k, a.rows_k, a.kv_heads, a.dim, a.k_row, a.k_head) ||
      !make_head_map(&v, a.v, a.rows_k, a.kv_heads, a.dim, a.v_row, a.v_head))
    return RMN_ERR_UNSUPPORTED;
  if (a.dim <= 64) return launch_fwd<64, 1>(q, k, v, a, stream);
  // two query tiles a block read the keys half as often, one leaves two blocks an SM: 16 heads of 128, one causal sample of 8192
  // rows 249 us with two and 260 with one (262 with two since the waits are votes); 100 samples of 256 rows, 8 heads, 76 and 66.5; 12 of
  // 2048 the same
  const bool two = a.rows_q / 2048 >= a.sequences;
  return two ? launch_fwd<128, 2>(q, k, v, a, stream) : launch_fwd<128, 1>(q, k, v, a, stream);
}

}  // namespace rmn
