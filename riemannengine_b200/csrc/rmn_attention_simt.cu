// Attention within packed samples by multiply-adds in fp32: every type, head size up to 256, stride and alignment.
//
// Forward: a block takes BM query rows of one head and walks over the keys they see, BM at a time, with the running maximum m
// and sum l of each row's softmax: scores s = scale q k^T, m' = max(m, max s), p = exp(s - m'), l = l exp(m - m') + sum p,
// o = o exp(m - m') + p v; at the end o / l and lse = m + log l. Nothing of the scores reaches memory.
// Backward, without atomics: one kernel per query tile (delta = sum grad * out, dq = scale sum ds k) and one per key tile
// (dv = sum p^T grad, dk = scale sum ds^T q over the query heads that share the key head), p = exp(s - lse),
// ds = p * (grad v^T - delta); each makes the scores anew, which costs 7 products where 5 would do, and every gradient is
// written once, in a fixed order of sums.
//
// 4096 rows, 8 heads of 64: forward 992 us, 35 TFLOP/s, backward 3597 us, 24 by the five products of the formula.
// Bound by the multiply-adds and their operands in shared memory: a thread's 4 x 4 outputs take 8 16-byte reads per 32 multiply-adds
// of pairs; rows are padded by 16 bytes, and a thread's columns are 16 apart, so that the reads of a warp meet no bank twice.
// Where the tiles are few, a cluster of blocks shares one: each walks over every second or fourth tile of the other side, and their
// parts are joined through shared memory, in the order of the blocks.
#include "rmn_attention.cuh"
#include "rmn_pair.cuh"

#include <math_constants.h>

#include <type_traits>

namespace rmn {
namespace {

constexpr int kSimtThreads = 256;  // 16 x 16 threads over a tile
// Up to 64 channels two blocks share an SM, held to 128 registers a thread (100 samples of 200 rows, 8 heads of 32, backward: 739 us
// so, 1017 with the 164 registers that the compiler likes); wider tiles would spill more than that gains (0: no such limit).
template <int DP>
constexpr int kBlocksPerSM = DP <= 64 ? 2 : 0;

template <int DP, int BM>
struct SimtShape {
  static constexpr int R = BM / 16;                 // rows, and columns of scores, of a thread
  static constexpr int CW = DP >= 64 ? 4 : DP / 16; // neighbouring channels of a thread
  static constexpr int NC = DP / (16 * CW);         // groups of them, 16 CW apart
  static constexpr int LD = DP + 4, LP = BM + 4;
  static constexpr size_t tile = (size_t)BM * LD * sizeof(float), square = (size_t)BM * LP * sizeof(float);
};

__device__ __forceinline__ void store_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// A thread's share of a tile of rows in registers: fetch() asks for them, put() makes them fp32 numbers in shared memory, so that
// the loads of a tile run behind the arithmetic on the one before (4096 rows, 8 heads of 128, backward: 8890 us without that, 7310
// with it; 8 heads of 32, forward: 732, 683).
template <typename T, int DP, int BM>
struct Share {
  static constexpr int Q = DP / 4, N = BM * Q / kSimtThreads, LD = SimtShape<DP, BM>::LD;
  using Four = std::conditional_t<sizeof(T) == 4, float4, uint2>;
  Four v[N];

  // rows [0, n) of `from`, `row` elements apart; zeros behind them and behind `dim`
  __device__ __forceinline__ void fetch(const T* from, int64_t row, int n, int dim) {
    const bool wide = ((uintptr_t)from % (4 * sizeof(T))) == 0 && row % 4 == 0 && dim % 4 == 0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = threadIdx.x + k * kSimtThreads, r = i / Q, c = (i % Q) * 4;
      T* as = reinterpret_cast<T*>(&v[k]);
      v[k] = Four{};
      if (r >= n || c >= dim) continue;
      const T* p = from + (int64_t)r * row + c;
      if (wide) {
        v[k] = __ldg(reinterpret_cast<const Four*>(p));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < dim) as[e] = p[e];
      }
    }
  }
  // times `scale` into dst [BM][LD]
  __device__ __forceinline__ void put(float* dst, float scale) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = threadIdx.x + k * kSimtThreads, r = i / Q, c = (i % Q) * 4;
      float4 x;
      if constexpr (sizeof(T) == 4) {
        x = v[k];
      } else {
        const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v[k].x));
        const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v[k].y));
        x = make_float4(lo.x, lo.y, hi.x, hi.y);
      }
      x.x *= scale; x.y *= scale; x.z *= scale; x.w *= scale;
      *reinterpret_cast<float4*>(dst + r * LD + c) = x;
    }
  }
};
template <typename T, int DP, int BM>
__device__ __forceinline__ void load_tile(float* dst, const T* from, int64_t row, int n, int dim, float scale) {
  Share<T, DP, BM> share;
  share.fetch(from, row, n, dim);
  share.put(dst, scale);
}

__device__ __forceinline__ Pair low_pair(const float4& v) { return make_pair(v.x, v.y); }
__device__ __forceinline__ Pair high_pair(const float4& v) { return make_pair(v.z, v.w); }

// s[i][j] = row (ty + 16 i) of a times row (tx + 16 j) of b
template <int DP, int BM, int R = SimtShape<DP, BM>::R>
__device__ __forceinline__ void product_rows(const float* a, const float* b, int tx, int ty, float (&s)[R][R]) {
  constexpr int LD = SimtShape<DP, BM>::LD;
  Pair t[R][R];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) t[i][j] = make_pair(0.f, 0.f);
#pragma unroll 4
  for (int c = 0; c < DP; c += 4) {
    float4 x[R], y[R];
#pragma unroll
    for (int i = 0; i < R; ++i) x[i] = *reinterpret_cast<const float4*>(a + (ty + 16 * i) * LD + c);
#pragma unroll
    for (int j = 0; j < R; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * LD + c);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < R; ++j) {
        t[i][j] = fma(low_pair(x[i]), low_pair(y[j]), t[i][j]);
        t[i][j] = fma(high_pair(x[i]), high_pair(y[j]), t[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) s[i][j] = total(t[i][j]);
}

// o[i][channels of the thread] += sum_j p[ty + 16 i][j] b[j][channels], j < n rounded up to 4 (zeros there)
template <int DP, int BM, int R = SimtShape<DP, BM>::R, int NC = SimtShape<DP, BM>::NC, int CW = SimtShape<DP, BM>::CW>
__device__ __forceinline__ void product_columns(const float* p, const float* b, int n, int tx, int ty, Pair (&o)[R][NC][CW / 2]) {
  constexpr int LD = SimtShape<DP, BM>::LD, LP = SimtShape<DP, BM>::LP;
  for (int j = 0; j < n; j += 4) {
    float4 w[R];
#pragma unroll
    for (int i = 0; i < R; ++i) w[i] = *reinterpret_cast<const float4*>(p + (ty + 16 * i) * LP + j);
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      const float* row = b + (j + jj) * LD + tx * CW;
      Pair y[NC][CW / 2];
#pragma unroll
      for (int g = 0; g < NC; ++g) {
        if constexpr (CW == 4) {
          const float4 v = *reinterpret_cast<const float4*>(row + g * 16 * CW);
          y[g][0] = low_pair(v);
          y[g][1] = high_pair(v);
        } else {
          const float2 v = *reinterpret_cast<const float2*>(row + g * 16 * CW);
          y[g][0] = make_pair(v.x, v.y);
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float f = jj == 0 ? w[i].x : jj == 1 ? w[i].y : jj == 2 ? w[i].z : w[i].w;
        const Pair ff = make_pair(f, f);
#pragma unroll
        for (int g = 0; g < NC; ++g)
#pragma unroll
          for (int e = 0; e < CW / 2; ++e) o[i][g][e] = fma(ff, y[g][e], o[i][g][e]);
      }
    }
  }
}
template <int R, int NC, int H>
__device__ __forceinline__ void clear(Pair (&o)[R][NC][H]) {
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int g = 0; g < NC; ++g)
#pragma unroll
      for (int e = 0; e < H; ++e) o[i][g][e] = make_pair(0.f, 0.f);
}
// the pairs as single numbers
template <int R, int NC, int H>
__device__ __forceinline__ void singles(const Pair (&o)[R][NC][H], float (&x)[R][NC][2 * H]) {
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int g = 0; g < NC; ++g)
#pragma unroll
      for (int e = 0; e < H; ++e) parts(o[i][g][e], x[i][g][2 * e], x[i][g][2 * e + 1]);
}

// A cluster's parts of a tile, each in its block's shared memory at `part` [BM][LD]: puts this block's there. Behind a cluster_sync,
// sum_parts adds up those of rows ty + 16 i with i % blocks == rank, times weight(i, block).
template <int DP, int BM, int R = SimtShape<DP, BM>::R, int NC = SimtShape<DP, BM>::NC, int CW = SimtShape<DP, BM>::CW>
__device__ __forceinline__ void put_part(float* part, int tx, int ty, const float (&x)[R][NC][CW]) {
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int g = 0; g < NC; ++g)
#pragma unroll
      for (int e = 0; e < CW; ++e) part[(ty + 16 * i) * SimtShape<DP, BM>::LD + g * 16 * CW + tx * CW + e] = x[i][g][e];
}
template <int DP, int BM, class Weight, int R = SimtShape<DP, BM>::R, int NC = SimtShape<DP, BM>::NC, int CW = SimtShape<DP, BM>::CW>
__device__ __forceinline__ void sum_parts(const float* part, int tx, int ty, int rank, int blocks, float (&x)[R][NC][CW],
                                          Weight&& weight) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i % blocks != rank) continue;
#pragma unroll
    for (int g = 0; g < NC; ++g)
#pragma unroll
      for (int e = 0; e < CW; ++e) x[i][g][e] = 0.f;
    for (int k = 0; k < blocks; ++k) {
      const float f = weight(i, k);
#pragma unroll
      for (int g = 0; g < NC; ++g)
#pragma unroll
        for (int e = 0; e < CW; ++e)
          x[i][g][e] = fmaf(float_of_block(part + (ty + 16 * i) * SimtShape<DP, BM>::LD + g * 16 * CW + tx * CW + e, (uint32_t)k), f,
                            x[i][g][e]);
    }
  }
}

// o times `by` into rows [0, n) of `to`, `row` elements apart: those of this block of the cluster
template <typename T, int DP, int BM, int R = SimtShape<DP, BM>::R, int NC = SimtShape<DP, BM>::NC, int CW = SimtShape<DP, BM>::CW>
__device__ __forceinline__ void store_tile(T* to, int64_t row, int n, int dim, int tx, int ty, int rank, int blocks,
                                           const float (&o)[R][NC][CW], const float (&by)[R]) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (ty + 16 * i >= n || i % blocks != rank) continue;
#pragma unroll
    for (int g = 0; g < NC; ++g)
#pragma unroll
      for (int e = 0; e < CW; ++e) {
        const int c = g * 16 * CW + tx * CW + e;
        if (c < dim) store_f32(to + (int64_t)(ty + 16 * i) * row + c, o[i][g][e] * by[i]);
      }
  }
}

template <typename T, int DP, int BM>
__global__ void __launch_bounds__(kSimtThreads, kBlocksPerSM<DP>) k_attention_simt(const AttnArgs a) {
  using S = SimtShape<DP, BM>;
  constexpr int R = S::R, NC = S::NC, CW = S::CW;
  extern __shared__ __align__(16) float smem[];
  __shared__ FoundTile found;
  __shared__ int32_t warp_sums[kSimtThreads / 32];
  float* s_q = smem;
  float* s_kv = s_q + BM * S::LD;
  float* s_p = s_kv + BM * S::LD;
  after_previous_kernel();
  const int blocks = (int)cluster_size(), rank = (int)cluster_rank(), tile = blockIdx.x / blocks;
  const int head = tile % a.heads;
  if (!find_tile<kSimtThreads, TilesOf::kQueries>(a, tile / a.heads, BM, &found, warp_sums)) return;
  const Segment g = found.g;
  const int first = (found.tiles - 1 - found.tile) * BM;  // the tiles with the most keys first
  const int rows = min(BM, g.n_q - first);
  const int kv = head / (a.heads / a.kv_heads);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  load_tile<T, DP, BM>(s_q, static_cast<const T*>(a.q) + (int64_t)(g.q0 + first) * a.q_row + head * a.q_head, a.q_row, rows,
                       a.dim, a.scale);
  Pair o[R][NC][CW / 2];
  clear(o);
  float m[R], l[R];
  int seen[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -CUDART_INF_F;
    l[i] = 0.f;
    seen[i] = ty + 16 * i < rows ? visible_keys(g, first + ty + 16 * i, a.causal) : 0;
  }
  const int keys = visible_keys(g, first + rows - 1, a.causal);  // of the last row: the most
  const T* k0 = static_cast<const T*>(a.k) + (int64_t)g.k0 * a.k_row + kv * a.k_head;
  const T* v0 = static_cast<const T*>(a.v) + (int64_t)g.k0 * a.v_row + kv * a.v_head;
  Share<T, DP, BM> share;
  share.fetch(k0 + (int64_t)rank * BM * a.k_row, a.k_row, min(BM, keys - rank * BM), a.dim);
  for (int j0 = rank * BM; j0 < keys; j0 += blocks * BM) {
    const int n = min(BM, keys - j0);
    __syncthreads();  // the products with the tile before are done
    share.put(s_kv, 1.f);
    share.fetch(v0 + (int64_t)j0 * a.v_row, a.v_row, n, a.dim);
    __syncthreads();
    float s[R][R];
    product_rows<DP, BM>(s_q, s_kv, tx, ty, s);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float top = -CUDART_INF_F;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (j0 + tx + 16 * j >= seen[i]) s[i][j] = -CUDART_INF_F;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w, 16));
      const float m_new = fmaxf(m[i], top);
      const float base = m_new == -CUDART_INF_F ? 0.f : m_new;  // a row that sees nothing yet
      const float shrink = expf(m[i] - base);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const float p = expf(s[i][j] - base);
        s_p[(ty + 16 * i) * S::LP + tx + 16 * j] = p;
        sum += p;
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w, 16);
      l[i] = l[i] * shrink + sum;
      m[i] = m_new;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < CW / 2; ++e) o[i][c][e] = mul(o[i][c][e], make_pair(shrink, shrink));
    }
    __syncthreads();  // the keys have been read
    share.put(s_kv, 1.f);
    share.fetch(k0 + (int64_t)(j0 + blocks * BM) * a.k_row, a.k_row, min(BM, keys - j0 - blocks * BM), a.dim);
    __syncthreads();
    product_columns<DP, BM>(s_p, s_kv, n, tx, ty, o);
  }
  float x[R][NC][CW], by[R];
  singles(o, x);
  if (blocks > 1) {
    __shared__ float s_m[BM], s_l[BM];
    __syncthreads();  // q has been read
    put_part<DP, BM>(s_q, tx, ty, x);
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (tx == 0) {
        s_m[ty + 16 * i] = m[i];
        s_l[ty + 16 * i] = l[i];
      }
    cluster_sync();
    float m_of[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = ty + 16 * i;
      float top = -CUDART_INF_F;
      for (int k = 0; k < blocks; ++k) top = fmaxf(top, float_of_block(s_m + r, (uint32_t)k));
      l[i] = 0.f;
      for (int k = 0; k < blocks; ++k) {
        // (a block without a visible key has summed nothing; one with NaN scores has no maximum, but a sum that is NaN)
        const float mk = float_of_block(s_m + r, (uint32_t)k), lk = float_of_block(s_l + r, (uint32_t)k);
        l[i] += mk == -CUDART_INF_F ? lk : lk * expf(mk - top);
      }
      m_of[i] = top;
    }
    sum_parts<DP, BM>(s_q, tx, ty, rank, blocks, x, [&](int i, int k) {
      const float mk = float_of_block(s_m + ty + 16 * i, (uint32_t)k);
      return mk == -CUDART_INF_F ? 0.f : expf(mk - m_of[i]);
    });
#pragma unroll
    for (int i = 0; i < R; ++i) m[i] = m_of[i];
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    by[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
    if (a.lse && tx == 0 && ty + 16 * i < rows && i % blocks == rank)
      a.lse[(size_t)head * a.rows_q + g.q0 + first + ty + 16 * i] = l[i] == 0.f ? -CUDART_INF_F : m[i] + logf(l[i]);
  }
  const int64_t out_row = (int64_t)a.heads * a.dim;
  const int64_t at = (int64_t)(g.q0 + first) * out_row + (int64_t)head * a.dim;
  store_tile<T, DP, BM>(static_cast<T*>(a.out) + at, out_row, rows, a.dim, tx, ty, rank, blocks, x, by);
  if (sizeof(T) == 2 && a.low) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < CW; ++e) {
          const float v = x[i][c][e] * by[i];
          x[i][c][e] = v - __bfloat162float(__float2bfloat16_rn(v));
        }
#pragma unroll
    for (int i = 0; i < R; ++i) by[i] = 1.f;
    store_tile<T, DP, BM>(static_cast<T*>(a.low) + at, out_row, rows, a.dim, tx, ty, rank, blocks, x, by);
  }
  if (blocks > 1) cluster_sync();  // no block leaves while another reads its part
}

// dq of a query tile, and delta of its rows for the kernel of the key tiles
template <typename T, int DP, int BM>
__global__ void __launch_bounds__(kSimtThreads, kBlocksPerSM<DP>) k_attention_simt_dq(const AttnArgs a) {
  using S = SimtShape<DP, BM>;
  constexpr int R = S::R, NC = S::NC, CW = S::CW;
  extern __shared__ __align__(16) float smem[];
  __shared__ FoundTile found;
  __shared__ int32_t warp_sums[kSimtThreads / 32];
  float* s_q = smem;
  float* s_g = s_q + BM * S::LD;
  float* s_k = s_g + BM * S::LD;
  float* s_v = s_k + BM * S::LD;
  float* s_p = s_v + BM * S::LD;
  after_previous_kernel();
  const int blocks = (int)cluster_size(), rank = (int)cluster_rank(), tile = blockIdx.x / blocks;
  const int head = tile % a.heads;
  if (!find_tile<kSimtThreads, TilesOf::kQueries>(a, tile / a.heads, BM, &found, warp_sums)) return;
  const Segment g = found.g;
  const int first = (found.tiles - 1 - found.tile) * BM;
  const int rows = min(BM, g.n_q - first);
  const int kv = head / (a.heads / a.kv_heads);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t out_row = (int64_t)a.heads * a.dim;
  load_tile<T, DP, BM>(s_q, static_cast<const T*>(a.q) + (int64_t)(g.q0 + first) * a.q_row + head * a.q_head, a.q_row, rows,
                       a.dim, a.scale);
  load_tile<T, DP, BM>(s_g, static_cast<const T*>(a.grad) + (int64_t)(g.q0 + first) * a.grad_row + head * a.grad_head,
                       a.grad_row, rows, a.dim, 1.f);
  load_tile<T, DP, BM>(s_k, static_cast<const T*>(a.fwd_out) + (int64_t)(g.q0 + first) * out_row + (int64_t)head * a.dim,
                       out_row, rows, a.dim, 1.f);
  if (a.low)
    load_tile<T, DP, BM>(s_v, static_cast<const T*>(a.low) + (int64_t)(g.q0 + first) * out_row + (int64_t)head * a.dim, out_row,
                         rows, a.dim, 1.f);
  __syncthreads();
  Pair o[R][NC][CW / 2];
  clear(o);
  float delta[R], lse[R];
  int seen[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = ty + 16 * i;
    float d = 0.f;
    for (int c = tx; c < DP; c += 16)
      d = fmaf(s_g[r * S::LD + c], s_k[r * S::LD + c] + (a.low ? s_v[r * S::LD + c] : 0.f), d);
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w, 16);
    delta[i] = d;
    seen[i] = r < rows ? visible_keys(g, first + r, a.causal) : 0;
    const size_t at = (size_t)head * a.rows_q + g.q0 + first + r;
    lse[i] = r < rows ? __ldg(a.lse + at) : 0.f;
    if (r < rows && tx == 0 && rank == 0) a.delta[at] = d;
  }
  const int keys = visible_keys(g, first + rows - 1, a.causal);
  const T* k0 = static_cast<const T*>(a.k) + (int64_t)g.k0 * a.k_row + kv * a.k_head;
  const T* v0 = static_cast<const T*>(a.v) + (int64_t)g.k0 * a.v_row + kv * a.v_head;
  Share<T, DP, BM> next_k, next_v;
  auto fetch = [&](int j) {
    next_k.fetch(k0 + (int64_t)j * a.k_row, a.k_row, min(BM, keys - j), a.dim);
    next_v.fetch(v0 + (int64_t)j * a.v_row, a.v_row, min(BM, keys - j), a.dim);
  };
  fetch(rank * BM);
  for (int j0 = rank * BM; j0 < keys; j0 += blocks * BM) {
    const int n = min(BM, keys - j0);
    __syncthreads();
    next_k.put(s_k, 1.f);
    next_v.put(s_v, 1.f);
    fetch(j0 + blocks * BM);
    __syncthreads();
    float s[R][R], dp[R][R];
    product_rows<DP, BM>(s_q, s_k, tx, ty, s);
    product_rows<DP, BM>(s_g, s_v, tx, ty, dp);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const bool see = j0 + tx + 16 * j < seen[i];
        s_p[(ty + 16 * i) * S::LP + tx + 16 * j] = see ? expf(s[i][j] - lse[i]) * (dp[i][j] - delta[i]) : 0.f;
      }
    __syncthreads();
    product_columns<DP, BM>(s_p, s_k, n, tx, ty, o);
  }
  float x[R][NC][CW], by[R];
  singles(o, x);
  if (blocks > 1) {
    __syncthreads();  // q has been read
    put_part<DP, BM>(s_q, tx, ty, x);
    cluster_sync();
    sum_parts<DP, BM>(s_q, tx, ty, rank, blocks, x, [](int, int) { return 1.f; });
  }
#pragma unroll
  for (int i = 0; i < R; ++i) by[i] = a.scale;
  store_tile<T, DP, BM>(static_cast<T*>(a.dq) + (int64_t)(g.q0 + first) * out_row + (int64_t)head * a.dim, out_row, rows, a.dim,
                        tx, ty, rank, blocks, x, by);
  if (blocks > 1) cluster_sync();  // no block leaves while another reads its part
}

// dk and dv of a key tile: the queries of all heads that share its head
template <typename T, int DP, int BM>
__global__ void __launch_bounds__(kSimtThreads, kBlocksPerSM<DP>) k_attention_simt_dkv(const AttnArgs a) {
  using S = SimtShape<DP, BM>;
  constexpr int R = S::R, NC = S::NC, CW = S::CW;
  extern __shared__ __align__(16) float smem[];
  __shared__ FoundTile found;
  __shared__ int32_t warp_sums[kSimtThreads / 32];
  float* s_k = smem;
  float* s_v = s_k + BM * S::LD;
  float* s_q = s_v + BM * S::LD;
  float* s_g = s_q + BM * S::LD;
  float* s_p = s_g + BM * S::LD;
  after_previous_kernel();
  const int blocks = (int)cluster_size(), rank = (int)cluster_rank(), tile = blockIdx.x / blocks;
  const int kv = tile % a.kv_heads;
  if (!find_tile<kSimtThreads, TilesOf::kSlots>(a, tile / a.kv_heads, BM, &found, warp_sums)) return;
  const Segment g = found.g;
  const int first = found.tile * BM;  // the first keys are seen by the most queries
  const int rows = min(BM, g.k_slot - first), used = max(0, min(BM, g.n_k - first));
  const int group = a.heads / a.kv_heads;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  load_tile<T, DP, BM>(s_k, static_cast<const T*>(a.k) + (int64_t)(g.k0 + first) * a.k_row + kv * a.k_head, a.k_row, used,
                       a.dim, a.scale);
  load_tile<T, DP, BM>(s_v, static_cast<const T*>(a.v) + (int64_t)(g.k0 + first) * a.v_row + kv * a.v_head, a.v_row, used,
                       a.dim, 1.f);
  Pair dk[R][NC][CW / 2], dv[R][NC][CW / 2];
  clear(dk);
  clear(dv);
  // tiles of queries that see any of these keys, over all heads: every block of the cluster takes its own
  const int from = first_query(g, first, a.causal) / BM * BM;
  const int tiles = used > 0 ? max(0, (g.n_q - from + BM - 1) / BM) : 0;
  Share<T, DP, BM> next_q, next_g;
  auto fetch = [&](int turn) {
    const int h = kv * group + turn / max(tiles, 1), i = from + turn % max(tiles, 1) * BM;
    const int n = turn < tiles * group ? min(BM, g.n_q - i) : 0;
    next_q.fetch(static_cast<const T*>(a.q) + (int64_t)(g.q0 + i) * a.q_row + (int64_t)h * a.q_head, a.q_row, n, a.dim);
    next_g.fetch(static_cast<const T*>(a.grad) + (int64_t)(g.q0 + i) * a.grad_row + (int64_t)h * a.grad_head, a.grad_row, n, a.dim);
  };
  fetch(rank);
  for (int turn = rank; turn < tiles * group; turn += blocks) {
    const int h = kv * group + turn / tiles, i0 = from + turn % tiles * BM;
    const int n = min(BM, g.n_q - i0);
    __syncthreads();
    next_q.put(s_q, 1.f);
    next_g.put(s_g, 1.f);
    fetch(turn + blocks);
    __syncthreads();
    float s[R][R], dp[R][R];
    product_rows<DP, BM>(s_k, s_q, tx, ty, s);
    product_rows<DP, BM>(s_v, s_g, tx, ty, dp);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int qi = tx + 16 * j;
      const size_t at = (size_t)h * a.rows_q + g.q0 + i0 + qi;
      const float lse = qi < n ? __ldg(a.lse + at) : 0.f, delta = qi < n ? __ldg(a.delta + at) : 0.f;
      const int seen = qi < n ? visible_keys(g, i0 + qi, a.causal) : 0;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float p = first + ty + 16 * i < seen ? expf(s[i][j] - lse) : 0.f;
        s[i][j] = p;
        dp[i][j] = p == 0.f ? 0.f : p * (dp[i][j] - delta);
        s_p[(ty + 16 * i) * S::LP + qi] = p;
      }
    }
    __syncthreads();
    product_columns<DP, BM>(s_p, s_g, n, tx, ty, dv);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < R; ++j) s_p[(ty + 16 * i) * S::LP + tx + 16 * j] = dp[i][j];
    __syncthreads();
    product_columns<DP, BM>(s_p, s_q, n, tx, ty, dk);
  }
  float x[R][NC][CW], y[R][NC][CW], by_k[R], by_v[R];
  singles(dk, x);
  singles(dv, y);
  if (blocks > 1) {
    __syncthreads();  // the tiles have been read
    put_part<DP, BM>(s_q, tx, ty, x);
    put_part<DP, BM>(s_g, tx, ty, y);
    cluster_sync();
    sum_parts<DP, BM>(s_q, tx, ty, rank, blocks, x, [](int, int) { return 1.f; });
    sum_parts<DP, BM>(s_g, tx, ty, rank, blocks, y, [](int, int) { return 1.f; });
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    by_k[i] = a.scale;
    by_v[i] = 1.f;
  }
  const int64_t kv_row = (int64_t)a.kv_heads * a.dim, at = (int64_t)(g.k0 + first) * kv_row + (int64_t)kv * a.dim;
  store_tile<T, DP, BM>(static_cast<T*>(a.dk) + at, kv_row, rows, a.dim, tx, ty, rank, blocks, x, by_k);
  store_tile<T, DP, BM>(static_cast<T*>(a.dv) + at, kv_row, rows, a.dim, tx, ty, rank, blocks, y, by_v);
  if (blocks > 1) cluster_sync();  // no block leaves while another reads its part
}

// Blocks that share a tile: twice as many as long as they fit the GPU at once and each has a tile of the other side (`other`: its
// rows a sample, over all heads) to walk over, or as long as they are four times that and each has `least` such tiles: the pieces
// of samples of different lengths then fill the SMs to the end. At most the rows of a thread, which divide them at the end. 3 samples
// of 400 ... 1200 rows, 8 / 2 heads of 64, causal: 157 + 801 us with the first rule alone, 117 + 483 with both; 4096 rows, 8 heads
// of 64: 1122 + 4002 and 992 + 3597, with 16 times as many blocks as fit 1090 + 3864.
int blocks_a_tile(uint64_t rows, int heads, uint64_t other, int BM, uint64_t least) {
  const uint64_t steps = (other + BM - 1) / BM;
  int n = 1;
  for (int twice = 2; twice <= BM / 16; twice *= 2) {
    const uint64_t blocks = rows / BM * heads * twice;
    if (steps < twice * (blocks <= 148 * 2 ? 1 : least) || blocks > 148 * 8) break;
    n = twice;
  }
  return n;
}

template <class Kernel>
int launch_simt(Kernel kern, SmemOptIn& opt_in, const AttnArgs& a, uint64_t tiles, int cluster, size_t smem, cudaStream_t stream) {
  const uint64_t blocks = tiles * cluster;
  if (blocks > 0x7fffffffull) return RMN_ERR_UNSUPPORTED;
  if (smem > 48 * 1024 - 1024) RMN_CUDA_TRY(opt_in.apply(reinterpret_cast<const void*>(kern), smem));
  RMN_CUDA_TRY(launch_overlapped_clusters(kern, (uint32_t)cluster, dim3((uint32_t)blocks), dim3(kSimtThreads), smem, stream, a));
  RMN_LAUNCH_CHECK();
  return RMN_OK;
}

template <typename T, int DP, int BM>
int forward(const AttnArgs& a, cudaStream_t stream) {
  using S = SimtShape<DP, BM>;
  static SmemOptIn opt_in;
  const uint64_t samples = a.sequences ? a.sequences : 1;
  return launch_simt(k_attention_simt<T, DP, BM>, opt_in, a, most_tiles(a.rows_q, a.sequences, BM) * a.heads,
                     blocks_a_tile(a.rows_q, a.heads, a.rows_k / samples, BM, 4), 2 * S::tile + S::square, stream);
}
template <typename T, int DP, int BM>
int backward(const AttnArgs& a, cudaStream_t stream) {
  using S = SimtShape<DP, BM>;
  static SmemOptIn opt_q, opt_kv;
  const uint64_t samples = a.sequences ? a.sequences : 1, group = a.heads / a.kv_heads;
  const int st = launch_simt(k_attention_simt_dq<T, DP, BM>, opt_q, a, most_tiles(a.rows_q, a.sequences, BM) * a.heads,
                             blocks_a_tile(a.rows_q, a.heads, a.rows_k / samples, BM, 2), 4 * S::tile + S::square, stream);
  if (st != RMN_OK) return st;
  return launch_simt(k_attention_simt_dkv<T, DP, BM>, opt_kv, a, most_tiles(a.rows_k, a.sequences, BM) * a.kv_heads,
                     blocks_a_tile(a.rows_k, a.kv_heads, a.rows_q / samples * group, BM, 2), 4 * S::tile + S::square, stream);
}

}  // namespace

#define RMN_SIMT_SHAPES(F)                                                             \
  if (a.dim <= 32) return dtype == RMN_F32 ? F<float, 32, 64>(a, stream) : F<__nv_bfloat16, 32, 64>(a, stream);     \
  if (a.dim <= 64) return dtype == RMN_F32 ? F<float, 64, 64>(a, stream) : F<__nv_bfloat16, 64, 64>(a, stream);     \
  if (a.dim <= 128) return dtype == RMN_F32 ? F<float, 128, 64>(a, stream) : F<__nv_bfloat16, 128, 64>(a, stream);  \
  if (a.dim <= 256) return dtype == RMN_F32 ? F<float, 256, 32>(a, stream) : F<__nv_bfloat16, 256, 32>(a, stream);  \
  return RMN_ERR_UNSUPPORTED;

int attention_simt_forward(const AttnArgs& a, int dtype, cudaStream_t stream) { RMN_SIMT_SHAPES(forward) }
int attention_simt_backward(const AttnArgs& a, int dtype, cudaStream_t stream) { RMN_SIMT_SHAPES(backward) }

}  // namespace rmn
