// Layer norm over the channels of every row of a feature matrix, forward and backward (the reference wraps torch's layer,
// engine/nn/normalization.hpp; it stands beside the batch norm of rmn_norm.cu).
//
//   mean = sum_c x / C,  inv = 1 / sqrt(sum_c (x - mean)^2 / C + eps),  xhat = (x - mean) * inv,  y = xhat * gamma + beta
//   g = dy * gamma,  dx = inv * (g - sum_c g / C - xhat * sum_c g xhat / C),  dgamma = sum_r dy xhat,  dbeta = sum_r dy
//
// Bound by memory: the forward pass reads x and writes y, the backward pass reads x and dy and writes dx. A row stays in the
// registers of L threads (L a power of two up to a warp, or a whole block for wide rows), 16 bytes a load, so each value is
// read once; the variance is taken around the mean in a second pass over the registers, in fp32. A thread of the backward pass
// keeps the same channels over all the rows it visits, so dgamma and dbeta are sums in its registers; they are added up over
// the block in a fixed order, and a second kernel adds the blocks' sums in order: no atomics, the same bits every time.
#include "rmn_common.cuh"

#include <cuda_bf16.h>

namespace rmn {
namespace {

constexpr int kNormThreads = 256;
constexpr int kMaxVectors = 4;          // vectors of a row that one thread holds
constexpr uint32_t kMaxBackwardBlocks = 148 * 4;

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else return __float2bfloat16_rn(v);
}
// element i of a parameter vector of either type
__device__ __forceinline__ float param(const void* p, int bf16, int i) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}
// V parameters from channel c on, `missing` where there are none
template <int V>
__device__ __forceinline__ void params(const void* p, int bf16, int c, float missing, float (&out)[V]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = missing;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = param(p, bf16, c + j);
  }
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  if constexpr (sizeof(T) * V == 16) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
    r = *reinterpret_cast<const Pack<T, V>*>(&w);
  } else {
    r = *reinterpret_cast<const Pack<T, V>*>(p);
  }
  return r;
}

// Sum over the threads of a row: L lanes of a warp, or (kBlock) the whole block. N sums at once; every thread gets them.
template <bool kBlock, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], int L, float* red) {
  const int width = kBlock ? 32 : L;
  for (int o = width >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
  }
  if constexpr (kBlock) {
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();  // the sums before these have been read
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[i * 32 + warp] = s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = lane < warps ? red[i * 32 + lane] : 0.f;
      for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      s[i] = t;
    }
  }
}

// U rows of L threads are in flight at once (kBlock: one row a block).
template <typename T, int V, int NV, int U, bool kBlock>
__global__ void __launch_bounds__(kBlock ? 1024 : kNormThreads)
    k_layer_norm(const T* __restrict__ x, int64_t ld, uint32_t n, int C, int L, const void* __restrict__ gamma,
                 const void* __restrict__ beta, int param_bf16, float eps, T* __restrict__ out, float* __restrict__ mean_out,
                 float* __restrict__ inv_out) {
  __shared__ float red[32];
  after_previous_kernel();
  const int group = kBlock ? 0 : threadIdx.x / L, at = kBlock ? threadIdx.x : threadIdx.x % L;
  const int groups = kBlock ? 1 : kNormThreads / L;
  const int nvec = C / V;
  const float inv_c = 1.f / (float)C;
  Pack<T, V> raw[U][NV];
  uint32_t row[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t r = ((uint64_t)blockIdx.x * U + u) * groups + group;
    row[u] = r < n ? (uint32_t)r : 0xffffffffu;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = at + i * L;
      if (row[u] != 0xffffffffu && v < nvec) raw[u][i] = load_pack<T, V>(x + (int64_t)row[u] * ld + (int64_t)v * V);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool ok = row[u] != 0xffffffffu;
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (ok && at + i * L < nvec)
#pragma unroll
        for (int j = 0; j < V; ++j) s[0] += to_f32(raw[u][i].v[j]);
    row_sum<kBlock>(s, L, red);
    const float mean = s[0] * inv_c;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (ok && at + i * L < nvec)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = to_f32(raw[u][i].v[j]) - mean;
          s[0] = fmaf(d, d, s[0]);
        }
    row_sum<kBlock>(s, L, red);
    const float inv = 1.f / sqrtf(s[0] * inv_c + eps);
    if (!ok) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = at + i * L;
      if (v >= nvec) continue;
      float g[V], b[V];
      params<V>(gamma, param_bf16, v * V, 1.f, g);
      params<V>(beta, param_bf16, v * V, 0.f, b);
      Pack<T, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j) o.v[j] = from_f32<T>(fmaf((to_f32(raw[u][i].v[j]) - mean) * inv, g[j], b[j]));
      *reinterpret_cast<Pack<T, V>*>(out + (size_t)row[u] * C + (size_t)v * V) = o;
    }
    if (at == 0 && mean_out) {
      mean_out[row[u]] = mean;
      inv_out[row[u]] = inv;
    }
  }
}

// Every block visits rows blockIdx.x * groups + group, + gridDim.x * groups, ...; partial[block][0][c] = its part of dgamma,
// [1][c] of dbeta (kSums: wanted).
template <typename T, int V, int NV, bool kBlock, bool kSums>
__global__ void __launch_bounds__(kBlock ? 1024 : kNormThreads)
    k_layer_norm_backward(const T* __restrict__ dy, int64_t ld_dy, const T* __restrict__ x, int64_t ld_x, uint32_t n, int C,
                          int L, const void* __restrict__ gamma, int param_bf16, const float* __restrict__ mean_in,
                          const float* __restrict__ inv_in, T* __restrict__ dx, float* __restrict__ partial) {
  extern __shared__ float sums[];  // [2][C] (kSums)
  __shared__ float red[64];
  after_previous_kernel();
  const int group = kBlock ? 0 : threadIdx.x / L, at = kBlock ? threadIdx.x : threadIdx.x % L;
  const int groups = kBlock ? 1 : kNormThreads / L;
  const int nvec = C / V;
  const float inv_c = 1.f / (float)C;
  float dg[kSums ? NV : 1][V], db[kSums ? NV : 1][V];
  if constexpr (kSums) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) dg[i][j] = db[i][j] = 0.f;
  }
  // whole groups of rows, so that all threads of a warp meet in the sums
  for (uint64_t first = (uint64_t)blockIdx.x * groups; first < n; first += (uint64_t)gridDim.x * groups) {
    const uint64_t r = first + group;
    const bool ok = r < n;
    Pack<T, V> rx[NV], rd[NV];
    float mean = 0.f, inv = 0.f;
    if (ok) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = at + i * L;
        if (v < nvec) {
          rx[i] = load_pack<T, V>(x + (int64_t)r * ld_x + (int64_t)v * V);
          rd[i] = load_pack<T, V>(dy + (int64_t)r * ld_dy + (int64_t)v * V);
        }
      }
      mean = __ldg(mean_in + r);
      inv = __ldg(inv_in + r);
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = at + i * L;
      if (!ok || v >= nvec) continue;
      float g[V];
      params<V>(gamma, param_bf16, v * V, 1.f, g);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xhat = (to_f32(rx[i].v[j]) - mean) * inv, d = to_f32(rd[i].v[j]);
        if constexpr (kSums) {
          dg[i][j] = fmaf(d, xhat, dg[i][j]);
          db[i][j] += d;
        }
        s[0] = fmaf(d, g[j], s[0]);
        s[1] = fmaf(d * g[j], xhat, s[1]);
      }
    }
    if (!dx) continue;  // (the same for all threads)
    row_sum<kBlock>(s, L, red);
    const float a = s[0] * inv_c, b = s[1] * inv_c;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = at + i * L;
      if (!ok || v >= nvec) continue;
      float g[V];
      params<V>(gamma, param_bf16, v * V, 1.f, g);
      Pack<T, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xhat = (to_f32(rx[i].v[j]) - mean) * inv;
        o.v[j] = from_f32<T>(inv * (fmaf(to_f32(rd[i].v[j]), g[j], -a) - xhat * b));
      }
      *reinterpret_cast<Pack<T, V>*>(dx + (size_t)r * C + (size_t)v * V) = o;
    }
  }
  if constexpr (kSums) {
    if constexpr (!kBlock) {  // the groups of a warp hold the same channels
      for (int o = L; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            dg[i][j] += __shfl_xor_sync(0xffffffffu, dg[i][j], o);
            db[i][j] += __shfl_xor_sync(0xffffffffu, db[i][j], o);
          }
    }
    const int turns = kBlock ? 1 : kNormThreads / 32;
    const bool mine = kBlock || (threadIdx.x & 31) < L;
    for (int w = 0; w < turns; ++w) {  // the warps one after the other
      if (mine && (kBlock || (int)(threadIdx.x >> 5) == w)) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int v = at + i * L;
          if (v >= nvec) continue;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int c = v * V + j;
            sums[c] = w ? sums[c] + dg[i][j] : dg[i][j];
            sums[C + c] = w ? sums[C + c] + db[i][j] : db[i][j];
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * C; c += blockDim.x) partial[(size_t)blockIdx.x * 2 * C + c] = sums[c];
  }
}

// dgamma[c], dbeta[c] = the blocks' sums in the order of the blocks: eight slices of them, in fp64, then the slices.
__global__ void __launch_bounds__(256) k_layer_norm_sums(const float* __restrict__ partial, uint32_t blocks, int C,
                                                         int param_bf16, void* __restrict__ dgamma,
                                                         void* __restrict__ dbeta) {
  __shared__ double part[8][32];
  after_previous_kernel();
  const int slice = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x * 32 + lane;
  double t = 0.0;
  if (i < 2 * C)
    for (uint32_t b = slice; b < blocks; b += 8) t += (double)__ldg(partial + (size_t)b * 2 * C + i);
  part[slice][lane] = t;
  __syncthreads();
  if (slice != 0 || i >= 2 * C) return;
  for (int k = 1; k < 8; ++k) t += part[k][lane];
  void* to = i < C ? dgamma : dbeta;
  if (!to) return;
  const int c = i < C ? i : i - C;
  if (param_bf16) static_cast<__nv_bfloat16*>(to)[c] = __float2bfloat16_rn((float)t);
  else static_cast<float*>(to)[c] = (float)t;
}

// How a row of C channels is laid over threads: V channels a load (16 bytes where alignment and C allow, else one), L threads a
// row, each with nv loads. Of the powers of two up to a warp the one that leaves the fewest threads idle, the largest of
// several; rows that a warp's registers cannot hold take a whole block.
struct RowLayout {
  int V, L, nv;
  bool block;
};
bool row_layout(int C, int elem, bool aligned, RowLayout* out) {
  const int wide = 16 / elem;
  const int V = aligned && C % wide == 0 ? wide : 1;
  const int nvec = C / V;
  int best = 0, best_nv = 0;
  for (int L = 32; L >= 1; L >>= 1) {
    const int nv = (nvec + L - 1) / L;
    if (nv > kMaxVectors) break;
    if (!best || (long long)L * nv < (long long)best * best_nv) { best = L; best_nv = nv; }
  }
  if (best) {
    *out = {V, best, best_nv, false};
    return true;
  }
  // the fewest warps whose threads hold the row
  const int threads = ((nvec + kMaxVectors - 1) / kMaxVectors + 31) / 32 * 32;
  if (threads > 1024) return false;
  *out = {V, threads, (nvec + threads - 1) / threads, true};
  return true;
}

bool aligned16(const void* p, int64_t ld, int elem) { return ((uintptr_t)p & 15) == 0 && (ld * elem) % 16 == 0; }
bool norm_args_ok(int C, int dtype, int param_dtype) {
  return C >= 1 && C <= 65536 && (dtype == RMN_F32 || dtype == RMN_BF16) &&
         (param_dtype == RMN_F32 || param_dtype == RMN_BF16);
}
uint32_t backward_blocks(uint32_t n, int groups) {
  const uint64_t want = ((uint64_t)n + groups - 1) / groups;
  return (uint32_t)(want < kMaxBackwardBlocks ? want : kMaxBackwardBlocks);
}

template <typename T, int V, int NV, bool kBlock>
int launch_forward(const RowLayout& a, const void* x, int64_t ld, uint32_t n, int C, const void* gamma, const void* beta,
                   int param_bf16, float eps, void* out, float* mean, float* inv, cudaStream_t stream) {
  constexpr int U = kBlock ? 1 : NV == 1 ? 4 : NV == 2 ? 2 : 1;
  const int threads = kBlock ? a.L : kNormThreads;
  const uint64_t rows = (uint64_t)U * (kBlock ? 1 : kNormThreads / a.L);
  const uint32_t grid = (uint32_t)(((uint64_t)n + rows - 1) / rows);
  RMN_CUDA_TRY(launch_overlapped(k_layer_norm<T, V, NV, U, kBlock>, dim3(grid), dim3(threads), 0, stream,
                                 static_cast<const T*>(x), ld, n, C, a.L, gamma, beta, param_bf16, eps, static_cast<T*>(out),
                                 mean, inv));
  RMN_LAUNCH_CHECK();
  return RMN_OK;
}

template <typename T, int V, int NV, bool kBlock>
int launch_backward(const RowLayout& a, const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, uint32_t n, int C,
                    const void* gamma, int param_bf16, const float* mean, const float* inv, void* dx, float* partial,
                    uint32_t grid, cudaStream_t stream) {
  const int threads = kBlock ? a.L : kNormThreads;
  const size_t smem = partial ? (size_t)2 * C * sizeof(float) : 0;
  auto go = [&](auto kern, SmemOptIn& opt_in) -> int {
    if (smem > 48 * 1024 - 512) RMN_CUDA_TRY(opt_in.apply(reinterpret_cast<const void*>(kern), smem));
    RMN_CUDA_TRY(launch_overlapped(kern, dim3(grid), dim3(threads), smem, stream, static_cast<const T*>(dy), ld_dy,
                                   static_cast<const T*>(x), ld_x, n, C, a.L, gamma, param_bf16, mean, inv,
                                   static_cast<T*>(dx), partial));
    RMN_LAUNCH_CHECK();
    return RMN_OK;
  };
  static SmemOptIn with_sums, without;
  return partial ? go(k_layer_norm_backward<T, V, NV, kBlock, true>, with_sums)
                 : go(k_layer_norm_backward<T, V, NV, kBlock, false>, without);
}

// f(type tag, V, NV, block) of the layout
template <class F>
int dispatch_row(const RowLayout& a, int dtype, F&& f) {
  auto by_nv = [&](auto t, auto v, auto block) -> int {
    switch (a.nv) {
      case 1: return f(t, v, std::integral_constant<int, 1>{}, block);
      case 2: return f(t, v, std::integral_constant<int, 2>{}, block);
      case 3: return f(t, v, std::integral_constant<int, 3>{}, block);
      default: return f(t, v, std::integral_constant<int, 4>{}, block);
    }
  };
  auto by_block = [&](auto t, auto v) -> int {
    return a.block ? by_nv(t, v, std::true_type{}) : by_nv(t, v, std::false_type{});
  };
  if (dtype == RMN_F32)
    return a.V == 1 ? by_block(float{}, std::integral_constant<int, 1>{}) : by_block(float{}, std::integral_constant<int, 4>{});
  return a.V == 1 ? by_block(__nv_bfloat16{}, std::integral_constant<int, 1>{})
                  : by_block(__nv_bfloat16{}, std::integral_constant<int, 8>{});
}

}  // namespace
}  // namespace rmn

using namespace rmn;

extern "C" int rmn_layer_norm_forward(const void* d_x, int64_t ld_x, uint32_t n_rows, int channels, const void* d_gamma,
                                      const void* d_beta, int param_dtype, float eps, void* d_out, float* d_mean,
                                      float* d_inv, int dtype, void* stream_) {
  if (!norm_args_ok(channels, dtype, param_dtype) || n_rows > 0x7fffffffu || ld_x < 0 || !(eps >= 0.f) ||
      (d_mean == nullptr) != (d_inv == nullptr))
    return RMN_ERR_BAD_ARG;
  if (n_rows == 0) return RMN_OK;
  if (!d_x || !d_out) return RMN_ERR_BAD_ARG;
  const int elem = dtype == RMN_F32 ? 4 : 2;
  RowLayout a;
  if (!row_layout(channels, elem, aligned16(d_x, ld_x, elem) && aligned16(d_out, channels, elem), &a))
    return RMN_ERR_UNSUPPORTED;
  return dispatch_row(a, dtype, [&](auto t, auto v, auto nv, auto block) {
    return launch_forward<decltype(t), v.value, nv.value, block.value>(a, d_x, ld_x, n_rows, channels, d_gamma, d_beta,
                                                                       param_dtype == RMN_BF16, eps, d_out, d_mean, d_inv,
                                                                       (cudaStream_t)stream_);
  });
}

extern "C" size_t rmn_layer_norm_backward_workspace_bytes(uint32_t n_rows, int channels) {
  if (channels < 1 || channels > 65536) return 0;
  const uint32_t blocks = n_rows < kMaxBackwardBlocks ? n_rows : kMaxBackwardBlocks;  // at most one block a row
  return (size_t)blocks * 2 * channels * sizeof(float);
}

extern "C" int rmn_layer_norm_backward(const void* d_dy, int64_t ld_dy, const void* d_x, int64_t ld_x, uint32_t n_rows,
                                       int channels, const void* d_gamma, int param_dtype, const float* d_mean,
                                       const float* d_inv, void* d_dx, void* d_dgamma, void* d_dbeta, int dtype,
                                       void* d_workspace, size_t workspace_bytes, void* stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  if (!norm_args_ok(channels, dtype, param_dtype) || n_rows > 0x7fffffffu || ld_dy < 0 || ld_x < 0) return RMN_ERR_BAD_ARG;
  const bool sums = d_dgamma || d_dbeta;
  if (n_rows == 0) {
    const size_t bytes = (size_t)channels * (param_dtype == RMN_BF16 ? 2 : 4);
    if (d_dgamma) RMN_CUDA_TRY(cudaMemsetAsync(d_dgamma, 0, bytes, stream));
    if (d_dbeta) RMN_CUDA_TRY(cudaMemsetAsync(d_dbeta, 0, bytes, stream));
    return RMN_OK;
  }
  if (!d_dx && !sums) return RMN_OK;
  if (!d_dy || !d_x || !d_mean || !d_inv) return RMN_ERR_BAD_ARG;
  if (sums) {
    if (!d_workspace || ((uintptr_t)d_workspace & 15)) return RMN_ERR_BAD_ARG;
    if (workspace_bytes < rmn_layer_norm_backward_workspace_bytes(n_rows, channels)) return RMN_ERR_ALLOC;
  }
  const int elem = dtype == RMN_F32 ? 4 : 2;
  RowLayout a;
  if (!row_layout(channels, elem,
                  aligned16(d_dy, ld_dy, elem) && aligned16(d_x, ld_x, elem) && (!d_dx || aligned16(d_dx, channels, elem)), &a))
    return RMN_ERR_UNSUPPORTED;
  if (sums && (size_t)2 * channels * sizeof(float) > 200 * 1024) return RMN_ERR_UNSUPPORTED;
  const uint32_t grid = backward_blocks(n_rows, a.block ? 1 : kNormThreads / a.L);
  float* partial = sums ? static_cast<float*>(d_workspace) : nullptr;
  const int st = dispatch_row(a, dtype, [&](auto t, auto v, auto nv, auto block) {
    return launch_backward<decltype(t), v.value, nv.value, block.value>(a, d_dy, ld_dy, d_x, ld_x, n_rows, channels, d_gamma,
                                                                        param_dtype == RMN_BF16, d_mean, d_inv, d_dx, partial,
                                                                        grid, stream);
  });
  if (st != RMN_OK || !sums) return st;
  RMN_CUDA_TRY(launch_overlapped(k_layer_norm_sums, dim3((2 * channels + 31) / 32), dim3(256), 0, stream,
                                 static_cast<const float*>(partial), grid, channels, (int)(param_dtype == RMN_BF16), d_dgamma,
                                 d_dbeta));
  RMN_LAUNCH_CHECK();
  return RMN_OK;
}
