// Layer norm over the channels of every row of a feature matrix, forward and backward (the reference wraps torch's layer,
// engine/nn/normalization.hpp; it stands beside the batch norm of rmn_norm.cu).
//
//   mean = sum_c x / C,  inv = 1 / sqrt(sum_c (x - mean)^2 / C + eps),  xhat = (x - mean) * inv,  y = xhat * gamma + beta
//   g = dy * gamma,  dx = inv * (g - sum_c g / C - xhat * sum_c g xhat / C),  dgamma = sum_r dy xhat,  dbeta = sum_r dy
//
// Bound by memory: the forward pass reads x and writes y, the backward pass reads x and dy and writes dx. A row stays in the
// registers of L threads (L a power of two, from one thread to a block), 16 bytes a load, so each value is read once; the
// variance is taken around the mean in a second pass over the registers, in fp32. A thread has the same channels of all the rows
// it visits: gamma and beta are loaded once, and dgamma and dbeta are sums in its registers, which are added up over the block in a
// fixed order; a second kernel adds the blocks' sums in order: no atomics, the same bits every time.
#include "rmn_common.cuh"
#include "rmn_pair.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace rmn {
namespace {

constexpr int kNormThreads = 256;
constexpr int kMaxVectors = 4;                 // loads of a row by one thread
constexpr uint32_t kMaxBackwardBlocks = 148 * 4;
constexpr size_t kMaxSums = 200 * 1024;        // bytes of a block's sums of dgamma and dbeta

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// The arithmetic is on pairs of fp32 numbers (in bf16 it bounds as much as memory: 1.2 M x 64 forward 74 us with single ones, 62.5
// with pairs); rows read one number at a time use plain floats in their place.
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ float fma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float total(float a) { return a; }
template <int V>
using Number = std::conditional_t<V == 1, float, Pair>;
template <int V>
constexpr int kNumbers = V == 1 ? 1 : V / 2;  // of a load
template <int V>
__device__ __forceinline__ Number<V> splat(float x) {
  if constexpr (V == 1) return x;
  else return make_pair(x, x);
}
// number k of a load, and a load's worth of them back
template <typename T, int V>
__device__ __forceinline__ Number<V> number(const Pack<T, V>& p, int k) {
  if constexpr (V == 1) {
    return (float)p.v[0];
  } else if constexpr (sizeof(T) == 4) {
    return make_pair(p.v[2 * k], p.v[2 * k + 1]);
  } else {
    const uint32_t w = reinterpret_cast<const uint32_t*>(&p)[k];
    return make_pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
}
template <typename T, int V>
__device__ __forceinline__ void set_number(Pack<T, V>& p, int k, Number<V> x) {
  if constexpr (V == 1) {
    if constexpr (sizeof(T) == 4) p.v[0] = x;
    else p.v[0] = __float2bfloat16_rn(x);
  } else {
    float lo, hi;
    parts(x, lo, hi);
    if constexpr (sizeof(T) == 4) {
      p.v[2 * k] = lo;
      p.v[2 * k + 1] = hi;
    } else {
      reinterpret_cast<__nv_bfloat162*>(&p)[k] = __floats2bfloat162_rn(lo, hi);
    }
  }
}
// the parameters (of either type) from channel c on, `missing` where there are none
template <int V>
__device__ __forceinline__ void params(const void* p, int bf16, int c, float missing, Number<V> (&out)[kNumbers<V>]) {
  float x[V];
#pragma unroll
  for (int j = 0; j < V; ++j)
    x[j] = !p ? missing : bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c + j]) : static_cast<const float*>(p)[c + j];
#pragma unroll
  for (int k = 0; k < kNumbers<V>; ++k) {
    if constexpr (V == 1) out[k] = x[0];
    else out[k] = make_pair(x[2 * k], x[2 * k + 1]);
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

// Sums over the L threads of a row, N at once; every thread gets them. Rows of more than a warp go through shared memory: `red` is
// [2][32][N], its halves used in turn, so that one barrier does.
template <int N>
__device__ __forceinline__ void row_sum(float (&s)[N], int L, float* red, uint32_t& turn) {
  for (int o = min(L, 32) >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
  }
  if (L > 32) {
    const int warps = L >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* buf = red + (turn++ & 1u) * 32 * N;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) buf[warp * N + i] = s[i];
    }
    __syncthreads();
    const int from = (warp & ~(warps - 1)) + (lane & (warps - 1));
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = buf[from * N + i];
    for (int o = warps >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
    }
  }
}

// Rows in flight at once: their loads are issued together, and (rows of several warps) their sums share a barrier. As many as
// leave registers for four blocks an SM: 1.2 M x 64 bf16 forward with 2 / 4 / 6 rows 68 / 62.5 / 67 us, backward with
// 1 / 2 / 3 / 4 rows 101 / 94 / 87 / 94.
constexpr int forward_rows(int nv) { return nv == 1 ? 4 : nv <= 3 ? 2 : 1; }
constexpr int backward_rows(int nv) { return nv == 1 ? 3 : nv == 2 ? 2 : 1; }

template <typename T, int V, int NV, int kMost>
__global__ void __launch_bounds__(kMost)
    k_layer_norm(const T* __restrict__ x, int64_t ld, uint32_t n, int C, int L, const void* __restrict__ gamma,
                 const void* __restrict__ beta, int param_bf16, float eps, T* __restrict__ out, float* __restrict__ mean_out,
                 float* __restrict__ inv_out) {
  constexpr int U = forward_rows(NV);
  __shared__ float red[2 * 32 * U];
  after_previous_kernel();
  const int group = threadIdx.x / L, at = threadIdx.x % L, groups = blockDim.x / L;
  const int nvec = C / V;
  const float inv_c = 1.f / (float)C;
  uint32_t turn = 0;
  constexpr int N = kNumbers<V>;
  Number<V> g[NV][N], b[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (at + i * L < nvec) {
      params<V>(gamma, param_bf16, (at + i * L) * V, 1.f, g[i]);
      params<V>(beta, param_bf16, (at + i * L) * V, 0.f, b[i]);
    }
  // whole batches of rows, so that all threads of a block meet in the sums
  for (uint64_t first = (uint64_t)blockIdx.x * groups * U; first < n; first += (uint64_t)gridDim.x * groups * U) {
    Pack<T, V> raw[U][NV];
    float s[U], mean[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t r = first + u * groups + group;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = at + i * L;
        if (r < n && v < nvec) raw[u][i] = load_pack<T, V>(x + (int64_t)r * ld + (int64_t)v * V);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Number<V> t = splat<V>(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (at + i * L < nvec)
#pragma unroll
          for (int k = 0; k < N; ++k) {
            t = add(t, number(raw[u][i], k));
          }
      s[u] = total(t);
    }
    row_sum(s, L, red, turn);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mean[u] = s[u] * inv_c;
      const Number<V> minus = splat<V>(-mean[u]);
      Number<V> t = splat<V>(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (at + i * L < nvec)
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const Number<V> d = add(number(raw[u][i], k), minus);
            t = fma(d, d, t);
          }
      s[u] = total(t);
    }
    row_sum(s, L, red, turn);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t r = first + u * groups + group;
      if (r >= n) continue;
      const float inv = 1.f / sqrtf(s[u] * inv_c + eps);
      const Number<V> by = splat<V>(inv), minus = splat<V>(-mean[u]);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = at + i * L;
        if (v >= nvec) continue;
        Pack<T, V> o;
#pragma unroll
        for (int k = 0; k < N; ++k) set_number(o, k, fma(mul(add(number(raw[u][i], k), minus), by), g[i][k], b[i][k]));
        *reinterpret_cast<Pack<T, V>*>(out + (size_t)r * C + (size_t)v * V) = o;
      }
      if (at == 0 && mean_out) {
        mean_out[r] = mean[u];
        inv_out[r] = inv;
      }
    }
  }
}

// partial[block][0][c] = the block's part of dgamma, [1][c] of dbeta (kSums: wanted)
template <typename T, int V, int NV, int kMost, bool kSums>
__global__ void __launch_bounds__(kMost)
    k_layer_norm_backward(const T* __restrict__ dy, int64_t ld_dy, const T* __restrict__ x, int64_t ld_x, uint32_t n, int C,
                          int L, const void* __restrict__ gamma, int param_bf16, const float* __restrict__ mean_in,
                          const float* __restrict__ inv_in, T* __restrict__ dx, float* __restrict__ partial) {
  constexpr int U = backward_rows(NV);
  // 16 bytes are made into fp32 again for the second pass over them; keeping fp32 takes the registers of rows in flight
  constexpr bool kKeep = V == 1;
  extern __shared__ float sums[];  // [2][C] (kSums)
  __shared__ float red[2 * 32 * 2 * U];
  after_previous_kernel();
  const int group = threadIdx.x / L, at = threadIdx.x % L, groups = blockDim.x / L;
  const int nvec = C / V;
  const float inv_c = 1.f / (float)C;
  uint32_t turn = 0;
  constexpr int N = kNumbers<V>;
  Number<V> g[NV][N], dg[kSums ? NV : 1][N], db[kSums ? NV : 1][N];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (at + i * L < nvec) params<V>(gamma, param_bf16, (at + i * L) * V, 1.f, g[i]);
  if constexpr (kSums) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) dg[i][k] = db[i][k] = splat<V>(0.f);
  }
  // whole batches of rows, so that all threads of a block meet in the sums
  for (uint64_t first = (uint64_t)blockIdx.x * groups * U; first < n; first += (uint64_t)gridDim.x * groups * U) {
    Pack<T, V> rx[U][NV], rd[U][NV];
    Number<V> kept[kKeep ? U : 1][kKeep ? NV : 1][2];  // xhat, dy * gamma
    float mean[U], inv[U], s[2 * U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t r = first + u * groups + group;
      mean[u] = inv[u] = s[2 * u] = s[2 * u + 1] = 0.f;
      if (r >= n) continue;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = at + i * L;
        if (v >= nvec) continue;
        rx[u][i] = load_pack<T, V>(x + (int64_t)r * ld_x + (int64_t)v * V);
        rd[u][i] = load_pack<T, V>(dy + (int64_t)r * ld_dy + (int64_t)v * V);
      }
      mean[u] = __ldg(mean_in + r);
      inv[u] = __ldg(inv_in + r);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (first + u * groups + group >= n) continue;
      const Number<V> minus = splat<V>(-mean[u]), by = splat<V>(inv[u]);
      Number<V> t0 = splat<V>(0.f), t1 = splat<V>(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (at + i * L >= nvec) continue;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const Number<V> h = mul(add(number(rx[u][i], k), minus), by), d = number(rd[u][i], k);
          if constexpr (kSums) {
            dg[i][k] = fma(d, h, dg[i][k]);
            db[i][k] = add(db[i][k], d);
          }
          const Number<V> e = mul(d, g[i][k]);
          if constexpr (kKeep) {
            kept[u][i][0] = h;
            kept[u][i][1] = e;
          }
          t0 = add(t0, e);
          t1 = fma(e, h, t1);
        }
      }
      s[2 * u] = total(t0);
      s[2 * u + 1] = total(t1);
    }
    if (!dx) continue;  // (the same for all threads)
    row_sum(s, L, red, turn);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t r = first + u * groups + group;
      if (r >= n) continue;
      const Number<V> a = splat<V>(-s[2 * u] * inv_c), b = splat<V>(-s[2 * u + 1] * inv_c), by = splat<V>(inv[u]), minus = splat<V>(-mean[u]);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = at + i * L;
        if (v >= nvec) continue;
        Pack<T, V> o;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          if constexpr (kKeep) {
            set_number(o, k, mul(by, fma(kept[u][i][0], b, add(kept[u][i][1], a))));
          } else {
            const Number<V> h = mul(add(number(rx[u][i], k), minus), by);
            set_number(o, k, mul(by, fma(h, b, fma(number(rd[u][i], k), g[i][k], a))));
          }
        }
        *reinterpret_cast<Pack<T, V>*>(dx + (size_t)r * C + (size_t)v * V) = o;
      }
    }
  }
  if constexpr (kSums) {
    float wg[NV][V], wb[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if constexpr (V == 1) {
          wg[i][k] = dg[i][k];
          wb[i][k] = db[i][k];
        } else {
          parts(dg[i][k], wg[i][2 * k], wg[i][2 * k + 1]);
          parts(db[i][k], wb[i][2 * k], wb[i][2 * k + 1]);
        }
      }
    for (int o = L; o < 32; o <<= 1) {  // the groups of a warp hold the same channels
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          wg[i][j] += __shfl_xor_sync(0xffffffffu, wg[i][j], o);
          wb[i][j] += __shfl_xor_sync(0xffffffffu, wb[i][j], o);
        }
    }
    // those that hold the same channels one after the other: warps, or groups of them
    const int wide = max(L, 32), turns = blockDim.x / wide;
    for (int w = 0; w < turns; ++w) {
      if ((int)threadIdx.x / wide == w && (int)(threadIdx.x % wide) < L) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int v = at + i * L;
          if (v >= nvec) continue;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int c = v * V + j;
            sums[c] = w ? sums[c] + wg[i][j] : wg[i][j];
            sums[C + c] = w ? sums[C + c] + wb[i][j] : wb[i][j];
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * C; c += blockDim.x) partial[(size_t)blockIdx.x * 2 * C + c] = sums[c];
  }
}

// dgamma[c], dbeta[c] = the blocks' sums in a fixed order: 32 slices of them, in fp64, then the slices.
__global__ void __launch_bounds__(1024) k_layer_norm_sums(const float* __restrict__ partial, uint32_t blocks, int C,
                                                          int param_bf16, void* __restrict__ dgamma,
                                                          void* __restrict__ dbeta) {
  __shared__ double part[32][33];
  after_previous_kernel();
  const int slice = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x * 32 + lane;
  double t = 0.0;
  if (i < 2 * C)
#pragma unroll 8
    for (uint32_t b = slice; b < blocks; b += 32) t += (double)__ldg(partial + (size_t)b * 2 * C + i);
  part[slice][lane] = t;
  __syncthreads();
  t = part[lane][slice];  // column `slice` by the warp of that number
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const int out = blockIdx.x * 32 + slice;
  if (lane != 0 || out >= 2 * C) return;
  void* to = out < C ? dgamma : dbeta;
  if (!to) return;
  const int c = out < C ? out : out - C;
  if (param_bf16) static_cast<__nv_bfloat16*>(to)[c] = __float2bfloat16_rn((float)t);
  else static_cast<float*>(to)[c] = (float)t;
}

// How a row of C channels is laid over threads: V channels a load (16 bytes where alignment and C allow, else one), L threads a
// row (a power of two), each with nv loads. The number of loads up to three that leaves the fewest threads idle, the smallest of
// several (48503 x 96 fp32 forward with one load, a quarter idle, 10.4 us, with three 6.3); but a row that fits a warp stays in one,
// which saves the barriers (16411 x 1024 bf16 forward in 128 threads 18 us, in 32 with four loads 14.2), in the backward pass as long
// as that takes two loads in bf16, three in fp32 (a thread keeps 3 V nv numbers there: the same rows 30 us against 47). Four loads for
// the widest rows.
struct RowLayout {
  int V, L, nv;
};
bool row_layout(int C, int elem, bool aligned, bool backward, RowLayout* out) {
  const int wide = 16 / elem;
  const int V = aligned && C % wide == 0 ? wide : 1;
  const int nvec = C / V;
  const int in_warp = !backward ? kMaxVectors : V == 8 ? 2 : 3;  // loads that a row may take to stay in a warp
  const int most = nvec > 512 * kMaxVectors ? 1024 : 512;  // (a thread of 1024 has 64 registers: only where nothing else holds the row)
  int best = 0, best_nv = 0;
  for (int nv = most == 1024 ? 3 : 1; nv <= kMaxVectors; ++nv) {
    int L = 1;
    while (L * nv < nvec) L *= 2;
    if (L > most) continue;
    const bool into_warp = best > 32 && L <= 32 && nv <= in_warp;
    if (nv == kMaxVectors && best && !into_warp) break;
    if (!best || into_warp || (long long)L * nv < (long long)best * best_nv) { best = L; best_nv = nv; }
  }
  if (!best) return false;
  *out = {V, best, best_nv};
  return true;
}
int row_threads(const RowLayout& a) { return a.L > kNormThreads ? a.L : kNormThreads; }

bool aligned16(const void* p, int64_t ld, int elem) { return ((uintptr_t)p & 15) == 0 && (ld * elem) % 16 == 0; }
bool norm_args_ok(int C, int dtype, int param_dtype) {
  return C >= 1 && C <= 65536 && (dtype == RMN_F32 || dtype == RMN_BF16) &&
         (param_dtype == RMN_F32 || param_dtype == RMN_BF16);
}
// As many blocks as fit the GPU, at most one for every `rows` rows. `known`: what registers allow an SM, asked once (blocks of one
// kernel have the same size but for rows of 512 threads and more, where one block more or less a time does not count).
template <class Kernel>
uint32_t resident_blocks(Kernel kern, std::atomic<int>& known, int threads, size_t smem, uint32_t n, uint64_t rows, uint32_t most) {
  int per_sm = known.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, 0) != cudaSuccess || per_sm < 1) {
      cudaGetLastError();
      per_sm = 1;
    }
    known.store(per_sm, std::memory_order_relaxed);
  }
  const uint64_t need = ((uint64_t)n + rows - 1) / rows;
  const uint64_t by_smem = std::max<uint64_t>(1, 227 * 1024 / (smem + 2048));
  return (uint32_t)std::min<uint64_t>({need, 148 * std::min<uint64_t>(per_sm, by_smem), most});
}

template <typename T, int V, int NV, int kMost>
int launch_forward(const RowLayout& a, const void* x, int64_t ld, uint32_t n, int C, const void* gamma, const void* beta,
                   int param_bf16, float eps, void* out, float* mean, float* inv, cudaStream_t stream) {
  auto kern = k_layer_norm<T, V, NV, kMost>;
  const int threads = row_threads(a);
  static std::atomic<int> known{0};
  const uint32_t grid = resident_blocks(kern, known, threads, 0, n, (uint64_t)forward_rows(NV) * (threads / a.L), 0xffffffffu);
  RMN_CUDA_TRY(launch_overlapped(kern, dim3(grid), dim3(threads), 0, stream, static_cast<const T*>(x), ld, n, C, a.L, gamma, beta,
                                 param_bf16, eps, static_cast<T*>(out), mean, inv));
  RMN_LAUNCH_CHECK();
  return RMN_OK;
}

template <typename T, int V, int NV, int kMost>
int launch_backward(const RowLayout& a, const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, uint32_t n, int C,
                    const void* gamma, int param_bf16, const float* mean, const float* inv, void* dx, float* partial,
                    uint32_t* grid_out, cudaStream_t stream) {
  const int threads = row_threads(a);
  const size_t smem = partial ? (size_t)2 * C * sizeof(float) : 0;
  auto go = [&](auto kern, SmemOptIn& opt_in, std::atomic<int>& known) -> int {
    // the most that any row takes: the attribute is set once for all of them
    if (smem > 46 * 1024) RMN_CUDA_TRY(opt_in.apply(reinterpret_cast<const void*>(kern), kMaxSums));
    *grid_out = resident_blocks(kern, known, threads, smem, n, (uint64_t)backward_rows(NV) * (threads / a.L), kMaxBackwardBlocks);
    RMN_CUDA_TRY(launch_overlapped(kern, dim3(*grid_out), dim3(threads), smem, stream, static_cast<const T*>(dy), ld_dy,
                                   static_cast<const T*>(x), ld_x, n, C, a.L, gamma, param_bf16, mean, inv,
                                   static_cast<T*>(dx), partial));
    RMN_LAUNCH_CHECK();
    return RMN_OK;
  };
  static SmemOptIn with_sums, without;
  static std::atomic<int> known_with{0}, known_without{0};
  return partial ? go(k_layer_norm_backward<T, V, NV, kMost, true>, with_sums, known_with)
                 : go(k_layer_norm_backward<T, V, NV, kMost, false>, without, known_without);
}

// f(type tag, V, NV, threads at most) of the layout
template <class F>
int dispatch_row(const RowLayout& a, int dtype, F&& f) {
  auto by_nv = [&](auto t, auto v, auto most) -> int {
    switch (a.nv) {
      case 1: return f(t, v, std::integral_constant<int, 1>{}, most);
      case 2: return f(t, v, std::integral_constant<int, 2>{}, most);
      case 3: return f(t, v, std::integral_constant<int, 3>{}, most);
      default: return f(t, v, std::integral_constant<int, 4>{}, most);
    }
  };
  auto by_threads = [&](auto t, auto v) -> int {
    if (a.L > 512) {
      using Most = std::integral_constant<int, 1024>;
      return a.nv == 3 ? f(t, v, std::integral_constant<int, 3>{}, Most{}) : f(t, v, std::integral_constant<int, 4>{}, Most{});
    }
    return a.L > kNormThreads ? by_nv(t, v, std::integral_constant<int, 512>{})
                              : by_nv(t, v, std::integral_constant<int, kNormThreads>{});
  };
  if (dtype == RMN_F32)
    return a.V == 1 ? by_threads(float{}, std::integral_constant<int, 1>{}) : by_threads(float{}, std::integral_constant<int, 4>{});
  return a.V == 1 ? by_threads(__nv_bfloat16{}, std::integral_constant<int, 1>{})
                  : by_threads(__nv_bfloat16{}, std::integral_constant<int, 8>{});
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
  if (!row_layout(channels, elem, aligned16(d_x, ld_x, elem) && aligned16(d_out, channels, elem), false, &a))
    return RMN_ERR_UNSUPPORTED;
  return dispatch_row(a, dtype, [&](auto t, auto v, auto nv, auto most) {
    return launch_forward<decltype(t), v.value, nv.value, most.value>(a, d_x, ld_x, n_rows, channels, d_gamma, d_beta,
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
                  aligned16(d_dy, ld_dy, elem) && aligned16(d_x, ld_x, elem) && (!d_dx || aligned16(d_dx, channels, elem)), true,
                  &a))
    return RMN_ERR_UNSUPPORTED;
  if (sums && (size_t)2 * channels * sizeof(float) > kMaxSums) return RMN_ERR_UNSUPPORTED;
  float* partial = sums ? static_cast<float*>(d_workspace) : nullptr;
  uint32_t grid = 0;
  const int st = dispatch_row(a, dtype, [&](auto t, auto v, auto nv, auto most) {
    return launch_backward<decltype(t), v.value, nv.value, most.value>(a, d_dy, ld_dy, d_x, ld_x, n_rows, channels, d_gamma,
                                                                        param_dtype == RMN_BF16, d_mean, d_inv, d_dx, partial,
                                                                        &grid, stream);
  });
  if (st != RMN_OK || !sums) return st;
  RMN_CUDA_TRY(launch_overlapped(k_layer_norm_sums, dim3((2 * channels + 31) / 32), dim3(1024), 0, stream,
                                 static_cast<const float*>(partial), grid, channels, (int)(param_dtype == RMN_BF16), d_dgamma,
                                 d_dbeta));
  RMN_LAUNCH_CHECK();
  return RMN_OK;
}
