// Rotary positions with several axes, alone or behind a norm of every head (queries and keys of attention), forward and backward.
//
//   angle(row, pair) = positions[row][axis of the pair] * frequency(pair)
//   y0 = x0 cos - x1 sin,  y1 = x1 cos + x0 sin,  channels behind the pairs as they are
//   norm: x is replaced by x inv w, inv = 1 / sqrt(sum x^2 / dim + eps) over the channels of a head
//   backward: g = the output's gradient turned back, a = g w, xhat = x inv, dx = inv (a - xhat sum(a xhat) / dim),
//   dw = sum over rows and heads of g xhat
//
// The angle in whole turns is a product of integers: the frequency as a fraction of a turn in 64 bits, so that the product wraps around
// where a turn is full. No bits are lost however far the position is, and no range has to be reduced. What is left of a turn is cut into
// quarters; sine and cosine of up to an eighth either way are their Taylor polynomials (off by less than 2e-9).
//
// Bound by memory: every value is read once and written once. A head's channels lie over L lanes (a power of two), each with units of V
// pairs, 16 bytes a load where sizes and alignment allow. Such a group takes a row's heads one after the other, U of them in flight,
// so that the angles of a row are made once; few rows are dealt out to several groups a row, each with every second, fourth ... head. The
// norm's sums go over the L lanes. dw is summed in registers over the rows that a thread visits, over the block in a fixed order and over
// the blocks by a second kernel: no atomics, the same bits every time.
#include "rmn_common.cuh"

#include <cuda_bf16.h>

#include <algorithm>

namespace rmn {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMostBackwardBlocks = 148 * 4;
constexpr int kMostAxes = 8;

struct Heads {  // [rows, heads, dim]
  const void* x;
  int64_t row, head;
  const void* grad;  // backward: of the output
  int64_t grad_row, grad_head;
  const void* weight;  // NULL: ones
  void* out;           // no gaps; backward: the gradient of x
  int heads;
};
struct RotaryArgs {
  Heads part[2];  // queries, keys (0 heads: none)
  uint32_t rows;
  int dim, pairs, lanes, per_row;  // lanes of a head, groups of lanes of a row
  const int32_t* positions;
  int64_t position_row, position_axis;
  const double* frequencies;
  int ends[kMostAxes];  // the pair behind the last one of an axis
  int weight_bf16, back;  // back: turned the other way (without a norm the gradient is nothing else)
  float eps;
  float* sums;  // backward: [block][2][dim]
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  if constexpr (sizeof(r) == 16) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
    r = *reinterpret_cast<const Pack<T, V>*>(&w);
  } else if constexpr (sizeof(r) == 8) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    r = *reinterpret_cast<const Pack<T, V>*>(&w);
  } else if constexpr (sizeof(r) == 4) {
    const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(p));
    r = *reinterpret_cast<const Pack<T, V>*>(&w);
  } else {
    r = *reinterpret_cast<const Pack<T, V>*>(p);
  }
  return r;
}
__device__ __forceinline__ float number(float v) { return v; }
__device__ __forceinline__ float number(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T rounded(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else return __float2bfloat16_rn(v);
}

// One pair's frequency as a 64-bit fraction of a turn.
__device__ __forceinline__ uint64_t fraction_of_turn(double radians) {
  const double turns = radians * 0.15915494309189533577;  // 1 / (2 pi)
  return __double2ull_rz((turns - floor(turns)) * 18446744073709551616.0);
}
// cos and sin of position * fraction (a full turn: 2^64)
__device__ __forceinline__ void turn_of(int32_t position, uint64_t fraction, float& c, float& s) {
  const uint32_t t = (uint32_t)(((uint64_t)(int64_t)position * fraction) >> 32);
  const uint32_t quarter = (t + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(t - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float y = x * x;
  float sine = fmaf(y, 2.7557319e-6f, -1.9841270e-4f), cosine = fmaf(y, -2.7557319e-7f, 2.4801587e-5f);
  sine = fmaf(y, sine, 8.3333333e-3f);
  cosine = fmaf(y, cosine, -1.3888889e-3f);
  sine = fmaf(y, sine, -1.6666667e-1f);
  cosine = fmaf(y, cosine, 4.1666667e-2f);
  sine = fmaf(x * y, sine, x);
  cosine = fmaf(y, cosine, -0.5f);
  cosine = fmaf(y, cosine, 1.f);
  const float a = quarter & 1u ? sine : cosine, b = quarter & 1u ? cosine : sine;
  c = (quarter + 1u) & 2u ? -a : a;
  s = quarter & 2u ? -b : b;
}

// A unit: V pairs of a lane, as 2 V numbers in two loads of V channels. Halves: the first numbers of the pairs, then the second ones.
template <int V, bool kNext>  // kNext: a pair's numbers are neighbours
struct Unit {
  int lo, hi;  // channels of the two loads
  __device__ __forceinline__ Unit(int u, int pairs, int dim) {
    if (kNext) {
      lo = 2 * u * V;
      hi = lo + V;
    } else if (u * V < pairs) {
      lo = u * V;
      hi = lo + pairs;
    } else {  // what stays as it is
      lo = u * V + pairs;
      hi = lo + dim / 2 - pairs;
    }
  }
  static constexpr int first(int j) { return kNext ? 2 * j : j; }
  static constexpr int second(int j) { return kNext ? 2 * j + 1 : V + j; }
};

template <int V, bool kNext>
__device__ __forceinline__ void rotate(const float (&x)[2 * V], const float (&c)[V], const float (&s)[V], int turned, float (&y)[2 * V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    constexpr auto first = Unit<V, kNext>::first;
    constexpr auto second = Unit<V, kNext>::second;
    const float a = x[first(j)], b = x[second(j)];
    y[first(j)] = j < turned ? fmaf(a, c[j], -(b * s[j])) : a;
    y[second(j)] = j < turned ? fmaf(b, c[j], a * s[j]) : b;
  }
}

// The angles of a lane's pairs.
template <int V, int NU>
struct Angles {
  uint64_t fraction[NU][V];
  int axis[NU][V];
  int turned[NU];  // pairs of the unit that turn
  __device__ __forceinline__ void begin(const RotaryArgs& a, int lane) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int p0 = (lane + i * a.lanes) * V;
      turned[i] = min(max(a.pairs - p0, 0), V);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        fraction[i][j] = p0 + j < a.pairs ? fraction_of_turn(__ldg(a.frequencies + p0 + j)) : 0;
        axis[i][j] = 0;
#pragma unroll
        for (int k = 0; k < kMostAxes - 1; ++k) axis[i][j] += p0 + j >= a.ends[k] && p0 + j < a.pairs ? 1 : 0;
      }
    }
  }
  __device__ __forceinline__ void of_row(const RotaryArgs& a, uint64_t row, float (&c)[NU][V], float (&s)[NU][V]) const {
    const int32_t* at = a.positions + (int64_t)row * a.position_row;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      int32_t place = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (j < turned[i] && (j == 0 || axis[i][j] != axis[i][j - 1])) place = __ldg(at + (int64_t)axis[i][j] * a.position_axis);
        turn_of(place, fraction[i][j], c[i][j], s[i][j]);
        if (a.back) s[i][j] = -s[i][j];
      }
    }
  }
};

// w of a lane's channels
template <int V, bool kNext, int NU>
__device__ __forceinline__ void weights(const RotaryArgs& a, const void* w, int lane, float (&out)[NU][2 * V]) {
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int u = lane + i * a.lanes;
    const Unit<V, kNext> unit(u, a.pairs, a.dim);
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) {
      const int ch = j < V ? unit.lo + j : unit.hi + j - V;
      out[i][j] = !w || u * V >= a.dim / 2 ? 1.f
                  : a.weight_bf16          ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[ch])
                                           : static_cast<const float*>(w)[ch];
    }
  }
}
// the sum over the lanes of a head; every one gets it
__device__ __forceinline__ float over_lanes(float v, int lanes, uint32_t mask) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
  return v;
}

template <typename T, int V, int NU>
__device__ __forceinline__ void load_units(const T* from, const int (&lo)[NU], const int (&hi)[NU], bool here, const bool (&has)[NU],
                                           Pack<T, V> (&x)[NU][2]) {
#pragma unroll
  for (int i = 0; i < NU; ++i)
    if (here && has[i]) {
      x[i][0] = load_pack<T, V>(from + lo[i]);
      x[i][1] = load_pack<T, V>(from + hi[i]);
    }
}

template <typename T, int V, int NU, bool kNext, bool kNorm>
__global__ void __launch_bounds__(kThreads) k_rotary(const __grid_constant__ RotaryArgs a) {
  constexpr int U = NU == 1 ? 4 : 2;  // heads in flight
  after_previous_kernel();
  const int lane = threadIdx.x & (a.lanes - 1);
  const uint64_t group = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) / a.lanes, groups = (uint64_t)gridDim.x * (kThreads / a.lanes);
  const uint32_t mask = a.lanes == 32 ? 0xffffffffu : ((1u << a.lanes) - 1u) << (threadIdx.x & 31 & ~(a.lanes - 1));
  const int head0 = (int)(group % a.per_row);
  const float inv_dim = 1.f / (float)a.dim;
  Angles<V, NU> angles;
  angles.begin(a, lane);
  int lo[NU], hi[NU];
  bool has[NU];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const Unit<V, kNext> unit(lane + i * a.lanes, a.pairs, a.dim);
    lo[i] = unit.lo;
    hi[i] = unit.hi;
    has[i] = (lane + i * a.lanes) * V < a.dim / 2;
  }
  float w[2][NU][2 * V];
  if constexpr (kNorm) {
    weights<V, kNext, NU>(a, a.part[0].weight, lane, w[0]);
    weights<V, kNext, NU>(a, a.part[1].weight, lane, w[1]);
  }
  for (uint64_t row = group / a.per_row; row < a.rows; row += groups / a.per_row) {
    float c[NU][V], s[NU][V];
    angles.of_row(a, row, c, s);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const Heads& p = a.part[which];
      const T* from = static_cast<const T*>(p.x) + (int64_t)row * p.row;
      T* to = static_cast<T*>(p.out) + row * (uint64_t)p.heads * a.dim;
      for (int h0 = head0; h0 < p.heads; h0 += U * a.per_row) {
        Pack<T, V> raw[U][NU][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * a.per_row;
          load_units<T, V, NU>(from + (int64_t)h * p.head, lo, hi, h < p.heads, has, raw[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * a.per_row;
          if (h >= p.heads) break;
          float x[NU][2 * V];
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) {
              x[i][j] = has[i] ? number(raw[u][i][j / V].v[j % V]) : 0.f;
              if constexpr (kNorm) sum = fmaf(x[i][j], x[i][j], sum);
            }
          if constexpr (kNorm) {
            const float inv = 1.f / sqrtf(over_lanes(sum, a.lanes, mask) * inv_dim + a.eps);
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
              for (int j = 0; j < 2 * V; ++j) x[i][j] = x[i][j] * inv * w[which][i][j];
          }
#pragma unroll
          for (int i = 0; i < NU; ++i) {
            if (!has[i]) continue;
            float y[2 * V];
            rotate<V, kNext>(x[i], c[i], s[i], angles.turned[i], y);
            Pack<T, V> o[2];
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) o[j / V].v[j % V] = rounded<T>(y[j]);
            *reinterpret_cast<Pack<T, V>*>(to + (int64_t)h * a.dim + lo[i]) = o[0];
            *reinterpret_cast<Pack<T, V>*>(to + (int64_t)h * a.dim + hi[i]) = o[1];
          }
        }
      }
    }
  }
}

// dx of the norm and the rotation (a.back is set: gradients are turned back), and a block's part of dw of both.
template <typename T, int V, int NU, bool kNext>
__global__ void __launch_bounds__(kThreads) k_rotary_backward(const __grid_constant__ RotaryArgs a) {
  constexpr int U = NU == 1 ? 2 : 1;
  __shared__ float block_sums[2 * 256];
  after_previous_kernel();
  const int lane = threadIdx.x & (a.lanes - 1);
  const uint64_t group = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) / a.lanes, groups = (uint64_t)gridDim.x * (kThreads / a.lanes);
  const uint32_t mask = a.lanes == 32 ? 0xffffffffu : ((1u << a.lanes) - 1u) << (threadIdx.x & 31 & ~(a.lanes - 1));
  const int head0 = (int)(group % a.per_row);
  const float inv_dim = 1.f / (float)a.dim;
  Angles<V, NU> angles;
  angles.begin(a, lane);
  int lo[NU], hi[NU];
  bool has[NU];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const Unit<V, kNext> unit(lane + i * a.lanes, a.pairs, a.dim);
    lo[i] = unit.lo;
    hi[i] = unit.hi;
    has[i] = (lane + i * a.lanes) * V < a.dim / 2;
  }
  float w[2][NU][2 * V], dw[2][NU][2 * V];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    weights<V, kNext, NU>(a, a.part[which].weight, lane, w[which]);
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) dw[which][i][j] = 0.f;
  }
  for (uint64_t row = group / a.per_row; row < a.rows; row += groups / a.per_row) {
    float c[NU][V], s[NU][V];
    angles.of_row(a, row, c, s);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const Heads& p = a.part[which];
      const T* from = static_cast<const T*>(p.x) + (int64_t)row * p.row;
      const T* grad = static_cast<const T*>(p.grad) + (int64_t)row * p.grad_row;
      T* to = static_cast<T*>(p.out) + row * (uint64_t)p.heads * a.dim;
      for (int h0 = head0; h0 < p.heads; h0 += U * a.per_row) {
        Pack<T, V> raw[U][NU][2], dy[U][NU][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * a.per_row;
          load_units<T, V, NU>(from + (int64_t)h * p.head, lo, hi, h < p.heads, has, raw[u]);
          load_units<T, V, NU>(grad + (int64_t)h * p.grad_head, lo, hi, h < p.heads, has, dy[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * a.per_row;
          if (h >= p.heads) break;
          float x[NU][2 * V], g[NU][2 * V];
          float sum = 0.f, dot = 0.f;
#pragma unroll
          for (int i = 0; i < NU; ++i) {
            float y[2 * V];
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) {
              x[i][j] = has[i] ? number(raw[u][i][j / V].v[j % V]) : 0.f;
              y[j] = has[i] ? number(dy[u][i][j / V].v[j % V]) : 0.f;
              sum = fmaf(x[i][j], x[i][j], sum);
            }
            rotate<V, kNext>(y, c[i], s[i], angles.turned[i], g[i]);
          }
          const float inv = 1.f / sqrtf(over_lanes(sum, a.lanes, mask) * inv_dim + a.eps);
#pragma unroll
          for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) {
              x[i][j] *= inv;
              dw[which][i][j] = fmaf(g[i][j], x[i][j], dw[which][i][j]);
              g[i][j] *= w[which][i][j];
              dot = fmaf(g[i][j], x[i][j], dot);
            }
          dot = over_lanes(dot, a.lanes, mask) * inv_dim;
#pragma unroll
          for (int i = 0; i < NU; ++i) {
            if (!has[i]) continue;
            Pack<T, V> o[2];
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) o[j / V].v[j % V] = rounded<T>(inv * fmaf(-dot, x[i][j], g[i][j]));
            *reinterpret_cast<Pack<T, V>*>(to + (int64_t)h * a.dim + lo[i]) = o[0];
            *reinterpret_cast<Pack<T, V>*>(to + (int64_t)h * a.dim + hi[i]) = o[1];
          }
        }
      }
    }
  }
  if (!a.sums) return;  // (the same for all threads)
  // the groups of a warp hold the same channels; then the warps one after the other
#pragma unroll
  for (int which = 0; which < 2; ++which)
    for (int o = a.lanes; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) dw[which][i][j] += __shfl_xor_sync(0xffffffffu, dw[which][i][j], o);
  for (int t = 0; t < kThreads / 32; ++t) {
    if ((int)threadIdx.x / 32 == t && (int)(threadIdx.x & 31) < a.lanes) {
#pragma unroll
      for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int i = 0; i < NU; ++i) {
          if (!has[i]) continue;
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) {
            float* at = block_sums + which * a.dim + (j < V ? lo[i] + j : hi[i] + j - V);
            *at = t ? *at + dw[which][i][j] : dw[which][i][j];
          }
        }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * a.dim; i += kThreads) a.sums[(size_t)blockIdx.x * 2 * a.dim + i] = block_sums[i];
}

// dw of queries and keys = the blocks' sums in a fixed order: 32 slices of them, in fp64, then the slices.
__global__ void __launch_bounds__(1024) k_rotary_sums(const float* __restrict__ sums, uint32_t blocks, int dim, int bf16,
                                                      void* __restrict__ dwq, void* __restrict__ dwk) {
  __shared__ double part[32][33];
  after_previous_kernel();
  const int slice = threadIdx.x >> 5, lane = threadIdx.x & 31, i = blockIdx.x * 32 + lane;
  double t = 0.0;
  if (i < 2 * dim)
#pragma unroll 8
    for (uint32_t b = slice; b < blocks; b += 32) t += (double)__ldg(sums + (size_t)b * 2 * dim + i);
  part[slice][lane] = t;
  __syncthreads();
  t = part[lane][slice];  // number `slice` by the warp of that number
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const int out = blockIdx.x * 32 + slice;
  if (lane != 0 || out >= 2 * dim) return;
  void* to = out < dim ? dwq : dwk;
  if (!to) return;
  const int c = out < dim ? out : out - dim;
  if (bf16) static_cast<__nv_bfloat16*>(to)[c] = __float2bfloat16_rn((float)t);
  else static_cast<float*>(to)[c] = (float)t;
}

bool stride_ok(int64_t s) { return s >= 0 && s <= (int64_t(1) << 40); }

// the problem as the kernels take it; RMN_OK or what is wrong with it
int arguments(const rmn_rotary* p, RotaryArgs* a) {
  if (!p || p->rows > 0x7fffffffu || p->heads < 1 || p->kv_heads < 0 || p->heads > 65536 || p->kv_heads > 65536 || p->dim < 2 || p->dim % 2 ||
      (p->dtype != RMN_F32 && p->dtype != RMN_BF16) || p->axes < 0 || p->axes > kMostAxes || (p->axes && !p->sections))
    return RMN_ERR_BAD_ARG;
  const int64_t strides[] = {p->q_row, p->q_head, p->k_row, p->k_head, p->position_row, p->position_axis};
  for (int64_t s : strides)
    if (!stride_ok(s)) return RMN_ERR_BAD_ARG;
  if (p->rows && (!p->q || (p->kv_heads && !p->k))) return RMN_ERR_BAD_ARG;
  if (p->norm && (!(p->eps >= 0.f) || (p->weight_dtype != RMN_F32 && p->weight_dtype != RMN_BF16))) return RMN_ERR_BAD_ARG;
  *a = {};
  int pairs = 0;
  for (int i = 0; i < kMostAxes; ++i) {
    if (i < p->axes) {
      if (p->sections[i] < 0 || p->sections[i] > p->dim / 2 - pairs) return RMN_ERR_BAD_ARG;
      pairs += p->sections[i];
    }
    a->ends[i] = pairs;
  }
  if (pairs && (!p->frequencies || ((uintptr_t)p->frequencies & 7) || (p->rows && !p->positions))) return RMN_ERR_BAD_ARG;
  if (p->dim > 256) return RMN_ERR_UNSUPPORTED;
  a->part[0].x = p->q; a->part[0].row = p->q_row; a->part[0].head = p->q_head; a->part[0].heads = p->heads;
  a->part[1].x = p->k; a->part[1].row = p->k_row; a->part[1].head = p->k_head; a->part[1].heads = p->kv_heads;
  if (p->norm) {
    a->part[0].weight = p->q_weight;
    a->part[1].weight = p->k_weight;
  }
  a->rows = p->rows;
  a->dim = p->dim;
  a->pairs = pairs;
  a->positions = p->positions;
  a->position_row = p->position_row;
  a->position_axis = p->position_axis;
  a->frequencies = p->frequencies;
  a->weight_bf16 = p->weight_dtype == RMN_BF16;
  a->eps = p->eps;
  return RMN_OK;
}

// The most pairs that a load may hold: 16 bytes, or half, a quarter ... of them where sizes, strides or pointers ask for that.
int pairs_a_load(const RotaryArgs& a, int elem, bool next) {
  auto fits = [&](int v) {
    if (next ? a.dim / 2 % v : a.pairs % v || (a.dim / 2 - a.pairs) % v) return false;
    for (const Heads& p : a.part) {
      if (!p.heads) continue;
      if (p.heads > 1 && (p.head % v || (p.grad && p.grad_head % v))) return false;
      if (a.rows > 1 && (p.row % v || (p.grad && p.grad_row % v))) return false;
      if ((uintptr_t)p.x % (v * elem) || (uintptr_t)p.grad % (v * elem) || (uintptr_t)p.out % (v * elem)) return false;
    }
    return true;
  };
  int v = 16 / elem;
  while (v > 1 && !fits(v)) v /= 2;
  return v;
}

// Lanes of a head, groups of a row: as many as the heads allow until the groups of all rows are 8 warps for every SM.
void lay_out(RotaryArgs* a, int V, int units_a_lane) {
  const int units = a->dim / 2 / V, heads = a->part[0].heads + a->part[1].heads;
  a->lanes = 1;
  while (a->lanes * units_a_lane < units) a->lanes *= 2;
  a->per_row = 1;
  while (a->per_row < heads && a->per_row * a->lanes < kThreads &&
         (uint64_t)a->rows * a->per_row * a->lanes < (uint64_t)148 * kThreads)
    a->per_row *= 2;
}
uint32_t blocks_of(const RotaryArgs& a, uint32_t most) {
  const uint64_t threads = (uint64_t)a.rows * a.per_row * a.lanes;
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>((threads + kThreads - 1) / kThreads, most));
}

template <typename T, int V, int NU>
int launch(RotaryArgs& a, bool next, bool norm, bool backward, cudaStream_t stream, uint32_t* blocks) {
  lay_out(&a, V, NU);
  *blocks = blocks_of(a, backward ? kMostBackwardBlocks : 148 * 16);
  void (*kern)(RotaryArgs);
  if (backward) kern = next ? k_rotary_backward<T, V, NU, true> : k_rotary_backward<T, V, NU, false>;
  else if (norm) kern = next ? k_rotary<T, V, NU, true, true> : k_rotary<T, V, NU, false, true>;
  else kern = next ? k_rotary<T, V, NU, true, false> : k_rotary<T, V, NU, false, false>;
  RMN_CUDA_TRY(launch_overlapped(kern, dim3(*blocks), dim3(kThreads), 0, stream, a));
  RMN_LAUNCH_CHECK();
  return RMN_OK;
}
int run(RotaryArgs& a, int dtype, bool next, bool norm, bool backward, cudaStream_t stream, uint32_t* blocks) {
  const int v = pairs_a_load(a, dtype == RMN_F32 ? 4 : 2, next);
  if (dtype == RMN_F32)
    return v == 4   ? launch<float, 4, 1>(a, next, norm, backward, stream, blocks)
           : v == 2 ? launch<float, 2, 2>(a, next, norm, backward, stream, blocks)
                    : launch<float, 1, 4>(a, next, norm, backward, stream, blocks);
  using B = __nv_bfloat16;
  return v == 8   ? launch<B, 8, 1>(a, next, norm, backward, stream, blocks)
         : v == 4 ? launch<B, 4, 1>(a, next, norm, backward, stream, blocks)
         : v == 2 ? launch<B, 2, 2>(a, next, norm, backward, stream, blocks)
                  : launch<B, 1, 4>(a, next, norm, backward, stream, blocks);
}

}  // namespace
}  // namespace rmn

using namespace rmn;

extern "C" int rmn_rotary_forward(const rmn_rotary* problem, void* d_q_out, void* d_k_out, void* stream_) {
  RotaryArgs a;
  const int st = arguments(problem, &a);
  if (st != RMN_OK) return st;
  if (a.rows == 0) return RMN_OK;
  if (!d_q_out || (problem->kv_heads && !d_k_out)) return RMN_ERR_BAD_ARG;
  a.part[0].out = d_q_out;
  a.part[1].out = d_k_out;
  uint32_t blocks;
  return run(a, problem->dtype, problem->interleaved != 0, problem->norm != 0, false, (cudaStream_t)stream_, &blocks);
}

extern "C" size_t rmn_rotary_backward_workspace_bytes(const rmn_rotary* problem) {
  return problem && problem->norm && problem->dim > 0 ? (size_t)kMostBackwardBlocks * 2 * (size_t)problem->dim * sizeof(float) : 0;
}

extern "C" int rmn_rotary_backward(const rmn_rotary* problem, const void* d_grad_q, int64_t grad_q_row, int64_t grad_q_head,
                                   const void* d_grad_k, int64_t grad_k_row, int64_t grad_k_head, void* d_dq, void* d_dk,
                                   void* d_dq_weight, void* d_dk_weight, void* d_workspace, size_t workspace_bytes, void* stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  rmn_rotary plain;
  const bool norm = problem && problem->norm;
  if (problem && !norm) {  // the gradients are what is turned (back): x itself is not looked at
    plain = *problem;
    plain.q = d_grad_q; plain.q_row = grad_q_row; plain.q_head = grad_q_head;
    plain.k = d_grad_k; plain.k_row = grad_k_row; plain.k_head = grad_k_head;
    if (d_dq_weight || d_dk_weight) return RMN_ERR_BAD_ARG;
  }
  RotaryArgs a;
  const int st = arguments(problem && !norm ? &plain : problem, &a);
  if (st != RMN_OK) return st;
  const int64_t strides[] = {grad_q_row, grad_q_head, grad_k_row, grad_k_head};
  for (int64_t s : strides)
    if (!stride_ok(s)) return RMN_ERR_BAD_ARG;
  const bool sums = d_dq_weight || d_dk_weight, keys = problem->kv_heads != 0;
  if (d_dk_weight && !keys) return RMN_ERR_BAD_ARG;
  if (a.rows && (!d_grad_q || !d_dq || (keys && (!d_grad_k || !d_dk)))) return RMN_ERR_BAD_ARG;
  if (sums && (!d_workspace || ((uintptr_t)d_workspace & 15))) return RMN_ERR_BAD_ARG;
  if (sums && workspace_bytes < rmn_rotary_backward_workspace_bytes(problem)) return RMN_ERR_ALLOC;
  a.part[0].out = d_dq;
  a.part[1].out = d_dk;
  a.back = 1;
  uint32_t blocks = 0;
  if (a.rows && !norm) return run(a, problem->dtype, problem->interleaved != 0, false, false, stream, &blocks);
  if (a.rows) {
    a.part[0].grad = d_grad_q; a.part[0].grad_row = grad_q_row; a.part[0].grad_head = grad_q_head;
    a.part[1].grad = d_grad_k; a.part[1].grad_row = grad_k_row; a.part[1].grad_head = grad_k_head;
    a.sums = sums ? static_cast<float*>(d_workspace) : nullptr;
    const int launched = run(a, problem->dtype, problem->interleaved != 0, true, true, stream, &blocks);
    if (launched != RMN_OK) return launched;
  }
  if (!sums) return RMN_OK;
  RMN_CUDA_TRY(launch_overlapped(k_rotary_sums, dim3((uint32_t)(2 * a.dim + 31) / 32), dim3(1024), 0, stream,
                                 static_cast<const float*>(d_workspace), blocks, a.dim, a.weight_bf16, d_dq_weight, d_dk_weight));
  RMN_LAUNCH_CHECK();
  return RMN_OK;
}
