// C-ABI entry points of attention within packed samples: argument checks and the choice of the kernel; and the row ranges of
// the samples of a coordinate map.
#include "rmn_attention.cuh"

#include <algorithm>

namespace rmn {

const uint32_t* tc_status_device_address();  // defined in rmn_conv_tc.cu

namespace {

// Runs of equal batch indices: every block counts those that begin in its share of the rows, then places them behind the counts of
// the blocks before it. The rows are read twice, whatever the number of runs.
constexpr int kRunBlocks = 148 * 4, kRunThreads = 256;

__device__ __forceinline__ bool begins_run(const int32_t* __restrict__ coords, uint32_t i, int W) {
  return i == 0 || __ldg(coords + (size_t)i * W) != __ldg(coords + (size_t)(i - 1) * W);
}
__device__ __forceinline__ uint32_t share_of(uint32_t n, uint32_t block) { return (uint32_t)((uint64_t)n * block / kRunBlocks); }

__global__ void __launch_bounds__(kRunThreads) k_count_runs(const int32_t* __restrict__ coords, uint32_t n, int W,
                                                            uint32_t* __restrict__ counts) {
  after_previous_kernel();
  const uint32_t end = share_of(n, blockIdx.x + 1);
  uint32_t mine = 0;
  for (uint32_t first = share_of(n, blockIdx.x); first < end; first += kRunThreads) {
    const uint32_t i = first + threadIdx.x;
    mine += (uint32_t)__syncthreads_count(i < end && begins_run(coords, i, W));
  }
  if (threadIdx.x == 0) counts[blockIdx.x] = mine;
}
// offsets = the first row of every run (`most` of them: n behind the last), n, the number of runs
__global__ void __launch_bounds__(kRunThreads) k_sample_offsets(const int32_t* __restrict__ coords, uint32_t n, int W, uint32_t most,
                                                                const uint32_t* __restrict__ counts, int32_t* __restrict__ offsets) {
  constexpr int kWarps = kRunThreads / 32;
  __shared__ uint32_t s_before[kWarps], s_all[kWarps], s_warp[2][kWarps];
  after_previous_kernel();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t before = 0, all = 0;
  for (uint32_t b = threadIdx.x; b < kRunBlocks; b += kRunThreads) {
    const uint32_t c = counts[b];
    all += c;
    if (b < blockIdx.x) before += c;
  }
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if (lane == 0) {
    s_before[warp] = before;
    s_all[warp] = all;
  }
  __syncthreads();
  before = all = 0;
  for (int w = 0; w < kWarps; ++w) {
    before += s_before[w];
    all += s_all[w];
  }
  const uint32_t end = share_of(n, blockIdx.x + 1);
  uint32_t turn = 0;
  for (uint32_t first = share_of(n, blockIdx.x); first < end; first += kRunThreads, turn ^= 1u) {
    const uint32_t i = first + threadIdx.x;
    const bool begins = i < end && begins_run(coords, i, W);
    const uint32_t votes = __ballot_sync(0xffffffffu, begins);
    if (lane == 0) s_warp[turn][warp] = (uint32_t)__popc(votes);
    __syncthreads();
    uint32_t at = before + (uint32_t)__popc(votes & ((1u << lane) - 1u));
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) at += s_warp[turn][w];
      before += s_warp[turn][w];
    }
    if (begins && at < most) offsets[at] = (int32_t)i;
  }
  for (uint64_t i = (uint64_t)all + blockIdx.x * kRunThreads + threadIdx.x; i < most; i += kRunBlocks * kRunThreads)
    offsets[i] = (int32_t)n;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    offsets[most] = (int32_t)n;
    offsets[most + 1] = (int32_t)min(all, 0x7fffffffu);
  }
}

bool stride_ok(int64_t s) { return s >= 0 && s <= (int64_t(1) << 40); }

// the problem as the kernels take it; RMN_OK or what is wrong with it
int arguments(const rmn_attention* p, AttnArgs* a) {
  if (!p) return RMN_ERR_BAD_ARG;
  if (p->heads < 1 || p->kv_heads < 1 || p->heads > 65536 || p->heads % p->kv_heads || p->dim < 1 ||
      (p->dtype != RMN_F32 && p->dtype != RMN_BF16) || p->rows_q > 0x7fffffffu || p->rows_k > 0x7fffffffu ||
      p->sequences > 0x7ffffffdu || !p->offsets)
    return RMN_ERR_BAD_ARG;
  if (p->dim > 256) return RMN_ERR_UNSUPPORTED;
  const int64_t strides[6] = {p->q_row, p->q_head, p->k_row, p->k_head, p->v_row, p->v_head};
  for (int64_t s : strides)
    if (!stride_ok(s)) return RMN_ERR_BAD_ARG;
  if ((p->rows_q && !p->q) || (p->rows_k && (!p->k || !p->v))) return RMN_ERR_BAD_ARG;
  if (!p->kv_offsets && p->rows_k != p->rows_q) return RMN_ERR_BAD_ARG;
  if (!(p->scale == p->scale)) return RMN_ERR_BAD_ARG;
  *a = {};
  a->q = p->q; a->k = p->k; a->v = p->v;
  a->q_row = p->q_row; a->q_head = p->q_head;
  a->k_row = p->k_row; a->k_head = p->k_head;
  a->v_row = p->v_row; a->v_head = p->v_head;
  a->rows_q = p->rows_q; a->rows_k = p->rows_k; a->sequences = p->sequences;
  a->heads = p->heads; a->kv_heads = p->kv_heads; a->dim = p->dim;
  a->offsets = p->offsets;
  a->kv_offsets = p->kv_offsets ? p->kv_offsets : p->offsets;
  a->kv_lengths = p->kv_lengths;
  a->causal = p->causal != 0;
  a->scale = p->scale;
  return RMN_OK;
}
int find_status(AttnArgs* a) {
  a->status = const_cast<uint32_t*>(tc_status_device_address());
  return a->status ? RMN_OK : RMN_ERR_CUDA;
}


// dK and dV of the sinks of the samples that are cut: the sums of their chunks' parts, in order.
constexpr int kSumThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kSumThreads) k_attention_sinks_sum(const AttnArgs a) {
  __shared__ FoundTile found;
  __shared__ int32_t warp_sums[kSumThreads / 32];
  after_previous_kernel();
  const int kv = blockIdx.x % a.kv_heads;
  if (!find_tile<kSumThreads, TilesOf::kLongQueries>(a, blockIdx.x / a.kv_heads, a.sink_chunk, &found, warp_sums)) return;
  const Segment g = found.g;
  // each of a sample's chunks has a block, which sums a share of its sinks' channels
  const int64_t sinks = min(a.sinks, g.n_k), n = 2 * sinks * a.dim;
  for (int64_t i = (int64_t)found.tile * kSumThreads + threadIdx.x; i < n; i += (int64_t)found.tiles * kSumThreads) {
    const int which = i >= sinks * a.dim;
    const int64_t at = i - which * sinks * a.dim;  // of the sinks' channels
    float sum = 0.f;
#pragma unroll 4
    for (int c = 0; c < found.tiles; ++c) sum += __ldg(a.sink_parts + sink_part(a, g.q0, c, kv) + (int64_t)which * a.sink_most * a.dim + at);
    const int64_t key = at / a.dim, to = ((g.k0 + key) * a.kv_heads + kv) * a.dim + at % a.dim;
    if (!which) sum *= a.scale;
    void* out = which ? a.dv : a.dk;
    if constexpr (sizeof(T) == 4) static_cast<float*>(out)[to] = sum;
    else static_cast<__nv_bfloat16*>(out)[to] = __float2bfloat16_rn(sum);
  }
}

}  // namespace

int attention_sinks_sum(const AttnArgs& a, int dtype, cudaStream_t stream) {
  const uint64_t blocks = (uint64_t)a.sink_chunks * a.kv_heads;
  if (blocks > 0x7fffffffull) return RMN_ERR_UNSUPPORTED;
  RMN_CUDA_TRY(launch_overlapped(dtype == RMN_F32 ? k_attention_sinks_sum<float> : k_attention_sinks_sum<__nv_bfloat16>, dim3((uint32_t)blocks),
                                 dim3(kSumThreads), 0, stream, a));
  RMN_LAUNCH_CHECK();
  return RMN_OK;
}

}  // namespace rmn

using namespace rmn;

extern "C" size_t rmn_sample_offsets_workspace_bytes(uint32_t) { return kRunBlocks * sizeof(uint32_t); }

extern "C" int rmn_sample_offsets(const int32_t* d_coords, uint32_t n_rows, int W, uint32_t n_samples, int32_t* d_offsets,
                                  void* d_workspace, size_t workspace_bytes, void* stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  if (W < 2 || W > RMN_MAX_W || n_rows > 0x7fffffffu || n_samples > 0x7ffffff0u || !d_offsets || !d_workspace ||
      (n_rows && !d_coords) || ((uintptr_t)d_workspace & 3))
    return RMN_ERR_BAD_ARG;
  if (workspace_bytes < rmn_sample_offsets_workspace_bytes(n_samples)) return RMN_ERR_ALLOC;
  uint32_t* counts = static_cast<uint32_t*>(d_workspace);
  RMN_CUDA_TRY(launch_overlapped(k_count_runs, dim3(kRunBlocks), dim3(kRunThreads), 0, stream, d_coords, n_rows, W, counts));
  RMN_LAUNCH_CHECK();
  RMN_CUDA_TRY(launch_overlapped(k_sample_offsets, dim3(kRunBlocks), dim3(kRunThreads), 0, stream, d_coords, n_rows, W, n_samples,
                                 static_cast<const uint32_t*>(counts), d_offsets));
  RMN_LAUNCH_CHECK();
  return RMN_OK;
}

namespace {
constexpr int32_t kMostSinks = 1 << 30;
bool window_ok(int32_t window, int32_t sinks) { return window >= 1 && sinks >= 0 && sinks < kMostSinks; }

// window 0: none
size_t forward_workspace(const rmn_attention* p, int32_t window, int32_t sinks) {
  if (!p || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads || p->dim < 1) return 0;
  return attention_rows_workspace(p->rows_q, p->rows_k, p->sequences, p->heads, p->kv_heads, p->dim, p->dtype, p->causal, window, sinks);
}
int forward(const rmn_attention* problem, int32_t window, int32_t sinks, void* d_out, void* d_low, float* d_lse, void* d_workspace,
            size_t workspace_bytes, cudaStream_t stream) {
  AttnArgs a;
  const int st = arguments(problem, &a);
  if (st != RMN_OK) return st;
  if (a.rows_q == 0) return RMN_OK;
  const size_t need = forward_workspace(problem, window, sinks);
  if (!d_out || (need && (!d_workspace || ((uintptr_t)d_workspace & 15)))) return RMN_ERR_BAD_ARG;
  if (workspace_bytes < need) return RMN_ERR_ALLOC;
  const int found = find_status(&a);
  if (found != RMN_OK) return found;
  a.window = window;
  a.sinks = sinks;
  a.out = d_out;
  a.low = problem->dtype == RMN_BF16 ? d_low : nullptr;
  a.lse = d_lse;
  if (need) {
    const int rows = attention_rows_forward(a, problem->dtype, d_workspace, stream);
    if (rows != RMN_ERR_UNSUPPORTED) return rows;
  }
  if (problem->dtype == RMN_BF16) {
    const int tc = attention_tc_forward(a, stream);
    if (tc != RMN_ERR_UNSUPPORTED) return tc;
  }
  return attention_simt_forward(a, problem->dtype, stream);
}

// delta, and behind it the sinks' parts
size_t delta_bytes(const rmn_attention* p) { return (size_t)p->heads * p->rows_q * sizeof(float); }
size_t parts_at(const rmn_attention* p) { return (delta_bytes(p) + 255) / 256 * 256; }
SinkPlan sinks_of(const rmn_attention* p, int32_t window, int32_t sinks) {
  return sink_plan(p->rows_q, p->rows_k, p->sequences, p->kv_heads, p->dim, p->causal, window, sinks);
}
size_t backward_workspace(const rmn_attention* p, int32_t window, int32_t sinks) {
  if (!p || p->heads < 1) return 0;
  if (!window || p->kv_heads < 1 || p->dim < 1) return delta_bytes(p);
  const SinkPlan plan = sinks_of(p, window, sinks);
  return plan.parts ? parts_at(p) + plan.parts * sizeof(float) : delta_bytes(p);
}
int backward(const rmn_attention* problem, int32_t window, int32_t sinks, const void* d_out, const void* d_low, const float* d_lse,
             const void* d_grad_out, int64_t grad_row, int64_t grad_head, void* d_dq, void* d_dk, void* d_dv, void* d_workspace,
             size_t workspace_bytes, cudaStream_t stream) {
  AttnArgs a;
  const int st = arguments(problem, &a);
  if (st != RMN_OK) return st;
  if ((a.rows_q && !d_dq) || (a.rows_k && (!d_dk || !d_dv)) || !stride_ok(grad_row) || !stride_ok(grad_head))
    return RMN_ERR_BAD_ARG;
  const size_t elem = problem->dtype == RMN_F32 ? 4 : 2;
  if (a.rows_q == 0 || a.rows_k == 0) {  // nothing attends to anything
    if (a.rows_q) RMN_CUDA_TRY(cudaMemsetAsync(d_dq, 0, (size_t)a.rows_q * a.heads * a.dim * elem, stream));
    if (a.rows_k) {
      RMN_CUDA_TRY(cudaMemsetAsync(d_dk, 0, (size_t)a.rows_k * a.kv_heads * a.dim * elem, stream));
      RMN_CUDA_TRY(cudaMemsetAsync(d_dv, 0, (size_t)a.rows_k * a.kv_heads * a.dim * elem, stream));
    }
    return RMN_OK;
  }
  if (!d_out || !d_lse || !d_grad_out || !d_workspace || ((uintptr_t)d_workspace & 15)) return RMN_ERR_BAD_ARG;
  if (workspace_bytes < backward_workspace(problem, window, sinks)) return RMN_ERR_ALLOC;
  const int found = find_status(&a);
  if (found != RMN_OK) return found;
  a.window = window;
  a.sinks = sinks;
  a.fwd_out = d_out;
  a.low = problem->dtype == RMN_BF16 ? const_cast<void*>(d_low) : nullptr;
  a.lse = const_cast<float*>(d_lse);
  a.grad = d_grad_out;
  a.grad_row = grad_row;
  a.grad_head = grad_head;
  a.delta = static_cast<float*>(d_workspace);
  const SinkPlan plan = sinks_of(problem, window, sinks);
  a.sink_chunk = plan.chunk;
  a.sink_most = plan.most;
  a.sink_chunks = (int32_t)std::min<int64_t>(plan.chunks, 0x7fffffff);
  a.sink_parts = plan.parts ? reinterpret_cast<float*>(static_cast<char*>(d_workspace) + parts_at(problem)) : nullptr;
  a.dq = d_dq; a.dk = d_dk; a.dv = d_dv;
  int done = problem->dtype == RMN_BF16 ? attention_tc_backward(a, stream) : RMN_ERR_UNSUPPORTED;
  if (done == RMN_ERR_UNSUPPORTED) done = attention_simt_backward(a, problem->dtype, stream);
  return done == RMN_OK && a.sink_chunk ? attention_sinks_sum(a, problem->dtype, stream) : done;
}
}  // namespace

extern "C" size_t rmn_attention_forward_workspace_bytes(const rmn_attention* problem) { return forward_workspace(problem, 0, 0); }

extern "C" int rmn_attention_forward(const rmn_attention* problem, void* d_out, void* d_low, float* d_lse, void* d_workspace,
                                     size_t workspace_bytes, void* stream) {
  return forward(problem, 0, 0, d_out, d_low, d_lse, d_workspace, workspace_bytes, (cudaStream_t)stream);
}

extern "C" size_t rmn_attention_backward_workspace_bytes(const rmn_attention* problem) { return backward_workspace(problem, 0, 0); }

extern "C" int rmn_attention_backward(const rmn_attention* problem, const void* d_out, const void* d_low, const float* d_lse,
                                      const void* d_grad_out, int64_t grad_row, int64_t grad_head, void* d_dq, void* d_dk,
                                      void* d_dv, void* d_workspace, size_t workspace_bytes, void* stream) {
  return backward(problem, 0, 0, d_out, d_low, d_lse, d_grad_out, grad_row, grad_head, d_dq, d_dk, d_dv, d_workspace, workspace_bytes,
                  (cudaStream_t)stream);
}

extern "C" size_t rmn_window_attention_forward_workspace_bytes(const rmn_attention* problem, int32_t window, int32_t sinks) {
  return window_ok(window, sinks) ? forward_workspace(problem, window, sinks) : 0;
}

extern "C" int rmn_window_attention_forward(const rmn_attention* problem, int32_t window, int32_t sinks, void* d_out, void* d_low,
                                            float* d_lse, void* d_workspace, size_t workspace_bytes, void* stream) {
  if (!window_ok(window, sinks)) return RMN_ERR_BAD_ARG;
  return forward(problem, window, sinks, d_out, d_low, d_lse, d_workspace, workspace_bytes, (cudaStream_t)stream);
}

extern "C" size_t rmn_window_attention_backward_workspace_bytes(const rmn_attention* problem, int32_t window, int32_t sinks) {
  return window_ok(window, sinks) ? backward_workspace(problem, window, sinks) : 0;
}

extern "C" int rmn_window_attention_backward(const rmn_attention* problem, int32_t window, int32_t sinks, const void* d_out,
                                             const void* d_low, const float* d_lse, const void* d_grad_out, int64_t grad_row,
                                             int64_t grad_head, void* d_dq, void* d_dk, void* d_dv, void* d_workspace,
                                             size_t workspace_bytes, void* stream) {
  if (!window_ok(window, sinks)) return RMN_ERR_BAD_ARG;
  return backward(problem, window, sinks, d_out, d_low, d_lse, d_grad_out, grad_row, grad_head, d_dq, d_dk, d_dv, d_workspace,
                  workspace_bytes, (cudaStream_t)stream);
}
