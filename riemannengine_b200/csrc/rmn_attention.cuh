// What the attention kernels share: the arguments as the kernels take them, the samples' row ranges, and the search of the
// tile of rows that a block works on.
#pragma once

#include "rmn_common.cuh"

#include <cuda_bf16.h>

namespace rmn {

// One attention problem, as rmn_attention describes it, with what backward passes add.
struct AttnArgs {
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  uint32_t rows_q, rows_k, sequences;
  int heads, kv_heads, dim;
  const int32_t *offsets, *kv_offsets, *kv_lengths;     // kv_offsets never NULL here
  int causal;
  float scale;                                          // of the scores
  uint32_t* status;                                     // device status word
  void* out;                                            // [rows_q, heads, dim]
  void* low;                                            // what rounding took from out (bf16; may be NULL)
  float* lse;                                           // [heads, rows_q], natural logarithm (forward: may be NULL)
  // backward
  const void* grad;                                     // of the output
  int64_t grad_row, grad_head;
  const void* fwd_out;
  float* delta;                                         // [heads, rows_q]: sum over the channels of grad * out
  void *dq, *dk, *dv;                                   // contiguous
};

// Row ranges of one sample. Every row of the tensors belongs to exactly one segment: segments 0 ... S - 1 are the samples,
// segment S the rows behind the last sample and S + 1 those before the first; the last two have no keys to attend to, so that
// their outputs come out as zeros by the same code.
struct Segment {
  int32_t q0, n_q;    // query rows
  int32_t k0, n_k;    // key rows in use
  int32_t k_slot;     // key rows from k0 to the next sample's
};

__device__ __forceinline__ int32_t clamp_row(int32_t v, uint32_t rows) { return max(0, min(v, (int32_t)rows)); }

// Offsets that do not ascend or leave the tensor are set right here, so that no row outside the tensors is touched whatever
// they say, and recorded in the status word. descends: set where a sample's rows would lie before those of the one before it.
__device__ __forceinline__ Segment segment(const AttnArgs& a, uint32_t s, bool* descends = nullptr) {
  Segment g;
  const uint32_t S = a.sequences;
  if (s > S) {
    g.q0 = 0;
    g.n_q = clamp_row(a.offsets[0], a.rows_q);
    g.k0 = 0;
    g.k_slot = clamp_row(a.kv_offsets[0], a.rows_k);
    g.n_k = 0;
    return g;
  }
  const int32_t q_lo = a.offsets[s], k_lo = a.kv_offsets[s];
  const int32_t q_hi = s < S ? a.offsets[s + 1] : (int32_t)a.rows_q, k_hi = s < S ? a.kv_offsets[s + 1] : (int32_t)a.rows_k;
  g.q0 = clamp_row(q_lo, a.rows_q);
  g.k0 = clamp_row(k_lo, a.rows_k);
  g.n_q = clamp_row(q_hi, a.rows_q) - g.q0;
  g.k_slot = clamp_row(k_hi, a.rows_k) - g.k0;
  if (descends) *descends = *descends || g.n_q < 0 || g.k_slot < 0;
  g.n_q = max(0, g.n_q);
  g.k_slot = max(0, g.k_slot);
  bool bad = q_lo < 0 || q_hi < q_lo || q_hi > (int32_t)a.rows_q || k_lo < 0 || k_hi < k_lo || k_hi > (int32_t)a.rows_k;
  g.n_k = s < S ? g.k_slot : 0;
  if (s < S && a.kv_lengths) {
    const int32_t len = a.kv_lengths[s];
    bad = bad || len < 0 || len > g.k_slot;
    g.n_k = max(0, min(len, g.k_slot));
  }
  if (bad) atomicMax(a.status, (uint32_t)RMN_ERR_BAD_ARG);
  return g;
}

// Keys that query row i of a segment attends to are 0 ... visible(i) - 1: all, or (causal, aligned at the end) those up to
// its own place.
__device__ __forceinline__ int32_t visible_keys(const Segment& g, int32_t i, int causal) {
  return causal ? max(0, min(g.n_k, i + 1 - (g.n_q - g.n_k))) : g.n_k;
}
// The first query row that attends to key j.
__device__ __forceinline__ int32_t first_query(const Segment& g, int32_t j, int causal) {
  return causal ? max(0, j - (g.n_k - g.n_q)) : 0;
}

__device__ __forceinline__ int32_t tiles_of(int32_t rows, int tile_rows) {
  return (int32_t)(((uint32_t)rows + (uint32_t)tile_rows - 1) / (uint32_t)tile_rows);
}

// The tile of `tile_rows` rows that a block works on: of query rows, or of key rows (whole slots, in use or not).
enum class TilesOf { kQueries, kSlots };
struct FoundTile {
  Segment g;
  int32_t tile, tiles;  // number of the tile in its segment, and the segment's tiles
};
template <TilesOf kOf>
__device__ __forceinline__ int32_t segment_tiles(const Segment& g, int tile_rows) {
  return tiles_of(kOf == TilesOf::kQueries ? g.n_q : g.k_slot, tile_rows);
}
// Sums stop at the largest number: offsets that descend may give a row to many samples.
__device__ __forceinline__ int32_t add_tiles(int32_t a, int32_t b) { return (int32_t)min((uint32_t)a + (uint32_t)b, 0x7fffffffu); }
// The inclusive sum of the threads before (`first`) and of all (`all`), for all kThreads threads of a block; `any`: of a flag.
template <int kThreads>
__device__ __forceinline__ void scan_block(int32_t mine, int32_t* warp_sums, int32_t& first, int32_t& all, bool& any) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto = add_tiles(upto, v);
  }
  if (lane == 31) warp_sums[warp] = upto;
  any = __syncthreads_or(any);
  first = __shfl_up_sync(0xffffffffu, upto, 1);
  if (lane == 0) first = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) first = add_tiles(first, warp_sums[w]);
    all = add_tiles(all, warp_sums[w]);
  }
}

// Up to kCountedSamples samples: every thread counts the tiles of a run of segments, a scan over the block places them, and the
// numbers behind the last tile are of no tile. Beyond, counting would cost the square of the samples: segment j in the order of the
// rows (those before the first sample, the samples, those behind) begins at row b(j) and has the numbers from b(j) / tile_rows + j
// on, as many as it has tiles or one more, which is of no tile; every warp searches for its number, 32 places at a time. Numbers
// without a tile cost a block each, and the search leaves them among the others. 8 heads of 64, backward, with counts and with the
// search: 128 samples of 96 rows 81 and 94 us; 256, 512, 1024, 4096 samples of 64 rows 115 and 122, 240 and 238, 523 and 476,
// 3650 and 1885.
constexpr uint32_t kCountedSamples = 384;
template <int kThreads, TilesOf kOf>
__device__ __forceinline__ bool find_tile(const AttnArgs& a, uint32_t want, int tile_rows, FoundTile* found, int32_t* warp_sums) {
  const uint32_t n = a.sequences + 2;
  if (a.sequences <= kCountedSamples) {
    const uint32_t per = (n + kThreads - 1) / kThreads;
    const uint32_t lo = min(threadIdx.x * per, n), hi = min(lo + per, n);
    int32_t mine = 0, first, all;
    Segment g = {};
    for (uint32_t s = lo; s < hi; ++s) {
      g = segment(a, s);
      mine = add_tiles(mine, segment_tiles<kOf>(g, tile_rows));
    }
    bool unused = false;
    scan_block<kThreads>(mine, warp_sums, first, all, unused);
    if (want >= (uint32_t)all) return false;
    if ((int32_t)want >= first && (int32_t)want - first < mine) {
      for (uint32_t s = lo; s < hi; ++s) {
        if (hi - lo > 1) g = segment(a, s);
        const int32_t tiles = segment_tiles<kOf>(g, tile_rows);
        if ((int32_t)want - first < tiles) {
          *found = {g, (int32_t)want - first, tiles};
          break;
        }
        first += tiles;
      }
    }
  } else {
    const int32_t* at = kOf == TilesOf::kQueries ? a.offsets : a.kv_offsets;
    const uint32_t rows = kOf == TilesOf::kQueries ? a.rows_q : a.rows_k, lane = threadIdx.x & 31;
    if (want < n && threadIdx.x == 0) segment(a, want);  // every segment is looked at: the search may step over some that are wrong
    auto number = [&](uint32_t j) { return j == 0 ? 0u : (uint32_t)clamp_row(__ldg(at + j - 1), rows) / (uint32_t)tile_rows + j; };
    uint32_t lo = 0, len = n;  // number(lo) <= want
    while (len > 1) {
      const uint32_t step = (len + 31) / 32, p = lane * step;
      const uint32_t below = __ballot_sync(0xffffffffu, p < len && number(lo + p) <= want);
      const uint32_t skip = (31 - __clz((int)(below | 1u))) * step;
      lo += skip;
      len = min(step, len - skip);
    }
    const Segment g = segment(a, lo == 0 ? a.sequences + 1 : lo - 1);
    const int32_t tiles = segment_tiles<kOf>(g, tile_rows), tile = (int32_t)(want - number(lo));
    if (tile < 0 || tile >= tiles) return false;
    if (threadIdx.x == 0) *found = {g, tile, tiles};
  }
  __syncthreads();
  return true;
}
// How many tile numbers there are at most.
inline uint64_t most_tiles(uint64_t rows, uint64_t sequences, uint32_t tile_rows) { return rows / tile_rows + sequences + 2; }

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// 16 bytes at this address of another block's shared memory
__device__ __forceinline__ float4 load_of_block(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}

// the number at this place of another block's shared memory
__device__ __forceinline__ float float_of_block(const float* p, uint32_t rank) {
  float v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
      : "=f"(v)
      : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank)
      : "memory");
  return v;
}

// The kernels behind rmn_attention_*: RMN_ERR_UNSUPPORTED where they do not cover the call.
int attention_simt_forward(const AttnArgs& a, int dtype, cudaStream_t stream);
int attention_simt_backward(const AttnArgs& a, int dtype, cudaStream_t stream);
int attention_tc_forward(const AttnArgs& a, cudaStream_t stream);  // bf16
int attention_tc_backward(const AttnArgs& a, cudaStream_t stream);
// few query rows a sample: chunks of the keys, then their sum. Scratch bytes, 0 where this form is not meant for the sizes
size_t attention_rows_workspace(uint32_t rows_q, uint32_t rows_k, uint32_t sequences, int heads, int kv_heads, int dim, int dtype);
int attention_rows_forward(const AttnArgs& a, int dtype, void* workspace, cudaStream_t stream);

}  // namespace rmn
