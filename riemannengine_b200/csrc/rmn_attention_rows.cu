// Attention of few query rows a sample against long keys (a token at a time): forward pass, fp32 and bf16, head sizes up to 128.
//
// Bound by memory: the keys and values are read once, whatever the number of heads that share them. All keys in use, in tiles of 64,
// are dealt out evenly to as many blocks as fit the GPU, so that samples of very different lengths keep all of it busy to the end;
// neighbouring blocks take the same tiles of neighbouring key heads (whose rows are neighbours in memory). A block walks through its
// run of tiles, which is a piece of one sample or of several, with all query rows and heads that go with them, up to 16 of them at
// a time as the rows of warp-wide matrix products (their rate does not bound here: 16 rows cost one product for 8 keys). Bulk copies bring a tile's keys and values into a ring in shared memory, some 100 KB in
// flight for a block, across the borders of pieces; each of four warps takes 16 of the 64 keys and has a
// running maximum and sum of its own. The warps are joined in shared memory, and the pieces of a sample that several blocks
// share by a second kernel, in a fixed order. 16 samples of 509 ... 30011 keys, 16 query and 4 key heads of 128 (336 MB in bf16):
// 62 us, 5.4 TB/s, and 8 us for the second kernel; in fp32 163 us for both, where the three products of every operand take longer
// than its bytes.
//
// Keys and values go from shared memory to registers as 16-byte loads that are product operands as they stand: which of a row's
// channels is which k of a product is free as long as q has the same order, and which channel is which column of the output is free
// as long as the store undoes it. In bf16 a thread's 8 adjacent channels of a key are its operands of two products; of the values
// it has 8 channels of the four keys whose weights it holds, paired by a byte permutation. In fp32 every operand is the sum of two
// tf32 numbers (its leading 11 bits and the next 11), and a product is three: high high + high low + low high, an error of 2^-22.
#include "rmn_attention_tc.cuh"

#include <math_constants.h>

#include <algorithm>
#include <cmath>

namespace rmn {
namespace {

using namespace tc;

constexpr int kSumWarps = 8, kSumThreads = kSumWarps * 32;
constexpr int kTileKeys = 64;
constexpr int kMostRows = 32;    // of a sample and a key head (queries times heads): on average, and for the sum of pieces
constexpr float kRescale = 8.f;  // log2 of how far a row's maximum may rise before the output is scaled

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = high + low + what is below 2^-22 of it
__device__ __forceinline__ void split_tf32(float x, uint32_t& high, uint32_t& low) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(high) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(low) : "f"(x - __uint_as_float(high)));
}
// d += a b of numbers in two parts
__device__ __forceinline__ void mma_split(float (&d)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], float b0, float b1) {
  uint32_t h0, l0, h1, l1;
  split_tf32(b0, h0, l0);
  split_tf32(b1, h1, l1);
  mma_tf32(d, al, h0, h1);
  mma_tf32(d, ah, l0, l1);
  mma_tf32(d, ah, h0, h1);
}
__device__ __forceinline__ uint4 load16(const void* p, bool ok) {
  return ok ? __ldg(static_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
}

// The ring: a slot is 64 rows of keys and 64 of values, each as columns of 128-byte swizzled lines.
template <typename T, int DP>
struct RowsShape {
  // with keys of their own, 16 of every tile: a warp waits for all phases of a slot's barrier. (Two fours of warps that took turns at the
  // tiles of a ring of three slots waited for every second phase of each; the parity of the one before lets such a wait pass early.)
  static constexpr int WARPS = 4;
  static constexpr int THREADS = WARPS * 32 + 32;                   // and one warp for the copies
  static constexpr int BLOCKS = sizeof(T) == 4 ? 1 : 2;             // an SM
  static constexpr int LINES = DP * (int)sizeof(T) / 128;           // of a row
  static constexpr uint32_t LINE = kTileKeys * 128, HALF = LINES * LINE, SLOT = 2 * HALF;
  static constexpr int SLOTS = SLOT >= 32 * 1024 ? 3 : 6;
  static constexpr uint32_t Q = SLOTS * SLOT;                       // fp32: q as operands
  static constexpr uint32_t JOIN = Q + (sizeof(T) == 4 ? DP / 8 * 1024 : 0);  // 16 rows of the output, fp32
  static constexpr uint32_t TAIL = JOIN + 16 * (DP + 4) * 4;
  static constexpr size_t SMEM = TAIL + 256 + 1024;
};

struct RowsWork {  // scratch, and how the keys are cut
  int blocks;           // of the first kernel, for each key head
  int most_queries;     // rows of a sample whose pieces are summed by the second kernel
  int32_t* starts;      // [blocks][3]: the sample that a block of the first head begins in, the tiles before that; all tiles
  float* sums;          // [piece][group * most_queries][2]: maximum (log 2), sum
  float* parts;         // [piece][group * most_queries][dim]: not yet divided by the sum
};
// Of `tiles` tiles, block b of a head takes those from first_of(b) to first_of(b + 1).
__device__ __forceinline__ int64_t first_of(const RowsWork& w, int64_t tiles, int64_t block) { return tiles * block / w.blocks; }
// The tile that a block begins with, by counts over all samples.
struct Begin {
  int32_t all;          // tiles; 0 where the samples' rows are out of order
  Segment g;            // of the tile, its sample, its number in it, the sample's tiles
  uint32_t s;
  int32_t tile, tiles;
};
// All threads of the block count: each a run of samples, a scan over the block places them.
template <int kThreads>
__device__ __forceinline__ void find_begin(const AttnArgs& a, const RowsWork& w, int block, Begin* found, int32_t* warp_sums, bool* in_order) {
  const uint32_t per = (a.sequences + kThreads - 1) / kThreads;
  const uint32_t lo = min(threadIdx.x * per, a.sequences), hi = min(lo + per, a.sequences);
  int32_t mine = 0;
  Segment g = {};
  bool descends = false;
  for (uint32_t s = lo; s < hi; ++s) {
    g = segment(a, s, &descends);
    mine = add_tiles(mine, tiles_of(g.n_k, kTileKeys));
  }
  int32_t first, all;
  scan_block<kThreads>(mine, warp_sums, first, all, descends);
  *in_order = !descends;
  const int32_t want = all ? (int32_t)first_of(w, all, block) : 0;
  if (*in_order && want >= first && want - first < mine) {
    for (uint32_t s = lo; s < hi; ++s) {
      if (hi - lo > 1) g = segment(a, s);
      const int32_t tiles = tiles_of(g.n_k, kTileKeys);
      if (want - first < tiles) {
        *found = {all, g, s, want - first, tiles};
        break;
      }
      first += tiles;
    }
  }
  if (threadIdx.x == 0 && (all == 0 || !*in_order)) found->all = 0;
  __syncthreads();
}
// The block whose run holds a tile.
__device__ __forceinline__ int32_t block_of(const RowsWork& w, int64_t tiles, int64_t tile) {
  return (int32_t)(((tile + 1) * w.blocks - 1) / tiles);
}
// Places of row r (of group * n_q) of a piece: of a block's run only the first piece and the last can be parts of a sample.
__device__ __forceinline__ size_t part_at(const AttnArgs& a, const RowsWork& w, int64_t block, int kv, bool first, int r) {
  const int64_t piece = 2 * ((int64_t)kv * w.blocks + block) + (first ? 0 : 1);
  return (size_t)piece * (a.heads / a.kv_heads * w.most_queries) + r;
}

// A run of tiles as pieces of samples: the same walk by the warp that copies and those that compute.
struct Piece {
  Segment g;
  uint32_t s;
  int32_t tile, tiles;  // the next tile of the sample, and its tiles
  int32_t left;         // tiles of the block's run from there on
  bool first;           // of the block's run
  // what belongs to this piece
  int32_t from, to;     // tiles of keys
  uint32_t row, step;   // the first of its rows, sixteen at a time, and how far the next sixteen are
  bool skip, split;

  // (all: the number of tiles)
  __device__ __forceinline__ void set(const RowsWork& w, int32_t all, int block) {
    from = tile;
    to = tile + min(tiles - tile, left);
    split = to - from < tiles;
    skip = g.n_q == 0;
    row = 0;
    step = 16;
    if (split && g.n_q > w.most_queries) {
      // no room for its pieces: the blocks that share its tiles walk over all of them, and take its rows in turn
      split = false;
      from = 0;
      to = tiles;
      if (all < w.blocks) {  // (a tile to a block then, and blocks without)
        row = 16 * (uint32_t)tile;
        step = 16 * (uint32_t)tiles;
      } else {
        const int64_t at = first_of(w, all, block + 1) - left - tile;  // its first tile
        const int32_t b = block_of(w, all, at);
        row = 16 * (uint32_t)(block - b);
        step = 16 * (uint32_t)(block_of(w, all, at + tiles - 1) - b + 1);
      }
    }
  }
  __device__ __forceinline__ bool next(const AttnArgs& a, const RowsWork& w, int32_t all, int block) {
    left -= min(tiles - tile, left);
    if (left <= 0) return false;
    do {
      if (++s >= a.sequences) return false;
      g = segment(a, s);
      tiles = tiles_of(g.n_k, kTileKeys);
    } while (tiles == 0);
    tile = 0;
    first = false;
    set(w, all, block);
    return true;
  }
};

template <typename T>
__device__ __forceinline__ void store_row(const AttnArgs& a, size_t at, int c, float v) {
  if constexpr (sizeof(T) == 4) {
    static_cast<float*>(a.out)[at + c] = v;
  } else {
    const __nv_bfloat16 h = __float2bfloat16_rn(v);
    static_cast<__nv_bfloat16*>(a.out)[at + c] = h;
    if (a.low) static_cast<__nv_bfloat16*>(a.low)[at + c] = __float2bfloat16_rn(v - __bfloat162float(h));
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(RowsShape<T, DP>::THREADS, RowsShape<T, DP>::BLOCKS)
    k_attention_rows(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttnArgs a,
                     const RowsWork w) {
  using C = RowsShape<T, DP>;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int KC = kF32 ? DP / 16 : DP / 32;  // 16-byte loads of a key row by one thread
  constexpr int VC = C::LINES;                  // ... of a value row
  constexpr int VJ = kF32 ? 4 : 8;              // column tiles of a value load
  constexpr int E = 16 / sizeof(T);
  constexpr int LD = DP + 4, WARPS = C::WARPS;
  __shared__ int s_timed_out;
  __shared__ Begin found;
  __shared__ Piece s_piece[WARPS + 1];
  __shared__ int32_t warp_sums[WARPS + 1];
  __shared__ float s_m[WARPS][16], s_l[WARPS][16];
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* s_o = reinterpret_cast<float*>(smem + C::JOIN);  // [16][LD]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::TAIL);
  uint64_t* empty = full + C::SLOTS;
  if (threadIdx.x == 0) {
    s_timed_out = 0;
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  after_previous_kernel();
  const int kv = blockIdx.x % a.kv_heads, block = blockIdx.x / a.kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, c = lane & 3;
  const int group = a.heads / a.kv_heads;
  bool in_order;
  find_begin<C::THREADS>(a, w, block, &found, warp_sums, &in_order);
  if (kv == 0 && threadIdx.x == 0) w.starts[3 * block + 2] = found.all;
  if (!in_order) return;  // (rows of several samples: no bound on the work)
  // rows of segments without keys become zeros, while the first copies are on their way: a warp looks at 32 segments at a time
  const uint32_t looked_at = warp < WARPS ? a.sequences + 2 : 0;
  for (uint32_t s0 = (uint32_t)(block * WARPS + warp) * 32; s0 < looked_at; s0 += (uint32_t)w.blocks * WARPS * 32) {
    Segment g = {};
    if (s0 + lane < looked_at) g = segment(a, s0 + lane);
    for (uint32_t some = __ballot_sync(0xffffffffu, g.n_k == 0 && g.n_q > 0); some; some &= some - 1) {
      const int from = __ffs(some) - 1, q0 = __shfl_sync(0xffffffffu, g.q0, from), n_q = __shfl_sync(0xffffffffu, g.n_q, from);
      for (int r = 0; r < group * n_q; ++r) {
        const int i = q0 + r / group, h = kv * group + r % group;
        for (int d = lane; d < a.dim; d += 32) store_row<T>(a, ((size_t)i * a.heads + h) * a.dim, d, 0.f);
        if (lane == 0 && a.lse) a.lse[(size_t)h * a.rows_q + i] = -CUDART_INF_F;
      }
    }
  }
  if (found.all == 0) return;
  const int32_t want = (int32_t)first_of(w, found.all, block), end = (int32_t)first_of(w, found.all, block + 1);
  if (kv == 0 && threadIdx.x == 0) {
    w.starts[3 * block] = (int32_t)found.s;
    w.starts[3 * block + 1] = want - found.tile;
  }
  if (want == end) return;
  // in shared memory, a copy for every warp: registers are short
  Piece& piece = s_piece[warp];
  if (lane == 0) {
    piece.g = found.g;
    piece.s = found.s;
    piece.tile = found.tile;
    piece.tiles = found.tiles;
    piece.left = end - want;
    piece.first = true;
    piece.set(w, found.all, block);
  }
  __syncwarp();

  const float scale = a.scale * kLog2e;
  const uint32_t ring = smem_u32(smem);
  bool timed_out = false;
  uint32_t it = 0;  // slots used so far

  if (warp == WARPS) {
    // ------------------------------ bulk copies ----------------------------------------
    if (lane == 0) {
      for (bool more = true; more && !timed_out; more = piece.next(a, w, found.all, block)) {
        if (piece.skip) continue;
        for (uint32_t r = piece.row; r < (uint32_t)(group * piece.g.n_q) && !timed_out; r += piece.step) {
          for (int t = piece.from; t < piece.to; ++t, ++it) {
            const uint32_t s = it % C::SLOTS;
            if (!mbar_wait(&empty[s], ((it / C::SLOTS) & 1u) ^ 1u)) { timed_out = true; break; }
            mbar_arrive_expect_tx(&full[s], C::SLOT);
#pragma unroll
            for (int b = 0; b < C::LINES; ++b) {
              const uint32_t at = ring + s * C::SLOT + b * C::LINE;
              tma_load_3d(at, &map_k, &full[s], b * 8 * E, kv, piece.g.k0 + t * kTileKeys);
              tma_load_3d(at + C::HALF, &map_v, &full[s], b * 8 * E, kv, piece.g.k0 + t * kTileKeys);
            }
          }
        }
      }
      if (timed_out)  // no copy may be in flight when the block ends
        for (uint32_t k = it > C::SLOTS ? it - C::SLOTS : 0; k < it; ++k) mbar_wait(&full[k % C::SLOTS], (k / C::SLOTS) & 1u);
    }
    if (timed_out) atomicExch(a.status, (uint32_t)RMN_ERR_TIMEOUT);
    return;
  }

  auto sync_warps = [] { asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory"); };  // those that compute
  const int mine16 = warp * 16;                                                            // this warp's keys of a tile
  auto next_piece = [&] {
    __syncwarp();
    bool more = false;
    if (lane == 0) more = piece.next(a, w, found.all, block);
    return __any_sync(0xffffffffu, more) != 0;  // (a barrier of the warp, too)
  };
  for (bool more = true; more && !timed_out; more = next_piece()) {
    __syncwarp();
    if (piece.skip) continue;
    const Segment& g = piece.g;
    const int hi = g.n_k, first_tile = piece.from, last_tile = piece.to;
    const int rows = group * g.n_q;
    for (uint32_t from = piece.row; from < (uint32_t)rows && !timed_out; from += piece.step) {
      const int r0 = (int)from;
      // q of rows gr and gr + 8 as operands
      uint32_t q[kF32 ? 1 : 2 * KC][4];
      int see[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = r0 + gr + 8 * e;
        const bool ok = r < rows;
        const int i = ok ? r / group : 0, h = kv * group + (ok ? r % group : 0);
        see[e] = ok ? visible_keys(g, i, a.causal) : 0;
        const T* from = static_cast<const T*>(a.q) + (int64_t)(g.q0 + i) * a.q_row + (int64_t)h * a.q_head;
        if constexpr (!kF32) {
#pragma unroll
          for (int b = 0; b < KC; ++b) {
            const uint4 x = load16(from + b * 32 + c * 8, ok && b * 32 + c * 8 < a.dim);
            q[2 * b][e] = x.x;
            q[2 * b][2 + e] = x.y;
            q[2 * b + 1][e] = x.z;
            q[2 * b + 1][2 + e] = x.w;
          }
        } else if (warp == 0) {
          // two parts of each number, in the order of the operands: [step][part][lane][4]
          uint32_t* s_q = reinterpret_cast<uint32_t*>(smem + C::Q);
#pragma unroll
          for (int b = 0; b < KC; ++b) {
            const uint4 x = load16(from + b * 16 + c * 4, ok && b * 16 + c * 4 < a.dim);
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // numbers 0, 1 belong to step 2 b, 2, 3 to step 2 b + 1
              uint32_t high, low;
              split_tf32(__uint_as_float(xs[k]), high, low);
              const int at = ((2 * b + (k >> 1)) * 2 * 32 + lane) * 4 + e + 2 * (k & 1);
              s_q[at] = high;
              s_q[at + 128] = low;
            }
          }
        }
      }
      if constexpr (kF32) sync_warps();
      float o[VC * VJ][4];
#pragma unroll
      for (int j = 0; j < VC * VJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
      float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};

      for (int t64 = first_tile; t64 < last_tile; ++t64) {
        const uint32_t load = it + (uint32_t)(t64 - first_tile), slot = load % C::SLOTS;
        const bool here = mbar_wait(&full[slot], (load / C::SLOTS) & 1u);
        if (!__all_sync(0xffffffffu, here)) {
          timed_out = true;
          break;
        }
        const int k0 = t64 * kTileKeys + mine16;
        const uint8_t* s_k = smem + slot * C::SLOT;
        // row and 16-byte piece of a tile, swizzled
        auto read16 = [&](uint32_t half, int row, int line, int at) {
          return *reinterpret_cast<const uint4*>(s_k + half + line * C::LINE + row * 128 + ((at ^ (row & 7)) << 4));
        };
        // 16 keys: two column tiles of scores
        float s[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
#pragma unroll
          for (int b = 0; b < KC; ++b) {
            const uint4 kx = read16(0, mine16 + t * 8 + gr, b >> 1, (b & 1) * 4 + c);
            if constexpr (!kF32) {
              mma_bf16(s[t], q[2 * b], kx.x, kx.y);
              mma_bf16(s[t], q[2 * b + 1], kx.z, kx.w);
            } else {
              const uint4* s_q = reinterpret_cast<const uint4*>(smem + C::Q);
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const uint4 h = s_q[(2 * b + half) * 64 + lane], lw = s_q[(2 * b + half) * 64 + 32 + lane];
                const uint32_t ah[4] = {h.x, h.y, h.z, h.w}, al[4] = {lw.x, lw.y, lw.z, lw.w};
                mma_split(s[t], ah, al, __uint_as_float(half ? kx.z : kx.x), __uint_as_float(half ? kx.w : kx.y));
              }
            }
          }
        }
        // the values of four keys (bf16) or two of them
        uint4 vx[kF32 ? 2 : 4][VC];
        auto read_values = [&](int from, int n) {
#pragma unroll
          for (int u = 0; u < n; ++u) {
            const int t = from + u, row = mine16 + (t >> 1) * 8 + 2 * c + (t & 1);
#pragma unroll
            for (int b = 0; b < VC; ++b) vx[u][b] = read16(C::HALF, row, b, gr);
            if (k0 + 16 > hi && t64 * kTileKeys + row >= hi) {  // what lies behind the last key: a weight of zero needs a number
#pragma unroll
              for (int b = 0; b < VC; ++b) vx[u][b] = make_uint4(0u, 0u, 0u, 0u);
            }
          }
        };
        auto release = [&] {
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[slot]);
        };
        if constexpr (!kF32) {
          read_values(0, 4);
          release();
        }
        float shrink[2];
        bool rise = false;
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // rows gr, gr + 8
          float top = -CUDART_INF_F;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float& x = s[t][2 * e + k];
              x = k0 + t * 8 + 2 * c + k < min(see[e], hi) ? x * scale : -CUDART_INF_F;
              top = fmaxf(top, x);
            }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          shrink[e] = 1.f;
          if (top > m[e] + kRescale) {
            shrink[e] = exp2_approx(m[e] - top);
            m[e] = top;
            l[e] *= shrink[e];
            rise = true;
          }
          const float base = m[e] == -CUDART_INF_F ? 0.f : m[e];
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float& x = s[t][2 * e + k];
              x = kF32 ? exp2f(x - base) : exp2_approx(x - base);
              l[e] += x;
            }
        }
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
          for (int j = 0; j < VC * VJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] *= shrink[e >> 1];
        }
        if constexpr (!kF32) {
          const uint32_t p[4] = {pack_bf16(s[0][0], s[0][1]), pack_bf16(s[0][2], s[0][3]), pack_bf16(s[1][0], s[1][1]),
                                 pack_bf16(s[1][2], s[1][3])};
#pragma unroll
          for (int b = 0; b < VC; ++b) {
            const uint32_t v0[4] = {vx[0][b].x, vx[0][b].y, vx[0][b].z, vx[0][b].w};
            const uint32_t v1[4] = {vx[1][b].x, vx[1][b].y, vx[1][b].z, vx[1][b].w};
            const uint32_t v2[4] = {vx[2][b].x, vx[2][b].y, vx[2][b].z, vx[2][b].w};
            const uint32_t v3[4] = {vx[3][b].x, vx[3][b].y, vx[3][b].z, vx[3][b].w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // channel j of the thread's 8: the two keys of each pair in one register
              const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
              mma_bf16(o[b * 8 + j], p, __byte_perm(v0[j >> 1], v1[j >> 1], sel), __byte_perm(v2[j >> 1], v3[j >> 1], sel));
            }
          }
        } else {
#pragma unroll
          for (int t = 0; t < 2; ++t) {  // k = c is key 2 c, k = c + 4 is key 2 c + 1
            read_values(2 * t, 2);
            if (t == 1) release();
            uint32_t ph[4], pl[4];
            split_tf32(s[t][0], ph[0], pl[0]);
            split_tf32(s[t][2], ph[1], pl[1]);
            split_tf32(s[t][1], ph[2], pl[2]);
            split_tf32(s[t][3], ph[3], pl[3]);
#pragma unroll
            for (int b = 0; b < VC; ++b) {
              const uint32_t v0[4] = {vx[0][b].x, vx[0][b].y, vx[0][b].z, vx[0][b].w};
              const uint32_t v1[4] = {vx[1][b].x, vx[1][b].y, vx[1][b].z, vx[1][b].w};
#pragma unroll
              for (int j = 0; j < 4; ++j) mma_split(o[b * 4 + j], ph, pl, __uint_as_float(v0[j]), __uint_as_float(v1[j]));
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      }
      it += (uint32_t)(last_tile - first_tile);
      // the warps, joined in their order
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (c == 0) {
          s_m[warp][gr + 8 * e] = m[e];
          s_l[warp][gr + 8 * e] = l[e];
        }
      if (timed_out) s_timed_out = 1;
      sync_warps();
      timed_out = s_timed_out != 0;  // all warps leave together
      float mine[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -CUDART_INF_F;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) top = fmaxf(top, s_m[k][gr + 8 * e]);
        mine[e] = m[e] == -CUDART_INF_F ? 0.f : exp2f(m[e] - top);
      }
      for (int k = 0; k < WARPS; ++k) {
        if (warp == k) {
#pragma unroll
          for (int e2 = 0; e2 < 2; ++e2) {
            if (r0 + gr + 8 * e2 >= rows) continue;
            // column 2 c + e of tile j is channel j of the 16 bytes of lane group 2 c + e
            float4* row = reinterpret_cast<float4*>(s_o + (gr + 8 * e2) * LD + 2 * c * E);
            float4 x[VC * 2 * VJ / 4];
            if (k) {
#pragma unroll
              for (int i = 0; i < VC * 2 * VJ / 4; ++i) x[i] = row[i / (VJ / 2) * 2 * E + i % (VJ / 2)];
            } else {
#pragma unroll
              for (int i = 0; i < VC * 2 * VJ / 4; ++i) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int i = 0; i < VC * 2 * VJ / 4; ++i) {
              const int b = i / (VJ / 2), e = i % (VJ / 2) / (VJ / 4), j = i % (VJ / 4) * 4;
              x[i].x = fmaf(o[b * VJ + j][2 * e2 + e], mine[e2], x[i].x);
              x[i].y = fmaf(o[b * VJ + j + 1][2 * e2 + e], mine[e2], x[i].y);
              x[i].z = fmaf(o[b * VJ + j + 2][2 * e2 + e], mine[e2], x[i].z);
              x[i].w = fmaf(o[b * VJ + j + 3][2 * e2 + e], mine[e2], x[i].w);
            }
#pragma unroll
            for (int i = 0; i < VC * 2 * VJ / 4; ++i) row[i / (VJ / 2) * 2 * E + i % (VJ / 2)] = x[i];
          }
        }
        sync_warps();
      }
      for (int r = warp; r < 16 && r0 + r < rows && !timed_out; r += WARPS) {
        float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) top = fmaxf(top, s_m[k][r]);
#pragma unroll
        for (int k = 0; k < WARPS; ++k)
          // (a warp without a visible key has summed nothing; one with NaN scores has no maximum either, but a sum that is NaN)
          sum += s_m[k][r] == -CUDART_INF_F ? s_l[k][r] : s_l[k][r] * exp2f(s_m[k][r] - top);
        const int i = (r0 + r) / group, h = kv * group + (r0 + r) % group;
        const size_t part = piece.split ? part_at(a, w, block, kv, piece.first, r0 + r) : 0;
        const size_t at = ((size_t)(g.q0 + i) * a.heads + h) * a.dim;
        for (int d = lane; d < a.dim; d += 32) {
          const float v = s_o[r * LD + d];
          if (piece.split) w.parts[part * a.dim + d] = v;
          else store_row<T>(a, at, d, sum == 0.f ? 0.f : v / sum);
        }
        if (lane == 0) {
          if (piece.split) {
            w.sums[part * 2] = top;
            w.sums[part * 2 + 1] = sum;
          } else if (a.lse) {
            a.lse[(size_t)h * a.rows_q + g.q0 + i] = sum == 0.f ? -CUDART_INF_F : (top + log2f(sum)) * kLn2;
          }
        }
      }
      sync_warps();  // before the next rows take their places
    }
  }
  if (timed_out) atomicExch(a.status, (uint32_t)RMN_ERR_TIMEOUT);
}

// Sums the pieces of the sample that the run of block b begins inside of, for one head and every gridDim.y-th row, each of eight
// warps every eighth piece; the first of several blocks that begin inside of one sample does it.
template <typename T>
__global__ void __launch_bounds__(kSumThreads) k_attention_rows_sum(const AttnArgs a, const RowsWork w) {
  __shared__ float s_m[kSumWarps], s_l[kSumWarps], s_o[kSumWarps][128];
  after_previous_kernel();
  const int h = blockIdx.x % a.heads, group = a.heads / a.kv_heads, kv = h / group;
  const int block = 1 + blockIdx.x / a.heads;
  const uint32_t s = (uint32_t)__ldg(w.starts + 3 * block);
  const int32_t at0 = __ldg(w.starts + 3 * block + 1), all = __ldg(w.starts + 3 * block + 2);
  if (all <= 0 || first_of(w, all, block) == at0 || first_of(w, all, block - 1) > at0) return;
  const Segment g = segment(a, s);
  if (g.n_q > w.most_queries) return;  // stored by the first kernel
  const int32_t end = at0 + tiles_of(g.n_k, kTileKeys);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = block - 1;
  const bool whole = first_of(w, all, first) == at0;  // its run begins with this sample
  // the blocks k with first_of(k) < end
  const int64_t past = ((int64_t)end * w.blocks + all - 1) / all;
  const int pieces = (int)min(past, (int64_t)w.blocks) - first;
  auto has_none = [&](int k) { return all < w.blocks && first_of(w, all, k) == first_of(w, all, k + 1); };  // more blocks than tiles
  for (int i = blockIdx.y; i < g.n_q; i += gridDim.y) {
    const size_t at = ((size_t)(g.q0 + i) * a.heads + h) * a.dim;
    const int r = i * group + h % group;
    float top = -CUDART_INF_F, sum = 0.f;
    for (int k = warp * 32 + lane; k < pieces; k += kSumThreads) {
      if (!has_none(first + k)) top = fmaxf(top, __ldg(w.sums + part_at(a, w, first + k, kv, k > 0 || whole, r) * 2));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    __syncthreads();  // what the row before left has been read
    if (lane == 0) s_m[warp] = top;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSumWarps; ++k) top = fmaxf(top, s_m[k]);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = warp; k < pieces; k += kSumWarps) {
      if (has_none(first + k)) continue;
      const size_t part = part_at(a, w, first + k, kv, k > 0 || whole, r);
      const float mk = __ldg(w.sums + part * 2), lk = __ldg(w.sums + part * 2 + 1);
      const float by = mk == -CUDART_INF_F ? 0.f : exp2f(mk - top);
      sum += mk == -CUDART_INF_F ? lk : lk * by;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < a.dim) v[e] += __ldg(w.parts + part * a.dim + lane + 32 * e) * by;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s_o[warp][lane + 32 * e] = v[e];
    if (lane == 0) s_l[warp] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < kSumWarps; ++k) sum += s_l[k];
    const int d = threadIdx.x;
    if (d < a.dim) {
      float x = 0.f;
#pragma unroll
      for (int k = 0; k < kSumWarps; ++k) x += s_o[k][d];
      store_row<T>(a, at, d, sum == 0.f ? 0.f : x / sum);
    }
    if (threadIdx.x == 0 && a.lse)
      a.lse[(size_t)h * a.rows_q + g.q0 + i] = sum == 0.f ? -CUDART_INF_F : (top + log2f(sum)) * kLn2;
  }
}

struct RowsSizes {
  int blocks, most_queries;
  size_t sums_at, parts_at, total;
};
// As many blocks as fit the SMs at once, but two tiles for each at least (of as many tiles as there may be: 512 samples of 4 keys,
// 8 / 2 heads of 64, 154 us by the tiles of their rows together).
RowsSizes rows_sizes(uint32_t rows_k, uint32_t sequences, int heads, int kv_heads, int dim, int dtype) {
  RowsSizes z;
  const uint64_t pairs = ((uint64_t)rows_k / kTileKeys + sequences + 1) / 2, fit = 148 * (dtype == RMN_F32 ? 1 : 2) / kv_heads;
  z.blocks = (int)std::max<uint64_t>(1, std::min(pairs, fit));
  z.most_queries = std::max(1, kMostRows / (heads / kv_heads));
  const size_t parts = z.blocks > 1 ? (size_t)z.blocks * 2 * heads * z.most_queries : 0;  // (one block: whole samples)
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  z.sums_at = up((size_t)z.blocks * 3 * sizeof(int32_t));
  z.parts_at = up(z.sums_at + parts * 2 * sizeof(float));
  z.total = up(z.parts_at + parts * dim * sizeof(float));
  return z;
}

template <typename T, int DP>
int launch_rows(const CUtensorMap& k, const CUtensorMap& v, const AttnArgs& a, const RowsWork& w, cudaStream_t stream) {
  constexpr size_t smem = RowsShape<T, DP>::SMEM;
  static SmemOptIn opt_in;
  RMN_CUDA_TRY(opt_in.apply(reinterpret_cast<const void*>(k_attention_rows<T, DP>), smem));
  RMN_CUDA_TRY(launch_overlapped(k_attention_rows<T, DP>, dim3((uint32_t)(w.blocks * a.kv_heads)), dim3(RowsShape<T, DP>::THREADS), smem, stream, k, v, a, w));
  RMN_LAUNCH_CHECK();
  if (w.blocks == 1) return RMN_OK;  // every sample is one piece
  const uint32_t rows = (a.rows_q + a.sequences - 1) / a.sequences;  // of a sample, on average
  RMN_CUDA_TRY(launch_overlapped(k_attention_rows_sum<T>, dim3((uint32_t)(w.blocks - 1) * (uint32_t)a.heads, rows),
                                 dim3(kSumThreads), 0, stream, a, w));
  RMN_LAUNCH_CHECK();
  return RMN_OK;
}

}  // namespace

namespace {
// Whether this form takes less time than whole tiles of a head's queries (bf16 128 of them on the tensor cores, fp32 64), both
// estimated in us from averages over the samples: here sixteen rows of a sample and key head pass over its keys at a time, 64 keys a
// step, all SMs taking their share; there every query head passes once, and the longest sample's chain is not cut. Measured in bf16
// (here, there): 16 samples of one row and 509 ... 30011 keys, 16 / 4 heads of 128, 71 and 503 us; 16 samples of 5 rows and 8000 keys
// (16 x 5 / 8000), 8 heads of 64, 59 and 102; 512 x 4 / 4, 8 / 2 heads of 64, 32 and 85; 512 x 16 / 16, 8 heads of 64, 81 and 88; but
// 64 x 20 / 1024 94 and 38, 256 x 32 / 32 84 and 46, 4 x 8 / 60 7.5 and 6.1. In fp32, 8 heads of 64: 64 x 20 / 1024 178 and 318,
// 256 x 1 / 200 123 and 489, but 256 x 32 / 32 183 and 70, 512 x 1 / 4 136 and 106.
bool rows_take_less(uint32_t rows_q, uint32_t rows_k, uint32_t sequences, int heads, int kv_heads, int dim, int dtype) {
  const double n = sequences, rows = std::ceil(rows_q / n) * (heads / kv_heads), keys = rows_k / n, pass_rows = std::min(16.0, rows);
  const bool wide = dim > 64, f32 = dtype == RMN_F32;
  const double places = f32 ? 148 : 2 * 148, pieces = std::max(1.0, n * kv_heads / places);
  const double tiles = std::max(1.0, n * kv_heads * std::max(1.0, keys / kTileKeys) / places);  // a block
  const double piece = f32 ? (wide ? 6.0 : 4.0) + 0.15 * pass_rows : 1.5 + 0.22 * pass_rows;
  const double here = 4 + std::ceil(rows / 16) * (pieces * piece + tiles * (wide ? 1.8 : 1.2));
  const double there = f32 ? std::max(1.0, n * heads / (wide ? 148 : 2 * 148)) * (std::max(1.0, keys / 64) * (wide ? 14 : 10.5) - 2)
                           : std::max(1.0, n * heads / (2 * 148)) * (5.5 + std::max(1.0, keys / 128) * (wide ? 1.9 : 1.1));
  return here < there;
}
}  // namespace

size_t attention_rows_workspace(uint32_t rows_q, uint32_t rows_k, uint32_t sequences, int heads, int kv_heads, int dim, int dtype) {
  if (!rows_q || !rows_k || !sequences || dim > 128 || dim % (dtype == RMN_F32 ? 4 : 8)) return 0;
  const uint64_t rows = ((uint64_t)rows_q + sequences - 1) / sequences * (heads / kv_heads);
  if (rows > kMostRows) return 0;
  if (!rows_take_less(rows_q, rows_k, sequences, heads, kv_heads, dim, dtype)) return 0;
  if ((uint64_t)rows_q * heads > 0x7fffffffull) return 0;
  return rows_sizes(rows_k, sequences, heads, kv_heads, dim, dtype).total;
}

int attention_rows_forward(const AttnArgs& a, int dtype, void* workspace, cudaStream_t stream) {
  const int elem = dtype == RMN_F32 ? 4 : 2;
  if (((uintptr_t)a.q & 15) || a.q_row * elem % 16 || a.q_head * elem % 16 || !(a.scale > 0.f)) return RMN_ERR_UNSUPPORTED;
  CUtensorMap k, v;
  if (!make_head_map(&k, a.k, a.rows_k, a.kv_heads, a.dim, a.k_row, a.k_head, kTileKeys, elem) ||
      !make_head_map(&v, a.v, a.rows_k, a.kv_heads, a.dim, a.v_row, a.v_head, kTileKeys, elem))
    return RMN_ERR_UNSUPPORTED;
  const RowsSizes z = rows_sizes(a.rows_k, a.sequences, a.heads, a.kv_heads, a.dim, dtype);
  char* base = static_cast<char*>(workspace);
  const RowsWork w = {z.blocks, z.most_queries, reinterpret_cast<int32_t*>(base), reinterpret_cast<float*>(base + z.sums_at),
                      reinterpret_cast<float*>(base + z.parts_at)};
  if (dtype == RMN_F32)
    return a.dim <= 32   ? launch_rows<float, 32>(k, v, a, w, stream)
           : a.dim <= 64 ? launch_rows<float, 64>(k, v, a, w, stream)
                         : launch_rows<float, 128>(k, v, a, w, stream);
  return a.dim <= 64 ? launch_rows<__nv_bfloat16, 64>(k, v, a, w, stream)
                     : launch_rows<__nv_bfloat16, 128>(k, v, a, w, stream);
}

}  // namespace rmn
