// Attention of few query rows a sample against long keys (a token at a time): forward pass, fp32 and bf16, head sizes up to 128.
//
// Bound by memory: the keys and values are read once, whatever the number of heads that share them. All keys in use, in tiles of 64,
// are dealt out evenly to as many blocks as fit the GPU, so that samples of very different lengths keep all of it busy to the end;
// neighbouring blocks take the same tiles of neighbouring key heads (whose rows are neighbours in memory). A block walks through its
// run of tiles, which is a piece of one sample or of several, with all query rows and heads that go with them, up to 16 of them at
// a time. Bulk copies bring a tile's keys and values into a ring in shared memory, some 100 KB in flight for a block, across the borders
// of pieces; each of four warps takes 16 of the 64 keys (in fp32 each of eight takes 8) and has a running maximum and sum of its own. The
// warps are joined in shared memory, and the pieces of a sample that several blocks share by a second kernel, in a fixed order.
// 16 samples of 509 ... 30011 keys, 16 query and 4 key heads of 128 (336 MB in bf16): 62 us, 5.4 TB/s, and 8 us for the second kernel;
// in fp32 123 us, 5.5 TB/s, and 8.
//
// In bf16 the rows are those of warp-wide matrix products (their rate does not bound here: 16 rows cost one product for 8 keys). Keys
// and values go from shared memory to registers as 16-byte loads that are product operands as they stand: which of a row's
// channels is which k of a product is free as long as q has the same order, and which channel is which column of the output is free
// as long as the store undoes it. A thread's 8 adjacent channels of a key are its operands of two products; of the values
// it has 8 channels of the four keys whose weights it holds, paired by a byte permutation.
// In fp32 they are multiplied and added in fp32 (Rows32): of up to 4 rows that takes less time than the bytes, of 16 rows it bounds (such
// samples with one key head: 93 us for 160 MB).
#include "rmn_attention_tc.cuh"

#include <math_constants.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace rmn {
namespace {

using namespace tc;

constexpr int kSumWarps = 8, kSumThreads = kSumWarps * 32;
constexpr int kTileKeys = 64;
constexpr int kMostRows = 32;    // of a sample and a key head (queries times heads): on average, and for the sum of pieces
constexpr float kRescale = 8.f;  // how far a row's maximum (bf16: its log2) may rise before the output is scaled

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Maxima are of the scores in fp32, of the scores times log2 e in bf16: the exponentials of differences to them, and the logarithm of a
// sum with the maximum it was taken at.
template <typename T>
__device__ __forceinline__ float exp_of(float x) {
  return sizeof(T) == 4 ? expf(x) : exp2f(x);
}
template <typename T>
__device__ __forceinline__ float lse_of(float top, float sum) {
  return sum == 0.f ? -CUDART_INF_F : sizeof(T) == 4 ? top + logf(sum) : (top + log2f(sum)) * kLn2;
}
__device__ __forceinline__ uint4 load16(const void* p, bool ok) {
  return ok ? __ldg(static_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
}

// The ring: a slot is 64 rows of keys and 64 of values, each as columns of 128-byte swizzled lines.
template <typename T, int DP>
struct RowsShape {
  // Each with keys of its own of every tile: a warp waits for all phases of a slot's barrier. (Two fours of warps that take turns at the
  // tiles of a ring of three slots wait for every second phase of each; the parity of the one before lets such a wait pass early.)
  static constexpr int WARPS = sizeof(T) == 4 ? 8 : 4;
  static constexpr int THREADS = WARPS * 32 + 32;                   // and one warp for the copies
  static constexpr int BLOCKS = sizeof(T) == 4 ? 1 : 2;             // an SM
  static constexpr int LINES = DP * (int)sizeof(T) / 128;           // of a row
  static constexpr uint32_t LINE = kTileKeys * 128, HALF = LINES * LINE, SLOT = 2 * HALF;
  static constexpr int SLOTS = SLOT >= 32 * 1024 ? 3 : 6;
  static constexpr uint32_t JOIN = SLOTS * SLOT;                    // rows of the output, fp32
  static constexpr uint32_t TAIL = JOIN + (sizeof(T) == 4 ? 32 : 16) * (DP + 4) * 4;
  static constexpr size_t SMEM = TAIL + 256 + 1024;
};

struct RowsWork {  // scratch, and how the keys are cut
  int blocks;           // of the first kernel, for each key head
  int most_queries;     // rows of a sample whose pieces are summed by the second kernel
  int32_t* starts;      // [blocks][3]: the sample that a block of the first head begins in, the tiles before that; all tiles
  float* sums;          // [piece][group * most_queries][2]: maximum, sum
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

// fp32, a warp's K keys of a tile (8 or 16) against R query rows (4 or 8): multiply-adds, so that products, sums and infinite values are
// what they are in the other fp32 kernels. DL lanes hold a row's channels, W neighbouring ones each, of all R rows and of the outputs, so
// that a key or a value is read once from shared memory; up to 64 channels the halves of a warp take half of the keys each.
// A lane's part of a score is of its channels. The parts of DL scores (KB keys, R rows) are added up by exchanges, of 16 numbers, of 8 ...,
// behind which lane i has the score of key i / R and row i % R. What is where makes every exchange one shuffle without a choice: lane i
// has the rows (and goes through the keys) in an order of its own, number r being row r ^ (i % R), number k key k ^ (i / R); so the number
// that it gives at distance n is the one that lane i ^ n keeps, and the weight that it needs for number (k, r) is in lane i ^ (k R + r).
template <int DP, int R, int K>
struct Rows32 {
  static constexpr int W = DP == 32 ? 2 : 4, DL = DP / W, KG = 32 / DL;
  static constexpr int KEYS = K / KG, KB = DL / R, NB = KEYS / KB;  // keys of a lane's half, of a batch of scores; batches
  Pair q[R / 2][W], o[R / 2][W];                                    // of two rows each
  float m, l;                                                       // of row lane % R; l: the lane's part
  int see;

  static __device__ __forceinline__ int ch() { return (threadIdx.x & 31) % DL; }
  static __device__ __forceinline__ int half() { return (threadIdx.x & 31) / DL; }
  static __device__ __forceinline__ int row_of(int r) { return r ^ (ch() % R); }
  static __device__ __forceinline__ int key_of(int k) { return k ^ (ch() / R); }
  static __device__ __forceinline__ Pair both(float x) { return make_pair(x, x); }
  // x of lane i ^ n
  static __device__ __forceinline__ float from(float x, int n) { return __shfl_xor_sync(0xffffffffu, x, n); }
  static __device__ __forceinline__ Pair from(Pair p, int n) {
    float x, y;
    parts(p, x, y);
    return make_pair(from(x, n), from(y, n));
  }
  // what row lane % R has, for rows 2 i and 2 i + 1 of the lane's order
  static __device__ __forceinline__ Pair of_rows(float x, int i) { return make_pair(from(x, 2 * i), from(x, 2 * i + 1)); }
  // the lane's channels at p
  static __device__ __forceinline__ void channels(const float* p, float (&x)[W]) {
    if constexpr (W == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(p);
      x[0] = v.x; x[1] = v.y;
    }
  }

  // rows r0 ... of the piece's `rows`
  __device__ __forceinline__ void begin(const AttnArgs& a, const Segment& g, int kv, int group, int r0, int rows) {
#pragma unroll
    for (int i = 0; i < R / 2; ++i) {
      float x[2][W];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = r0 + row_of(2 * i + t);
#pragma unroll
        for (int e = 0; e < W; ++e) x[t][e] = 0.f;
        if (r < rows && ch() * W < a.dim)
          channels(static_cast<const float*>(a.q) + (int64_t)(g.q0 + r / group) * a.q_row + (int64_t)(kv * group + r % group) * a.q_head + ch() * W,
                   x[t]);
      }
#pragma unroll
      for (int e = 0; e < W; ++e) {
        q[i][e] = make_pair(x[0][e] * a.scale, x[1][e] * a.scale);
        o[i][e] = both(0.f);
      }
    }
    const int mine = r0 + ch() % R;
    see = mine < rows ? visible_keys(g, mine / group, a.causal) : 0;
    m = -CUDART_INF_F;
    l = 0.f;
  }
  // the lane's channels of key (or value) `row` of a tile of 128-byte swizzled lines, LINE bytes apart
  template <uint32_t LINE>
  static __device__ __forceinline__ void read(const uint8_t* tile, int row, float (&x)[W]) {
    const int piece = ch() * W / 4;
    channels(reinterpret_cast<const float*>(tile + piece / 8 * LINE + row * 128 + (((piece % 8) ^ (row & 7)) << 4)) + ch() * W % 4, x);
  }
  // keys k0 ... k0 + K - 1 of the sample, rows first ... of the tile, of which those up to hi are in use
  template <uint32_t LINE, class Release>
  __device__ __forceinline__ void step(const uint8_t* keys, const uint8_t* values, int first, int k0, int hi, Release&& release) {
    float s[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      Pair v[DL / 2];
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        float x[W];
        read<LINE>(keys, first + half() * KEYS + b * KB + key_of(k), x);
#pragma unroll
        for (int i = 0; i < R / 2; ++i) {
          Pair t = mul(q[i][0], both(x[0]));
#pragma unroll
          for (int e = 1; e < W; ++e) t = fma(q[i][e], both(x[e]), t);
          v[k * R / 2 + i] = t;
        }
      }
#pragma unroll
      for (int n = DL / 2; n > 1; n /= 2)
#pragma unroll
        for (int i = 0; i < n / 2; ++i) v[i] = add(v[i], from(v[i + n / 2], n));
      float x, y;
      parts(v[0], x, y);
      s[b] = x + from(y, 1);
    }
    float top = -CUDART_INF_F;
    const int left = min(see, hi) - k0 - half() * KEYS - key_of(0);  // keys that the row sees from the lane's first one on
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (b * KB >= left) s[b] = -CUDART_INF_F;
      top = fmaxf(top, s[b]);
    }
#pragma unroll
    for (int n = R; n < 32; n *= 2) top = fmaxf(top, from(top, n));
    const bool rise = top > m + kRescale;
    if (__any_sync(0xffffffffu, rise)) {
      const float shrink = rise ? expf(m - top) : 1.f;
      if (rise) m = top;
      l *= shrink;
#pragma unroll
      for (int i = 0; i < R / 2; ++i) {
        const Pair f = of_rows(shrink, i);
#pragma unroll
        for (int e = 0; e < W; ++e) o[i][e] = mul(o[i][e], f);
      }
    }
    const float base = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      s[b] = expf(s[b] - base);
      l += s[b];
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const int row = half() * KEYS + b * KB + key_of(k);
        float x[W];
        read<LINE>(values, first + row, x);
        if (k0 + row >= hi) {  // what lies behind the last key: a weight of zero needs a number
#pragma unroll
          for (int e = 0; e < W; ++e) x[e] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < R / 2; ++i) {
          const Pair f = make_pair(from(s[b], k * R + 2 * i), from(s[b], k * R + 2 * i + 1));
#pragma unroll
          for (int e = 0; e < W; ++e) o[i][e] = fma(f, both(x[e]), o[i][e]);
        }
      }
    release();
  }
  // the lanes' parts put together: l whole in every lane of a row, o whole in every lane of its channels
  __device__ __forceinline__ void end() {
#pragma unroll
    for (int n = R; n < 32; n *= 2) l += from(l, n);
    if constexpr (KG == 2) {
#pragma unroll
      for (int i = 0; i < R / 2; ++i)
#pragma unroll
        for (int e = 0; e < W; ++e) o[i][e] = add(o[i][e], from(o[i][e], 16));
    }
  }
  // o, times what row lane % R has in `by`, into rows of `to`, LD apart, or on top of what is there
  template <int LD>
  __device__ __forceinline__ void put(float* to, float by, bool on_top) const {
#pragma unroll
    for (int i = 0; i < R / 2; ++i) {
      const Pair f = of_rows(by, i);
      if (half()) continue;
      float x[2][W];
#pragma unroll
      for (int e = 0; e < W; ++e) parts(mul(o[i][e], f), x[0][e], x[1][e]);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float* row = to + row_of(2 * i + t) * LD + ch() * W;
        if (on_top) {
          float before[W];
          channels(row, before);
#pragma unroll
          for (int e = 0; e < W; ++e) x[t][e] += before[e];
        }
        if constexpr (W == 4) *reinterpret_cast<float4*>(row) = make_float4(x[t][0], x[t][1], x[t][2], x[t][3]);
        else *reinterpret_cast<float2*>(row) = make_float2(x[t][0], x[t][1]);
      }
    }
  }
};

template <typename T, int DP>
__global__ void __launch_bounds__(RowsShape<T, DP>::THREADS, RowsShape<T, DP>::BLOCKS)
    k_attention_rows(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttnArgs a,
                     const RowsWork w) {
  using C = RowsShape<T, DP>;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int KC = DP / 32;  // bf16: 16-byte loads of a key row by one thread
  constexpr int VC = C::LINES; // ... of a value row
  constexpr int VJ = 8;        // column tiles of a value load
  constexpr int E = 16 / sizeof(T);
  constexpr int LD = DP + 4, WARPS = C::WARPS;
  __shared__ int s_timed_out;
  __shared__ Begin found;
  __shared__ Piece s_piece[WARPS + 1];
  __shared__ int32_t warp_sums[WARPS + 1];
  __shared__ float s_m[WARPS][16], s_l[WARPS][16];
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* s_o = reinterpret_cast<float*>(smem + C::JOIN);  // [parts][rows at once][LD]
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
  if (!in_order) {  // rows of several samples: no bound on the work. The call is reported; its outputs are those of rows without keys
    const uint64_t rows = (uint64_t)a.rows_q * a.heads, first = (uint64_t)blockIdx.x * C::THREADS + threadIdx.x;
    const uint64_t all = (uint64_t)gridDim.x * C::THREADS;
    for (uint64_t i = first; i < rows * a.dim; i += all) store_row<T>(a, i, 0, 0.f);
    if (a.lse)
      for (uint64_t i = first; i < rows; i += all) a.lse[i] = -CUDART_INF_F;
    return;
  }
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
  const int mine16 = (warp & 3) * 16;                                                      // bf16: this warp's keys of a tile
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
      // the tiles of this piece, as f(keys and values of the tile, its first key, what releases its place)
      auto walk = [&](auto&& f) {
        for (int t64 = first_tile; t64 < last_tile; ++t64) {
          const uint32_t slot = it % C::SLOTS;
          const bool here = mbar_wait(&full[slot], (it / C::SLOTS) & 1u);
          if (!__all_sync(0xffffffffu, here)) {
            timed_out = true;
            break;
          }
          f(smem + slot * C::SLOT, t64 * kTileKeys, [&] {
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[slot]);
          });
          ++it;
        }
      };
      // the warps leave together where a wait ran out
      auto meet = [&] {
        if (timed_out) s_timed_out = 1;
        sync_warps();
        timed_out = s_timed_out != 0;
      };
      // the largest of the warps' maxima of row r
      auto top_of = [&](int r) {
        float top = -CUDART_INF_F;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) top = fmaxf(top, s_m[k][r]);
        return top;
      };
      int n_parts = 1, part_rows = 16;  // of s_o
      if constexpr (kF32) {
        // Up to 4 rows: a warp has 8 keys; more: 16 keys, and two fours of warps half of the rows each (the registers of 9 warps do not
        // hold 16).
        auto fp32 = [&](auto rows_at_once, auto keys_at_once) {
          constexpr int R = decltype(rows_at_once)::value, K = decltype(keys_at_once)::value;
          constexpr int SHARE = kTileKeys / K, ROWS = R * WARPS / SHARE;  // warps that have a row; rows of all
          using Rows = Rows32<DP, R, K>;
          const int mine0 = warp / SHARE * R, part = warp % SHARE;
          Rows x;
          x.begin(a, g, kv, group, r0 + mine0, rows);
          walk([&](const uint8_t* tile, int k64, auto&& release) {
            x.template step<C::LINE>(tile, tile + C::HALF, part * K, k64 + part * K, hi, release);
          });
          x.end();
          // the warps' parts of a row side by side, as many as there is room for, the others on top of them
          if (lane < 16) {
            const bool here = lane >= mine0 && lane < mine0 + R;
            s_m[warp][lane] = here ? x.m : -CUDART_INF_F;  // (R divides mine0: lane's row is lane % R)
            s_l[warp][lane] = here ? x.l : 0.f;
          }
          meet();
          const float mine = x.m == -CUDART_INF_F ? 0.f : expf(x.m - top_of(mine0 + lane % R));
          n_parts = min(SHARE, 32 / ROWS);
          part_rows = ROWS;
          for (int k = 0; k < SHARE; k += n_parts) {
            if (part >= k && part < k + n_parts) x.template put<LD>(s_o + ((part - k) * ROWS + mine0) * LD, mine, k > 0);
            sync_warps();
          }
        };
        using Four = std::integral_constant<int, 4>;
        using Eight = std::integral_constant<int, 8>;
        using Sixteen = std::integral_constant<int, 16>;
        if (rows - r0 <= 4) fp32(Four{}, Eight{});
        else if (rows - r0 <= 8) fp32(Four{}, Sixteen{});
        else fp32(Eight{}, Sixteen{});
      } else {
        // q of rows gr and gr + 8 as operands
        uint32_t q[2 * KC][4];
        int see[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = r0 + gr + 8 * e;
          const bool ok = r < rows;
          const int i = ok ? r / group : 0, h = kv * group + (ok ? r % group : 0);
          see[e] = ok ? visible_keys(g, i, a.causal) : 0;
          const T* from = static_cast<const T*>(a.q) + (int64_t)(g.q0 + i) * a.q_row + (int64_t)h * a.q_head;
#pragma unroll
          for (int b = 0; b < KC; ++b) {
            const uint4 x = load16(from + b * 32 + c * 8, ok && b * 32 + c * 8 < a.dim);
            q[2 * b][e] = x.x;
            q[2 * b][2 + e] = x.y;
            q[2 * b + 1][e] = x.z;
            q[2 * b + 1][2 + e] = x.w;
          }
        }
        float o[VC * VJ][4];
#pragma unroll
        for (int j = 0; j < VC * VJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
        float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};

        walk([&](const uint8_t* s_k, int k64, auto&& release) {
          const int k0 = k64 + mine16;
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
              mma_bf16(s[t], q[2 * b], kx.x, kx.y);
              mma_bf16(s[t], q[2 * b + 1], kx.z, kx.w);
            }
          }
          uint4 vx[4][VC];  // the values of four keys
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int row = mine16 + (t >> 1) * 8 + 2 * c + (t & 1);
#pragma unroll
            for (int b = 0; b < VC; ++b) vx[t][b] = read16(C::HALF, row, b, gr);
            if (k0 + 16 > hi && k64 + row >= hi) {  // what lies behind the last key: a weight of zero needs a number
#pragma unroll
              for (int b = 0; b < VC; ++b) vx[t][b] = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          release();
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
                x = exp2_approx(x - base);
                l[e] += x;
              }
          }
          if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int j = 0; j < VC * VJ; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[j][e] *= shrink[e >> 1];
          }
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
        });
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
          l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        }
        // the warps, joined in their order
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (c == 0) {
            s_m[warp][gr + 8 * e] = m[e];
            s_l[warp][gr + 8 * e] = l[e];
          }
        meet();
        float mine[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mine[e] = m[e] == -CUDART_INF_F ? 0.f : exp2f(m[e] - top_of(gr + 8 * e));
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
      }
      for (int r = warp; r < 16 && r0 + r < rows && !timed_out; r += WARPS) {
        const float top = top_of(r);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k)
          // (a warp without a visible key has summed nothing; one with NaN scores has no maximum either, but a sum that is NaN)
          sum += s_m[k][r] == -CUDART_INF_F ? s_l[k][r] : s_l[k][r] * exp_of<T>(s_m[k][r] - top);
        const int i = (r0 + r) / group, h = kv * group + (r0 + r) % group;
        const size_t part = piece.split ? part_at(a, w, block, kv, piece.first, r0 + r) : 0;
        const size_t at = ((size_t)(g.q0 + i) * a.heads + h) * a.dim;
        for (int d = lane; d < a.dim; d += 32) {
          float v = s_o[r * LD + d];
          for (int k = 1; k < n_parts; ++k) v += s_o[(k * part_rows + r) * LD + d];
          if (piece.split) w.parts[part * a.dim + d] = v;
          else store_row<T>(a, at, d, sum == 0.f ? 0.f : v / sum);
        }
        if (lane == 0) {
          if (piece.split) {
            w.sums[part * 2] = top;
            w.sums[part * 2 + 1] = sum;
          } else if (a.lse) {
            a.lse[(size_t)h * a.rows_q + g.q0 + i] = lse_of<T>(top, sum);
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
      const float by = mk == -CUDART_INF_F ? 0.f : exp_of<T>(mk - top);
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
      a.lse[(size_t)h * a.rows_q + g.q0 + i] = lse_of<T>(top, sum);
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
// 64 x 20 / 1024 94 and 38, 256 x 32 / 32 84 and 46, 4 x 8 / 60 7.5 and 6.1. In fp32, 8 heads of 64: 64 x 20 / 1024 204 and 325,
// 256 x 1 / 200 101 and 495, 64 x 1 / 100 32 and 65, 512 x 1 / 4 118 and 118, but 256 x 32 / 32 225 and 80.
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
