// What the tensor-core attention kernels share.
#pragma once

#include "rmn_attention.cuh"
#include "rmn_pair.cuh"
#include "rmn_tma.cuh"

namespace rmn {

void count_tc_launch();  // defined in rmn_conv_tc.cu

namespace tc {

constexpr uint32_t kAtomBytes = 128 * 128;  // 128 rows of 64 bf16: one 128-byte swizzled box
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_approx(float x) {  // 2 ulp; results below 2^-126 are zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ Pair pair_of(uint32_t x, uint32_t y) { return make_pair(__uint_as_float(x), __uint_as_float(y)); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

#define RMN_TC_REGS16(r, o)                                                                                               \
  "r"(r[o + 0]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7]), \
      "r"(r[o + 8]), "r"(r[o + 9]), "r"(r[o + 10]), "r"(r[o + 11]), "r"(r[o + 12]), "r"(r[o + 13]), "r"(r[o + 14]),       \
      "r"(r[o + 15])
// 16 (32) columns of the warp's 32 lanes: register i of thread t is column i of lane t
template <int FIRST, int N>
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[N]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      RMN_TC_REGS16(r, FIRST)
      : "memory");
}
template <int FIRST, int N>
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&r)[N]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      RMN_TC_REGS16(r, FIRST), RMN_TC_REGS16(r, FIRST + 16)
      : "memory");
}
#undef RMN_TC_REGS16

// 32 columns into r[FIRST ... FIRST + 31]
template <int FIRST, int N>
__device__ __forceinline__ void tc_ld32_at(uint32_t taddr, uint32_t (&r)[N]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[FIRST + 0]), "=r"(r[FIRST + 1]), "=r"(r[FIRST + 2]), "=r"(r[FIRST + 3]), "=r"(r[FIRST + 4]),
        "=r"(r[FIRST + 5]), "=r"(r[FIRST + 6]), "=r"(r[FIRST + 7]), "=r"(r[FIRST + 8]), "=r"(r[FIRST + 9]),
        "=r"(r[FIRST + 10]), "=r"(r[FIRST + 11]), "=r"(r[FIRST + 12]), "=r"(r[FIRST + 13]), "=r"(r[FIRST + 14]),
        "=r"(r[FIRST + 15]), "=r"(r[FIRST + 16]), "=r"(r[FIRST + 17]), "=r"(r[FIRST + 18]), "=r"(r[FIRST + 19]),
        "=r"(r[FIRST + 20]), "=r"(r[FIRST + 21]), "=r"(r[FIRST + 22]), "=r"(r[FIRST + 23]), "=r"(r[FIRST + 24]),
        "=r"(r[FIRST + 25]), "=r"(r[FIRST + 26]), "=r"(r[FIRST + 27]), "=r"(r[FIRST + 28]), "=r"(r[FIRST + 29]),
        "=r"(r[FIRST + 30]), "=r"(r[FIRST + 31])
      : "r"(taddr)
      : "memory");
}

// A wait of a whole warp, left by all lanes together: what follows is executed by whole warps (tcgen05, elect), also when it ran out.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  if (__all_sync(0xffffffffu, mbar_try_wait(addr, parity))) return true;
  const unsigned long long t0 = global_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
      if (__all_sync(0xffffffffu, mbar_try_wait(addr, parity))) return true;
    if (__any_sync(0xffffffffu, global_ns() - t0 > 2000000000ull)) return false;
  }
}

// The address field of a shared-memory descriptor. In a block of a cluster other than its first, addresses have bits above the
// block's own window, which would run into the next field.
__device__ __forceinline__ uint64_t desc_address(uint32_t addr) { return (addr >> 4) & 0x3FFFu; }
// D[128, n] (+)= A[128, 16 steps] B[n, 16 steps]^T, both K-major tiles in shared memory: A of 128 rows, B of B_ROWS, as atoms of 64
// channels (128-byte swizzled lines)
template <int B_ROWS = 128>
__device__ __forceinline__ void mma_rows(uint32_t d_tmem, uint32_t a_s, uint32_t b_s, uint32_t idesc, int steps) {
  constexpr uint64_t DESC = smem_desc_sw_const(16, 1024, 2u);
  for (int j = 0; j < steps; ++j) {
    const uint32_t in = (uint32_t)(j & 3) * 32u;
    tc_mma_bf16_elect(d_tmem, DESC + desc_address(a_s + (uint32_t)(j >> 2) * kAtomBytes + in),
                      DESC + desc_address(b_s + (uint32_t)(j >> 2) * (B_ROWS * 128u) + in), idesc, j != 0);
  }
}
// D[128, n] (+)= A[128, ROWS] B[ROWS, n]: A in tensor memory, its pieces of 32 columns (64 values) HALF apart, B a tile whose ROWS
// rows are summed over (MN-major)
template <int ROWS = 128, int HALF = 32>
__device__ __forceinline__ void mma_columns(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_s, uint32_t idesc, bool accumulate) {
  constexpr uint64_t DESC = smem_desc_sw_const(ROWS * 128, 1024, 2u);
#pragma unroll
  for (int j = 0; j < ROWS / 16; ++j)
    tc_mma_bf16_ta_elect(d_tmem, a_tmem + (j >> 2) * HALF + (j & 3) * 8, DESC + desc_address(b_s + (uint32_t)j * 2048u), idesc,
                         accumulate || j != 0);
}

// One warp: rows [from, ROWS) of a tile of `atoms` atoms become zeros (a masked weight of zero times what lies there must be zero)
template <int ROWS = 128>
__device__ __forceinline__ void zero_rows(uint32_t tile_s, int from, int atoms) {
  const int lane = threadIdx.x & 31;
  for (int a = 0; a < atoms; ++a)
    for (uint32_t at = (uint32_t)from * 128u + lane * 16u; at < ROWS * 128u; at += 512u)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile_s + a * (ROWS * 128u) + at), "r"(0u) : "memory");
  fence_proxy_async();
  __syncwarp();
}

// [rows, heads, dim] (bf16, or fp32 where elem is 4) as a tensor map with boxes of 128 bytes of channels of one head in box_rows
// rows; columns behind `dim` and rows behind `rows` read as zeros. False where strides or alignment do not allow it.
inline bool make_head_map(CUtensorMap* map, const void* base, uint32_t rows, int heads, int dim, int64_t row, int64_t head,
                          int box_rows = 128, int elem = 2) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (heads == 1) head = dim;
  if (rows == 1) row = dim;
  const int unit = 16 / elem;
  if (!fn || ((uintptr_t)base & 15) || dim % unit || row % unit || head % unit || row <= 0 || head <= 0) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)head * elem, (cuuint64_t)row * elem};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / elem), 1, (cuuint32_t)box_rows}, estr[3] = {1, 1, 1};
  return fn(map, elem == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims,
            strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tc
}  // namespace rmn
