// Pieces shared by the tcgen05 attention kernels: tile sizes, tensor-memory layout and instruction descriptors, tensor-memory
// accesses with four threads per row, and the packing of a row's probabilities.
#pragma once
#include "tcgen05.cuh"

namespace pmm {

using bf16 = __nv_bfloat16;

constexpr int kAtKeys = 128;    // keys per tile
constexpr int kAtBox = 64;      // keys per TMA box (inside one page)
constexpr int kAtDhBlock = 64;  // head-size columns per sub-tile (128 bytes of bfloat16)
constexpr float kAtLazy = 8.f;  // how far (log2) a row's maximum may run ahead of the one in use
constexpr int kAtBoxCap = 512;  // boxes of the block's key range whose rows of the pool are kept in shared memory
constexpr int kAtKvSub = kAtKeys * kAtDhBlock * 2;  // 16 KB: 128 keys x 64 head-size columns
constexpr int kAtRing = 3;                          // K and V tiles in flight
__host__ __device__ constexpr int at_q_sub(int rows) { return rows * kAtDhBlock * 2; }      // a sub-tile of Q (64 head-size columns) or of P (64 keys)
__host__ __device__ constexpr int at_threads(int rows) { return 64 + 2 * rows; }            // producer, issuer, a warp per 16 rows
__host__ __device__ constexpr size_t at_smem(int dh, int rows) {  // Q, the ring (each head size / 64 sub-tiles), P
  return static_cast<size_t>(dh / kAtDhBlock) * (at_q_sub(rows) + kAtRing * kAtKvSub) + 2 * at_q_sub(rows) + 1024 /*alignment*/;
}
// Tensor memory.  128 rows: S in columns 0..127, O behind it.  64 rows: a product leaves row i in lane 32 (i / 16) + i % 16,
// so S takes the lower 16 lanes of every warp's 32 and O the upper 16 of the same columns.
__host__ __device__ constexpr int at_tmem_cols(int rows) { return rows == 64 ? 128 : 256; }
__host__ __device__ constexpr unsigned at_o_offset(int rows) { return rows == 64 ? (16u << 16) : static_cast<unsigned>(kAtKeys); }

// kind::f16 instruction descriptors: float accumulate, bfloat16 operands, A K-major.
__host__ __device__ constexpr unsigned at_idesc_s(int rows) {  // B = K tile, K-major
  return (1u << 4) | (1u << 7) | (1u << 10) | ((kAtKeys >> 3) << 17) | (static_cast<unsigned>(rows >> 4) << 24);
}
__host__ __device__ constexpr unsigned at_idesc_o(int rows) {  // B = 64 columns of the V tile, MN-major
  return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((kAtDhBlock >> 3) << 17) | (static_cast<unsigned>(rows >> 4) << 24);
}

__device__ __forceinline__ float at_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned at_pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&v);
}
// Byte offset of 16-byte chunk `chunk` (0..7) of row `row` in a [rows][64] bfloat16 tile with the
// 128-byte swizzle that TMA and the tensor core use (8-row groups of 1024 bytes).
__device__ __forceinline__ int at_swizzled(int row, int chunk) {
  return (row >> 3) * 1024 + (row & 7) * 128 + ((chunk ^ (row & 7)) << 4);
}

// 16 lanes of tensor memory x 64 columns: lane l of the warp gets columns 4 i + l % 4 of rows l / 4 (r[2 i]) and l / 4 + 8 (r[2 i + 1]).
__device__ __forceinline__ void at_tmem_ld(unsigned taddr, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x128b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// The same for 32 columns, and its store.
__device__ __forceinline__ void at_tmem_ld32(unsigned taddr, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x128b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void at_tmem_st32(unsigned taddr, const unsigned* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Two columns' values of one row, k = column % 4 of this lane: columns 4 i + k (x0) and 4 i + 4 + k (x1), i even, become the
// word (two neighbouring bfloat16) of the row's 16-byte piece i / 2 that this lane owns, word 2 (k & 1) + (k >> 1).
__device__ __forceinline__ unsigned at_pair(float x0, float x1, unsigned sel) {
  const unsigned own = at_pack(x0, x1);
  return __byte_perm(own, __shfl_xor_sync(0xffffffffu, own, 1), sel);
}
__device__ __forceinline__ float at_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Place of a tile among the copies: K_0, K_1, V_0, K_2, V_1, ..., K_{n-1}, V_{n-2}, V_{n-1}, the order of the products.
__device__ __forceinline__ int at_k_item(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int at_v_item(int j, int n) { return j + 1 < n ? 2 * j + 2 : 2 * j + 1; }

}  // namespace pmm
