// Pieces shared by the tcgen05 attention kernels: tiles of keys in the 128-byte swizzle, the exponential and its packing, the maximum.
#pragma once
#include "tcgen05.cuh"

namespace pmm {

using bf16 = __nv_bfloat16;

constexpr int kAtKeys = 128;    // keys per tile
constexpr int kAtBox = 64;      // keys per TMA box (inside one page)
constexpr int kAtDhBlock = 64;  // head-size columns per sub-tile (128 bytes of bfloat16)
constexpr float kAtLazy = 8.f;  // how far (log2) a row's maximum may run ahead of the one in use
constexpr int kAtKvSub = kAtKeys * kAtDhBlock * 2;  // 16 KB: 128 keys x 64 head-size columns

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
__device__ __forceinline__ float at_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

}  // namespace pmm
