// Shared by the kernels that work on 4-bit codes: the warp-level matrix step they use and the way codes reach it.
//
// A 32-bit word holds eight codes, code i in bits 4i..4i+3.  `word & 0x000f000f` is two codes that, read as f16,
// are the denormals c * 2^-24; `word & 0x00f000f0` is two codes as c * 2^-20.  The matrix unit multiplies f16
// denormals exactly and sums in f32, so a code costs five integer operations per eight (two masks, one shift, two
// masks) and no conversion: the power of two goes into the scale that the f32 result is multiplied by anyway.
//
// mma.sync (m16n8k16, f32 accumulate) is used instead of tcgen05.mma because these products have 1 to 16 columns and
// are bound by the bytes of the codes: tcgen05 takes its operands from shared or tensor memory, and writing the
// widened codes there and reading them back would move eight times the bytes that arrive from HBM, more than
// shared memory delivers at the HBM rate.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ph {

constexpr uint32_t Q4_LO = 0x000f000fu, Q4_HI = 0x00f000f0u;
constexpr float Q4_LO_UNIT = 16777216.0f;  // 2^24: what a low-nibble product is multiplied by
constexpr float Q4_HI_UNIT = 1048576.0f;   // 2^20: the same for a high-nibble one

// D (16 x 8, f32) += A (16 x 16, f16) B (16 x 8, f16).  Lane 4g + t holds of A rows g (a0, a2) and g + 8 (a1, a3),
// columns 2t, 2t + 1 (a0, a1) and 2t + 8, 2t + 9 (a2, a3); of B the same rows-of-k in column g; of D rows g (c0, c1)
// and g + 8 (c2, c3), columns 2t, 2t + 1.
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with D = A B.
__device__ __forceinline__ void mma_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// Transposes an 8 x 8 matrix of 16-bit values held two to a lane (lane 4r + t: row r, columns 2t, 2t + 1).
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace ph
