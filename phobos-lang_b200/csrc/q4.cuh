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

// Sum of x_k w_nk, k < K, where the kernels' split into sum x c - z sum x came to NaN: an infinity in x makes it inf - inf, the
// definition an infinity unless a weight it meets is zero.  Beside x values that are not finite, and groups whose scale or
// zero is not, the other terms do not matter.  Without either `v` stands.  One thread looks through a whole row of X and
// of W (blocks as at the top of gemv_q4.cu); a call without such values never comes here.  (With an infinity in every row of X:
// 1 x 28672 x 8192 111 us in place of 30, 64 x 16384 x 8192 5 ms in place of 58 us.)
inline __device__ float q4_not_finite(float v, const __half* x, const uint8_t* W, int n, int K, int kblocks, int G) {
  const int block_bytes = 1024 + 64 * (128 / G), r = n & 15;
  const uint8_t* blocks = W + static_cast<long long>(n >> 4) * kblocks * block_bytes;
  float sum = 0.0f;
  bool found = false;
  for (int k0 = 0; k0 < K; k0 += 32) {  // (a group has 32 columns or a multiple)
    const uint8_t* block = blocks + static_cast<long long>(k0 >> 7) * block_bytes;
    const float2 sz = __half22float2(reinterpret_cast<const __half2*>(block + 1024)[((k0 & 127) / G) * 16 + r]);
    const bool all = !isfinite(sz.x) || !isfinite(sz.y);
    bool odd = all;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint4 xs = reinterpret_cast<const uint4*>(x + k0)[i];
      const uint32_t word[4] = {xs.x, xs.y, xs.z, xs.w};
#pragma unroll
      for (int j = 0; j < 4; j++) odd = odd || (~word[j] & 0x7c00u) == 0 || (~word[j] & 0x7c000000u) == 0;
    }
    if (!odd) continue;
#pragma unroll 1
    for (int i = 0; i < 32; i++) {
      const float xi = __half2float(x[k0 + i]);
      if (!all && isfinite(xi)) continue;
      const int k = (k0 & 127) + i, w = (k >> 5) * 2 + ((i >> 2) & 1), lane = (r & 7) * 4 + (i >> 3);
      const int in_word = (i & 1) * 2 + ((i >> 1) & 1);  // columns stand in byte order 0, 2, 1, 3
      const uint8_t byte = block[(w >> 2) * 512 + lane * 16 + (w & 3) * 4 + in_word];
      const float c = static_cast<float>((byte >> (4 * (r >> 3))) & 15);
      sum += xi * (sz.x * (c - sz.y));
      found = true;
    }
    if (sum != sum) return sum;
  }
  return found ? sum : v;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace ph
