// Products with 4-bit weights: Y[M,N] = alpha * X[M,K] W[N,K]^T + beta * Y, W[n,k] = s[n,k/G] (c[n,k] - z[n,k/G]).
//
//   sum_k x_k s (c_k - z) = s ( sum_k x_k c_k - z sum_k x_k )      within a group of G columns
// so the matrix unit sees the bare codes, a group's sum is scaled once in f32, and nothing is rounded between X and Y
// but the f32 sums.
//
// Packed weights: blocks of 16 rows x 128 columns, [N / 16][K / 128], each 1024 bytes of codes and then [128 / G][16]
// (scale, zero) pairs of f16.  Lane 4g + t of a warp finds in words w = 2 S + e (bytes (w / 4) * 512 + lane * 16 +
// (w % 4) * 4) the columns 32 S + 8 t + 4 e + {0, 1, 2, 3} of rows g (low nibbles) and g + 8 (high nibbles), columns in
// byte order 0, 2, 1, 3: the A operand of one matrix step from one word.
#include "common.cuh"
#include "kernels.h"
#include "q4.cuh"

namespace ph {
namespace {

constexpr int GV_WARPS = 8;
constexpr uint32_t ONES = 0x3c003c00u;

struct GemvParams {
  const __half* X;
  const uint8_t* W;
  void* Y;
  long long ldx, ldy;
  int M, N, K, G, block_bytes, kblocks;
  float alpha, beta;
  int out_f32;
};

// One CTA: 16 rows of W, 8 * NT rows of X; its warps share the columns out block by block.
template <int NT>
__global__ void __launch_bounds__(GV_WARPS * 32) gemv_q4_kernel(GemvParams p) {
  __shared__ float part[GV_WARPS][16][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int m0 = blockIdx.y * 8 * NT;
  const uint8_t* tile = p.W + static_cast<long long>(blockIdx.x) * p.kblocks * p.block_bytes;
  const int steps_per_group = p.G / 16;
  float y[NT][4] = {};
  for (int kb = warp; kb < p.kblocks; kb += GV_WARPS) {
    const uint8_t* blk = tile + static_cast<long long>(kb) * p.block_bytes;
    uint4 w4[2] = {reinterpret_cast<const uint4*>(blk)[lane], reinterpret_cast<const uint4*>(blk + 512)[lane]};
    const uint32_t* w = reinterpret_cast<const uint32_t*>(w4);
    const __half2* par = reinterpret_cast<const __half2*>(blk + 1024);
    float acc[NT][4] = {}, one[NT][4] = {};
#pragma unroll
    for (int S = 0; S < 4; S++) {
      const int k = kb * 128 + S * 32 + t * 8;
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const int m = m0 + n * 8 + g;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (m < p.M && k < p.K) x = *reinterpret_cast<const uint4*>(p.X + static_cast<long long>(m) * p.ldx + k);
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t c = w[2 * S + e], b0 = e ? x.z : x.x, b1 = e ? x.w : x.y;
          mma_16816(acc[n], c & Q4_LO, c & Q4_HI, (c >> 8) & Q4_LO, (c >> 8) & Q4_HI, b0, b1);
          mma_16816(one[n], ONES, ONES, ONES, ONES, b0, b1);
        }
      }
      if ((2 * S + 2) % steps_per_group == 0) {
        const int grp = (2 * S + 1) / steps_per_group;
        if (kb * 128 + grp * p.G < p.K) {
          const float2 lo = __half22float2(par[grp * 16 + g]), hi = __half22float2(par[grp * 16 + g + 8]);
#pragma unroll
          for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              y[n][i] = fmaf(lo.x, fmaf(-lo.y, one[n][i], acc[n][i] * Q4_LO_UNIT), y[n][i]);
              y[n][2 + i] = fmaf(hi.x, fmaf(-hi.y, one[n][i], acc[n][2 + i] * Q4_HI_UNIT), y[n][2 + i]);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) acc[n][i] = one[n][i] = 0.0f;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int i = 0; i < 4; i++) part[warp][g + (i >> 1) * 8][n * 8 + 2 * t + (i & 1)] = y[n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 8 * NT; i += GV_WARPS * 32) {
    const int r = i & 15, m = m0 + (i >> 4), n = blockIdx.x * 16 + r;
    if (m >= p.M || n >= p.N) continue;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < GV_WARPS; w++) s += part[w][r][i >> 4];
    s *= p.alpha;
    const long long at = m * p.ldy + n;
    if (p.out_f32) {
      float* o = static_cast<float*>(p.Y) + at;
      *o = p.beta == 0.0f ? s : fmaf(p.beta, *o, s);
    } else {
      __half* o = static_cast<__half*>(p.Y) + at;
      *o = __float2half_rn(p.beta == 0.0f ? s : fmaf(p.beta, __half2float(*o), s));
    }
  }
}

struct PackParams {
  const uint8_t* codes;
  const __half* scales;
  const __half* zeros;  // may be null: 8
  uint8_t* out;
  long long ldc, lds, ldz;
  int N, K, G, block_bytes, kblocks;
};

// One CTA of 256 threads: one block; thread i writes one 4-byte word of codes (eight codes of two rows).
__global__ void __launch_bounds__(256) q4_pack_kernel(PackParams p) {
  const int kb = blockIdx.x % p.kblocks, tile = blockIdx.x / p.kblocks, tid = threadIdx.x;
  uint8_t* blk = p.out + static_cast<long long>(blockIdx.x) * p.block_bytes;
  const int lane = (tid & 127) >> 2, w = (tid >> 7) * 4 + (tid & 3), g = lane >> 2, t = lane & 3;
  const int k = kb * 128 + (w >> 1) * 32 + t * 8 + (w & 1) * 4;
  uint32_t word = 0;
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const int byte = c == 1 ? 2 : c == 2 ? 1 : c;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int n = tile * 16 + h * 8 + g;
      const uint32_t v = n < p.N && k + c < p.K ? p.codes[n * p.ldc + k + c] & 15u : 0u;
      word |= v << (byte * 8 + h * 4);
    }
  }
  reinterpret_cast<uint32_t*>(blk)[tid] = word;
  const int groups = 128 / p.G;
  if (tid < groups * 16) {
    const int n = tile * 16 + (tid & 15), grp = kb * groups + (tid >> 4);
    __half2 sz = __floats2half2_rn(0.0f, 0.0f);
    if (n < p.N && grp < p.K / p.G)
      sz = __halves2half2(p.scales[n * p.lds + grp], p.zeros ? p.zeros[n * p.ldz + grp] : __float2half_rn(8.0f));
    reinterpret_cast<__half2*>(blk + 1024)[tid] = sz;
  }
}

int launched(const char** err) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  *err = cudaGetErrorString(e);
  return -3;
}

}  // namespace

size_t q4_packed_bytes(long long N, long long K, int group) {
  return static_cast<size_t>((N + 15) / 16) * static_cast<size_t>((K + 127) / 128) * (1024 + 64 * (128 / group));
}

int launch_q4_pack(const void* codes, long long ldc, const void* scales, long long lds, const void* zeros, long long ldz,
                   void* out, int N, int K, int group, cudaStream_t stream, const char** err) {
  PackParams p{static_cast<const uint8_t*>(codes), static_cast<const __half*>(scales), static_cast<const __half*>(zeros),
               static_cast<uint8_t*>(out), ldc, lds, ldz, N, K, group, 1024 + 64 * (128 / group), (K + 127) / 128};
  const long long blocks = static_cast<long long>((N + 15) / 16) * p.kblocks;
  if (blocks > 0x7fffffffLL) {
    *err = "more than 2^31 - 1 blocks of weights";
    return -2;
  }
  q4_pack_kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p);
  return launched(err);
}

int launch_gemv_q4(const void* X, long long ldx, const void* W, void* Y, long long ldy, int out_f32, int M, int N, int K,
                   int group, float alpha, float beta, int sm_count, uint32_t* status, cudaStream_t stream, const char** err) {
  GemvParams p{static_cast<const __half*>(X), static_cast<const uint8_t*>(W), Y, ldx, ldy, M, N, K, group,
               1024 + 64 * (128 / group), (K + 127) / 128, alpha, beta, out_f32};
  const unsigned tiles = (N + 15) / 16;
  const int nt = M <= 8 ? 1 : M <= 16 ? 2 : 4;
  const dim3 grid(tiles, (M + 8 * nt - 1) / (8 * nt));
  if (grid.y > 65535) {
    *err = "gemv_q4: too many rows of X";
    return -2;
  }
  if (nt == 1)
    gemv_q4_kernel<1><<<grid, GV_WARPS * 32, 0, stream>>>(p);
  else if (nt == 2)
    gemv_q4_kernel<2><<<grid, GV_WARPS * 32, 0, stream>>>(p);
  else
    gemv_q4_kernel<4><<<grid, GV_WARPS * 32, 0, stream>>>(p);
  return launched(err);
}

}  // namespace ph
