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
// The kernel: a CTA of eight multiplying warps and one that copies.  The multiplying warps form WR x WK: WR along the rows
// of W (RT tiles of 16 each), WK along the columns (a block of 128 each).  A stage of the ring holds WR RT x WK blocks and
// the WK * 128 columns of up to 8 NT rows of X, brought by bulk copies; X rows stand 64 bytes off a multiple of 128
// apart, so that a lane's 16-byte reads (the B operand of two matrix steps) meet no bank twice.  CTAs stay: each takes
// row groups in turn, and the copying warp runs ahead into the next group while the last one is written.
#include <atomic>

#include "common.cuh"
#include "kernels.h"
#include "q4.cuh"

namespace ph {
namespace {

constexpr int GV_WARPS = 8;                            // multiplying warps
constexpr int GV_THREADS = (GV_WARPS + 1) * 32;
constexpr uint32_t ONES = 0x3c003c00u;                 // two f16 ones
enum : uint32_t { SITE_GEMV_FULL = 0x42, SITE_GEMV_EMPTY = 0x43 };

struct GemvParams {
  const __half* X;
  const uint8_t* W;
  void* Y;
  long long ldx, ldy;
  int M, N, K, G, block_bytes, kblocks, tiles;         // tiles of 16 rows
  int row_groups, m_groups;
  float alpha, beta;
  int out_f32;
  uint32_t* status;
};

template <int NT, int RT, int WR>
struct GemvShape {
  static constexpr int WK = GV_WARPS / WR, TILES = RT * WR, ROWS = 16 * TILES, COLS = 8 * NT;
  static constexpr int X_PITCH = WK * 256 + 64, X_BYTES = COLS * X_PITCH;
  static constexpr int W_MOST = TILES * WK * (1024 + 256);  // (at G = 32)
  static constexpr int STAGE = (X_BYTES + W_MOST + 127) / 128 * 128;
  static constexpr int OUT_PITCH = ROWS + 4, OUT = WK * COLS * OUT_PITCH * 4;
  static constexpr int HEAD = 256;
  static constexpr int TWO = (226 * 1024 / 2 - 1024 - HEAD - OUT) / STAGE;  // stages with two CTAs on an SM
  static constexpr int ROOM = TWO >= 2 ? TWO : (226 * 1024 - HEAD - OUT) / STAGE;
  static constexpr int STAGES = ROOM > 6 ? 6 : ROOM;
  static constexpr int SMEM = HEAD + STAGES * STAGE + OUT;
  static_assert(STAGES >= 2 && SMEM <= 227 * 1024, "stages of the ring");
};

__device__ __forceinline__ void gemv_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int NT, int RT, int WR>
__global__ void __launch_bounds__(GV_THREADS) gemv_q4_kernel(GemvParams p) {
  using S = GemvShape<NT, RT, WR>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty = full + S::STAGES;
  uint32_t* abort_flag = reinterpret_cast<uint32_t*>(smem + 192);
  uint8_t* ring = smem + S::HEAD;
  float* out = reinterpret_cast<float*>(ring + S::STAGES * S::STAGE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (threadIdx.x < S::STAGES) {
    mbar_init(full + threadIdx.x, 1);
    mbar_init(empty + threadIdx.x, GV_WARPS);
  }
  if (threadIdx.x == 0) *abort_flag = 0;
  fence_mbar_init();
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const WaitCtx ctx{abort_flag, p.status};
  const int chunks = (p.kblocks + S::WK - 1) / S::WK, groups = p.row_groups * p.m_groups;
  uint32_t it = 0;
  if (warp == GV_WARPS) {
    // ---- copies ---------------------------------------------------------------------------------------------------------
    for (int grp = blockIdx.x; grp < groups; grp += gridDim.x) {
      // neighbours take the same rows of W for other rows of X: W comes from HBM once
      const int tile0 = grp / p.m_groups * S::TILES, m0 = grp % p.m_groups * S::COLS;
      const int n_tiles = min(S::TILES, p.tiles - tile0), n_m = min(S::COLS, p.M - m0);
      for (int c = 0; c < chunks; c++, it++) {
        const int st = it % S::STAGES, kb = c * S::WK;
        if (it >= S::STAGES && !mbar_wait_warp(empty + st, (it / S::STAGES - 1) & 1, SITE_GEMV_EMPTY, ctx)) return;
        const int n_kb = min(S::WK, p.kblocks - kb);
        const uint32_t w_bytes = n_kb * p.block_bytes, x_bytes = min(n_kb * 128, p.K - kb * 128) * 2;
        uint8_t* stage = ring + st * S::STAGE;
        if (lane == 0) mbar_arrive_expect_tx(full + st, n_tiles * w_bytes + n_m * x_bytes);
        __syncwarp();
        for (int i = lane; i < n_tiles + n_m; i += 32) {
          if (i < n_tiles)
            gemv_bulk_load(stage + S::X_BYTES + i * S::WK * p.block_bytes,
                           p.W + (static_cast<long long>(tile0 + i) * p.kblocks + kb) * p.block_bytes, w_bytes, full + st);
          else
            gemv_bulk_load(stage + (i - n_tiles) * S::X_PITCH, p.X + (m0 + i - n_tiles) * p.ldx + kb * 128, x_bytes, full + st);
        }
      }
    }
    return;
  }
  // ---- products -----------------------------------------------------------------------------------------------------------
  const int wr = warp / S::WK, wk = warp % S::WK;
  const int steps_per_group = p.G / 16;
  for (int grp = blockIdx.x; grp < groups; grp += gridDim.x) {
    const int tile0 = grp / p.m_groups * S::TILES, m0 = grp % p.m_groups * S::COLS;
    float y[RT][NT][4];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) y[r][n][i] = 0.0f;
#pragma unroll 1
    for (int c = 0; c < chunks; c++, it++) {
      const int st = it % S::STAGES, kb = c * S::WK + wk;
      const bool ok = mbar_wait_warp(full + st, (it / S::STAGES) & 1, SITE_GEMV_FULL, ctx);  // else recorded; nothing hangs
      const uint8_t* stage = ring + st * S::STAGE;
      if (ok && kb < p.kblocks) {
        const uint8_t* x_at = stage + g * S::X_PITCH + wk * 256 + t * 16;
        const uint8_t* blk[RT];
        uint32_t w[RT][8];
#pragma unroll
        for (int r = 0; r < RT; r++) {
          blk[r] = stage + S::X_BYTES + ((wr * RT + r) * S::WK + wk) * p.block_bytes;
          const uint4 lo = reinterpret_cast<const uint4*>(blk[r])[lane], hi = reinterpret_cast<const uint4*>(blk[r] + 512)[lane];
          w[r][0] = lo.x; w[r][1] = lo.y; w[r][2] = lo.z; w[r][3] = lo.w;
          w[r][4] = hi.x; w[r][5] = hi.y; w[r][6] = hi.z; w[r][7] = hi.w;
        }
        float acc[RT][NT][4], one[NT][4];
#pragma unroll
        for (int s = 0; s < 4; s++) {
          if ((2 * s) % steps_per_group == 0) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
              for (int i = 0; i < 4; i++) {
                one[n][i] = 0.0f;
#pragma unroll
                for (int r = 0; r < RT; r++) acc[r][n][i] = 0.0f;
              }
          }
          uint4 x[NT];
#pragma unroll
          for (int n = 0; n < NT; n++) x[n] = *reinterpret_cast<const uint4*>(x_at + n * 8 * S::X_PITCH + s * 64);
#pragma unroll
          for (int e = 0; e < 2; e++) {
#pragma unroll
            for (int n = 0; n < NT; n++) mma_16816(one[n], ONES, ONES, ONES, ONES, e ? x[n].z : x[n].x, e ? x[n].w : x[n].y);
#pragma unroll
            for (int r = 0; r < RT; r++) {
              const uint32_t a = w[r][2 * s + e], a2 = a >> 8;
#pragma unroll
              for (int n = 0; n < NT; n++)
                mma_16816(acc[r][n], a & Q4_LO, a & Q4_HI, a2 & Q4_LO, a2 & Q4_HI, e ? x[n].z : x[n].x, e ? x[n].w : x[n].y);
            }
          }
          if ((2 * s + 2) % steps_per_group == 0) {
            const int in_block = (2 * s + 1) / steps_per_group;
            if (kb * 128 + in_block * p.G < p.K) {  // (behind K a stage holds whatever it held)
#pragma unroll
              for (int r = 0; r < RT; r++) {
                const __half2* par = reinterpret_cast<const __half2*>(blk[r] + 1024) + in_block * 16 + g;
                const float2 lo = __half22float2(par[0]), hi = __half22float2(par[8]);
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                  for (int i = 0; i < 2; i++) {
                    y[r][n][i] = fmaf(lo.x, fmaf(-lo.y, one[n][i], acc[r][n][i] * Q4_LO_UNIT), y[r][n][i]);
                    y[r][n][2 + i] = fmaf(hi.x, fmaf(-hi.y, one[n][i], acc[r][n][2 + i] * Q4_HI_UNIT), y[r][n][2 + i]);
                  }
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + st);
    }
    // ---- join the columns' warps, write ------------------------------------------------------------------------------------
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          out[(wk * S::COLS + n * 8 + 2 * t + (i & 1)) * S::OUT_PITCH + (wr * RT + r) * 16 + g + (i >> 1) * 8] = y[r][n][i];
    named_bar_sync(1, GV_WARPS * 32);
    for (int i = threadIdx.x; i < S::COLS * S::ROWS; i += GV_WARPS * 32) {
      const int row = i % S::ROWS, col = i / S::ROWS, m = m0 + col, n = tile0 * 16 + row;
      if (m >= p.M) break;
      if (n >= p.N) continue;
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < S::WK; k++) v += out[(k * S::COLS + col) * S::OUT_PITCH + row];
      v *= p.alpha;
      const long long at = m * p.ldy + n;
      if (p.out_f32) {
        float* o = static_cast<float*>(p.Y) + at;
        *o = p.beta == 0.0f ? v : fmaf(p.beta, *o, v);
      } else {
        __half* o = static_cast<__half*>(p.Y) + at;
        *o = __float2half_rn(p.beta == 0.0f ? v : fmaf(p.beta, __half2float(*o), v));
      }
    }
    named_bar_sync(1, GV_WARPS * 32);
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

namespace {

// CTAs of a kernel that share an SM, asked for once per device.
template <int NT, int RT, int WR>
cudaError_t per_sm_of(int* per_sm) {
  using S = GemvShape<NT, RT, WR>;
  auto kernel = gemv_q4_kernel<NT, RT, WR>;
  static std::atomic<int> known[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  *per_sm = dev < 64 ? known[dev].load(std::memory_order_acquire) : 0;
  if (*per_sm > 0) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, kernel, GV_THREADS, S::SMEM);
  if (e != cudaSuccess) return e;
  *per_sm = *per_sm < 1 ? 1 : *per_sm;
  if (dev < 64) known[dev].store(*per_sm, std::memory_order_release);
  return cudaSuccess;
}

template <int NT, int RT, int WR>
cudaError_t launch_shape(GemvParams& p, int sm_count, cudaStream_t stream) {
  using S = GemvShape<NT, RT, WR>;
  int per_sm = 0;
  const cudaError_t e = per_sm_of<NT, RT, WR>(&per_sm);
  if (e != cudaSuccess) return e;
  p.row_groups = (p.tiles + S::TILES - 1) / S::TILES;
  p.m_groups = (p.M + S::COLS - 1) / S::COLS;
  const long long groups = static_cast<long long>(p.row_groups) * p.m_groups;
  const long long room = static_cast<long long>(sm_count) * per_sm;
  return launch_with_pdl(gemv_q4_kernel<NT, RT, WR>, dim3(static_cast<unsigned>(groups < room ? groups : room)), dim3(GV_THREADS),
                         S::SMEM, stream, p);
}

// As many rows of W to a CTA as leave every SM one: fewer rows mean that more CTAs read X, more that some SMs have none.
template <int NT>
cudaError_t launch_rows_of(GemvParams& p, int sm_count, cudaStream_t stream) {
  if constexpr (NT == 8) {
    if (p.tiles >= 8 * sm_count) return launch_shape<NT, 1, 8>(p, sm_count, stream);
    if (p.tiles >= 4 * sm_count) return launch_shape<NT, 1, 4>(p, sm_count, stream);
  } else {
    if (p.tiles >= 8 * sm_count) return launch_shape<NT, 2, 4>(p, sm_count, stream);
    if (p.tiles >= 4 * sm_count) return launch_shape<NT, 2, 2>(p, sm_count, stream);
  }
  if constexpr (NT == 8) {  // (sixteen rows a CTA would leave no room for two stages)
    return launch_shape<NT, 1, 2>(p, sm_count, stream);
  } else {
    if (p.tiles >= 2 * sm_count) return launch_shape<NT, 1, 2>(p, sm_count, stream);
    return launch_shape<NT, 1, 1>(p, sm_count, stream);
  }
}

}  // namespace

int launch_gemv_q4(const void* X, long long ldx, const void* W, void* Y, long long ldy, int out_f32, int M, int N, int K,
                   int group, float alpha, float beta, int sm_count, uint32_t* status, cudaStream_t stream, const char** err) {
  GemvParams p{static_cast<const __half*>(X), static_cast<const uint8_t*>(W), Y, ldx, ldy, M, N, K, group,
               1024 + 64 * (128 / group), (K + 127) / 128, (N + 15) / 16, 0, 0, alpha, beta, out_f32, status};
  cudaError_t e = M <= 8    ? launch_rows_of<1>(p, sm_count, stream)
                  : M <= 16 ? launch_rows_of<2>(p, sm_count, stream)
                  : M <= 32 ? launch_rows_of<4>(p, sm_count, stream)
                            : launch_rows_of<8>(p, sm_count, stream);
  if (e == cudaSuccess) return 0;
  *err = cudaGetErrorString(e);
  return -3;
}

}  // namespace ph
