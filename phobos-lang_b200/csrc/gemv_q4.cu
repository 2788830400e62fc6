// Products with 4-bit weights: Y[M,N] = alpha * X[M,K] W[N,K]^T + beta * Y, W[n,k] = s[n,k/G] (c[n,k] - z[n,k/G]).
//
//   sum_k x_k s (c_k - z) = s ( sum_k x_k c_k - z sum_k x_k )      within a group of G columns
// so the matrix unit sees the bare codes, a group's sum is scaled once in f32, and nothing is rounded between X and Y
// but the f32 sums.  Where infinities in X make the two sums cancel to NaN, the sum is formed from the definition
// (q4_not_finite).
//
// Packed weights: blocks of 16 rows x 128 columns, [N / 16][K / 128], each 1024 bytes of codes and then [128 / G][16]
// (scale, zero) pairs of f16.  Lane 4g + t of a warp finds in words w = 2 S + e (bytes (w / 4) * 512 + lane * 16 +
// (w % 4) * 4) the columns 32 S + 8 t + 4 e + {0, 1, 2, 3} of rows g (low nibbles) and g + 8 (high nibbles), columns in
// byte order 0, 2, 1, 3: the A operand of one matrix step from one word.
// The kernel: a CTA of eight multiplying warps and one that copies.  The multiplying warps form WR x WK: WR along the rows
// of W (RT tiles of 16 each), WK along the columns (a block of 128 each).  A stage of the ring holds WR RT x WK blocks and
// WK * 128 columns of up to eight rows of X, brought by bulk copies; X rows stand 64 bytes off a multiple of 128 apart, so
// that a lane's 16-byte reads (the B operand of two matrix steps) meet no bank twice.  The tiles of W are dealt out evenly
// over a grid that fills the GPU.  A CTA whose share is not a multiple of WR RT does the products of the places without a
// tile all the same, on what the ring held; that is part of what 5 x 11001 x 4096, G = 64, pays: its CTAs have two or three
// tiles in a shape of four, and it takes 10.9 us, 7.9 with the products left out, where the bytes are 3.9.
// Measured: 1 x 28672 x 8192, G = 128: 27.9 us, 4.5 TB/s (23.4 us without the products; 122 instructions for a block of 16 x
// 128, half of them masks and shifts; neither HBM nor a pipe nor the issue slots are full: half of them, by four warps a
// scheduler that wait for loads and for the pipes in turn); 1 x 4096 x 4096: 4.9 us back to back in a graph.  Four tiles a
// warp (x read and summed once for all of them) took 31 us where two took 34, sixteen rows a CTA in every case 37.
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "q4.cuh"

namespace ph {
namespace {

constexpr int GV_WARPS = 8;                            // multiplying warps
constexpr int GV_PER_SM = 2;                            // CTAs that share an SM
constexpr int GV_THREADS = (GV_WARPS + 1) * 32;
constexpr uint32_t ONES = 0x3c003c00u;                 // two f16 ones
enum : uint32_t { SITE_GEMV_FULL = 0x42, SITE_GEMV_EMPTY = 0x43 };

struct GemvParams {
  const __half* X;
  const uint8_t* W;
  void* Y;
  long long ldx, ldy;
  int M, N, K, kblocks, tiles;         // tiles of 16 rows
  int stages, stage_bytes;
  float alpha, beta;
  int out_f32;
  uint32_t* status;
};

template <int RT, int WR, int GS>
struct GemvShape {
  static constexpr int WK = GV_WARPS / WR, TILES = RT * WR, ROWS = 16 * TILES;
  static constexpr int X_PITCH = WK * 256 + 64;
  static constexpr int BLOCK = 1024 + 64 * (8 / GS);   // GS matrix steps of 16 columns are a group
  static constexpr int W_BYTES = TILES * WK * BLOCK;
  static constexpr int OUT_PITCH = ROWS + 4, OUT = WK * 8 * OUT_PITCH * 4;
  static constexpr int HEAD = 256, MOST_STAGES = 8;
  static_assert(X_PITCH % 128 == 64 && W_BYTES % 64 == 0, "shared memory layout");
};

// CTA (x, y): its share of the tiles of W, rows 8y .. 8y + 7 of X.
template <int RT, int WR, int GS>
__global__ void __launch_bounds__(GV_THREADS, GV_PER_SM) gemv_q4_kernel(GemvParams p) {
  using S = GemvShape<RT, WR, GS>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty = full + S::MOST_STAGES;
  uint32_t* abort_flag = reinterpret_cast<uint32_t*>(smem + 192);
  static_assert(16 * S::MOST_STAGES <= 192, "shared memory head");
  float* out = reinterpret_cast<float*>(smem + S::HEAD);
  uint8_t* ring = smem + S::HEAD + S::OUT;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (threadIdx.x < p.stages) {
    mbar_init(full + threadIdx.x, 1);
    mbar_init(empty + threadIdx.x, GV_WARPS);
  }
  if (threadIdx.x == 0) abort_flag[0] = abort_flag[1] = 0;
  fence_mbar_init();
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const WaitCtx ctx{abort_flag, p.status};
  const int chunks = (p.kblocks + S::WK - 1) / S::WK;
  const int first = static_cast<int>(static_cast<long long>(p.tiles) * blockIdx.x / gridDim.x);
  const int last = static_cast<int>(static_cast<long long>(p.tiles) * (blockIdx.x + 1) / gridDim.x);
  const int m0 = blockIdx.y * 8, n_m = min(8, p.M - m0);
  const int x_bytes = n_m * S::X_PITCH;  // of a stage
  int st = 0;
  uint32_t parity = 0;
  if (warp == GV_WARPS) {
    // ---- copies ---------------------------------------------------------------------------------------------------------
    bool refill = false;
    for (int tile0 = first; tile0 < last; tile0 += S::TILES) {
      const int n_tiles = min(S::TILES, last - tile0);
      for (int c = 0; c < chunks; c++) {
        const int kb = c * S::WK, n_kb = min(S::WK, p.kblocks - kb);
        if (refill && !mbar_wait_warp(empty + st, parity ^ 1, SITE_GEMV_EMPTY, ctx)) return;
        const uint32_t w_each = n_kb * S::BLOCK, x_each = min(n_kb * 128, p.K - kb * 128) * 2;
        uint8_t* stage = ring + st * p.stage_bytes;
        if (lane == 0) mbar_arrive_expect_tx(full + st, n_tiles * w_each + n_m * x_each);
        __syncwarp();
        if (lane < n_tiles)
          bulk_load(stage + x_bytes + lane * S::WK * S::BLOCK, p.W + (static_cast<long long>(tile0 + lane) * p.kblocks + kb) * S::BLOCK,
                         w_each, full + st);
        else if (lane - n_tiles < n_m)
          bulk_load(stage + (lane - n_tiles) * S::X_PITCH, p.X + (m0 + lane - n_tiles) * p.ldx + kb * 128, x_each, full + st);
        if (++st == p.stages) {
          st = 0;
          parity ^= 1;
          refill = true;
        }
      }
    }
    return;
  }
  // ---- products -----------------------------------------------------------------------------------------------------------
  static_assert(S::TILES + 8 <= 32, "a lane for every copy");
  const int wr = warp / S::WK, wk = warp % S::WK;
  const int x_row = min(g, n_m - 1) * S::X_PITCH;  // columns of the product behind the last row repeat it
  for (int tile0 = first; tile0 < last; tile0 += S::TILES) {
    float y[RT][4];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int i = 0; i < 4; i++) y[r][i] = 0.0f;
#pragma unroll 1
    for (int c = 0; c < chunks; c++) {
      const int kb = c * S::WK + wk;
      const bool ok = mbar_wait_copies(full + st, parity, SITE_GEMV_FULL, ctx, abort_flag + 1);  // else recorded; nothing hangs
      const uint8_t* stage = ring + st * p.stage_bytes;
      auto block = [&](auto whole) {  // (behind K a stage holds whatever it held)
        const uint8_t* x_at = stage + x_row + wk * 256 + t * 16;
        const uint8_t* blk = stage + x_bytes + (wr * S::WK + wk) * S::BLOCK;  // of tile wr; the warp's next is WR further
        constexpr int NEXT = WR * S::WK * S::BLOCK;
        float acc[RT][4], one[4];
#pragma unroll
        for (int half = 0; half < 2; half++) {
          uint32_t w[RT][4];
#pragma unroll
          for (int r = 0; r < RT; r++) {
            const uint4 v = reinterpret_cast<const uint4*>(blk + r * NEXT + half * 512)[lane];
            w[r][0] = v.x; w[r][1] = v.y; w[r][2] = v.z; w[r][3] = v.w;
          }
#pragma unroll
          for (int s = 2 * half; s < 2 * half + 2; s++) {
            const uint4 x = *reinterpret_cast<const uint4*>(x_at + s * 64);
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const bool fresh = (2 * s + e) % GS == 0;
              const uint32_t b0 = e ? x.z : x.x, b1 = e ? x.w : x.y;
              if (fresh)
                mma_16816_first(one, ONES, ONES, ONES, ONES, b0, b1);
              else
                mma_16816(one, ONES, ONES, ONES, ONES, b0, b1);
#pragma unroll
              for (int r = 0; r < RT; r++) {
                const uint32_t a = w[r][(2 * s + e) & 3], a2 = a >> 8;
                if (fresh)
                  mma_16816_first(acc[r], a & Q4_LO, a & Q4_HI, a2 & Q4_LO, a2 & Q4_HI, b0, b1);
                else
                  mma_16816(acc[r], a & Q4_LO, a & Q4_HI, a2 & Q4_LO, a2 & Q4_HI, b0, b1);
              }
            }
            if ((2 * s + 2) % GS == 0) {
              const int in_block = (2 * s + 1) / GS;
              if (decltype(whole)::value || kb * 128 + in_block * (16 * GS) < p.K) {
#pragma unroll
                for (int r = 0; r < RT; r++) {
                  const __half2* par = reinterpret_cast<const __half2*>(blk + r * NEXT + 1024) + in_block * 16 + g;
                  const float2 lo = __half22float2(par[0]), hi = __half22float2(par[8]);
#pragma unroll
                  for (int i = 0; i < 2; i++) {
                    y[r][i] = fmaf(lo.x, fmaf(-lo.y, one[i], acc[r][i] * Q4_LO_UNIT), y[r][i]);
                    y[r][2 + i] = fmaf(hi.x, fmaf(-hi.y, one[i], acc[r][2 + i] * Q4_HI_UNIT), y[r][2 + i]);
                  }
                }
              }
            }
          }
        }
      };
      if (ok && kb < p.kblocks) {
        if (kb * 128 + 128 <= p.K)
          block(std::true_type{});
        else
          block(std::false_type{});
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + st);
      if (++st == p.stages) {
        st = 0;
        parity ^= 1;
      }
    }
    // ---- join the columns' warps, write ------------------------------------------------------------------------------------
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int i = 0; i < 4; i++) out[(wk * 8 + 2 * t + (i & 1)) * S::OUT_PITCH + (r * WR + wr) * 16 + g + (i >> 1) * 8] = y[r][i];
    bool nan = false;
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int i = 0; i < 4; i++) nan = nan || y[r][i] != y[r][i];
    nan = named_bar_or(1, GV_WARPS * 32, nan);
    const int n_rows = min(min(S::TILES, last - tile0) * 16, p.N - tile0 * 16);
    auto write = [&](auto look) {
      for (int i = threadIdx.x; i < n_m * S::ROWS; i += GV_WARPS * 32) {
        const int row = i % S::ROWS, col = i / S::ROWS;
        if (row >= n_rows) continue;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < S::WK; k++) v += out[(k * 8 + col) * S::OUT_PITCH + row];
        if (decltype(look)::value && v != v)
          v = q4_not_finite(v, p.X + (m0 + col) * p.ldx, p.W, tile0 * 16 + row, p.K, p.kblocks, GS * 16);
        v *= p.alpha;
        const long long at = (m0 + col) * p.ldy + tile0 * 16 + row;
        if (p.out_f32) {
          float* o = static_cast<float*>(p.Y) + at;
          *o = p.beta == 0.0f ? v : fmaf(p.beta, *o, v);
        } else {
          __half* o = static_cast<__half*>(p.Y) + at;
          *o = __float2half_rn(p.beta == 0.0f ? v : fmaf(p.beta, __half2float(*o), v));
        }
      }
    };
    if (__builtin_expect(nan, 0))
      write(std::true_type{});
    else
      write(std::false_type{});
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
  pdl_wait();
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
  const cudaError_t e = launch_with_pdl(q4_pack_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, p);
  if (e == cudaSuccess) return 0;
  *err = cudaGetErrorString(e);
  return -3;
}

namespace {

template <int RT, int WR, int GS>
cudaError_t launch_shape(GemvParams& p, int sm_count, cudaStream_t stream) {
  using S = GemvShape<RT, WR, GS>;
  constexpr int MOST = 227 * 1024 / GV_PER_SM - 1024;  // bytes of a CTA
  static std::atomic<bool> known[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !known[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(gemv_q4_kernel<RT, WR, GS>, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST);
    if (e != cudaSuccess) return e;
    if (dev < 64) known[dev].store(true, std::memory_order_release);
  }
  const int room = MOST - S::HEAD - S::OUT;
  static_assert((MOST - S::HEAD - S::OUT) / ((8 * S::X_PITCH + S::W_BYTES + 127) / 128 * 128) >= 2, "two stages at least");
  p.stage_bytes = ((p.M < 8 ? p.M : 8) * S::X_PITCH + S::W_BYTES + 127) / 128 * 128;
  p.stages = room / p.stage_bytes < S::MOST_STAGES ? room / p.stage_bytes : S::MOST_STAGES;
  const int ctas = p.tiles < GV_PER_SM * sm_count ? p.tiles : GV_PER_SM * sm_count;
  return launch_with_pdl(gemv_q4_kernel<RT, WR, GS>, dim3(ctas, (p.M + 7) / 8), dim3(GV_THREADS),
                         S::HEAD + S::OUT + p.stages * p.stage_bytes, stream, p);
}

// The shape whose tiles are at least a CTA's share, so that its share is one pass over X.
template <int GS>
cudaError_t launch_group(GemvParams& p, int sm_count, cudaStream_t stream) {
  const int share = (p.tiles + GV_PER_SM * sm_count - 1) / (GV_PER_SM * sm_count);
  if (share <= 1) return launch_shape<1, 1, GS>(p, sm_count, stream);
  if (share <= 2) return launch_shape<2, 1, GS>(p, sm_count, stream);
  if (share <= 4) return launch_shape<2, 2, GS>(p, sm_count, stream);
  if constexpr (GS == 2)
    return launch_shape<2, 4, GS>(p, sm_count, stream);  // (four tiles a warp leave no room for two stages)
  else
    return launch_shape<4, 2, GS>(p, sm_count, stream);
}

}  // namespace

int launch_gemv_q4(const void* X, long long ldx, const void* W, void* Y, long long ldy, int out_f32, int M, int N, int K,
                   int group, float alpha, float beta, int sm_count, uint32_t* status, cudaStream_t stream, const char** err) {
  // (more than 8 * 65535 rows of X are more than this kernel's grid holds)
  if (M > 8 && (M > 8 * 65535 || gemv_q4_tc_is_faster(M, N, K, group, sm_count)))
    return launch_gemv_q4_tc(X, ldx, W, Y, ldy, out_f32, M, N, K, group, alpha, beta, sm_count, status, stream, err);
  GemvParams p{static_cast<const __half*>(X), static_cast<const uint8_t*>(W), Y, ldx, ldy, M, N, K, (K + 127) / 128,
               (N + 15) / 16, 0, 0, alpha, beta, out_f32, status};
  const cudaError_t e = group == 128  ? launch_group<8>(p, sm_count, stream)
                        : group == 64 ? launch_group<4>(p, sm_count, stream)
                                      : launch_group<2>(p, sm_count, stream);
  if (e == cudaSuccess) return 0;
  *err = cudaGetErrorString(e);
  return -3;
}

}  // namespace ph
