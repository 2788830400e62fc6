// Products with 4-bit weights for more than eight rows of X, on the fifth-generation tensor cores (same operator and same
// packed weights as gemv_q4.cu).
//
// What bounds the warp-level form there: a 16 x 8 x 16 step takes the matrix unit of an SM quarter 8 cycles, so that 32
// rows of X cost more time in it than the weights take to arrive.  Here W is the A operand of tcgen05.mma: 128 rows of W
// x 16 columns in tensor memory, 16, 32 or 64 rows of X beside it in shared memory.  A lane of tensor memory is a row of
// W: a thread widens its row's codes in registers (two masks and a shift for four of them; a code stays c * 2^-24 or, for
// the rows of the high nibbles, c * 2^-20, which f16 holds as a subnormal) and stores them there, so the widened weights
// never cross shared memory.  Every group of G columns has an accumulator of its own in tensor memory,
//   Y[n] += s ( D - z sum_k x_k ),
// scaled in f32 by a second set of threads while the next group is multiplied.
//
// A CTA: warps 0-7 widen (two sets of four, a block of 128 columns each in turn), 8-11 scale and sum, 12 copies, 13 issues
// the products, 14 and 15 sum X over each group (with warp-level steps against ones).  Few rows of W are shared out along
// K over a cluster, whose CTAs add up through distributed shared memory.
#include <atomic>
#include <cuda.h>

#include "common.cuh"
#include "kernels.h"
#include "q4.cuh"

namespace ph {
namespace {

constexpr int QT_THREADS = 512;
constexpr int QT_TILES = 8;                                // tiles of 16 rows of W
constexpr int QT_KBS = 2;                                  // blocks of 128 columns in a stage: fewer, larger copies
constexpr int QT_A_SLOTS = 4, QT_A_COLS = 64;              // widened blocks in tensor memory: 128 columns of W each
constexpr int QT_D_SLOTS = 4;
constexpr int QT_TMEM = 512;
constexpr uint32_t ONES = 0x3c003c00u;                     // two f16 ones
enum : uint32_t {
  SITE_QT_FULL = 0x44, SITE_QT_EMPTY = 0x45, SITE_QT_A_FULL = 0x46, SITE_QT_A_EMPTY = 0x47, SITE_QT_D_FULL = 0x48,
  SITE_QT_D_EMPTY = 0x49, SITE_QT_SUMS = 0x4a
};

struct TcGemvParams {
  const __half* X;
  const uint8_t* W;
  void* Y;
  long long ldx, ldy;
  int M, N, K, kblocks, tiles, tiles_per_cta, split;       // split: CTAs of a cluster, along K
  float alpha, beta;
  int out_f32;
  uint32_t* status;
};

template <int NC, int GS>
struct TcGemvShape {
  static constexpr int GROUPS = 8 / GS;                    // of a block of 128 columns
  static constexpr int BLOCK = 1024 + 64 * GROUPS;
  static constexpr int PITCH = QT_KBS * BLOCK + 16;        // of tiles in a stage: see the widening warps
  static constexpr int X_BOX = NC * 128, X_BYTES = QT_KBS * 2 * X_BOX;
  static constexpr int STAGE = (X_BYTES + QT_TILES * PITCH + 1023) / 1024 * 1024;
  static constexpr int HEAD = 1024;                        // barriers, flags
  static constexpr int SUMS = QT_KBS * GROUPS * NC * 4;    // of a stage
  static constexpr int MOST = 227 * 1024 - 1024;
  static constexpr int ROOM = (MOST - HEAD - 1024) / (STAGE + SUMS);
  static constexpr int STAGES = ROOM > 8 ? 8 : ROOM;
  static constexpr int RED = 128 * (NC + 4) * 4;           // a CTA's sums for the cluster, in the drained ring
  static constexpr int SMEM = HEAD + 1024 + STAGES * (STAGE + SUMS);
  static_assert(SMEM > 114 * 1024, "one CTA to an SM: it takes all of tensor memory");
  static_assert(STAGES >= 3 && RED <= STAGES * STAGE && QT_A_SLOTS * QT_A_COLS + QT_D_SLOTS * NC <= QT_TMEM, "shape");
};

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// A slot of a ring: which one, and the parity its `full` barrier completes with.
struct Turn {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next(int slots) {
    if (++slot == slots) {
      slot = 0;
      parity ^= 1;
    }
  }
};

template <int NC, int GS>
__global__ void __launch_bounds__(QT_THREADS, 1) gemv_q4_tc_kernel(const __grid_constant__ CUtensorMap x_map, TcGemvParams p) {
  using S = TcGemvShape<NC, GS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);   // X tiles are swizzled: 1024-byte aligned
  uint8_t* ring = smem;
  float* sums = reinterpret_cast<float*>(ring + S::STAGES * S::STAGE);        // [STAGES][QT_KBS][GROUPS][NC]
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sums) + S::STAGES * S::SUMS);
  uint64_t* empty = full + S::STAGES;
  uint64_t* summed = empty + S::STAGES;
  uint64_t* a_full = summed + S::STAGES;
  uint64_t* a_empty = a_full + QT_A_SLOTS;
  uint64_t* d_full = a_empty + QT_A_SLOTS;
  uint64_t* d_empty = d_full + QT_D_SLOTS;
  uint32_t* abort_flag = reinterpret_cast<uint32_t*>(d_empty + QT_D_SLOTS);
  uint32_t* tmem_slot = abort_flag + 1;
  static_assert((3 * S::STAGES + 2 * QT_A_SLOTS + 2 * QT_D_SLOTS) * 8 + 16 <= S::HEAD, "barriers");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag[0] = abort_flag[2] = 0;  // (the word between them is tensor memory's address)
    for (int i = 0; i < S::STAGES; i++) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 8 + 4 + 2);       // widening, scaling (who have seen the products done) and summing warps
      mbar_init(summed + i, 2);
    }
    for (int i = 0; i < QT_A_SLOTS; i++) {
      mbar_init(a_full + i, 4);
      mbar_init(a_empty + i, 1);
    }
    for (int i = 0; i < QT_D_SLOTS; i++) {
      mbar_init(d_full + i, 1);
      mbar_init(d_empty + i, 4);
    }
  }
  fence_mbar_init();
  if (warp == 13) {
    tmem_alloc(tmem_slot, QT_TMEM);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_a = *tmem_slot, tmem_d = tmem_a + QT_A_SLOTS * QT_A_COLS;
  pdl_wait();
  pdl_launch_dependents();
  const WaitCtx ctx{abort_flag, p.status};
  const int rank = blockIdx.x % p.split, tile0 = blockIdx.x / p.split * p.tiles_per_cta, m0 = blockIdx.y * NC;
  const int n_tiles = min(p.tiles_per_cta, p.tiles - tile0);
  const int kb0 = static_cast<int>(static_cast<long long>(p.kblocks) * rank / p.split);
  const int kb1 = static_cast<int>(static_cast<long long>(p.kblocks) * (rank + 1) / p.split);
  // a block's groups that lie before K
  auto groups_of = [&](int kb) { return min(S::GROUPS, (p.K - kb * 128) / (16 * GS)); };
  float y[NC];  // the scaling warps' sums: of one row of W
#pragma unroll
  for (int n = 0; n < NC; n++) y[n] = 0.0f;

  if (warp == 12) {
    // ---- copies ---------------------------------------------------------------------------------------------------------
    Turn s;
    for (int kb = kb0; kb < kb1; kb += QT_KBS, s.next(S::STAGES)) {
      if (kb >= kb0 + S::STAGES * QT_KBS && !mbar_wait_soon(empty + s.slot, s.parity ^ 1, SITE_QT_EMPTY, ctx)) break;
      uint8_t* stage = ring + s.slot * S::STAGE;
      const int n_kb = min(QT_KBS, kb1 - kb);
      if (lane == 0) mbar_arrive_expect_tx(full + s.slot, n_kb * (2 * S::X_BOX + n_tiles * S::BLOCK));
      __syncwarp();
      if (lane < n_tiles)
        bulk_load(stage + S::X_BYTES + lane * S::PITCH, p.W + (static_cast<long long>(tile0 + lane) * p.kblocks + kb) * S::BLOCK,
                          n_kb * S::BLOCK, full + s.slot);
      else if (lane >= 16 && lane < 16 + 2 * n_kb)
        tma_load_2d(stage + (lane - 16) * S::X_BOX, &x_map, full + s.slot, kb * 128 + (lane - 16) * 64, m0);
    }
  } else if (warp == 13) {
    // ---- products -------------------------------------------------------------------------------------------------------
    constexpr uint32_t idesc = umma_idesc_f16(128, NC, true, false, false);
    const uint64_t x_desc = umma_smem_desc(smem_u32(ring), 16, 1024);
    Turn s, a, d;
    int done = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; kb++, a.next(QT_A_SLOTS)) {
      const int groups = groups_of(kb), in_stage = (kb - kb0) % QT_KBS;
      // (who widened the block has seen the stage arrive, X with it)
      ok = mbar_wait_soon(a_full + a.slot, a.parity, SITE_QT_A_FULL, ctx) && ok;
#pragma unroll
      for (int grp = 0; grp < S::GROUPS; grp++) {
        if (grp >= groups) break;
        if (done >= QT_D_SLOTS) ok = mbar_wait_soon(d_empty + d.slot, d.parity ^ 1, SITE_QT_D_EMPTY, ctx) && ok;
        tc_fence_after_sync();
        if (ok && elect_one()) {
          const uint64_t xd = x_desc + static_cast<uint64_t>((s.slot * S::STAGE + in_stage * 2 * S::X_BOX) >> 4);
#pragma unroll
          for (int k = 0; k < GS; k++) {
            const int step = grp * GS + k;  // 32 bytes of X further each; the second four steps are the second box
            umma_f16_ts(tmem_d + d.slot * NC, tmem_a + a.slot * QT_A_COLS + step * 8,
                        xd + static_cast<uint64_t>(((step >> 2) * S::X_BOX + (step & 3) * 32) >> 4), idesc, k > 0 ? 1u : 0u);
          }
          umma_commit(d_full + d.slot);
          if (grp == groups - 1) umma_commit(a_empty + a.slot);
        }
        __syncwarp();
        d.next(QT_D_SLOTS);
        done++;
      }
      if (in_stage == QT_KBS - 1) s.next(S::STAGES);
    }
  } else if (warp >= 14) {
    // ---- sums of X over the groups ------------------------------------------------------------------------------------------
    Turn s;
    const int g = lane >> 2, t = lane & 3, block = warp - 14;
    for (int kb = kb0; kb < kb1; kb += QT_KBS, s.next(S::STAGES)) {
      if (mbar_wait_copies(full + s.slot, s.parity, SITE_QT_FULL, ctx, abort_flag + 2) && kb + block < kb1) {
        const uint8_t* x = ring + s.slot * S::STAGE + block * 2 * S::X_BOX;
        float* out = sums + (s.slot * QT_KBS + block) * S::GROUPS * NC;
#pragma unroll
        for (int grp = 0; grp < S::GROUPS; grp++) {
          float one[NC / 8][4];
#pragma unroll
          for (int q = grp * GS / 2; q < (grp + 1) * GS / 2; q++) {  // 32 columns; which lane has which does not matter to a sum
            const int chunk = (q & 1) * 4 + t;
            uint4 v[NC / 8];
#pragma unroll
            for (int n = 0; n < NC / 8; n++)
              v[n] = *reinterpret_cast<const uint4*>(x + (q >> 1) * S::X_BOX + (n * 8 + g) * 128 + ((chunk ^ g) << 4));
#pragma unroll
            for (int n = 0; n < NC / 8; n++)
              if (q == grp * GS / 2)
                mma_16816_first(one[n], ONES, ONES, ONES, ONES, v[n].x, v[n].y);
              else
                mma_16816(one[n], ONES, ONES, ONES, ONES, v[n].x, v[n].y);
#pragma unroll
            for (int n = 0; n < NC / 8; n++) mma_16816(one[n], ONES, ONES, ONES, ONES, v[n].z, v[n].w);
          }
          if (g == 0)
#pragma unroll
            for (int n = 0; n < NC / 8; n++)
              *reinterpret_cast<float2*>(out + grp * NC + n * 8 + 2 * t) = make_float2(one[n][0], one[n][1]);
        }
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(summed + s.slot);
        mbar_arrive(empty + s.slot);
      }
    }
  } else {
    // Rows of tensor memory: quarter q holds rows 8 (q / 2) + 0..7 of tiles 4 (q % 2) + 0..3, lane l row 2 (l / 8) + l % 2 of
    // tile (l / 2) % 4.  Eight neighbouring lanes then read 16 bytes each of four tiles, 16 bytes off a multiple of 64 apart,
    // and two rows 64 bytes apart: no two in one bank.
    const int quarter = warp & 3, high = quarter >> 1, tile = 4 * (quarter & 1) + ((lane >> 1) & 3);
    const int g = 2 * (lane >> 3) + (lane & 1);
    const uint32_t tmem_row = static_cast<uint32_t>(quarter * 32) << 16;
    if (warp < 8) {
      // ---- widening -------------------------------------------------------------------------------------------------------
      const uint32_t mask = high ? Q4_HI : Q4_LO;
      Turn s, a;
      static_assert(QT_KBS == 2, "a set of widening warps for each block of a stage");
      const int set = warp >> 2;
      a.slot = set;
      for (int kb = kb0; kb < kb1; kb += 2, s.next(S::STAGES)) {
        // Both sets wait for every stage, the last one with a single block too: an arrival on `empty` for a stage that has not
        // come would count for the one before it in the slot, whose (scale, zero) pairs and sums are still being read.
        const bool ok = mbar_wait_copies(full + s.slot, s.parity, SITE_QT_FULL, ctx, abort_flag + 2);
        if (kb + set < kb1) {
          const bool ok_a = kb < kb0 + QT_A_SLOTS || mbar_wait_soon(a_empty + a.slot, a.parity ^ 1, SITE_QT_A_EMPTY, ctx);
          if (ok && ok_a) {
            tc_fence_after_sync();
            const uint8_t* row = ring + s.slot * S::STAGE + S::X_BYTES + tile * S::PITCH + set * S::BLOCK + g * 64;
#pragma unroll
            for (int half = 0; half < 2; half++) {
              uint32_t c[32];  // 64 columns of W
#pragma unroll
              for (int t = 0; t < 4; t++) {
                const uint4 v = *reinterpret_cast<const uint4*>(row + half * 512 + t * 16);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                  c[16 * (j >> 1) + 4 * t + 2 * (j & 1)] = w[j] & mask;
                  c[16 * (j >> 1) + 4 * t + 2 * (j & 1) + 1] = (w[j] >> 8) & mask;
                }
              }
              tmem_st_32x32b_x32(tmem_a + a.slot * QT_A_COLS + half * 32 + tmem_row, c);
            }
            tmem_st_wait();
            tc_fence_before_sync();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(a_full + a.slot);
          a.next(QT_A_SLOTS);
          a.next(QT_A_SLOTS);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + s.slot);
      }
    } else {
      // ---- scaling ----------------------------------------------------------------------------------------------------------
      const float unit = high ? Q4_HI_UNIT : Q4_LO_UNIT, per_unit = high ? -1.0f / Q4_HI_UNIT : -1.0f / Q4_LO_UNIT;
      Turn s, d;
      for (int kb = kb0; kb < kb1; kb++) {
        const int in_stage = (kb - kb0) % QT_KBS, groups = groups_of(kb);
        bool ok = in_stage != 0 || (mbar_wait_copies(full + s.slot, s.parity, SITE_QT_FULL, ctx, abort_flag + 2) &&
                                    mbar_wait_soon(summed + s.slot, s.parity, SITE_QT_SUMS, ctx));
        const __half2* par = reinterpret_cast<const __half2*>(ring + s.slot * S::STAGE + S::X_BYTES + tile * S::PITCH + in_stage * S::BLOCK + 1024) +
                             high * 8 + g;
        const float* sum = sums + (s.slot * QT_KBS + in_stage) * S::GROUPS * NC;
        for (int grp = 0; grp < groups; grp++, d.next(QT_D_SLOTS)) {
          const float2 sz = __half22float2(par[grp * 16]);
          const float scale = sz.x * unit, zero = sz.y * per_unit;  // D is in units of a code, 2^-24 or 2^-20
          ok = mbar_wait_soon(d_full + d.slot, d.parity, SITE_QT_D_FULL, ctx) && ok;
          tc_fence_after_sync();
          constexpr int PART = NC < 32 ? NC : 32;
#pragma unroll
          for (int n0 = 0; n0 < NC; n0 += PART) {
            uint32_t v[PART];
#pragma unroll
            for (int i = 0; i < PART; i += 16) tmem_ld_32x32b_x16(tmem_d + d.slot * NC + n0 + i + tmem_row, v + i);
            tmem_ld_wait();
            if (n0 + PART == NC) {
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive(d_empty + d.slot);
            }
            if (!ok) continue;
#pragma unroll
            for (int i = 0; i < PART; i += 4) {
              const float4 x = *reinterpret_cast<const float4*>(sum + grp * NC + n0 + i);
              y[n0 + i] = fmaf(scale, fmaf(zero, x.x, __uint_as_float(v[i])), y[n0 + i]);
              y[n0 + i + 1] = fmaf(scale, fmaf(zero, x.y, __uint_as_float(v[i + 1])), y[n0 + i + 1]);
              y[n0 + i + 2] = fmaf(scale, fmaf(zero, x.z, __uint_as_float(v[i + 2])), y[n0 + i + 2]);
              y[n0 + i + 3] = fmaf(scale, fmaf(zero, x.w, __uint_as_float(v[i + 3])), y[n0 + i + 3]);
            }
          }
        }
        if (in_stage == QT_KBS - 1 || kb == kb1 - 1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(empty + s.slot);
          s.next(S::STAGES);
        }
      }
    }
  }
  // ---- write; a cluster's CTAs add up first -----------------------------------------------------------------------------------
  const int quarter = warp & 3, tile = 4 * (quarter & 1) + ((lane >> 1) & 3), g = 2 * (lane >> 3) + (lane & 1);
  const int row = tile * 16 + (quarter >> 1) * 8 + g, n = tile0 * 16 + row;
  const bool mine = warp >= 8 && warp < 12 && tile < n_tiles && n < p.N;
  auto write = [&](int m, float v) {
    v *= p.alpha;
    const long long at = static_cast<long long>(m0 + m) * p.ldy + n;
    if (p.out_f32) {
      float* o = static_cast<float*>(p.Y) + at;
      *o = p.beta == 0.0f ? v : fmaf(p.beta, *o, v);
    } else {
      __half* o = static_cast<__half*>(p.Y) + at;
      *o = __float2half_rn(p.beta == 0.0f ? v : fmaf(p.beta, __half2float(*o), v));
    }
  };
  const int n_m = min(NC, p.M - m0);
  auto not_finite = [&](int m, float v) { return q4_not_finite(v, p.X + (m0 + m) * p.ldx, p.W, n, p.K, p.kblocks, GS * 16); };
  if (p.split == 1) {
    if (mine) {
      bool nan = false;
#pragma unroll
      for (int m = 0; m < NC; m++) nan = nan || y[m] != y[m];
      if (!nan) {
#pragma unroll
        for (int m = 0; m < NC; m++)
          if (m < n_m) write(m, y[m]);
      } else {
#pragma unroll 1
        for (int m = 0; m < n_m; m++) {
          float v = 0.0f;
#pragma unroll
          for (int i = 0; i < NC; i++) v = i == m ? y[i] : v;  // (y stays in registers)
          write(m, v == v ? v : not_finite(m, v));
        }
      }
    }
  } else {
    constexpr int PITCH = NC + 4;
    float* red = reinterpret_cast<float*>(ring);
    __syncthreads();  // the ring is drained
    if (warp >= 8 && warp < 12)
#pragma unroll
      for (int m = 0; m < NC; m += 4)
        *reinterpret_cast<float4*>(red + row * PITCH + m) = make_float4(y[m], y[m + 1], y[m + 2], y[m + 3]);
    cluster_sync_all();
    if (mine) {
      const uint32_t at = smem_u32(red + row * PITCH);
      for (int m = rank; m < n_m; m += p.split) {  // this CTA's columns
        float v = 0.0f;
        for (int r = 0; r < p.split; r++) v += ld_cluster_f32(mapa_u32(at + m * 4, r));
        write(m, v == v ? v : not_finite(m, v));
      }
    }
    __syncwarp();
    cluster_sync_all();  // until then the other CTAs read here
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 13) tmem_dealloc(tmem_a, QT_TMEM);
}

// How the rows of W and K are shared out.
struct TcGemvSplit {
  int tiles_per_cta, split, rounds;
};
TcGemvSplit tc_gemv_split(int tiles, int kblocks, int m_groups, int sm_count) {
  TcGemvSplit s;
  // as many rows of W to a CTA as fill whole rounds of the GPU evenly
  const long long rounds = (static_cast<long long>((tiles + QT_TILES - 1) / QT_TILES) * m_groups + sm_count - 1) / sm_count;
  const long long slots = rounds * sm_count / m_groups;
  const long long share = slots > 0 ? (tiles + slots - 1) / slots : QT_TILES;
  s.tiles_per_cta = share > QT_TILES ? QT_TILES : static_cast<int>(share);
  s.rounds = static_cast<int>(rounds);
  // too few rows for that: share K out as well, four blocks of columns to a CTA at least.  (Clusters of eight take longer to
  // start than they save: 1024 x 4096 for 32 rows of X 18.8 us in eights, 11.5 in fours, 16.6 in twos.)
  s.split = 1;
  if (rounds == 1 && s.tiles_per_cta < 4) {
    s.tiles_per_cta = tiles < 4 ? tiles : 4;
    const int ctas = (tiles + s.tiles_per_cta - 1) / s.tiles_per_cta * m_groups;
    while (s.split < 4 && ctas * s.split * 2 <= sm_count && kblocks / (s.split * 2) >= 4) s.split *= 2;
  }
  return s;
}

// Columns of the product.  (With four groups to a block sixteen of them never pay: 0.79 us a block and round for up to 1184
// tiles, which the other kernel takes 0.66 for.)
int columns_for(int M, int group) { return M <= 16 && group > 32 ? 16 : M <= 32 ? 32 : 64; }

template <int NC, int GS>
cudaError_t launch_shape(const CUtensorMap& x_map, TcGemvParams& p, int sm_count, cudaStream_t stream) {
  using S = TcGemvShape<NC, GS>;
  auto kernel = gemv_q4_tc_kernel<NC, GS>;
  static std::atomic<bool> known[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !known[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return e;
    if (dev < 64) known[dev].store(true, std::memory_order_release);
  }
  const int m_groups = (p.M + NC - 1) / NC;
  const TcGemvSplit s = tc_gemv_split(p.tiles, p.kblocks, m_groups, sm_count);
  p.tiles_per_cta = s.tiles_per_cta;
  p.split = s.split;
  return launch_clusters_with_pdl(kernel, dim3((p.tiles + p.tiles_per_cta - 1) / p.tiles_per_cta * p.split, m_groups), dim3(QT_THREADS), p.split,
                                  S::SMEM, stream, x_map, p);
}

template <int GS>
int launch_group(const void* X, long long ldx, TcGemvParams& p, int sm_count, cudaStream_t stream, const char** err) {
  const int nc = columns_for(p.M, 16 * GS);
  CUtensorMap x_map;
  if (!make_tmap_2d(&x_map, X, TMAP_F16, p.M, p.K, ldx, nc, 64, TMAP_SWIZZLE_128B)) {
    *err = "cuTensorMapEncodeTiled failed (alignment or driver entry point)";
    return -1;
  }
  cudaError_t e = cudaSuccess;
  if constexpr (GS > 2)
    if (nc == 16) e = launch_shape<16, GS>(x_map, p, sm_count, stream);
  if (nc == 32) e = launch_shape<32, GS>(x_map, p, sm_count, stream);
  if (nc == 64) e = launch_shape<64, GS>(x_map, p, sm_count, stream);
  if (e == cudaSuccess) return 0;
  *err = cudaGetErrorString(e);
  return -3;
}

}  // namespace

// Times of both kernels in us as they were measured (B200, weights not in L2), fitted: this one takes 4 us and then for each
// block of 128 columns in turn 0.25 us and for each of its groups 0.03 us and 6.5 ns a column of the product (16384 x 8192, G =
// 128: 31, 35, 55 us for 16, 32, 64 rows of X); the other 3.5 us and 0.28 ns for each 16 x 128 block and eight rows of X,
// which it reads the weights anew for (39, 76, 151 us; but 4096 x 4096: 9, 16, 30 us against 13, 17, 27).
bool gemv_q4_tc_is_faster(int M, int N, int K, int group, int sm_count) {
  const int nc = columns_for(M, group), m_groups = (M + nc - 1) / nc, tiles = (N + 15) / 16, kblocks = (K + 127) / 128;
  const TcGemvSplit s = tc_gemv_split(tiles, kblocks, m_groups, sm_count);
  const double here = 4.0 + (s.split > 1 ? 4.0 : 0.0) + static_cast<double>(s.rounds) * ((kblocks + s.split - 1) / s.split) *
                                                           (0.25 + 128 / group * (0.03 + 0.0065 * nc));
  const double there = 3.5 + 0.28e-3 * 148 / sm_count * tiles * kblocks * ((M + 7) / 8);
  return here < there;
}

int launch_gemv_q4_tc(const void* X, long long ldx, const void* W, void* Y, long long ldy, int out_f32, int M, int N, int K,
                      int group, float alpha, float beta, int sm_count, uint32_t* status, cudaStream_t stream, const char** err) {
  if (M > 64 * 65535) {
    *err = "gemv_q4: too many rows of X";
    return -2;
  }
  TcGemvParams p{static_cast<const __half*>(X), static_cast<const uint8_t*>(W), Y, ldx, ldy, M, N, K, (K + 127) / 128, (N + 15) / 16, 0, 0, alpha, beta, out_f32, status};
  return group == 128  ? launch_group<8>(X, ldx, p, sm_count, stream, err)
         : group == 64 ? launch_group<4>(X, ldx, p, sm_count, stream, err)
                       : launch_group<2>(X, ldx, p, sm_count, stream, err);
}

}  // namespace ph
