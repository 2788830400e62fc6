// Rows of keys and values into the 4-bit cache, and back.
//
//   scale = f16((max - min) / 15), zero = min, code = rint((x - min) / scale) in 0..15     per group of G dims
// Differences are rounded to f32, which only values far smaller than the minimum notice: x = -2^-23 beside a minimum of -2.3
// counts as 0, and one whose quotient then stands between two codes goes to the even one.
// The codes are found without a division: k = rint((x - min) * (1 / scale)) is right unless the product lies close to the
// middle between two codes; then e = (x - min) - k scale, exact in f32, says whether it is, and at e = scale / 2
// which neighbour is even.  (With a division for each value 25930 rows of 8 x 128, G = 32, took 186 us, bound by
// instructions; now 70, 2.0 TB/s, still bound by them.  Reading them back takes 41.)  A group whose range rounds to a scale of
// zero holds `zero` alone; a group with a value that is not finite reads back as NaN.
#include "kv4.cuh"

namespace ph {
namespace {

struct RowParams {
  Kv4View c;
  const __half* K;
  const __half* V;
  __half* Kout;
  __half* Vout;
  long long ldk, ldv;
  const int* slots;
  const int* ind;
  int T, n;
  uint32_t* status;
  bool images;  // whole units through shared memory
};

constexpr int ROW_WARPS = 8;

constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23: a sum's low bits are the other number, rounded

// rint(a / s) for a >= 0, s > 0 and quotients below 2^21, at most 15.
__device__ __forceinline__ uint32_t code_of(float a, float s, float per_s) {
  const float m = fmaf(a, per_s, MAGIC);
  int k = static_cast<int>(__float_as_uint(m) & 0x3fffffu);
  const float e = fmaf(-(m - MAGIC), s, a), off = fabsf(e), half = 0.5f * s;
  if (off > half || (off == half && (k & 1))) k += e > 0.0f ? 1 : -1;
  return static_cast<uint32_t>(min(k, 15));
}

// Which unit of which sequence a CTA works on.
struct Job {
  Kv4Rows rows;
  int unit;  // of the sequence; below 0 for rows whose token is not in the cache
};

// A sequence's new tokens stand in units (length - rows) / 16 .. (length - 1) / 16, rounded down.
__device__ __forceinline__ int units_of(const Kv4Rows& r, int* first) {
  const int n = r.end - r.begin;
  *first = (r.length - n) >> 4;
  return n > 0 ? ((r.length - 1) >> 4) - *first + 1 : 0;
}

// The job of CTA `at`: the sequences are walked a CTA's width at a time.  False behind the last.
__device__ bool find_job(const RowParams& p, int at, Job* job) {
  __shared__ int warp_sum[ROW_WARPS];
  __shared__ Job found;
  int first;
  if (!p.ind) {  // one row, so one unit each
    if (at >= p.n) return false;
    job->rows = kv4_rows(p.c, p.slots, p.ind, at, p.T, p.status);
    units_of(job->rows, &first);
    job->unit = first;
    return true;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int done = 0;
  for (int i0 = 0; i0 < p.n; i0 += ROW_WARPS * 32) {
    const int b = i0 + threadIdx.x;
    int count = 0;
    Kv4Rows rows{};
    if (b < p.n) {
      rows = kv4_rows(p.c, p.slots, p.ind, b, p.T, p.status);
      count = units_of(rows, &first);
    }
    int sum = count;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    int before = done, total = 0;
    for (int w = 0; w < ROW_WARPS; w++) {
      if (w < warp) before += warp_sum[w];
      total += warp_sum[w];
    }
    before += sum - count;
    if (at >= before && at < before + count) {
      found.rows = rows;
      found.unit = first + at - before;
    }
    done += total;
    __syncthreads();
    if (at < done) break;
  }
  if (at >= done) return false;
  *job = found;
  return true;
}

// One CTA: a unit of one sequence; each warp takes heads in turn.  D / 8 lanes work on a row's key and D / 8 on its value,
// eight dims each, in as many rows at once as a warp holds.  Where there are many, a unit whose sixteen tokens are all there
// goes through shared memory, one head to a warp, and is read or written in one piece of 16-byte words; of any other one only
// the rows' own bytes are touched, and its rows are shared out over the warps (350 rows of 4 heads: 12 us in whole units).
template <int D, bool READ>
__global__ void __launch_bounds__(ROW_WARPS * 32, 3) kv4_rows_kernel(RowParams p) {
  constexpr int W = D / 8, AT_ONCE = 32 / (2 * W), PASSES = KV4_UNIT / AT_ONCE, AHEAD = 4;
  __shared__ __align__(16) uint8_t image[ROW_WARPS][16 * D + 128 * (D / 32)];
  pdl_wait();
  Job job;
  if (!find_job(p, blockIdx.x, &job)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = job.rows.end - job.rows.begin, first = job.rows.length - n;
  const int r0 = max(first - job.unit * 16, 0), r1 = min(job.rows.length - job.unit * 16, 16);  // its tokens r0 .. r1 - 1 are rows
  const bool whole = r0 == 0 && r1 == 16 && p.images;
  const int page = job.unit >= 0 ? kv4_page(p.c, job.rows.slot, job.unit * 16, p.status) : -1;
  const int groups = D / p.c.G, unit_bytes = kv4_unit_bytes(D, p.c.G), page_units = 1 << (p.c.page_shift - 4);
  const bool value = (lane % (2 * W)) >= W;
  const int word = lane % W, grp = word * 8 / p.c.G;
  // of a unit that is not whole every warp takes one batch of rows of one head, so that all can have some
  constexpr int BATCH = AHEAD * AT_ONCE;
  const int batch0 = r0 / BATCH, batches = whole ? 1 : (r1 - 1) / BATCH - batch0 + 1, jobs = p.c.heads * batches;
  for (int at = warp; at < jobs; at += ROW_WARPS) {
    const int head = at / batches, pass0 = whole ? 0 : (batch0 + at % batches) * AHEAD;
    const int passes = whole ? PASSES : AHEAD;
    uint8_t* unit = p.c.pages + page * p.c.page_bytes +
                    (static_cast<long long>(head) * page_units + (job.unit & (page_units - 1))) * unit_bytes;
    uint8_t* to = whole ? image[warp] : unit;
    if (READ && whole && page >= 0) {
      __syncwarp();
      for (int i = lane; i < unit_bytes / 16; i += 32)
        reinterpret_cast<uint4*>(image[warp])[i] = reinterpret_cast<const uint4*>(unit)[i];
      __syncwarp();
    }
    uint4 rows[AHEAD];
#pragma unroll 4
    for (int k = 0; k < passes; k++) {
      const int r = (pass0 + k) * AT_ONCE + lane / (2 * W);
      const bool live = r >= r0 && r < r1;
      if constexpr (!READ) {
        if (k % AHEAD == 0) {
#pragma unroll
          for (int i = 0; i < AHEAD; i++) {
            const int ri = r + i * AT_ONCE;
            rows[i] = make_uint4(0, 0, 0, 0);
            if (ri >= r0 && ri < r1)
              rows[i] = *reinterpret_cast<const uint4*>((value ? p.V : p.K) + (job.rows.begin + job.unit * 16 + ri - first) * (value ? p.ldv : p.ldk) +
                                                        head * D + word * 8);
          }
        }
      }
      if (!whole && !__any_sync(0xffffffffu, live)) continue;
      // where this lane's eight codes and its group's pair stand in the unit
      const int k_at = (r >> 3) * 4 * D + ((r & 7) * 4 + (word & 3)) * W + (word >> 2) * 4;
      const int v_at = 8 * D + (r >> 3) * 4 * D + (2 * (word & 3) * 4 + ((r & 7) >> 1)) * W + (word >> 2) * 4 + (r & 1) * 2;
      const int par_at = 16 * D + (value ? 64 * groups : 0) + (r * groups + grp) * 4;
      if constexpr (READ) {
        if (!live) continue;
        uint4 out = make_uint4(0, 0, 0, 0);  // a row whose token is not in the cache reads as zero
        if (page >= 0) {
          uint32_t codes;
          if (value)
            codes = *reinterpret_cast<const uint16_t*>(to + v_at) |
                    static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(to + v_at + 4 * W)) << 16;
          else
            codes = *reinterpret_cast<const uint32_t*>(to + k_at);
          const float2 sz = __half22float2(*reinterpret_cast<const __half2*>(to + par_at));
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            x[i] = fmaf(sz.x, static_cast<float>((codes >> (4 * i)) & 15u), sz.y);
            // zero + 15 scale can pass the group's maximum by half a step of the f16 scale: not into infinity (NaN stays)
            if (x[i] > 65504.0f) x[i] = 65504.0f;
            if (x[i] < -65504.0f) x[i] = -65504.0f;
          }
          __half2* o = reinterpret_cast<__half2*>(&out);
#pragma unroll
          for (int i = 0; i < 4; i++) o[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        }
        *reinterpret_cast<uint4*>((value ? p.Vout : p.Kout) + (job.rows.begin + job.unit * 16 + r - first) * (value ? p.ldv : p.ldk) + head * D +
                                  word * 8) = out;
      } else {
        // the group's minimum and, negated, its maximum in one pair; NaN wins
        const __half2* h = reinterpret_cast<const __half2*>(&rows[k % AHEAD]);
        const __half2 even_odd = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3]));
        const __half2 neg = __hmin2_nan(__hmin2_nan(__hneg2(h[0]), __hneg2(h[1])), __hmin2_nan(__hneg2(h[2]), __hneg2(h[3])));
        __half2 ends = __hmin2_nan(__lows2half2(even_odd, neg), __highs2half2(even_odd, neg));
        for (int d = 1; d < p.c.G / 8; d *= 2) ends = __hmin2_nan(ends, __shfl_xor_sync(0xffffffffu, ends, d));  // its lanes are neighbours
        if (!live || page < 0) continue;
        const float lo = __low2float(ends), range = __fsub_rn(-__high2float(ends), lo);
        const bool bad = !(range <= 2.0f * 65504.0f);
        const __half scale = __float2half_rn(__fdiv_rn(range, 15.0f));
        const float s = __half2float(scale);
        uint32_t codes = 0;
        if (s > 0.0f && !bad) {
          float x[8];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(h[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
          }
          const float per_s = 1.0f / s;
          float off = range * per_s > 15.4f ? 1.0f : 0.0f;  // (a subnormal scale's error can lead past 15)
#pragma unroll
          for (int i = 7; i >= 0; i--) {
            const float a = __fsub_rn(x[i], lo), m = fmaf(a, per_s, MAGIC);
            off = fmaxf(off, fabsf(fmaf(a, per_s, MAGIC - m)));
            codes = codes << 4 | (__float_as_uint(m) & 15u);
          }
          if (off > 0.499f) {
            codes = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) codes |= code_of(__fsub_rn(x[i], lo), s, per_s) << (4 * i);
          }
        }
        if (value) {
          *reinterpret_cast<uint16_t*>(to + v_at) = static_cast<uint16_t>(codes);
          *reinterpret_cast<uint16_t*>(to + v_at + 4 * W) = static_cast<uint16_t>(codes >> 16);
        } else {
          *reinterpret_cast<uint32_t*>(to + k_at) = codes;
        }
        if (word * 8 % p.c.G == 0) {
          const __half nan = __ushort_as_half(0x7e00);
          *reinterpret_cast<__half2*>(to + par_at) = bad ? __halves2half2(nan, nan) : __halves2half2(scale, __float2half_rn(lo));
        }
      }
    }
    if (!READ && whole && page >= 0) {
      __syncwarp();
      for (int i = lane; i < unit_bytes / 16; i += 32)
        reinterpret_cast<uint4*>(unit)[i] = reinterpret_cast<const uint4*>(image[warp])[i];
      __syncwarp();
    }
  }
}

template <bool READ>
int launch_rows(const RowParams& rows, cudaStream_t stream, const char** err) {
  // an upper bound on the units that the rows stand in: a sequence's first and last may be partly theirs
  const long long jobs = rows.ind ? static_cast<long long>(rows.T) / KV4_UNIT + 2LL * rows.n : rows.n;
  if (jobs > 0x7fffffffLL) {
    *err = "kv4: too many rows";
    return -2;
  }
  RowParams p = rows;
  p.images = p.T >= 4096;  // 256 units, enough CTAs to fill the GPU
  const cudaError_t e = launch_with_pdl(p.c.D == 128 ? kv4_rows_kernel<128, READ> : kv4_rows_kernel<64, READ>, dim3(static_cast<unsigned>(jobs)),
                                        dim3(ROW_WARPS * 32), 0, stream, p);
  if (e == cudaSuccess) return 0;
  *err = cudaGetErrorString(e);
  return -3;
}

}  // namespace

int launch_kv4_append(const Kv4View& c, const void* K, long long ldk, const void* V, long long ldv, int T, const int* slots,
                      const int* ind, int n, uint32_t* status, cudaStream_t stream, const char** err) {
  const RowParams p{c, static_cast<const __half*>(K), static_cast<const __half*>(V), nullptr, nullptr, ldk, ldv, slots, ind, T, n, status, false};
  return launch_rows<false>(p, stream, err);
}

int launch_kv4_read(const Kv4View& c, void* K, long long ldk, void* V, long long ldv, int T, const int* slots, const int* ind,
                    int n, uint32_t* status, cudaStream_t stream, const char** err) {
  const RowParams p{c, nullptr, nullptr, static_cast<__half*>(K), static_cast<__half*>(V), ldk, ldv, slots, ind, T, n, status, false};
  return launch_rows<true>(p, stream, err);
}

}  // namespace ph
