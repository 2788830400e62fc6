// Rows of keys and values into the 4-bit cache, and back.
//
//   scale = f16((max - min) / 15), zero = min, code = rint((x - min) / scale) in 0..15     per group of G dims
// Differences and quotients are f32 with IEEE rounding, so the codes do not depend on how the work is split.  A group
// whose range rounds to a scale of zero holds `zero` alone; a group with a value that is not finite reads back as NaN.
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
};

constexpr int ROW_THREADS = 128;

// One warp: a row and one head of it (D = 128), or a row and two heads (D = 64).
template <int D, bool READ>
__global__ void __launch_bounds__(ROW_THREADS) kv4_rows_kernel(RowParams p) {
  constexpr int W = D / 8, PER = 32 / (2 * W);  // lanes of a key or value; heads of a warp
  const int lane = threadIdx.x & 31;
  const int head_groups = (p.c.heads + PER - 1) / PER;
  const long long job = static_cast<long long>(blockIdx.x) * (ROW_THREADS / 32) + (threadIdx.x >> 5);
  if (job >= static_cast<long long>(p.T) * head_groups) return;
  const int row = static_cast<int>(job / head_groups), hg = static_cast<int>(job % head_groups);
  const int b = kv4_find(p.ind, p.n, row);
  const Kv4Rows rows = kv4_rows(p.c, p.slots, p.ind, b, p.T, p.status);
  const int pos = rows.length - (rows.end - rows.begin) + (row - rows.begin);
  if (row < rows.begin || row >= rows.end) return;  // rows behind the last sequence stay as they are
  const int head = hg * PER + lane / (2 * W);
  const bool value = (lane % (2 * W)) >= W;
  const int word = lane % W;
  const bool live = head < p.c.heads;
  int page = -1;
  if (pos >= 0) page = kv4_page(p.c, rows.slot, pos, p.status);
  const int groups = D / p.c.G, grp = word * 8 / p.c.G;
  const int r = pos & 15, unit_bytes = kv4_unit_bytes(D, p.c.G), page_units = 1 << (p.c.page_shift - 4);
  uint8_t* unit = p.c.pages + page * p.c.page_bytes +
                  (static_cast<long long>(head) * page_units + ((pos & ((1 << p.c.page_shift) - 1)) >> 4)) * unit_bytes;
  // where this lane's eight codes and its group's pair stand in the unit
  const int k_at = (r >> 3) * 4 * D + ((r & 7) * 4 + (word & 3)) * W + (word >> 2) * 4;
  const int v_at = 8 * D + (r >> 3) * 4 * D + (2 * (word & 3) * 4 + ((r & 7) >> 1)) * W + (word >> 2) * 4 + (r & 1) * 2;
  const int par_at = 16 * D + (value ? 64 * groups : 0) + (r * groups + grp) * 4;
  const long long at = row * (value ? p.ldv : p.ldk) + head * D + word * 8;
  if constexpr (READ) {
    if (!live) return;
    uint4 out = make_uint4(0, 0, 0, 0);  // a row whose token is not in the cache reads as zero
    if (page >= 0) {
      uint32_t codes;
      if (value)
        codes = *reinterpret_cast<const uint16_t*>(unit + v_at) |
                static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(unit + v_at + 4 * W)) << 16;
      else
        codes = *reinterpret_cast<const uint32_t*>(unit + k_at);
      const float2 sz = __half22float2(*reinterpret_cast<const __half2*>(unit + par_at));
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
    *reinterpret_cast<uint4*>((value ? p.Vout : p.Kout) + at) = out;
  } else {
    uint4 in = make_uint4(0, 0, 0, 0);
    if (live) in = *reinterpret_cast<const uint4*>((value ? p.V : p.K) + at);
    const __half2* h = reinterpret_cast<const __half2*>(&in);
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(h[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
    float lo = x[0], hi = x[0];
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
      finite = finite && fabsf(x[i]) <= 65504.0f;
    }
    int bad = finite ? 0 : 1;
    for (int d = 1; d < p.c.G / 8; d *= 2) {  // the group's lanes are neighbours
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
      bad |= __shfl_xor_sync(0xffffffffu, bad, d);
    }
    if (!live || page < 0) return;
    const __half scale = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
    const float s = __half2float(scale);
    uint32_t codes = 0;
    if (s > 0.0f && !bad) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float c = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[i], lo), s)), 0.0f), 15.0f);
        codes |= static_cast<uint32_t>(c) << (4 * i);
      }
    }
    if (value) {
      *reinterpret_cast<uint16_t*>(unit + v_at) = static_cast<uint16_t>(codes);
      *reinterpret_cast<uint16_t*>(unit + v_at + 4 * W) = static_cast<uint16_t>(codes >> 16);
    } else {
      *reinterpret_cast<uint32_t*>(unit + k_at) = codes;
    }
    if (word * 8 % p.c.G == 0) {
      const __half nan = __ushort_as_half(0x7e00);
      *reinterpret_cast<__half2*>(unit + par_at) = bad ? __halves2half2(nan, nan) : __halves2half2(scale, __float2half_rn(lo));
    }
  }
}

template <bool READ>
int launch_rows(const RowParams& p, cudaStream_t stream, const char** err) {
  const int per = p.c.D == 128 ? 1 : 2;
  const long long jobs = static_cast<long long>(p.T) * ((p.c.heads + per - 1) / per);
  const long long blocks = (jobs + ROW_THREADS / 32 - 1) / (ROW_THREADS / 32);
  if (blocks > 0x7fffffffLL) {
    *err = "kv4: too many rows";
    return -2;
  }
  if (p.c.D == 128)
    kv4_rows_kernel<128, READ><<<static_cast<unsigned>(blocks), ROW_THREADS, 0, stream>>>(p);
  else
    kv4_rows_kernel<64, READ><<<static_cast<unsigned>(blocks), ROW_THREADS, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  *err = cudaGetErrorString(e);
  return -3;
}

}  // namespace

int launch_kv4_append(const Kv4View& c, const void* K, long long ldk, const void* V, long long ldv, int T, const int* slots,
                      const int* ind, int n, uint32_t* status, cudaStream_t stream, const char** err) {
  const RowParams p{c, static_cast<const __half*>(K), static_cast<const __half*>(V), nullptr, nullptr, ldk, ldv, slots, ind, T, n, status};
  return launch_rows<false>(p, stream, err);
}

int launch_kv4_read(const Kv4View& c, void* K, long long ldk, void* V, long long ldv, int T, const int* slots, const int* ind,
                    int n, uint32_t* status, cudaStream_t stream, const char** err) {
  const RowParams p{c, nullptr, nullptr, static_cast<__half*>(K), static_cast<__half*>(V), ldk, ldv, slots, ind, T, n, status};
  return launch_rows<true>(p, stream, err);
}

}  // namespace ph
