// Attention over the 4-bit cache: o = softmax(scale q K^T) V, one pass over the tokens with the running maximum and sum.
//
// A group of G dims of a token is zero + step * code, so
//   q . k = sum_G ( step (q . c) + zero (sum q) )         and       sum_j p_j v_j = sum_j (p_j step_j) c_j + sum_j p_j zero_j
// The matrix unit sees the bare codes of K against q, and the bare codes of V against p * step; zeros go through f32.
// S^T = K Q^T has the tokens as rows, so a K fragment is 16 tokens x 16 dims straight from the page, and P^T, whose
// accumulator layout is transposed by one movmatrix per 8 x 8, is the B operand of O^T = V^T P^T.
//
// p * step is rounded to f16 (half a step of 2^-11, as flash_attention rounds its p).  step can be small, so it is
// taken relative to a running power of two `e` (the largest exponent of a step so far, moved up like the maximum),
// with p * step * 2^(14 - e) < 2^15: a weight keeps its eleven bits down to 2^-28 of the largest.
#include "kv4.cuh"
#include "q4.cuh"

namespace ph {
namespace {

constexpr int AT_WARPS = 4;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^n for -126 <= n <= 127
__device__ __forceinline__ float pow2i(int n) { return __uint_as_float(static_cast<uint32_t>(n + 127) << 23); }

struct AttnParams {
  Kv4View c;
  Kv4AttnArgs a;
  int rep;
  uint32_t* status;
};

// Running state of eight query rows in one warp: lane 4g + t keeps rows 2t and 2t + 1.  Sums of p and of p * zero are
// the lane's own tokens' only, until the end.
template <int D, int NG>
struct RowState {
  float m[2], l[2], z[2][NG];
  float o[D / 16][4];  // dims 32p + 4g + {0, 2} (even i: low nibbles), + {1, 3} (odd i) of rows 2t, 2t + 1
  int e;
};

template <int D, int NG>
struct Queries {
  uint32_t b[D / 16][2];  // B operand: row g, the dims of matrix step i
  float sum[2][NG];       // sums of q over a group, rows 2t and 2t + 1
};

template <int D, int NG>
__device__ __forceinline__ void kv4_tile(const uint8_t* unit, int tok0, int lo0, int hi0, int lo1, int hi1, float cs,
                                         const Queries<D, NG>& q, RowState<D, NG>& s) {
  constexpr int J = D / 32, W = D / 8;
  const int lane = threadIdx.x & 31, g = lane >> 2;
  const uint32_t* kw0 = reinterpret_cast<const uint32_t*>(unit + lane * W);
  const uint32_t* kw1 = reinterpret_cast<const uint32_t*>(unit + 4 * D + lane * W);
  const uint32_t* vw0 = reinterpret_cast<const uint32_t*>(unit + 8 * D + lane * W);
  const uint32_t* vw1 = reinterpret_cast<const uint32_t*>(unit + 12 * D + lane * W);
  const __half2* kpar = reinterpret_cast<const __half2*>(unit + 16 * D);
  const __half2* vpar = reinterpret_cast<const __half2*>(unit + 16 * D + 64 * NG);
  // ---- S^T -------------------------------------------------------------------------------------------------------
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // tokens g (0, 1) and g + 8 (2, 3), rows 2t and 2t + 1
#pragma unroll
  for (int grp = 0; grp < NG; grp++) {
    float lo[4] = {}, hi[4] = {};
#pragma unroll
    for (int j = grp * J / NG; j < (grp + 1) * J / NG; j++) {
      const uint32_t a = kw0[j], b = kw1[j];
      mma_16816(lo, a & Q4_LO, b & Q4_LO, (a >> 8) & Q4_LO, (b >> 8) & Q4_LO, q.b[2 * j][0], q.b[2 * j][1]);
      mma_16816(hi, a & Q4_HI, b & Q4_HI, (a >> 8) & Q4_HI, (b >> 8) & Q4_HI, q.b[2 * j + 1][0], q.b[2 * j + 1][1]);
    }
    const float2 pa = __half22float2(kpar[g * NG + grp]), pb = __half22float2(kpar[(g + 8) * NG + grp]);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 p = i < 2 ? pa : pb;
      const float dot = fmaf(hi[i], 1.0f / 16.0f, lo[i]) * Q4_LO_UNIT;
      x[i] = fmaf(p.x, dot, fmaf(p.y, q.sum[i & 1][grp], x[i]));
    }
  }
  bool see[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int tok = tok0 + g + (i >> 1) * 8;
    see[i] = (i & 1) ? (tok >= lo1 && tok < hi1) : (tok >= lo0 && tok < hi0);
    x[i] = see[i] ? x[i] * cs : -INFINITY;
  }
  // ---- running maximum -----------------------------------------------------------------------------------------------
#pragma unroll
  for (int r = 0; r < 2; r++) {
    float m = fmaxf(x[r], x[2 + r]);
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
    m = fmaxf(m, s.m[r]);
    const float f = s.m[r] == m ? 1.0f : exp2_approx(s.m[r] - m);  // (also where both are -inf)
    s.m[r] = m;
    s.l[r] *= f;
#pragma unroll
    for (int grp = 0; grp < NG; grp++) s.z[r][grp] *= f;
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
      s.o[i][r] *= f;
      s.o[i][2 + r] *= f;
    }
  }
  float p[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    p[i] = see[i] ? exp2_approx(x[i] - s.m[i & 1]) : 0.0f;
    s.l[i & 1] += p[i];
  }
  // ---- the power of two that p * step is taken relative to ---------------------------------------------------------------
  float step[2][NG];
  uint32_t top = 0;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const bool any = see[2 * h] || see[2 * h + 1];
#pragma unroll
    for (int grp = 0; grp < NG; grp++) {
      const float2 v = __half22float2(vpar[(g + 8 * h) * NG + grp]);
      step[h][grp] = v.x;
      if (any && v.x <= 65504.0f) top = max(top, __float_as_uint(v.x) >> 23);
#pragma unroll
      for (int r = 0; r < 2; r++)
        if (see[2 * h + r]) s.z[r][grp] = fmaf(p[2 * h + r], v.y, s.z[r][grp]);
    }
  }
  const int e = max(s.e, static_cast<int>(__reduce_max_sync(0xffffffffu, top & 255u)) - 127);
  if (e != s.e) {
    const float f = pow2i(max(s.e - e, -126));
#pragma unroll
    for (int i = 0; i < D / 16; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) s.o[i][k] *= f;
    s.e = e;
  }
  const float up = pow2i(14 - e);
  // ---- O^T += V^T P^T -------------------------------------------------------------------------------------------------------
#pragma unroll
  for (int grp = 0; grp < NG; grp++) {
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = see[i] ? p[i] * (step[i >> 1][grp] * up) : 0.0f;
    const uint32_t b0 = transpose_8x8(pack_half2(w[0], w[1])), b1 = transpose_8x8(pack_half2(w[2], w[3]));
#pragma unroll
    for (int i = grp * J / NG; i < (grp + 1) * J / NG; i++) {
      const uint32_t a = vw0[i], b = vw1[i];
      mma_16816(s.o[2 * i], a & Q4_LO, (a >> 8) & Q4_LO, b & Q4_LO, (b >> 8) & Q4_LO, b0, b1);
      mma_16816(s.o[2 * i + 1], a & Q4_HI, (a >> 8) & Q4_HI, b & Q4_HI, (b >> 8) & Q4_HI, b0, b1);
    }
  }
}

// One CTA: eight query rows (a row is one query token and one head of a key/value head's heads) of one sequence and one
// key/value head; its warps share out the sequence's units and join at the end.
template <int D, int NG>
__global__ void __launch_bounds__(AT_WARPS * 32) kv4_attn_kernel(AttnParams p) {
  constexpr int J = D / 32, G = D / NG, UNIT = kv4_unit_bytes(D, G);
  __shared__ float so[AT_WARPS][8][D + 4];
  __shared__ float sm[AT_WARPS][8], sl[AT_WARPS][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int head = blockIdx.y;
  // ---- which sequence and rows --------------------------------------------------------------------------------------
  int b = -1, tile = blockIdx.x, base = 0;
  Kv4Rows rows{};
  for (int i0 = 0; i0 < p.a.n; i0 += 32) {
    int tiles = 0;
    if (i0 + lane < p.a.n) {
      const int begin = p.a.ind ? min(max(p.a.ind[i0 + lane], 0), p.a.T) : 0;
      const int end = p.a.ind ? min(max(p.a.ind[i0 + lane + 1], begin), p.a.T) : 1;
      tiles = ((end - begin) * p.rep + 7) / 8;
    }
    int sum = tiles;
    for (int d = 1; d < 32; d *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, base + sum > tile);
    if (past) {
      const int k = __ffs(past) - 1;
      b = i0 + k;
      tile -= base + __shfl_sync(0xffffffffu, sum - tiles, k);
      break;
    }
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (b < 0) return;
  rows = kv4_rows(p.c, p.a.slots, p.a.ind, b, p.a.T, p.status);
  const int n_rows = (rows.end - rows.begin) * p.rep, first = rows.length - (rows.end - rows.begin);
  // ---- queries ---------------------------------------------------------------------------------------------------------
  Queries<D, NG> q;
  const int my = tile * 8 + g;
  const __half* qp = static_cast<const __half*>(p.a.Q) + (rows.begin + min(my, n_rows - 1) / p.rep) * p.a.ldq +
                     (head * p.rep + min(my, n_rows - 1) % p.rep) * D;
  float sums[NG] = {};
#pragma unroll
  for (int j = 0; j < J; j++) {
    const uint4 v = *reinterpret_cast<const uint4*>(qp + (4 * j + t) * 8);
    // dims 0..7 of the word pair up as (0, 4), (2, 6) for the low nibbles' step and (1, 5), (3, 7) for the high ones'
    q.b[2 * j][0] = __byte_perm(v.x, v.z, 0x5410);
    q.b[2 * j][1] = __byte_perm(v.y, v.w, 0x5410);
    q.b[2 * j + 1][0] = __byte_perm(v.x, v.z, 0x7632);
    q.b[2 * j + 1][1] = __byte_perm(v.y, v.w, 0x7632);
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(h[i]);
      sums[j * NG / J] += f.x + f.y;
    }
  }
#pragma unroll
  for (int grp = 0; grp < NG; grp++) {
    sums[grp] += __shfl_xor_sync(0xffffffffu, sums[grp], 1);
    sums[grp] += __shfl_xor_sync(0xffffffffu, sums[grp], 2);
    q.sum[0][grp] = __shfl_sync(0xffffffffu, sums[grp], 8 * t);
    q.sum[1][grp] = __shfl_sync(0xffffffffu, sums[grp], 8 * t + 4);
  }
  // ---- what rows 2t and 2t + 1 see: tokens [lo, hi) ----------------------------------------------------------------------
  int lo[2], hi[2];
#pragma unroll
  for (int r = 0; r < 2; r++) {
    const int row = tile * 8 + 2 * t + r;
    const int pos = first + row / p.rep;
    const bool is = row < n_rows;
    hi[r] = is ? pos + 1 : 0;
    lo[r] = is && p.a.window > 0 ? max(pos + 1 - p.a.window, 0) : 0;
  }
  const int last_row = min(tile * 8 + 7, n_rows - 1);
  const int end = first + last_row / p.rep + 1;  // tokens that some row of this tile sees end here
  const int start = p.a.window > 0 ? max(first + tile * 8 / p.rep + 1 - p.a.window, 0) : 0;
  RowState<D, NG> s;
#pragma unroll
  for (int r = 0; r < 2; r++) {
    s.m[r] = -INFINITY;
    s.l[r] = 0.0f;
#pragma unroll
    for (int grp = 0; grp < NG; grp++) s.z[r][grp] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < D / 16; i++)
#pragma unroll
    for (int k = 0; k < 4; k++) s.o[i][k] = 0.0f;
  s.e = -24;
  const float cs = p.a.scale * LOG2E;
  const int page_units = 1 << (p.c.page_shift - 4);
  for (int u = start / 16 + warp; u * 16 < end; u += AT_WARPS) {
    const int page = kv4_page(p.c, rows.slot, u * 16, p.status);
    if (page < 0) continue;
    const uint8_t* unit = p.c.pages + page * p.c.page_bytes +
                          (static_cast<long long>(head) * page_units + (u & (page_units - 1))) * UNIT;
    kv4_tile<D, NG>(unit, u * 16, lo[0], hi[0], lo[1], hi[1], cs, q, s);
  }
  // ---- join ------------------------------------------------------------------------------------------------------------
#pragma unroll
  for (int r = 0; r < 2; r++) {
    s.l[r] += __shfl_xor_sync(0xffffffffu, s.l[r], 4);
    s.l[r] += __shfl_xor_sync(0xffffffffu, s.l[r], 8);
    s.l[r] += __shfl_xor_sync(0xffffffffu, s.l[r], 16);
#pragma unroll
    for (int grp = 0; grp < NG; grp++) {
      s.z[r][grp] += __shfl_xor_sync(0xffffffffu, s.z[r][grp], 4);
      s.z[r][grp] += __shfl_xor_sync(0xffffffffu, s.z[r][grp], 8);
      s.z[r][grp] += __shfl_xor_sync(0xffffffffu, s.z[r][grp], 16);
    }
    const float down = pow2i(s.e - 14);
#pragma unroll
    for (int i = 0; i < J; i++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const float zero = s.z[r][i * NG / J];
        so[warp][2 * t + r][32 * i + 4 * g + 2 * k] = fmaf(s.o[2 * i][2 * k + r] * Q4_LO_UNIT, down, zero);
        so[warp][2 * t + r][32 * i + 4 * g + 2 * k + 1] = fmaf(s.o[2 * i + 1][2 * k + r] * Q4_HI_UNIT, down, zero);
      }
    if (g == 0) {
      sm[warp][2 * t + r] = s.m[r];
      sl[warp][2 * t + r] = s.l[r];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * D; i += AT_WARPS * 32) {
    const int r = i / D, d = i % D, row = tile * 8 + r;
    if (row >= n_rows) break;
    float m = sm[0][r];
    for (int w = 1; w < AT_WARPS; w++) m = fmaxf(m, sm[w][r]);
    float l = 0.0f, o = 0.0f;
    for (int w = 0; w < AT_WARPS; w++) {
      const float f = sm[w][r] == -INFINITY ? 0.0f : exp2_approx(sm[w][r] - m);
      l = fmaf(sl[w][r], f, l);
      if (f != 0.0f) o = fmaf(so[w][r][d], f, o);
    }
    const long long out = rows.begin + row / p.rep;
    const int h = head * p.rep + row % p.rep;
    static_cast<__half*>(p.a.O)[out * p.a.ldo + h * D + d] = __float2half_rn(m == -INFINITY ? 0.0f : o / l);
    if (d == 0 && p.a.lse) p.a.lse[out * p.a.ldl + h] = m == -INFINITY ? -INFINITY : fmaf(m, LN2, logf(l));
  }
}

}  // namespace

size_t kv4_attention_workspace(const Kv4View& c, int T, int n, int q_heads, int sm_count) { return 0; }

int launch_kv4_attention(const Kv4View& c, const Kv4AttnArgs& a, void* workspace, size_t workspace_bytes, int sm_count,
                         uint32_t* status, cudaStream_t stream, const char** err) {
  AttnParams p{c, a, a.q_heads / c.heads, status};
  const long long tiles = a.ind ? (static_cast<long long>(a.T) * p.rep + 7) / 8 + a.n
                                : static_cast<long long>(a.n) * ((p.rep + 7) / 8);
  if (tiles > 0x7fffffffLL || c.heads > 65535) {
    *err = "kv4_attention: too many rows";
    return -2;
  }
  const dim3 grid(static_cast<unsigned>(tiles), c.heads);
  const int ng = c.D / c.G;
  if (c.D == 128) {
    if (ng == 1) kv4_attn_kernel<128, 1><<<grid, AT_WARPS * 32, 0, stream>>>(p);
    else if (ng == 2) kv4_attn_kernel<128, 2><<<grid, AT_WARPS * 32, 0, stream>>>(p);
    else kv4_attn_kernel<128, 4><<<grid, AT_WARPS * 32, 0, stream>>>(p);
  } else {
    if (ng == 1) kv4_attn_kernel<64, 1><<<grid, AT_WARPS * 32, 0, stream>>>(p);
    else kv4_attn_kernel<64, 2><<<grid, AT_WARPS * 32, 0, stream>>>(p);
  }
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  *err = cudaGetErrorString(e);
  return -3;
}

}  // namespace ph
