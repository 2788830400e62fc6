// Attention over the 4-bit cache: o = softmax(scale q K^T) V, one pass over the tokens with the running maximum and sum.
//
// A group of G dims of a token is zero + step * code, so
//   q . k = sum_G ( step (q . c) + zero (sum q) )
//   sum_j p_j v_j = sum_j (p_j step_j) (c_j - 8) + sum_j p_j (zero_j + 8 step_j)
// The matrix unit sees the bare codes of K against q, and the codes of V, centred, against p * step; the rest goes
// through f32.  (Uncentred, the sums of c cancel against the zeros: with 131072 tokens that cost o a relative error of
// 3.5e-3, from the cut of the matrix unit's running sum.)
// S^T = K Q^T has the tokens as rows, so a K fragment is 16 tokens x 16 dims straight from the page, and P^T, whose
// accumulator layout is transposed by one movmatrix per 8 x 8, is the B operand of O^T = V^T P^T.
//
// p * step is rounded to f16 (half a step of 2^-11, as flash_attention rounds its p); it multiplies c - 8, so a token's share
// is off by at most 2^-11 p step |c - 8|.  Keeping what the rounding takes in a second f16 operand costs 13 to 21 %
// (64 sequences 82 us against 73, 131072 tokens 77 against 64) and leaves 2.2e-4 of 2.4e-4 and 2.7e-4 of 2.9e-4 of the error,
// most of which is the rounding of O.  step can be small, so it is
// taken relative to a running power of two `e` (the largest exponent of a step so far, moved up like the maximum),
// with p * step * 2^(14 - e) < 2^15: a weight keeps its eleven bits down to 2^-28 of the largest.
//
// Work: a problem is one sequence, one key/value head and 8 NT query rows (a row is one query token and one of the
// heads that read the key/value head).  The units of 16 tokens of all problems form one line that is cut into equal
// pieces, one per warp of a grid that fills the GPU once.  On the line every problem stands behind AT_START places that
// hold no units: what starting one costs, so that a piece of many short sequences is not longer than one of a long
// sequence.  A problem whose units lie in one piece is finished there; one that was cut leaves (m, l, o) of its parts in
// the workspace for a second, small kernel.  Warps share nothing: each streams its units through a ring of its own in
// shared memory with bulk copies (one per unit, 2176 bytes at D = G = 128) that it issues itself.
// Measured: 64 sequences of 1..8192 tokens, 8 heads of 128, 291 MB: 62 us, 4.7 TB/s, bound by instructions (257 a unit, issued
// in half of all slots by 12 warps to an SM).  Eight rows a problem where no more can be there, else sixteen: the widening of
// the codes is then done once for both halves (64 query heads on 4, G = 32: 73 us against 90).  What holds these forms back
// is registers: at D = 128 and four groups 168 for eight rows (324 bytes of spills stored a thread, 448 loaded) and 255 for
// sixteen (208 and 196, eight warps to an SM); two groups at sixteen rows 255 (172 and 120); D = 64 up to 160 and 100.
// Every warp walks the batch 32 sequences at a time to find its piece, twice where there are more than 32: 256 and 1024
// sequences of 100 to 2000 tokens (8 heads of 128) take 87 and 290 us where the bytes take 44 and 177, 4096 of 25 to 500 tokens
// 634 against 180.
#include <atomic>

#include "kv4.cuh"
#include "q4.cuh"

namespace ph {
namespace {

constexpr int AT_WARPS = 4;
constexpr int AT_START = 8;             // places for starting a problem
constexpr int AT_PIECE = 4;             // a piece is at least that long: one tile
constexpr uint32_t EIGHT = 0x00080008u;  // 8 * 2^-24, as a low nibble's 8, two f16
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
enum : uint32_t { SITE_KV4_RING = 0x41 };

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^n for -126 <= n <= 127
__device__ __forceinline__ float pow2i(int n) { return __uint_as_float(static_cast<uint32_t>(n + 127) << 23); }

// Rounded to f16, at most +-65504 in size as kv4_read has it: zero + 15 step can pass the group's largest value by the
// rounding of the step, and must not become an infinity (a NaN stays).
__device__ __forceinline__ uint32_t pack_output(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* at) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(at);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    w[0] = v.x; w[1] = v.y;
  }
}

struct AttnParams {
  Kv4View c;
  Kv4AttnArgs a;
  int rep, pieces;
  struct Cut* cuts;  // per piece: the problem that it ends inside of
  float* part;       // per piece two parts: of the problem it begins inside of, and of the one it ends inside of
  uint32_t* status;
};

// What the joining kernel has to know of a problem that starts in one piece and goes on behind it.
struct Cut {
  int parts;          // 0: none, or its units lie in one piece
  int first;          // index of its first part in the workspace; the following ones are those that continue it in the
  int next;           // pieces after it: next, next + 2, ...
  int row_begin, n_rows, head, row0, unused;
};

// Units of every problem of sequence b, and their first; at least one, so that rows without a token are answered too.
__device__ __forceinline__ int seq_units(const AttnParams& p, const Kv4Rows& r, int* begin) {
  const int n = r.end - r.begin;
  *begin = p.a.window > 0 ? max(r.length - n + 1 - p.a.window, 0) / KV4_UNIT : 0;
  return max((r.length + KV4_UNIT - 1) / KV4_UNIT - *begin, 1);
}
template <int ROWS>
__device__ __forceinline__ int seq_problems(const AttnParams& p, const Kv4Rows& r) {
  return p.c.heads * (((r.end - r.begin) * p.rep + ROWS - 1) / ROWS);
}

// a / b for b > 0; most numbers here fit 32 bits, and a 64-bit division takes a hundred instructions.
__device__ __forceinline__ long long divide(long long a, int b) {
  return (a >> 32) == 0 ? static_cast<long long>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}

// 32 sequences, one to a lane, and where they stand on the line.
struct Chunk {
  int first;             // sequence of lane 0
  Kv4Rows rows;
  long long begin, end;  // the lane's places, counted from the chunk's
};
template <int ROWS>
__device__ void load_chunk(const AttnParams& p, int first, Chunk* c) {
  const int lane = threadIdx.x & 31;
  long long places = 0;
  c->first = first;
  if (first + lane < p.a.n) {
    c->rows = kv4_rows(p.c, p.a.slots, p.a.ind, first + lane, p.a.T, p.status);
    int begin;
    places = static_cast<long long>(seq_units(p, c->rows, &begin) + AT_START) * seq_problems<ROWS>(p, c->rows);
  }
  long long sum = places;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long v = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += v;
  }
  c->begin = sum - places;
  c->end = sum;
}
__device__ __forceinline__ long long length_of(const Chunk& c) { return __shfl_sync(0xffffffffu, c.end, 31); }

// Running state of 8 NT query rows in one warp: lane 4g + t keeps rows 8k + 2t and 8k + 2t + 1.  Sums of p and of
// p * zero are the lane's own tokens' only, until the end.
template <int D, int NG, int NT>
struct RowState {
  float m[2 * NT], l[2 * NT], z[2 * NT][NG];
  float o[NT][D / 16][4];  // dims 32p + 4g + {0, 2} (even i: low nibbles), + {1, 3} (odd i) of rows 2t, 2t + 1
  int e;
};
template <int D, int NG, int NT>
struct Queries {
  uint32_t b[NT][D / 16][2];  // B operand: row g, the dims of matrix step i
  float sum[2 * NT][NG];      // sums of q over a group
  int lo[2 * NT], hi[2 * NT]; // the tokens that a row sees
};

template <int D, int NG, int NT, int UN, bool MASKED>
__device__ __forceinline__ void kv4_tile(const uint8_t* stage, int tok0, uint32_t present, float cs, const Queries<D, NG, NT>& q,
                                         RowState<D, NG, NT>& s) {
  constexpr int J = D / 32, W = D / 8, UNIT = kv4_unit_bytes(D, D / NG);
  const int lane = threadIdx.x & 31, g = lane >> 2;
  // ---- S^T -------------------------------------------------------------------------------------------------------
  float x[UN][NT][4];  // tokens g (0, 1) and g + 8 (2, 3), rows 2t and 2t + 1
  constexpr int PAIR = UN % 2 == 0 ? 2 : 1;  // units whose matrix steps alternate: each unit's are a chain
#pragma unroll
  for (int u0 = 0; u0 < UN; u0 += PAIR) {
    uint32_t kw0[PAIR][J], kw1[PAIR][J];
#pragma unroll
    for (int v = 0; v < PAIR; v++) {
      load_words<J>(kw0[v], stage + (u0 + v) * UNIT + lane * W);
      load_words<J>(kw1[v], stage + (u0 + v) * UNIT + 4 * D + lane * W);
    }
#pragma unroll
    for (int grp = 0; grp < NG; grp++) {
      float lo[PAIR][NT][4], hi[PAIR][NT][4];
#pragma unroll
      for (int j = grp * J / NG; j < (grp + 1) * J / NG; j++)
#pragma unroll
        for (int v = 0; v < PAIR; v++) {
          const uint32_t a = kw0[v][j], b = kw1[v][j], a2 = a >> 8, b2 = b >> 8;
#pragma unroll
          for (int k = 0; k < NT; k++) {
            if (j == grp * J / NG) {
              mma_16816_first(lo[v][k], a & Q4_LO, b & Q4_LO, a2 & Q4_LO, b2 & Q4_LO, q.b[k][2 * j][0], q.b[k][2 * j][1]);
              mma_16816_first(hi[v][k], a & Q4_HI, b & Q4_HI, a2 & Q4_HI, b2 & Q4_HI, q.b[k][2 * j + 1][0], q.b[k][2 * j + 1][1]);
            } else {
              mma_16816(lo[v][k], a & Q4_LO, b & Q4_LO, a2 & Q4_LO, b2 & Q4_LO, q.b[k][2 * j][0], q.b[k][2 * j][1]);
              mma_16816(hi[v][k], a & Q4_HI, b & Q4_HI, a2 & Q4_HI, b2 & Q4_HI, q.b[k][2 * j + 1][0], q.b[k][2 * j + 1][1]);
            }
          }
        }
#pragma unroll
      for (int v = 0; v < PAIR; v++) {
        const __half2* kpar = reinterpret_cast<const __half2*>(stage + (u0 + v) * UNIT + 16 * D);
        const float2 pa = __half22float2(kpar[g * NG + grp]), pb = __half22float2(kpar[(g + 8) * NG + grp]);
        const float sa = pa.x * cs, sb = pb.x * cs;
#pragma unroll
        for (int k = 0; k < NT; k++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float dot = fmaf(hi[v][k][i], 1.0f / 16.0f, lo[v][k][i]), z = i < 2 ? pa.y : pb.y, qs = q.sum[2 * k + (i & 1)][grp];
            x[u0 + v][k][i] = fmaf(i < 2 ? sa : sb, dot, grp == 0 ? z * qs : fmaf(z, qs, x[u0 + v][k][i]));
          }
      }
    }
  }
  auto sees = [&](int u, int k, int i) {
    if (!MASKED) return true;
    const int tok = tok0 + u * KV4_UNIT + g + (i >> 1) * 8, r = 2 * k + (i & 1);
    return tok >= q.lo[r] && tok < q.hi[r] && ((present >> u) & 1u) != 0;
  };
  // ---- running maximum and weights -------------------------------------------------------------------------------------
  float f[2 * NT];
  bool moved = false;
#pragma unroll
  for (int r = 0; r < 2 * NT; r++) {
    float m = s.m[r];
#pragma unroll
    for (int u = 0; u < UN; u++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float& v = x[u][r >> 1][2 * h + (r & 1)];
        if (MASKED && !sees(u, r >> 1, 2 * h + (r & 1))) v = -INFINITY;
        m = fmaxf(m, v);
      }
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
    f[r] = s.m[r] == m ? 1.0f : exp2_approx(s.m[r] - m);  // (1 also where both are -inf)
    moved = moved || s.m[r] != m;
    s.m[r] = m;
  }
  // ---- the power of two that p * step is taken relative to ---------------------------------------------------------------
  uint32_t top = 0, vpar[UN][2][NG];
#pragma unroll
  for (int u = 0; u < UN; u++) {
    const uint32_t* at = reinterpret_cast<const uint32_t*>(stage + u * UNIT + 16 * D + 64 * NG);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      bool any = !MASKED;
#pragma unroll
      for (int k = 0; k < NT; k++) any = any || sees(u, k, 2 * h) || sees(u, k, 2 * h + 1);
#pragma unroll
      for (int grp = 0; grp < NG; grp++) {
        vpar[u][h][grp] = at[(g + 8 * h) * NG + grp];
        const uint32_t step = vpar[u][h][grp] & 0x7fffu;
        if (any && step < 0x7c00u) top = max(top, step);
      }
    }
  }
  // exponent of the largest finite step: a half's 2^(field - 15), and -14 for the subnormals
  const int e = max(s.e, max(static_cast<int>(__reduce_max_sync(0xffffffffu, top) >> 10), 1) - 15);
  if (__any_sync(0xffffffffu, moved) || e != s.e) {
    const float down = pow2i(s.e - e);
#pragma unroll
    for (int r = 0; r < 2 * NT; r++) {
      s.l[r] *= f[r];
#pragma unroll
      for (int grp = 0; grp < NG; grp++) s.z[r][grp] *= f[r];
      const float fd = f[r] * down;
#pragma unroll
      for (int i = 0; i < D / 16; i++) {
        s.o[r >> 1][i][r & 1] *= fd;
        s.o[r >> 1][i][2 + (r & 1)] *= fd;
      }
    }
    s.e = e;
  }
  const float up = pow2i(14 - e);
#pragma unroll
  for (int u = 0; u < UN; u++)
#pragma unroll
    for (int k = 0; k < NT; k++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float w = sees(u, k, i) ? exp2_approx(x[u][k][i] - s.m[2 * k + (i & 1)]) : 0.0f;
        x[u][k][i] = w;
        s.l[2 * k + (i & 1)] += w;
      }
  // ---- O^T += V^T P^T, and what the 8 of c - 8 comes to: the same product with 8 for every code ---------------------------
  float eight[NT][NG][4];
#pragma unroll
  for (int u = 0; u < UN; u++) {
    const uint8_t* unit = stage + u * UNIT;
    uint32_t vw0[J], vw1[J];
    load_words<J>(vw0, unit + 8 * D + lane * W);
    load_words<J>(vw1, unit + 12 * D + lane * W);
#pragma unroll
    for (int grp = 0; grp < NG; grp++) {
      uint32_t b0[NT], b1[NT];
      const float2 va = __half22float2(*reinterpret_cast<const __half2*>(&vpar[u][0][grp]));
      const float2 vb = __half22float2(*reinterpret_cast<const __half2*>(&vpar[u][1][grp]));
      const float za = fmaf(va.x, 8.0f, va.y), zb = fmaf(vb.x, 8.0f, vb.y), sa = va.x * up, sb = vb.x * up;
#pragma unroll
      for (int k = 0; k < NT; k++) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const bool see = sees(u, k, i);
          w[i] = see ? x[u][k][i] * (i < 2 ? sa : sb) : 0.0f;
          if (see) s.z[2 * k + (i & 1)][grp] = fmaf(x[u][k][i], i < 2 ? za : zb, s.z[2 * k + (i & 1)][grp]);
        }
        b0[k] = transpose_8x8(pack_half2(w[0], w[1]));
        b1[k] = transpose_8x8(pack_half2(w[2], w[3]));
      }
#pragma unroll
      for (int i = grp * J / NG; i < (grp + 1) * J / NG; i++) {
        const uint32_t a = vw0[i], b = vw1[i], a2 = a >> 8, b2 = b >> 8;
#pragma unroll
        for (int k = 0; k < NT; k++) {
          mma_16816(s.o[k][2 * i], a & Q4_LO, a2 & Q4_LO, b & Q4_LO, b2 & Q4_LO, b0[k], b1[k]);
          mma_16816(s.o[k][2 * i + 1], a & Q4_HI, a2 & Q4_HI, b & Q4_HI, b2 & Q4_HI, b0[k], b1[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < NT; k++) {
        if (u == 0)
          mma_16816_first(eight[k][grp], EIGHT, EIGHT, EIGHT, EIGHT, b0[k], b1[k]);
        else
          mma_16816(eight[k][grp], EIGHT, EIGHT, EIGHT, EIGHT, b0[k], b1[k]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < NT; k++)
#pragma unroll
    for (int i = 0; i < J; i++)
#pragma unroll
      for (int c = 0; c < 4; c++) {
        s.o[k][2 * i][c] -= eight[k][i * NG / J][c & 1];
        s.o[k][2 * i + 1][c] = fmaf(-16.0f, eight[k][i * NG / J][c & 1], s.o[k][2 * i + 1][c]);
      }
}

template <int D, int NG, int NT, int UN, int STAGES>
struct AttnShape {
  static constexpr int ROWS = 8 * NT, UNIT = kv4_unit_bytes(D, D / NG), STAGE = UN * UNIT, RING = STAGES * STAGE;
  static constexpr int HEAD = 256;           // barriers, abort flag
  static constexpr int SMEM = HEAD + AT_WARPS * RING;
  static constexpr int PART = ROWS * (D + 2);  // floats of a part in the workspace: o, m, l
};

template <int D, int NG, int NT, int UN, int STAGES>
__global__ void __launch_bounds__(AT_WARPS * 32, NT == 1 ? 3 : D == 64 ? 3 : 2) kv4_attn_kernel(AttnParams p) {
  using S = AttnShape<D, NG, NT, UN, STAGES>;
  constexpr int J = D / 32, ROWS = S::ROWS;
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);                 // [AT_WARPS][STAGES]
  uint32_t* abort_flag = reinterpret_cast<uint32_t*>(smem + 192);
  static_assert(AT_WARPS * STAGES * 8 <= 192 && 200 <= S::HEAD, "shared memory head");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + S::HEAD + warp * S::RING;
  uint64_t* bar = bars + warp * STAGES;
  if (threadIdx.x < AT_WARPS * STAGES) mbar_init(bars + threadIdx.x, 1);
  if (threadIdx.x == 0) abort_flag[0] = abort_flag[1] = 0;
  fence_mbar_init();
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  Chunk chunk;
  load_chunk<ROWS>(p, 0, &chunk);
  long long line = length_of(chunk);
  if (p.a.n > 32) {
    for (int i = 32; i < p.a.n; i += 32) {
      load_chunk<ROWS>(p, i, &chunk);
      line += length_of(chunk);
    }
    load_chunk<ROWS>(p, 0, &chunk);
  }
  const long long piece = max(divide(line + p.pieces - 1, p.pieces), static_cast<long long>(AT_PIECE));
  const int me = blockIdx.x * AT_WARPS + warp;  // this warp's piece
  long long at = piece * me;
  const long long stop = min(at + piece, line);
  if (lane == 0) p.cuts[me].parts = 0;
  if (at >= stop) return;
  const WaitCtx ctx{abort_flag, p.status};
  const float cq = p.a.scale * LOG2E, cs = cq * Q4_LO_UNIT;
  const int page_units = 1 << (p.c.page_shift - 4);
  uint32_t phase = 0;  // tiles this warp has taken from its ring so far
  long long chunk_at = 0;  // where the chunk stands on the line
  int next_chunk = -1;     // a chunk's registers are not held while a sequence is worked on
  while (at < stop) {
    // ---- the sequence at `at`, and its problems from there on --------------------------------------------------------------
    if (next_chunk >= 0) load_chunk<ROWS>(p, next_chunk, &chunk);
    next_chunk = chunk.first;
    const unsigned past = __ballot_sync(0xffffffffu, chunk_at + chunk.end > at);
    if (past == 0) {
      chunk_at += length_of(chunk);
      next_chunk += 32;
      if (next_chunk >= p.a.n) break;  // (not reached: the line ends with the last sequence)
      continue;
    }
    const int of = __ffs(past) - 1;
    const long long seq_at = chunk_at + __shfl_sync(0xffffffffu, chunk.begin, of);
    Kv4Rows rows;
    rows.begin = __shfl_sync(0xffffffffu, chunk.rows.begin, of);
    rows.end = __shfl_sync(0xffffffffu, chunk.rows.end, of);
    rows.length = __shfl_sync(0xffffffffu, chunk.rows.length, of);
    rows.slot = __shfl_sync(0xffffffffu, chunk.rows.slot, of);
    const int n_rows = (rows.end - rows.begin) * p.rep, first = rows.length - (rows.end - rows.begin);
    int u_begin;
    const int units = seq_units(p, rows, &u_begin), span = units + AT_START, problems = seq_problems<ROWS>(p, rows);
    const int tiles = problems / p.c.heads;
    for (int index = static_cast<int>(divide(at - seq_at, span)); index < problems && at < stop; index++) {
      const int head = index / tiles, row0 = (index - head * tiles) * ROWS;
      const long long start = seq_at + static_cast<long long>(index) * span;  // of the problem, on the line
      const bool continued = at > start;
      const int from = max(static_cast<int>(at - start) - AT_START, 0);
      const int upto = max(static_cast<int>(min(static_cast<long long>(span), stop - start)) - AT_START, 0);
      if (lane == 0 && !continued && start + span > stop) {
        // pieces [lo, hi] hold its units: this one does not if it ends among the empty places
        const long long lo = (start + AT_START) / piece, hi = (start + span - 1) / piece;
        Cut cut;
        cut.parts = hi > lo ? static_cast<int>(hi - lo) + 1 : 0;
        cut.first = static_cast<int>(lo * 2 + (lo == me ? 1 : 0));
        cut.next = static_cast<int>(lo * 2 + 2);
        cut.row_begin = rows.begin;
        cut.n_rows = min(n_rows - row0, ROWS);
        cut.head = head;
        cut.row0 = row0;
        cut.unused = 0;
        p.cuts[me] = cut;
      }
      at = min(start + span, stop);
      if (from >= upto) continue;  // the piece ends among the problem's empty places
      // ---- its units in this piece, their pages, and the first tiles under way ----------------------------------------------
      const int last_row = min(row0 + ROWS, n_rows) - 1;
      const int visible = (max(first + last_row / p.rep + 1, 0) + KV4_UNIT - 1) / KV4_UNIT;  // units that hold a seen token
      // (units before the window of the tile's first row, whose sequence's earliest row may reach further back, are left out)
      const int window_begin = p.a.window > 0 ? max(first + row0 / p.rep + 1 - p.a.window, 0) / KV4_UNIT : 0;
      const int w0 = max(u_begin + from, window_begin), w1 = min(u_begin + upto, visible);
      int base = w0;                     // lane i knows where unit base + i is, and copies it
      const uint8_t* source = nullptr;   // (null: not there)
      auto look_up = [&](int from_unit) {
        base = from_unit;
        const int u = base + lane, page = u < w1 ? kv4_page(p.c, rows.slot, u * KV4_UNIT, p.status) : -1;
        source = page < 0 ? nullptr
                          : p.c.pages + page * p.c.page_bytes +
                                (static_cast<long long>(head) * page_units + (u & (page_units - 1))) * S::UNIT;
      };
      auto issue = [&](int u, uint32_t st) {  // units [u, u + UN) into a stage; returns which are there
        if (u + UN > base + 32) look_up(u);
        const int of = u - base, k = lane - of;
        const bool is = k >= 0 && k < UN && source != nullptr;
        const uint32_t present = __ballot_sync(0xffffffffu, is) >> of;
        if (lane == 0) mbar_arrive_expect_tx(bar + st, __popc(present) * S::UNIT);
        __syncwarp();
        if (is) bulk_load(ring + st * S::STAGE + k * S::UNIT, source, S::UNIT, bar + st);
        return present;
      };
      const int n_tiles = w0 < w1 ? (w1 - w0 + UN - 1) / UN : 0;
      if (n_tiles > 0) look_up(w0);
      uint32_t present = 0;  // UN bits a stage
      for (int k = 0; k < STAGES && k < n_tiles; k++) present |= issue(w0 + k * UN, (phase + k) % STAGES) << ((phase + k) % STAGES * UN);
      // ---- queries -------------------------------------------------------------------------------------------------------
      Queries<D, NG, NT> q;
#pragma unroll
      for (int k = 0; k < NT; k++) {
        const int row = min(row0 + k * 8 + g, n_rows - 1), token = row / p.rep;
        const __half* qp = static_cast<const __half*>(p.a.Q) + (rows.begin + token) * p.a.ldq +
                           (head * p.rep + row - token * p.rep) * D;
        float sum[NG] = {};
#pragma unroll
        for (int j = 0; j < J; j++) {
          const uint4 v = *reinterpret_cast<const uint4*>(qp + (4 * j + t) * 8);
          // dims 0..7 of the word pair up as (0, 4), (2, 6) for the low nibbles' step and (1, 5), (3, 7) for the high ones'
          q.b[k][2 * j][0] = __byte_perm(v.x, v.z, 0x5410);
          q.b[k][2 * j][1] = __byte_perm(v.y, v.w, 0x5410);
          q.b[k][2 * j + 1][0] = __byte_perm(v.x, v.z, 0x7632);
          q.b[k][2 * j + 1][1] = __byte_perm(v.y, v.w, 0x7632);
          const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(h[i]);
            sum[j * NG / J] += f.x + f.y;
          }
        }
#pragma unroll
        for (int grp = 0; grp < NG; grp++) {
          sum[grp] += __shfl_xor_sync(0xffffffffu, sum[grp], 1);
          sum[grp] += __shfl_xor_sync(0xffffffffu, sum[grp], 2);
          q.sum[2 * k][grp] = __shfl_sync(0xffffffffu, sum[grp], 8 * t) * cq;
          q.sum[2 * k + 1][grp] = __shfl_sync(0xffffffffu, sum[grp], 8 * t + 4) * cq;
        }
      }
#pragma unroll
      for (int r = 0; r < 2 * NT; r++) {  // rows behind the last repeat it
        const int pos = first + min(row0 + (r >> 1) * 8 + 2 * t + (r & 1), n_rows - 1) / p.rep;
        q.hi[r] = pos + 1;
        q.lo[r] = p.a.window > 0 ? max(pos + 1 - p.a.window, 0) : 0;
      }
      // every row sees tokens [all_lo, all_hi)
      const int all_hi = first + row0 / p.rep + 1;
      const int all_lo = p.a.window > 0 ? max(first + last_row / p.rep + 1 - p.a.window, 0) : 0;
      RowState<D, NG, NT> s;
#pragma unroll
      for (int r = 0; r < 2 * NT; r++) {
        s.m[r] = -INFINITY;
        s.l[r] = 0.0f;
#pragma unroll
        for (int grp = 0; grp < NG; grp++) s.z[r][grp] = 0.0f;
      }
#pragma unroll
      for (int k = 0; k < NT; k++)
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
          for (int c = 0; c < 4; c++) s.o[k][i][c] = 0.0f;
      s.e = -14;
      // ---- tokens ----------------------------------------------------------------------------------------------------------
#pragma unroll 1
      for (int i = 0; i < n_tiles; i++) {
        const uint32_t n = phase + i, st = n % STAGES, here = (present >> (st * UN)) & ((1u << UN) - 1);
        if (!mbar_wait_copies(bar + st, (n / STAGES) & 1, SITE_KV4_RING, ctx, abort_flag + 1)) continue;  // recorded; nothing hangs
        const int tok0 = (w0 + i * UN) * KV4_UNIT;
        const uint8_t* stage = ring + st * S::STAGE;
        if (tok0 >= all_lo && tok0 + UN * KV4_UNIT <= all_hi && here == (1u << UN) - 1)
          kv4_tile<D, NG, NT, UN, false>(stage, tok0, here, cs, q, s);
        else
          kv4_tile<D, NG, NT, UN, true>(stage, tok0, here, cs, q, s);
        __syncwarp();
        if (i + STAGES < n_tiles) {
          present &= ~(((1u << UN) - 1) << (st * UN));
          present |= issue(w0 + (i + STAGES) * UN, st) << (st * UN);
        }
      }
      phase += n_tiles;
      // ---- rows 2t, 2t + 1: finish, or leave a part ---------------------------------------------------------------------------
      const bool whole = from == 0 && upto == units;
      float* part = p.part + (static_cast<long long>(me) * 2 + (continued ? 0 : 1)) * S::PART;
      const float down = pow2i(s.e - 14);
#pragma unroll
      for (int r = 0; r < 2 * NT; r++) {
        const int in_tile = (r >> 1) * 8 + 2 * t + (r & 1), row = row0 + in_tile;
        s.l[r] += __shfl_xor_sync(0xffffffffu, s.l[r], 4);
        s.l[r] += __shfl_xor_sync(0xffffffffu, s.l[r], 8);
        s.l[r] += __shfl_xor_sync(0xffffffffu, s.l[r], 16);
#pragma unroll
        for (int grp = 0; grp < NG; grp++) {
          s.z[r][grp] += __shfl_xor_sync(0xffffffffu, s.z[r][grp], 4);
          s.z[r][grp] += __shfl_xor_sync(0xffffffffu, s.z[r][grp], 8);
          s.z[r][grp] += __shfl_xor_sync(0xffffffffu, s.z[r][grp], 16);
        }
        if (row >= n_rows) continue;
        const int token = row / p.rep, h = head * p.rep + row - token * p.rep;
        const long long out = rows.begin + token;
        const float inv = s.l[r] == 0.0f ? 0.0f : 1.0f / s.l[r];  // (a row that saw nothing has only zeros)
#pragma unroll
        for (int i = 0; i < J; i++) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const float zero = s.z[r][i * NG / J];
            v[2 * k] = fmaf(s.o[r >> 1][2 * i][2 * k + (r & 1)] * Q4_LO_UNIT, down, zero);
            v[2 * k + 1] = fmaf(s.o[r >> 1][2 * i + 1][2 * k + (r & 1)] * Q4_HI_UNIT, down, zero);
          }
          if (whole)
            *reinterpret_cast<uint2*>(static_cast<__half*>(p.a.O) + out * p.a.ldo + h * D + 32 * i + 4 * g) =
                make_uint2(pack_output(v[0] * inv, v[1] * inv), pack_output(v[2] * inv, v[3] * inv));
          else
            *reinterpret_cast<float4*>(part + in_tile * D + 32 * i + 4 * g) = make_float4(v[0], v[1], v[2], v[3]);
        }
        if (g == 0) {
          if (!whole) {
            part[ROWS * D + in_tile] = s.m[r];
            part[ROWS * D + ROWS + in_tile] = s.l[r];
          } else if (p.a.lse) {
            p.a.lse[out * p.a.ldl + h] = s.l[r] == 0.0f ? -INFINITY : fmaf(s.m[r], LN2, logf(s.l[r]));
          }
        }
      }
    }
  }
}

constexpr int JOIN_THREADS = 512;

// Joins the parts of problems that were cut.  An item is one row of a problem; CTA b looks at items b, b + gridDim.x, ... all
// at once, for most pieces end without a cut, and joins those that there are: rows of up to JOIN_WARP parts a warp each, all
// warps at the same time (no barrier in it), then the longer ones with the whole block.  (With a block to every row the 96
// problems of 12 sequences of 1635 tokens, a dozen parts each, took 27 us to join.)
constexpr int JOIN_WARP = 32;

template <int D, int ROWS>
__global__ void __launch_bounds__(JOIN_THREADS) kv4_join_kernel(AttnParams p, int rows) {
  constexpr int PART = ROWS * (D + 2), GROUPS = JOIN_THREADS / D, WARPS = JOIN_THREADS / 32, DIMS = D / 32;
  __shared__ float weight[JOIN_THREADS], top[WARPS], so[GROUPS][D], sl[WARPS];
  __shared__ int list[JOIN_THREADS], listed;
  if (threadIdx.x == 0) listed = 0;
  __syncthreads();
  pdl_wait();
  {
    // (the launch sees to it that a CTA has at most JOIN_THREADS items)
    const int item = blockIdx.x + threadIdx.x * gridDim.x;
    if (item < p.pieces * rows) {
      const Cut& c = p.cuts[item / rows];
      if (c.parts > 0 && item % rows < c.n_rows) list[atomicAdd(&listed, 1)] = item;
    }
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto part_of = [&](const Cut& cut, int i) {
    return p.part + static_cast<long long>(i == 0 ? cut.first : cut.next + 2 * (i - 1)) * PART;
  };
  auto place = [&](const Cut& cut, int r, long long* out, int* h) {
    const int row = cut.row0 + r, token = row / p.rep;
    *out = cut.row_begin + token;
    *h = cut.head * p.rep + row - token * p.rep;
  };
  bool longer = false;
  for (int at = warp; at < listed; at += WARPS) {
    const Cut cut = p.cuts[list[at] / rows];
    const int n = cut.parts, r = list[at] % rows;
    if (n > JOIN_WARP) {
      longer = true;
      continue;
    }
    constexpr int AHEAD = 8;  // parts whose o is on its way while the weights are found
    float v[AHEAD][DIMS];
    auto fetch = [&](int k0) {
#pragma unroll
      for (int k = 0; k < AHEAD; k++)
        if (k0 + k < n) {
          const float* from = part_of(cut, k0 + k) + r * D + lane * DIMS;
#pragma unroll
          for (int d = 0; d < DIMS; d++) v[k][d] = from[d];
        }
    };
    fetch(0);
    float mi = -INFINITY, l = 0.0f;
    if (lane < n) {
      const float* part = part_of(cut, lane);
      mi = part[ROWS * D + r];
      l = part[ROWS * D + ROWS + r];
    }
    float m = mi, o[DIMS] = {};
#pragma unroll
    for (int k = 16; k > 0; k /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    const float f = l == 0.0f ? 0.0f : exp2_approx(mi - m);  // (the weight of a part that saw nothing)
    l = l == 0.0f ? 0.0f : l * f;
    for (int k0 = 0; k0 < n; k0 += AHEAD) {
      if (k0 > 0) fetch(k0);
#pragma unroll
      for (int k = 0; k < AHEAD; k++) {
        const float fk = __shfl_sync(0xffffffffu, f, k0 + k);
        if (k0 + k < n)
#pragma unroll
          for (int d = 0; d < DIMS; d++) o[d] = fmaf(v[k][d], fk, o[d]);
      }
    }
#pragma unroll
    for (int k = 16; k > 0; k /= 2) l += __shfl_xor_sync(0xffffffffu, l, k);
    long long out;
    int h;
    place(cut, r, &out, &h);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    __half* to = static_cast<__half*>(p.a.O) + out * p.a.ldo + h * D + lane * DIMS;
#pragma unroll
    for (int d = 0; d < DIMS; d += 2) *reinterpret_cast<uint32_t*>(to + d) = pack_output(o[d] * inv, o[d + 1] * inv);
    if (lane == 0 && p.a.lse) p.a.lse[out * p.a.ldl + h] = l == 0.0f ? -INFINITY : fmaf(m, LN2, logf(l));
  }
  if (!__syncthreads_or(longer)) return;
  const int d = threadIdx.x % D, group = threadIdx.x / D;
  for (int at = 0; at < listed; at++) {
    const Cut cut = p.cuts[list[at] / rows];
    const int n = cut.parts, r = list[at] % rows;
    if (n <= JOIN_WARP) continue;
    // the largest maximum, then every part's weight
    float m = -INFINITY;
    for (int i = threadIdx.x; i < n; i += JOIN_THREADS) m = fmaxf(m, part_of(cut, i)[ROWS * D + r]);
#pragma unroll
    for (int k = 16; k > 0; k /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    if (lane == 0) top[warp] = m;
    __syncthreads();
    for (int w = 0; w < WARPS; w++) m = fmaxf(m, top[w]);
    float l = 0.0f, o = 0.0f;
    for (int i0 = 0; i0 < n; i0 += JOIN_THREADS) {
      const int i = i0 + threadIdx.x;
      if (i < n) {
        const float* part = part_of(cut, i);
        const float mi = part[ROWS * D + r], li = part[ROWS * D + ROWS + r];
        const float f = li == 0.0f ? 0.0f : exp2_approx(mi - m);
        weight[threadIdx.x] = f;
        if (li != 0.0f) l = fmaf(li, f, l);
      }
      __syncthreads();
      const int end = min(n - i0, JOIN_THREADS);
#pragma unroll 8
      for (int k = group; k < end; k += GROUPS) o = fmaf(part_of(cut, i0 + k)[r * D + d], weight[k], o);
      __syncthreads();
    }
#pragma unroll
    for (int k = 16; k > 0; k /= 2) l += __shfl_xor_sync(0xffffffffu, l, k);
    if (lane == 0) sl[warp] = l;
    so[group][d] = o;
    __syncthreads();
    if (group == 0) {
      l = o = 0.0f;
      for (int w = 0; w < WARPS; w++) l += sl[w];
      for (int k = 0; k < GROUPS; k++) o += so[k][d];
      long long out;
      int h;
      place(cut, r, &out, &h);
      static_cast<__half*>(p.a.O)[out * p.a.ldo + h * D + d] = __ushort_as_half(static_cast<uint16_t>(pack_output(l == 0.0f ? 0.0f : o / l, 0.0f)));
      if (d == 0 && p.a.lse) p.a.lse[out * p.a.ldl + h] = l == 0.0f ? -INFINITY : fmaf(m, LN2, logf(l));
    }
    __syncthreads();
  }
}

constexpr int AT_MOST_PER_SM = 4;

// CTAs of a kernel that share an SM, asked for once per device.
template <int D, int NG, int NT, int UN, int STAGES>
cudaError_t per_sm_of(int* per_sm) {
  constexpr int smem = AttnShape<D, NG, NT, UN, STAGES>::SMEM;
  auto kernel = kv4_attn_kernel<D, NG, NT, UN, STAGES>;
  static std::atomic<int> known[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  *per_sm = dev < 64 ? known[dev].load(std::memory_order_acquire) : 0;
  if (*per_sm > 0) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, kernel, AT_WARPS * 32, smem);
  if (e != cudaSuccess) return e;
  *per_sm = *per_sm < 1 ? 1 : *per_sm > AT_MOST_PER_SM ? AT_MOST_PER_SM : *per_sm;
  if (dev < 64) known[dev].store(*per_sm, std::memory_order_release);
  return cudaSuccess;
}

template <int D, int NG, int NT, int UN, int STAGES>
cudaError_t launch_attn(AttnParams& p, int most_rows, int sm_count, cudaStream_t stream) {
  using S = AttnShape<D, NG, NT, UN, STAGES>;
  int per_sm = 0;
  cudaError_t e = per_sm_of<D, NG, NT, UN, STAGES>(&per_sm);
  if (e != cudaSuccess) return e;
  // no more warps than pieces of the smallest size, if the tables are narrow
  const long long most = (static_cast<long long>(p.c.table_width) << (p.c.page_shift - 4)) + AT_START;
  const long long problems = static_cast<long long>(p.c.heads) *
                             (p.a.ind ? static_cast<long long>(p.a.T) * p.rep / S::ROWS + p.a.n
                                      : static_cast<long long>(p.a.n) * ((p.rep + S::ROWS - 1) / S::ROWS));
  int ctas = sm_count * per_sm;
  if (problems < ctas * AT_WARPS) ctas = static_cast<int>(min(static_cast<long long>(ctas), (problems * most + AT_PIECE * AT_WARPS - 1) / (AT_PIECE * AT_WARPS)));
  p.pieces = ctas * AT_WARPS;
  e = launch_with_pdl(kv4_attn_kernel<D, NG, NT, UN, STAGES>, dim3(ctas), dim3(AT_WARPS * 32), S::SMEM, stream, p);
  if (e != cudaSuccess) return e;
  const int rows = min(most_rows, S::ROWS), join_ctas = min(p.pieces * rows, 4 * sm_count);
  static_assert(AT_MOST_PER_SM * AT_WARPS * S::ROWS <= 4 * JOIN_THREADS, "a CTA's items of the joining kernel");
  return launch_with_pdl(kv4_join_kernel<D, S::ROWS>, dim3(join_ctas), dim3(JOIN_THREADS), 0, stream, p, rows);
}

template <int D, int NG>
cudaError_t launch_rows_of(AttnParams& p, int nt, int most_rows, int sm_count, cudaStream_t stream) {
  return nt == 1 ? launch_attn<D, NG, 1, 4, 2>(p, most_rows, sm_count, stream) : launch_attn<D, NG, 2, 2, 2>(p, most_rows, sm_count, stream);
}

// Rows of a problem: eight where every sequence brings at most eight rows a key/value head, sixteen otherwise.
int row_tiles(const Kv4View& c, int T, int n, int q_heads, bool one_each) { return q_heads / c.heads > 8 || (!one_each && T > n) ? 2 : 1; }

}  // namespace

size_t kv4_attention_workspace(const Kv4View& c, int sm_count) {
  return static_cast<size_t>(sm_count) * AT_MOST_PER_SM * AT_WARPS * (sizeof(Cut) + 2 * (16 * (c.D + 2)) * sizeof(float));
}

int launch_kv4_attention(const Kv4View& c, const Kv4AttnArgs& a, void* workspace, int sm_count, uint32_t* status,
                         cudaStream_t stream, const char** err) {
  Cut* cuts = static_cast<Cut*>(workspace);
  AttnParams p{c, a, a.q_heads / c.heads, 0, cuts, reinterpret_cast<float*>(cuts + sm_count * AT_MOST_PER_SM * AT_WARPS), status};
  const int nt = row_tiles(c, a.T, a.n, a.q_heads, a.ind == nullptr);
  const int most_rows = a.ind ? 8 * nt : p.rep;  // rows of a problem that can be there
  const int ng = c.D / c.G;
  cudaError_t e;
  if (c.D == 128)
    e = ng == 1 ? launch_rows_of<128, 1>(p, nt, most_rows, sm_count, stream)
      : ng == 2 ? launch_rows_of<128, 2>(p, nt, most_rows, sm_count, stream)
                : launch_rows_of<128, 4>(p, nt, most_rows, sm_count, stream);
  else
    e = ng == 1 ? launch_rows_of<64, 1>(p, nt, most_rows, sm_count, stream) : launch_rows_of<64, 2>(p, nt, most_rows, sm_count, stream);
  if (e == cudaSuccess) return 0;
  *err = cudaGetErrorString(e);
  return -3;
}

}  // namespace ph
