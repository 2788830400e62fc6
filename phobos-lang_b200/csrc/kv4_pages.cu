// Pages of the 4-bit cache: extending, forking, freeing and compacting sequences.
//
// What is free is told by the reference counts alone (refs[page] == 0), so there is no list that can come apart from
// them, and a fresh page is always the lowest free one: the outcome does not depend on timing.  A change that needs
// pages is planned by one CTA (counts, prefix sums, the free pages in order) and is all or nothing; the pages' bytes
// are then moved by the whole GPU from the list that the plan left in the workspace.
// Measured: copying 16 sequences of 2000 tokens in 16 layers, 1 GB read and written: 165 us, 6.2 TB/s.  A plan
// takes 7 to 9 us for up to 48 rows and grows with them: extending 1000, 4096 and 65536 branches of one prompt takes 46, 126
// and 2281 us in all, as many sequences that share nothing 29, 69 and 1113.
#include "kv4.cuh"

namespace ph {
namespace {

constexpr int PLAN_THREADS = 1024;
constexpr int MOVE_THREADS = 256;

// Workspace: header | claims, one per sequence | rows, one per sequence | free pages / page map | moves (from, to).
struct Plan {
  int* n_moves;
  int* claim;   // [max_seqs] the first row of the call that names a sequence
  int* fresh;   // [max_seqs] fresh pages of a row, then where its fresh pages start
  int* last;    // [max_seqs] the shared, partly filled page that a row extends, or -1
  int* pages;   // [n_pages] free pages in order; for compaction a page's new place
  int2* moves;  // [n_pages]
};

__host__ __device__ inline size_t up16(size_t x) { return (x + 15) & ~size_t(15); }

__host__ inline Plan plan_of(const Kv4View& c, void* ws) {
  char* w = static_cast<char*>(ws);
  Plan p;
  p.n_moves = reinterpret_cast<int*>(w);
  w += 16;
  const size_t rows = up16(static_cast<size_t>(c.max_seqs) * 4);
  p.claim = reinterpret_cast<int*>(w);
  w += rows;
  p.fresh = reinterpret_cast<int*>(w);
  w += rows;
  p.last = reinterpret_cast<int*>(w);
  w += rows;
  p.pages = reinterpret_cast<int*>(w);
  w += up16(static_cast<size_t>(c.n_pages) * 4);
  p.moves = reinterpret_cast<int2*>(w);
  return p;
}

// The rows' arrays of a call stand in shared memory where they fit: a planning block reads back what it wrote three times,
// and each time costs a trip to L2 otherwise.
constexpr int PLAN_SHARED = 40 * 1024;  // (with what the kernels have besides, within the 48 KB that need no asking)
__host__ inline int plan_shared(const Kv4View& c) { return c.max_seqs <= PLAN_SHARED / 12 ? c.max_seqs * 12 : 0; }
__device__ __forceinline__ void use_shared(const Kv4View& c, Plan* p) {
  extern __shared__ int rows_of_call[];
  if (c.max_seqs > PLAN_SHARED / 12) return;
  p->claim = rows_of_call;
  p->fresh = rows_of_call + c.max_seqs;
  p->last = rows_of_call + 2 * c.max_seqs;
}

// Exclusive prefix sum over the CTA, and the total; all threads call.
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int warp_sum[33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int u = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += u;
  }
  __syncthreads();  // the previous scan's sums have been read
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  if (warp == 0) {
    const int w = warp_sum[lane];
    int x = w;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int u = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += u;
    }
    warp_sum[lane] = x - w;
    if (lane == 31) warp_sum[32] = x;
  }
  __syncthreads();
  *total = warp_sum[32];
  return warp_sum[warp] + s - v;
}

// Writes the lowest free pages to `out` until `want` are found; returns how many were found (want at most, exact below).
__device__ int collect_free(const int* refs, int n_pages, int want, int* out) {
  int found = 0;
  for (int i0 = 0; i0 < n_pages && found < want; i0 += 4 * PLAN_THREADS) {
    const int at = i0 + threadIdx.x * 4;
    bool free[4];
    int mine = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      free[k] = at + k < n_pages && refs[at + k] == 0;
      mine += free[k];
    }
    int total;
    int pos = found + block_scan(mine, &total);
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (free[k]) {
        if (pos < want) out[pos] = at + k;
        pos++;
      }
    found += total;
  }
  __syncthreads();
  return min(found, want);
}

__device__ __forceinline__ int pages_for(const Kv4View& c, int tokens) {
  return static_cast<int>((static_cast<long long>(tokens) + (1 << c.page_shift) - 1) >> c.page_shift);
}

// Claims every named sequence for the first row that names it.
__device__ void claim_rows(const Kv4View& c, const Plan& p, const int* slots, int n) {
  for (int i = threadIdx.x; i < c.max_seqs; i += PLAN_THREADS) p.claim[i] = n;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS)
    if (slots[i] >= 0 && slots[i] < c.max_seqs) atomicMin(&p.claim[slots[i]], i);
  __syncthreads();
}

// Turns p.fresh[0..n) into starts; returns the sum (which may pass 32 bits for nonsense counts).
__device__ long long scan_fresh(const Plan& p, int n) {
  long long base = 0;
  for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x;
    const int v = i < n ? p.fresh[i] : 0;
    int total;
    const int before = block_scan(v, &total);
    if (i < n) p.fresh[i] = static_cast<int>(base + before);
    base += total;
  }
  __syncthreads();
  return base;
}

__global__ void __launch_bounds__(PLAN_THREADS) extend_plan_kernel(Kv4View c, Plan p, const int* slots, const int* counts, int n,
                                                                   int* shortfall) {
  pdl_wait();
  pdl_launch_dependents();
  use_shared(c, &p);
  __shared__ int wrong, moves;
  if (threadIdx.x == 0) {
    wrong = 0;
    moves = 0;
    *p.n_moves = 0;
  }
  claim_rows(c, p, slots, n);
  const int in_page = (1 << c.page_shift) - 1;
  bool shares = false;
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int slot = slots[i], add = counts[i];
    int fresh = 0, last = -1;
    if (slot < 0 || slot >= c.max_seqs || p.claim[slot] != i || add < 0) {
      wrong = 1;
    } else {
      const int len = c.lens[slot];
      if (len < 0 || static_cast<long long>(len) + add > static_cast<long long>(c.table_width) << c.page_shift ||
          static_cast<long long>(len) + add > 0x7fffffffLL) {
        wrong = 1;
      } else {
        const int have = pages_for(c, len);
        fresh = pages_for(c, len + add) - have;
        if (add > 0 && (len & in_page)) {
          const int page = c.tables[static_cast<long long>(slot) * c.table_width + have - 1];
          if (page < 0 || page >= c.n_pages) {
            wrong = 1;
          } else if (c.refs[page] > 1) {
            last = page;
            shares = true;
            p.moves[page] = make_int2(0, -1);
          }
        }
      }
    }
    p.fresh[i] = fresh;
    p.last[i] = last;
  }
  // Of the rows that extend one shared page all copy it, but where they are all that hold it the last one keeps it: what doing
  // them one after another would give.  The moves' places are free until then and count the rows of each such page.
  if (__syncthreads_or(shares)) {
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS)
      if (p.last[i] >= 0) {
        atomicAdd(&p.moves[p.last[i]].x, 1);
        atomicMax(&p.moves[p.last[i]].y, i);
      }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
      const int last = p.last[i];
      if (last < 0) continue;
      const int2 rows = __ldcg(&p.moves[last]);
      if (rows.x > c.refs[last]) wrong = 1;  // (more tables name the page than its count says)
      if (rows.x < c.refs[last] || rows.y != i) p.fresh[i]++;
    }
    __syncthreads();
  }
  // a row's fresh pages beyond those its length asks for are the copy's
  const long long want = scan_fresh(p, n);
  if (wrong) {
    if (threadIdx.x == 0) *shortfall = -1;
    return;
  }
  const int ask = want > c.n_pages ? c.n_pages : static_cast<int>(want);
  const int found = collect_free(c.refs, c.n_pages, ask, p.pages);
  if (found < want) {
    if (threadIdx.x == 0) *shortfall = static_cast<int>(min(want - found, 0x7fffffffLL));
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = warp; i < n; i += PLAN_THREADS / 32) {
    const int slot = slots[i], len = c.lens[slot], have = pages_for(c, len);
    const int begin = p.fresh[i], end = i + 1 < n ? p.fresh[i + 1] : static_cast<int>(want);
    const bool copies = end - begin > pages_for(c, len + counts[i]) - have;
    int* row = c.tables + static_cast<long long>(slot) * c.table_width + have - (copies ? 1 : 0);
    for (int k = lane; k < end - begin; k += 32) {
      const int page = p.pages[begin + k];
      if (copies && k == 0) {
        p.moves[atomicAdd(&moves, 1)] = make_int2(row[0], page);
        atomicSub(&c.refs[row[0]], 1);
      }
      row[k] = page;
      c.refs[page] = 1;
    }
    __syncwarp();
    if (lane == 0) c.lens[slot] = len + counts[i];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    *p.n_moves = moves;
    *shortfall = 0;
  }
}

__global__ void __launch_bounds__(PLAN_THREADS) fork_plan_kernel(Kv4View c, Plan p, const int* src, const int* dst, int n,
                                                                 int deep, int* shortfall) {
  pdl_wait();
  pdl_launch_dependents();
  use_shared(c, &p);
  __shared__ int wrong;
  if (threadIdx.x == 0) {
    wrong = 0;
    *p.n_moves = 0;
  }
  claim_rows(c, p, dst, n);
  for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
    const int a = src[i], b = dst[i];
    int need = 0;
    if (a < 0 || a >= c.max_seqs || b < 0 || b >= c.max_seqs || p.claim[b] != i || c.lens[b] != 0 || c.lens[a] < 0 ||
        c.lens[a] > static_cast<long long>(c.table_width) << c.page_shift)
      wrong = 1;
    else
      need = pages_for(c, c.lens[a]);
    p.fresh[i] = need;
    if (!wrong) p.last[i] = c.lens[a];  // lengths as they are before any row changes
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (!wrong)  // every page that is to be shared or copied has to exist
    for (int i = warp; i < n; i += PLAN_THREADS / 32)
      for (int k = lane; k < p.fresh[i]; k += 32) {
        const int page = c.tables[static_cast<long long>(src[i]) * c.table_width + k];
        if (page < 0 || page >= c.n_pages) wrong = 1;
      }
  __syncthreads();
  const bool refused = wrong;
  const long long want = scan_fresh(p, n);
  if (refused) {
    if (threadIdx.x == 0) *shortfall = -1;
    return;
  }
  if (deep) {
    const int ask = want > c.n_pages ? c.n_pages : static_cast<int>(want);
    const int found = collect_free(c.refs, c.n_pages, ask, p.pages);
    if (found < want) {
      if (threadIdx.x == 0) *shortfall = static_cast<int>(min(want - found, 0x7fffffffLL));
      return;
    }
  }
  for (int i = warp; i < n; i += PLAN_THREADS / 32) {
    const int* from = c.tables + static_cast<long long>(src[i]) * c.table_width;
    int* to = c.tables + static_cast<long long>(dst[i]) * c.table_width;
    const int begin = p.fresh[i], need = pages_for(c, p.last[i]);
    for (int k = lane; k < need; k += 32) {
      const int page = from[k];
      if (deep) {
        const int fresh = p.pages[begin + k];
        p.moves[begin + k] = make_int2(page, fresh);
        c.refs[fresh] = 1;
        to[k] = fresh;
      } else {
        atomicAdd(&c.refs[page], 1);
        to[k] = page;
      }
    }
    if (lane == 0) c.lens[dst[i]] = p.last[i];
  }
  if (threadIdx.x == 0) {
    *p.n_moves = deep ? static_cast<int>(want) : 0;
    *shortfall = 0;
  }
}

// One CTA per row: gives back the pages behind the first `keep` tokens.
__global__ void __launch_bounds__(MOVE_THREADS) free_kernel(Kv4View c, const int* slots, const int* keep, int n) {
  pdl_wait();
  pdl_launch_dependents();
  const int i = blockIdx.x, slot = slots[i];
  if (slot < 0 || slot >= c.max_seqs) return;
  int earlier = 0;  // a sequence that is named twice goes by its first row
  for (int j = threadIdx.x; j < i; j += MOVE_THREADS) earlier |= slots[j] == slot;
  if (__syncthreads_or(earlier)) return;
  const int len = c.lens[slot], left = keep ? keep[i] : 0;
  if (left < 0 || left >= len) return;
  const int begin = pages_for(c, left), end = min(pages_for(c, len), c.table_width);
  for (int k = begin + threadIdx.x; k < end; k += MOVE_THREADS) {
    int* at = c.tables + static_cast<long long>(slot) * c.table_width + k;
    const int page = *at;
    *at = -1;
    if (page >= 0 && page < c.n_pages) atomicSub(&c.refs[page], 1);
  }
  __syncthreads();
  if (threadIdx.x == 0) c.lens[slot] = left;
}

// With L live pages: the live pages at L and above, in order, go to the free places below L, in order.
__global__ void __launch_bounds__(PLAN_THREADS) compact_plan_kernel(Kv4View c, Plan p, int* live_out) {
  pdl_wait();
  pdl_launch_dependents();
  int live = 0;
  for (int i0 = 0; i0 < c.n_pages; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x;
    live += __syncthreads_count(i < c.n_pages && c.refs[i] > 0);
  }
  int movers = 0, holes = 0;
  for (int i0 = 0; i0 < c.n_pages; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x;
    const bool is = i < c.n_pages && c.refs[i] > 0;
    const bool mover = is && i >= live, hole = i < live && !is;
    int total;
    const int packed = block_scan((mover ? 1 : 0) | (hole ? 1 << 16 : 0), &total);
    if (mover) p.moves[movers + (packed & 0xffff)].x = i;
    if (hole) p.moves[holes + (packed >> 16)].y = i;
    if (i >= live && i < c.n_pages && !is) p.pages[i] = i;
    movers += total & 0xffff;
    holes += total >> 16;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < movers; k += PLAN_THREADS) {
    const int2 m = p.moves[k];
    p.pages[m.x] = m.y;
    c.refs[m.y] = c.refs[m.x];
    c.refs[m.x] = 0;
  }
  if (threadIdx.x == 0) {
    *p.n_moves = movers;
    *live_out = live;
  }
}

// Moves pages of every layer; the list and its length come from the plan.  An item is 16 KB of one page.  After a
// compaction's plan (live not null) it also renames the pages at L = *live and above in the tables.
__global__ void __launch_bounds__(MOVE_THREADS) move_kernel(Kv4View c, Plan p, const int* live) {
  pdl_wait();
  pdl_launch_dependents();
  const int* n_moves = p.n_moves;
  const int2* moves = p.moves;
  if (live) {
    const int l = *live;
    for (int slot = blockIdx.x; slot < c.max_seqs; slot += gridDim.x) {
      const int used = min(pages_for(c, max(c.lens[slot], 0)), c.table_width);
      int* row = c.tables + static_cast<long long>(slot) * c.table_width;
      for (int k = threadIdx.x; k < used; k += MOVE_THREADS) {
        const int page = row[k];
        if (page >= l && page < c.n_pages) row[k] = p.pages[page];
      }
    }
  }
  constexpr int ITEM = 16384;
  const int chunks = static_cast<int>((c.page_bytes + ITEM - 1) / ITEM);
  const long long items = static_cast<long long>(*n_moves) * c.layers * chunks;
  for (long long it = blockIdx.x; it < items; it += gridDim.x) {
    const int chunk = static_cast<int>(it % chunks);
    const long long rest = it / chunks;
    const int layer = static_cast<int>(rest % c.layers);
    const int2 m = moves[rest / c.layers];
    uint8_t* base = c.pages + layer * c.layer_pitch + static_cast<long long>(chunk) * ITEM;
    const int n = static_cast<int>(min(static_cast<long long>(ITEM), c.page_bytes - static_cast<long long>(chunk) * ITEM)) / 16;
    const uint4* from = reinterpret_cast<const uint4*>(base + m.x * c.page_bytes);
    uint4* to = reinterpret_cast<uint4*>(base + m.y * c.page_bytes);
    uint4 v[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (threadIdx.x + k * MOVE_THREADS < n) v[k] = from[threadIdx.x + k * MOVE_THREADS];
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (threadIdx.x + k * MOVE_THREADS < n) to[threadIdx.x + k * MOVE_THREADS] = v[k];
  }
}

// Launches one after another; nothing more once one has failed.
struct Launches {
  cudaStream_t stream;
  cudaError_t error = cudaSuccess;
  template <typename... KArgs, typename... Args>
  void add(void (*kernel)(KArgs...), int blocks, int threads, int shared, Args... args) {
    if (error == cudaSuccess) error = launch_with_pdl(kernel, dim3(blocks), dim3(threads), shared, stream, args...);
  }
  void move(const Kv4View& c, const Plan& p, int sm_count, const int* live = nullptr) {
    add(move_kernel, sm_count * 8, MOVE_THREADS, 0, c, p, live);
  }
  int done(const char** err) const {
    if (error == cudaSuccess) return 0;
    *err = cudaGetErrorString(error);
    return -3;
  }
};

}  // namespace

size_t kv4_pages_workspace(const Kv4View& c) {
  return 16 + 3 * up16(static_cast<size_t>(c.max_seqs) * 4) + up16(static_cast<size_t>(c.n_pages) * 4) +
         static_cast<size_t>(c.n_pages) * 8;
}

int launch_kv4_extend(const Kv4View& c, const int* slots, const int* counts, int n, int* shortfall, void* workspace,
                      int sm_count, cudaStream_t stream, const char** err) {
  const Plan p = plan_of(c, workspace);
  Launches l{stream};
  l.add(extend_plan_kernel, 1, PLAN_THREADS, plan_shared(c), c, p, slots, counts, n, shortfall);
  l.move(c, p, sm_count);
  return l.done(err);
}

int launch_kv4_fork(const Kv4View& c, const int* src, const int* dst, int n, int deep, int* shortfall, void* workspace,
                    int sm_count, cudaStream_t stream, const char** err) {
  const Plan p = plan_of(c, workspace);
  Launches l{stream};
  l.add(fork_plan_kernel, 1, PLAN_THREADS, plan_shared(c), c, p, src, dst, n, deep, shortfall);
  if (deep) l.move(c, p, sm_count);
  return l.done(err);
}

int launch_kv4_free(const Kv4View& c, const int* slots, const int* keep, int n, cudaStream_t stream, const char** err) {
  Launches l{stream};
  l.add(free_kernel, n, MOVE_THREADS, 0, c, slots, keep, n);
  return l.done(err);
}

int launch_kv4_compact(const Kv4View& c, int* live, void* workspace, int sm_count, cudaStream_t stream, const char** err) {
  const Plan p = plan_of(c, workspace);
  Launches l{stream};
  l.add(compact_plan_kernel, 1, PLAN_THREADS, 0, c, p, live);
  l.move(c, p, sm_count, live);
  return l.done(err);
}

}  // namespace ph
