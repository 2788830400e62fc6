// The 4-bit key/value cache as the kernels see it.
//
// A page holds page_tokens tokens of every key/value head of one layer: [heads][page_tokens / 16] units, a unit being
// 16 tokens of one head:
//   K codes 8 D bytes | V codes 8 D bytes | K (scale, zero) [16][D / G] | V (scale, zero) [16][D / G]   (f16 pairs)
// value = zero + scale * code.  Codes stand in the order a warp feeds them to the matrix unit (lane 4g + t):
//   K, the A operand of S^T = K Q^T: token 8h + g, dims 8 (4j + t) .. + 7 are the 32-bit word at byte
//     4 D h + lane D / 8 + 4 j.  One matrix step takes the low nibbles of the words of both h, the next the high ones.
//   V, the A operand of O^T = V^T P^T: token 8h + 2t + l, dims 32 p + 4 g .. + 3 are the 16-bit word at byte
//     4 D h + lane D / 8 + 4 p + 2 l.  Low nibbles make one tile of 16 dims, high ones another.
// A token's bytes are its own (no byte holds two tokens), so tokens are written without reading their neighbours.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

namespace ph {

constexpr int KV4_UNIT = 16;  // tokens of a unit

// What a kernel found wrong in the caller's device-side data (recorded in the status word; the access is left out).
enum Kv4Site : uint32_t { SITE_KV4_SLOT = 0x81, SITE_KV4_PAGE = 0x82 };

__host__ __device__ constexpr int kv4_unit_bytes(int D, int G) { return 16 * D + 128 * (D / G); }

__device__ __forceinline__ void kv4_report(uint32_t* status, uint32_t site) {
  atomicCAS(status, 0u, site | (blockIdx.x << 8));
}

// Rows of a batch: rows [begin, end) of the caller's tensors are the last (end - begin) tokens of sequence `slot`.
struct Kv4Rows {
  int begin, end, length;  // length 0 for a slot that does not exist
  int slot;
};
__device__ __forceinline__ Kv4Rows kv4_rows(const Kv4View& c, const int* slots, const int* ind, int b, int T, uint32_t* status) {
  Kv4Rows r;
  r.begin = ind ? min(max(ind[b], 0), T) : b;
  r.end = ind ? min(max(ind[b + 1], r.begin), T) : b + 1;
  r.slot = slots[b];
  const bool ok = r.slot >= 0 && r.slot < c.max_seqs;
  if (!ok) kv4_report(status, SITE_KV4_SLOT);
  r.length = ok ? max(c.lens[r.slot], 0) : 0;
  return r;
}

// The page that holds token `pos` of a sequence, or -1 (recorded) where the table has none.
__device__ __forceinline__ int kv4_page(const Kv4View& c, int slot, int pos, uint32_t* status) {
  const int i = pos >> c.page_shift;
  const int page = i < c.table_width ? c.tables[static_cast<long long>(slot) * c.table_width + i] : -1;
  if (page >= 0 && page < c.n_pages) return page;
  kv4_report(status, SITE_KV4_PAGE);
  return -1;
}

}  // namespace ph
