// Internal launcher interface between api.cu and the kernel translation units.
#pragma once
#include <cstdlib>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ph {

// Launches `kernel` so that its prologue may overlap the tail of the kernel before it on the stream
// (programmatic stream serialization); the kernel calls pdl_wait() before its first dependent access.
// PHOBOS_PDL=0 falls back to an ordinary launch.
// launch_clusters_with_pdl: the same in clusters of `cluster` CTAs along x.
template <typename... KArgs, typename... Args>
cudaError_t launch_clusters_with_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, unsigned cluster, size_t smem, cudaStream_t stream,
                                     Args... args) {
  static const bool off = [] {
    const char* e = getenv("PHOBOS_PDL");
    return e && e[0] == '0';
  }();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (!off) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 0) {  // (0: the kernel is not one for clusters, or says itself of how many CTAs)
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    n++;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}
template <typename... KArgs, typename... Args>
cudaError_t launch_with_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  return launch_clusters_with_pdl(kernel, grid, block, 0, smem, stream, args...);
}


// gemm_tc.cu — f16 operands on tcgen05 tensor cores.
int launch_gemm_tc(const void* A, long long lda, const void* B, long long ldb, void* C, long long ldc, int M, int N,
                   int K, float alpha, float beta, bool acc_f16, bool c_f16, int sm_count,
                   uint32_t* status, cudaStream_t stream, const char** err);
// gemm_tc2.cu — the same operator on CTA pairs (cta_group::2), for large problems.  `workspace` (optional,
// gemm_tc_pair_workspace_bytes, 256-byte aligned) lets the kernel share out its last rounds of tiles by k-blocks.
int launch_gemm_tc_pair(const void* A, long long lda, const void* B, long long ldb, void* C, long long ldc, int M, int N,
                        int K, float alpha, float beta, bool acc_f16, bool c_f16, int sm_count, void* workspace,
                        size_t workspace_bytes, uint32_t* status, cudaStream_t stream, const char** err);
size_t gemm_tc_pair_workspace_bytes(int M, int N, int K, int sm_count);

// tmap.cu — TMA descriptors (cuTensorMapEncodeTiled through the runtime's driver entry point).
enum TmapType { TMAP_F16 = 0, TMAP_F32 = 1 };
enum TmapSwizzle { TMAP_SWIZZLE_NONE = 0, TMAP_SWIZZLE_32B = 1, TMAP_SWIZZLE_64B = 2, TMAP_SWIZZLE_128B = 3 };
// Row-major [rows, cols] tensor with row pitch ld_elems; box [box_rows, box_cols].
// tmap_out points at 128 bytes, 64-byte aligned (a CUtensorMap).
bool make_tmap_2d(void* tmap_out, const void* base, TmapType type, long long rows, long long cols,
                  long long ld_elems, int box_rows, int box_cols, TmapSwizzle swizzle);
// [batch, rows, cols] tensor: batch pitch in elements; box [1, box_rows, box_cols].
bool make_tmap_3d(void* tmap_out, const void* base, TmapType type, long long batch, long long rows, long long cols,
                  long long ld_elems, long long batch_pitch_elems, int box_rows, int box_cols, TmapSwizzle swizzle);

// gemm_f32.cu — FFMA GEMM and the matmul_init leaf.  With `workspace` of at least
// gemm_f32_workspace_bytes(M, K) bytes (256-byte aligned) a transposed copy of A is written there first and
// the faster form of the kernel runs; the result is bit-identical either way.
size_t gemm_f32_workspace_bytes(long long M, long long K);
int launch_gemm_f32(const float* A, long long lda, const float* B, long long ldb, float* C, long long ldc, int M,
                    int N, int K, float alpha, float beta, void* workspace, size_t workspace_bytes, uint32_t* status,
                    cudaStream_t stream, const char** err);
int launch_scale_f32(float* C, long long ldc, long long rows, long long cols, float beta, bool zero_fill,
                     cudaStream_t stream, const char** err);

// flash.cu — flash attention forward, f16 operands.
// out_f32 != 0: O is f32 (flash_fp32), otherwise f16.
int launch_flash_f16(const void* Q, const void* K, const void* V, void* O, int out_f32, long long batch_heads,
                     int Nq, int Nk, int D, float scale, int sm_count, uint32_t* status, cudaStream_t stream,
                     const char** err);

// selftest.cu — one CTA whose barrier wait must run out after limit_ns (bounded-wait self-test).
int launch_selftest_wait(unsigned long long limit_ns, uint32_t* status, cudaStream_t stream, const char** err);

// elementwise.cu — generator and conversions.
int launch_fill_random(void* out, int dtype_is_f16, unsigned long long n, unsigned long long seed,
                       unsigned long long first, float scale, int normal, cudaStream_t stream, const char** err);
int launch_fill_random_block(void* out, int dtype_is_f16, unsigned long long rows, unsigned long long cols,
                             unsigned long long ld_out, unsigned long long seed, unsigned long long first,
                             unsigned long long stream_pitch, float scale, cudaStream_t stream, const char** err);
int launch_f32_to_f16(const float* in, void* out, unsigned long long n, cudaStream_t stream, const char** err);
int launch_f16_to_f32(const void* in, float* out, unsigned long long n, cudaStream_t stream, const char** err);
// Chunkwise gated linear attention of one head (examples/kda_fp32.ph): Q, K, V, O [N, D], G [N, 1]; D = 64
int launch_kda(const float* Q, long long ldq, const float* K, long long ldk, const float* V, long long ldv, const float* G,
               long long ldg, float* O, long long ldo, int N, int D, float scale, cudaStream_t stream, const char** err);
// out = alpha * x + y, one rounded multiply and one rounded add per element
int launch_saxpy(const float* x, const float* y, float* out, unsigned long long n, float alpha, int sm_count,
                 cudaStream_t stream, const char** err);
// Strided 2-D f32 -> contiguous f16 (rows x cols), used to stage f32-stored tensor-core operands.
int launch_f32_to_f16_2d(const float* in, long long ld_in, void* out, long long rows, long long cols,
                         cudaStream_t stream, const char** err);

// gemv_q4.cu — products with 4-bit weights (block layout at the top of that file).
size_t q4_packed_bytes(long long N, long long K, int group);
int launch_q4_pack(const void* codes, long long ldc, const void* scales, long long lds, const void* zeros, long long ldz,
                   void* out, int N, int K, int group, cudaStream_t stream, const char** err);
int launch_gemv_q4(const void* X, long long ldx, const void* W, void* Y, long long ldy, int out_f32, int M, int N, int K,
                   int group, float alpha, float beta, int sm_count, uint32_t* status, cudaStream_t stream, const char** err);

// gemv_q4_tc.cu — the same for more than eight rows of X, on tcgen05, and whether its times are expected below those of
// gemv_q4.cu's kernel run for eight rows at a time.
bool gemv_q4_tc_is_faster(int M, int N, int K, int group, int sm_count);
int launch_gemv_q4_tc(const void* X, long long ldx, const void* W, void* Y, long long ldy, int out_f32, int M, int N, int K,
                      int group, float alpha, float beta, int sm_count, uint32_t* status, cudaStream_t stream, const char** err);

// The 4-bit key/value cache (layout in kv4.cuh): one layer of it for the kernels that read or write tokens.
struct Kv4View {
  uint8_t* pages;       // this layer's pages
  int* refs;
  int* tables;          // [max_seqs][table_width]
  int* lens;            // [max_seqs]
  long long page_bytes, layer_pitch;
  int layers, n_pages, page_shift, heads, D, G, max_seqs, table_width;
};

// kv4_cache.cu — quantise rows into the pages, read rows back.
int launch_kv4_append(const Kv4View& c, const void* K, long long ldk, const void* V, long long ldv, int T, const int* slots,
                      const int* ind, int n, uint32_t* status, cudaStream_t stream, const char** err);
int launch_kv4_read(const Kv4View& c, void* K, long long ldk, void* V, long long ldv, int T, const int* slots, const int* ind,
                    int n, uint32_t* status, cudaStream_t stream, const char** err);

// kv4_attn.cu — attention over the cache.
struct Kv4AttnArgs {
  const void* Q;
  void* O;
  float* lse;           // may be null
  long long ldq, ldo, ldl;
  int T, n, q_heads, window;
  const int* slots;
  const int* ind;       // may be null: one row per sequence
  float scale;
};
size_t kv4_attention_workspace(const Kv4View& c, int sm_count);  // for any batch
int launch_kv4_attention(const Kv4View& c, const Kv4AttnArgs& a, void* workspace, int sm_count, uint32_t* status,
                         cudaStream_t stream, const char** err);

// kv4_pages.cu — the pages' bookkeeping and moves.
size_t kv4_pages_workspace(const Kv4View& c);
int launch_kv4_extend(const Kv4View& c, const int* slots, const int* counts, int n, int* shortfall, void* workspace,
                      int sm_count, cudaStream_t stream, const char** err);
int launch_kv4_fork(const Kv4View& c, const int* src, const int* dst, int n, int deep, int* shortfall, void* workspace,
                    int sm_count, cudaStream_t stream, const char** err);
int launch_kv4_free(const Kv4View& c, const int* slots, const int* keep, int n, cudaStream_t stream, const char** err);
int launch_kv4_compact(const Kv4View& c, int* live, void* workspace, int sm_count, cudaStream_t stream, const char** err);

}  // namespace ph
