// extern "C" entry points of serving from 4-bit weights and a 4-bit cache: argument checks and launches.  See
// include/phobos_leaf.h for the contract of every function.
#include <cuda_runtime.h>

#include "../../include/phobos_leaf.h"
#include "host.h"
#include "kernels.h"
#include "kv4.cuh"

using namespace ph;

namespace {

// A rank-2 view with inner stride 1 whose rows start on `align` bytes; extents of zero rows are allowed.
struct Rows {
  char* base;
  long long rows, cols, ld;
  int dtype;
};

int rows_of(const PhTensor* t, const char* name, int align, Rows* v) {
  if (!t) return fail(PH_ERR_INVALID, "%s: null tensor descriptor", name);
  if (t->rank != 2) return fail(PH_ERR_INVALID, "%s: rank %d, expected 2", name, t->rank);
  const long long es = static_cast<long long>(phobos_dtype_bytes(t->dtype));
  if (es == 0) return fail(PH_ERR_UNSUPPORTED, "%s: unknown element type %d", name, t->dtype);
  if (t->sizes[0] < 0 || t->sizes[1] <= 0 || t->sizes[0] > 0x7fffffffLL || t->sizes[1] > 0x7fffffffLL)
    return fail(PH_ERR_INVALID, "%s: extent %lldx%lld", name, (long long)t->sizes[0], (long long)t->sizes[1]);
  if (t->sizes[1] > 1 && t->strides[1] != 1)
    return fail(PH_ERR_INVALID, "%s: inner stride %lld, expected 1", name, (long long)t->strides[1]);
  const bool one_row = t->sizes[0] <= 1;  // whose row stride means nothing
  if (!one_row && (t->strides[0] < t->sizes[1] || t->strides[0] > (1LL << 40)))
    return fail(PH_ERR_INVALID, "%s: row stride %lld for rows of %lld", name, (long long)t->strides[0], (long long)t->sizes[1]);
  if (t->offset < 0) return fail(PH_ERR_INVALID, "%s: negative offset", name);
  if (t->sizes[0] > 0 && !t->ptr) return fail(PH_ERR_INVALID, "%s: null data pointer", name);
  char* base = static_cast<char*>(t->ptr) + t->offset * es;
  if (reinterpret_cast<uintptr_t>(base) % align != 0 || (!one_row && (t->strides[0] * es) % align != 0))
    return fail(PH_ERR_INVALID, "%s: rows do not start on %d bytes", name, align);
  *v = Rows{base, t->sizes[0], t->sizes[1], one_row ? t->sizes[1] : t->strides[0], t->dtype};
  return PH_OK;
}

bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }

int packed_of(const PhTensor* t, size_t need, char** base) {
  if (!t || !t->ptr) return fail(PH_ERR_INVALID, "packed weights: null tensor");
  if (t->rank != 1 || (t->dtype != PH_I8 && t->dtype != PH_BOOL) || t->strides[0] != 1 || t->offset < 0)
    return fail(PH_ERR_INVALID, "packed weights: expected a contiguous rank-1 i8 tensor");
  if (t->sizes[0] < 0 || static_cast<size_t>(t->sizes[0]) < need)
    return fail(PH_ERR_INVALID, "packed weights: %lld bytes, these sizes need %zu", (long long)t->sizes[0], need);
  *base = static_cast<char*>(t->ptr) + t->offset;
  if (reinterpret_cast<uintptr_t>(*base) % 16 != 0) return fail(PH_ERR_INVALID, "packed weights: not 16-byte aligned");
  return PH_OK;
}

int view_of_cache(const PhKv4Cache* c, Kv4View* v) {
  if (!c) return fail(PH_ERR_INVALID, "kv4: null cache");
  const size_t page = phobos_kv4_page_bytes(c->kv_heads, c->head_dim, c->group, c->page_tokens);
  if (page == 0)
    return fail(PH_ERR_UNSUPPORTED, "kv4: %d heads of %d dims in groups of %d, pages of %d tokens", c->kv_heads, c->head_dim,
                c->group, c->page_tokens);
  if (!c->pages || !c->refs || !c->tables || !c->lens) return fail(PH_ERR_INVALID, "kv4: null array");
  if (c->layers < 1 || c->n_pages < 1 || c->max_seqs < 1 || c->table_width < 1)
    return fail(PH_ERR_INVALID, "kv4: %d layers, %d pages, %d sequences, tables of %d pages", c->layers, c->n_pages, c->max_seqs,
                c->table_width);
  if (c->table_width > (1 << 20) || static_cast<long long>(c->table_width) * c->page_tokens > 0x7fffffffLL)
    return fail(PH_ERR_UNSUPPORTED, "kv4: tables of %d pages of %d tokens", c->table_width, c->page_tokens);
  if (reinterpret_cast<uintptr_t>(c->pages) % 16 != 0) return fail(PH_ERR_INVALID, "kv4: pages are not 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(c->refs) % 4 != 0 || reinterpret_cast<uintptr_t>(c->tables) % 4 != 0 ||
      reinterpret_cast<uintptr_t>(c->lens) % 4 != 0)
    return fail(PH_ERR_INVALID, "kv4: refs, tables and lens hold 32-bit values");
  if (c->layers > 1 && (c->layer_pitch % 16 != 0 || c->layer_pitch < 0 ||
                        static_cast<unsigned long long>(c->layer_pitch) / page < static_cast<unsigned long long>(c->n_pages)))
    return fail(PH_ERR_INVALID, "kv4: layers %lld bytes apart for %d pages of %zu bytes", (long long)c->layer_pitch, c->n_pages, page);
  int shift = 4;
  while ((1 << shift) < c->page_tokens) shift++;
  *v = Kv4View{static_cast<uint8_t*>(c->pages), c->refs, c->tables, c->lens, static_cast<long long>(page), c->layer_pitch,
               c->layers, c->n_pages, shift, c->kv_heads, c->head_dim, c->group, c->max_seqs, c->table_width};
  return PH_OK;
}

int layer_of(const PhKv4Cache* c, int layer, Kv4View* v) {
  const int rc = view_of_cache(c, v);
  if (rc) return rc;
  if (layer < 0 || layer >= c->layers) return fail(PH_ERR_INVALID, "kv4: layer %d of %d", layer, c->layers);
  v->pages += layer * c->layer_pitch;
  return PH_OK;
}

int batch_of(const char* what, const int32_t* slots, const int32_t* indptr, int32_t n, long long T) {
  if (n < 0) return fail(PH_ERR_INVALID, "%s: %d sequences", what, n);
  if (n > 0 && !slots) return fail(PH_ERR_INVALID, "%s: null slots", what);
  if (reinterpret_cast<uintptr_t>(slots) % 4 != 0 || reinterpret_cast<uintptr_t>(indptr) % 4 != 0)
    return fail(PH_ERR_INVALID, "%s: slots and indptr hold 32-bit values", what);
  if (!indptr && T < n) return fail(PH_ERR_INVALID, "%s: %lld rows for %d sequences of one row each", what, T, n);
  return PH_OK;
}

int workspace_of(const char* what, void* ws, size_t got, size_t need) {
  if (need == 0) return PH_OK;
  if (!ws || got < need) return fail(PH_ERR_WORKSPACE, "%s needs %zu workspace bytes, got %zu", what, need, ws ? got : 0);
  if (reinterpret_cast<uintptr_t>(ws) % 256 != 0) return fail(PH_ERR_WORKSPACE, "workspace is not 256-byte aligned");
  return PH_OK;
}

int kv_rows(const PhKv4Cache* cache, int32_t layer, const PhTensor* K, const PhTensor* V, const int32_t* slots,
            const int32_t* indptr, int32_t n, bool read, void* stream) {
  clear_error();
  const char* what = read ? "kv4_read" : "kv4_append";
  Kv4View c;
  Rows k, v;
  int rc;
  if ((rc = layer_of(cache, layer, &c)) || (rc = rows_of(K, "K", 16, &k)) || (rc = rows_of(V, "V", 16, &v))) return rc;
  if (k.dtype != PH_F16 || v.dtype != PH_F16) return fail(PH_ERR_UNSUPPORTED, "%s takes f16 rows", what);
  const long long width = static_cast<long long>(c.heads) * c.D;
  if (k.cols != width || v.cols != width || k.rows != v.rows)
    return fail(PH_ERR_INVALID, "%s: K %lldx%lld, V %lldx%lld, expected rows of %lld", what, k.rows, k.cols, v.rows, v.cols, width);
  if ((rc = batch_of(what, slots, indptr, n, k.rows))) return rc;
  const long long T = indptr ? k.rows : n;
  int sms;
  uint32_t* status;
  if ((rc = device_props(&sms, &status))) return rc;
  if (T == 0 || n == 0) return PH_OK;
  const char* err = "";
  const auto s = static_cast<cudaStream_t>(stream);
  rc = read ? launch_kv4_read(c, k.base, k.ld, v.base, v.ld, static_cast<int>(T), slots, indptr, n, status, s, &err)
            : launch_kv4_append(c, k.base, k.ld, v.base, v.ld, static_cast<int>(T), slots, indptr, n, status, s, &err);
  return map_launch_rc(rc, what, err);
}

}  // namespace

extern "C" {

size_t phobos_q4_packed_bytes(int64_t N, int64_t K, int32_t group) {
  if (N <= 0 || K <= 0 || N > 0x7fffffffLL || K > 0x7fffffffLL || !group_ok(group) || K % group != 0) return 0;
  return q4_packed_bytes(N, K, group);
}

int phobos_q4_pack(const PhTensor* codes, const PhTensor* scales, const PhTensor* zeros, int32_t group, const PhTensor* packed,
                   void* stream) {
  clear_error();
  Rows c, s, z{nullptr, 0, 0, 0, PH_F16};
  int rc;
  if ((rc = rows_of(codes, "codes", 1, &c)) || (rc = rows_of(scales, "scales", 2, &s)) ||
      (zeros && (rc = rows_of(zeros, "zeros", 2, &z))))
    return rc;
  const size_t need = phobos_q4_packed_bytes(c.rows, c.cols, group);
  if (need == 0)
    return fail(PH_ERR_UNSUPPORTED, "q4_pack: %lldx%lld codes in groups of %d", c.rows, c.cols, group);
  if (phobos_dtype_bytes(c.dtype) != 1) return fail(PH_ERR_INVALID, "q4_pack: codes stand one to a byte");
  if (s.dtype != PH_F16 || z.dtype != PH_F16) return fail(PH_ERR_UNSUPPORTED, "q4_pack: scales and zeros are f16");
  if (s.rows != c.rows || s.cols != c.cols / group || (zeros && (z.rows != s.rows || z.cols != s.cols)))
    return fail(PH_ERR_INVALID, "q4_pack: scales and zeros of %lldx%lld codes are %lldx%lld", c.rows, c.cols, c.rows, c.cols / group);
  char* out;
  if ((rc = packed_of(packed, need, &out))) return rc;
  int sms;
  uint32_t* status;
  if ((rc = device_props(&sms, &status))) return rc;
  const char* err = "";
  rc = launch_q4_pack(c.base, c.ld, s.base, s.ld, z.base, z.ld, out, static_cast<int>(c.rows), static_cast<int>(c.cols), group,
                      static_cast<cudaStream_t>(stream), &err);
  return map_launch_rc(rc, "q4_pack", err);
}

int phobos_gemv_q4(const PhTensor* X, const PhTensor* packed, const PhTensor* Y, float alpha, float beta, int32_t group,
                   void* stream) {
  clear_error();
  Rows x, y;
  int rc;
  if ((rc = rows_of(X, "X", 16, &x)) || (rc = rows_of(Y, "Y", 1, &y))) return rc;
  if (x.dtype != PH_F16) return fail(PH_ERR_UNSUPPORTED, "gemv_q4 takes an f16 X");
  if (y.dtype != PH_F16 && y.dtype != PH_F32) return fail(PH_ERR_UNSUPPORTED, "gemv_q4 writes an f16 or f32 Y");
  if (reinterpret_cast<uintptr_t>(y.base) % phobos_dtype_bytes(y.dtype) != 0) return fail(PH_ERR_INVALID, "Y: not aligned to its elements");
  if (x.rows != y.rows) return fail(PH_ERR_INVALID, "gemv_q4: X has %lld rows, Y has %lld", x.rows, y.rows);
  const size_t need = phobos_q4_packed_bytes(y.cols, x.cols, group);
  if (need == 0) return fail(PH_ERR_UNSUPPORTED, "gemv_q4: weights of %lldx%lld in groups of %d", y.cols, x.cols, group);
  char* w;
  if ((rc = packed_of(packed, need, &w))) return rc;
  int sms;
  uint32_t* status;
  if ((rc = device_props(&sms, &status))) return rc;
  if (x.rows == 0) return PH_OK;
  const char* err = "";
  rc = launch_gemv_q4(x.base, x.ld, w, y.base, y.ld, y.dtype == PH_F32, static_cast<int>(x.rows), static_cast<int>(y.cols),
                      static_cast<int>(x.cols), group, alpha, beta, sms, status, static_cast<cudaStream_t>(stream), &err);
  return map_launch_rc(rc, "gemv_q4", err);
}

size_t phobos_kv4_page_bytes(int32_t kv_heads, int32_t head_dim, int32_t group, int32_t page_tokens) {
  if (kv_heads < 1 || kv_heads > 65535 || (head_dim != 64 && head_dim != 128) || !group_ok(group) || group > head_dim) return 0;
  if (page_tokens < 16 || page_tokens > 256 || (page_tokens & (page_tokens - 1)) != 0) return 0;
  return static_cast<size_t>(kv_heads) * (page_tokens / KV4_UNIT) * kv4_unit_bytes(head_dim, group);
}

int phobos_kv4_append(const PhKv4Cache* cache, int32_t layer, const PhTensor* K, const PhTensor* V, const int32_t* slots,
                      const int32_t* indptr, int32_t n, void* stream) {
  return kv_rows(cache, layer, K, V, slots, indptr, n, false, stream);
}

int phobos_kv4_read(const PhKv4Cache* cache, int32_t layer, const PhTensor* K, const PhTensor* V, const int32_t* slots,
                    const int32_t* indptr, int32_t n, void* stream) {
  return kv_rows(cache, layer, K, V, slots, indptr, n, true, stream);
}

size_t phobos_kv4_attention_workspace_bytes(const PhKv4Cache* cache, int64_t T, int32_t n, int32_t q_heads) {
  Kv4View c;
  if (view_of_cache(cache, &c) || T < 0 || T > 0x7fffffffLL || n < 0 || q_heads < 1 || q_heads % c.heads != 0) return 0;
  return kv4_attention_workspace(c, sm_count_or_default());
}

int phobos_kv4_attention(const PhKv4Cache* cache, int32_t layer, const PhTensor* Q, const PhTensor* O, const PhTensor* lse,
                         float scale, int32_t window, const int32_t* slots, const int32_t* indptr, int32_t n, void* workspace,
                         size_t workspace_bytes, void* stream) {
  clear_error();
  Kv4View c;
  Rows q, o, l{nullptr, 0, 0, 0, PH_F32};
  int rc;
  if ((rc = layer_of(cache, layer, &c)) || (rc = rows_of(Q, "Q", 16, &q)) || (rc = rows_of(O, "O", 16, &o)) ||
      (lse && (rc = rows_of(lse, "lse", 4, &l))))
    return rc;
  if (q.dtype != PH_F16 || o.dtype != PH_F16 || l.dtype != PH_F32)
    return fail(PH_ERR_UNSUPPORTED, "kv4_attention takes f16 Q and O and an f32 lse");
  if (q.rows != o.rows || q.cols != o.cols || q.cols % (static_cast<long long>(c.heads) * c.D) != 0)
    return fail(PH_ERR_INVALID, "kv4_attention: Q %lldx%lld, O %lldx%lld for %d key/value heads of %d", q.rows, q.cols, o.rows,
                o.cols, c.heads, c.D);
  const long long q_heads = q.cols / c.D;
  if (lse && (l.rows != q.rows || l.cols != q_heads))
    return fail(PH_ERR_INVALID, "kv4_attention: lse %lldx%lld, expected %lldx%lld", l.rows, l.cols, q.rows, q_heads);
  if (window < 0) return fail(PH_ERR_INVALID, "kv4_attention: window %d", window);
  // No sequence is longer than its table, so a window of that size hides nothing.  (The kernel takes windows from positions,
  // which are negative for rows in front of a sequence's first token: below 2^28 the difference stays within 32 bits.)
  if (window >= static_cast<long long>(c.table_width) << c.page_shift) window = 0;
  if ((rc = batch_of("kv4_attention", slots, indptr, n, q.rows))) return rc;
  const long long T = indptr ? q.rows : n;
  const size_t need = kv4_attention_workspace(c, sm_count_or_default());
  if ((rc = workspace_of("kv4_attention", workspace, workspace_bytes, need))) return rc;
  int sms;
  uint32_t* status;
  if ((rc = device_props(&sms, &status))) return rc;
  if (T == 0 || n == 0) return PH_OK;
  const Kv4AttnArgs a{q.base, o.base, reinterpret_cast<float*>(l.base), q.ld, o.ld, l.ld, static_cast<int>(T), n,
                      static_cast<int>(q_heads), window, slots, indptr, scale};
  const char* err = "";
  rc = launch_kv4_attention(c, a, workspace, sms, status, static_cast<cudaStream_t>(stream), &err);
  return map_launch_rc(rc, "kv4_attention", err);
}

size_t phobos_kv4_pages_workspace_bytes(const PhKv4Cache* cache) {
  Kv4View c;
  return view_of_cache(cache, &c) ? 0 : kv4_pages_workspace(c);
}

int phobos_kv4_extend(const PhKv4Cache* cache, const int32_t* slots, const int32_t* counts, int32_t n, int32_t* shortfall,
                      void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  Kv4View c;
  int rc, sms;
  uint32_t* status;
  if ((rc = view_of_cache(cache, &c))) return rc;
  if (n < 0 || n > c.max_seqs) return fail(PH_ERR_INVALID, "kv4_extend: %d rows for %d sequences", n, c.max_seqs);
  if (!shortfall || (n > 0 && (!slots || !counts))) return fail(PH_ERR_INVALID, "kv4_extend: null array");
  if ((rc = workspace_of("kv4_extend", workspace, workspace_bytes, kv4_pages_workspace(c)))) return rc;
  if ((rc = device_props(&sms, &status))) return rc;
  const char* err = "";
  rc = launch_kv4_extend(c, slots, counts, n, shortfall, workspace, sms, static_cast<cudaStream_t>(stream), &err);
  return map_launch_rc(rc, "kv4_extend", err);
}

int phobos_kv4_fork(const PhKv4Cache* cache, const int32_t* src, const int32_t* dst, int32_t n, int32_t deep,
                    int32_t* shortfall, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  Kv4View c;
  int rc, sms;
  uint32_t* status;
  if ((rc = view_of_cache(cache, &c))) return rc;
  if (n < 0 || n > c.max_seqs) return fail(PH_ERR_INVALID, "kv4_fork: %d rows for %d sequences", n, c.max_seqs);
  if (!shortfall || (n > 0 && (!src || !dst))) return fail(PH_ERR_INVALID, "kv4_fork: null array");
  if ((rc = workspace_of("kv4_fork", workspace, workspace_bytes, kv4_pages_workspace(c)))) return rc;
  if ((rc = device_props(&sms, &status))) return rc;
  const char* err = "";
  rc = launch_kv4_fork(c, src, dst, n, deep, shortfall, workspace, sms, static_cast<cudaStream_t>(stream), &err);
  return map_launch_rc(rc, "kv4_fork", err);
}

int phobos_kv4_free(const PhKv4Cache* cache, const int32_t* slots, const int32_t* keep, int32_t n, void* stream) {
  clear_error();
  Kv4View c;
  int rc, sms;
  uint32_t* status;
  if ((rc = view_of_cache(cache, &c))) return rc;
  if (n < 0 || (n > 0 && !slots)) return fail(PH_ERR_INVALID, "kv4_free: %d rows, slots %p", n, static_cast<const void*>(slots));
  if ((rc = device_props(&sms, &status))) return rc;
  if (n == 0) return PH_OK;
  const char* err = "";
  rc = launch_kv4_free(c, slots, keep, n, static_cast<cudaStream_t>(stream), &err);
  return map_launch_rc(rc, "kv4_free", err);
}

int phobos_kv4_compact(const PhKv4Cache* cache, int32_t* live, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  Kv4View c;
  int rc, sms;
  uint32_t* status;
  if ((rc = view_of_cache(cache, &c))) return rc;
  if (!live) return fail(PH_ERR_INVALID, "kv4_compact: null output");
  if ((rc = workspace_of("kv4_compact", workspace, workspace_bytes, kv4_pages_workspace(c)))) return rc;
  if ((rc = device_props(&sms, &status))) return rc;
  const char* err = "";
  rc = launch_kv4_compact(c, live, workspace, sms, static_cast<cudaStream_t>(stream), &err);
  return map_launch_rc(rc, "kv4_compact", err);
}

}  // extern "C"
