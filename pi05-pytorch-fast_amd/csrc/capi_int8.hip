// extern "C" entry points of the 8-bit operators (declared in include/pi05_w4a4.h): every bound
// that the kernels and their grids rely on is checked here, before anything is launched.

#include <cmath>

#include "../../include/pi05_w4a4.h"
#include "int8_internal.h"

using namespace w4a4;

namespace {

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int check_elem(int32_t elem) {
  if (elem != PI05W4A4_FP16 && elem != PI05W4A4_BF16)
    return capi_fail(PI05W4A4_EINVAL, "elem must be PI05W4A4_FP16 or PI05W4A4_BF16, got %d", elem);
  return PI05W4A4_OK;
}

int check_strides(const void* p, const int64_t* s, const char* name) {
  if (p == nullptr || s == nullptr) return capi_fail(PI05W4A4_EINVAL, "null pointer argument");
  if (!aligned(p, 16)) return capi_fail(PI05W4A4_EINVAL, "%s must be 16-byte aligned", name);
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || s[i] % 8 != 0)
      return capi_fail(PI05W4A4_EINVAL, "%s strides must be multiples of 8 elements, got %lld", name, (long long)s[i]);
  return PI05W4A4_OK;
}

int check_cache(const KvCache8& c, int32_t b, int32_t t) {
  if (c.d != 64 && c.d != 128 && c.d != 256)
    return capi_fail(PI05W4A4_EINVAL, "the int8 KV cache takes head_dim 64, 128 or 256, got %d", c.d);
  if (b < 0 || t < 0 || b > 65535 || c.kvh <= 0 || c.kvh > 32767)
    return capi_fail(PI05W4A4_EINVAL, "batch %d (at most 65535), tokens %d or KV heads %d out of range", b, t, c.kvh);
  if (c.pages < 0 || c.table_pages < 0 || c.table_stride < 0 || c.table_pages > (1 << 24))
    return capi_fail(PI05W4A4_EINVAL, "pages and table sizes must be >= 0, table rows at most 2^24 pages");
  if (t > (1 << 24)) return capi_fail(PI05W4A4_EINVAL, "at most 2^24 tokens a call, got %d", t);
  return PI05W4A4_OK;
}

int check_cache_pointers(const KvCache8& c) {
  if (c.lens == nullptr || (c.table_pages > 0 && c.table == nullptr)) return capi_fail(PI05W4A4_EINVAL, "null pointer argument");
  if (c.pages > 0 && (c.k == nullptr || c.v == nullptr || c.ks == nullptr || c.vs == nullptr))
    return capi_fail(PI05W4A4_EINVAL, "null pointer argument");
  if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.ks, 4) || !aligned(c.vs, 4) || !aligned(c.table, 4) || !aligned(c.lens, 4))
    return capi_fail(PI05W4A4_EINVAL, "the KV cache must be 16-byte aligned");
  return PI05W4A4_OK;
}

}  // namespace

extern "C" int pi05w4a4_int8_rows(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* norm_w,
                                  float eps, int32_t unit_offset, int32_t elem, int64_t m, int32_t k, void* q,
                                  float* scale, void* h_out, void* stream) {
  if (int rc = check_elem(elem)) return rc;
  if (m < 0 || m > 0x7fffffffLL) return capi_fail(PI05W4A4_EINVAL, "M must be in [0, 2^31), got %lld", (long long)m);
  if (k <= 0 || k % 8 != 0 || k > 32768)
    return capi_fail(PI05W4A4_EINVAL, "K must be a multiple of 8 of at most 32768, got %d", k);
  // A launch holds fewer than 2^32 threads: 64, 256 or 1024 of them a row.
  if (m * (k <= 2048 ? 64 : k <= 8192 ? 256 : 1024) >= 1LL << 32)
    return capi_fail(PI05W4A4_EINVAL, "M=%lld rows of K=%d are more than one launch holds", (long long)m, k);
  if (residual != nullptr && (norm_w == nullptr || h_out == nullptr))
    return capi_fail(PI05W4A4_EINVAL, "a residual needs a norm weight and an output for the sum");
  if (m == 0) return capi_ok();
  if (x == nullptr || q == nullptr || scale == nullptr) return capi_fail(PI05W4A4_EINVAL, "null pointer argument");
  if (!aligned(x, 16) || !aligned(residual, 16) || !aligned(norm_w, 16) || !aligned(q, 8) || !aligned(scale, 4) || !aligned(h_out, 16))
    return capi_fail(PI05W4A4_EINVAL, "x, residual, norm weight and outputs must be 16-byte aligned");
  if (ldx < 0 || ldx % 8 != 0 || ldr < 0 || ldr % 8 != 0)
    return capi_fail(PI05W4A4_EINVAL, "row strides must be multiples of 8 elements, got %lld and %lld", (long long)ldx, (long long)ldr);
  const Int8RowsParams p{x, residual, norm_w, ldx, ldr, m, k, eps, unit_offset != 0, static_cast<int8_t*>(q), scale, h_out};
  return capi_hip(launch_int8_rows(p, elem, static_cast<hipStream_t>(stream)), "int8_rows launch");
}

extern "C" size_t pi05w4a4_int8_gemm_workspace_bytes(int64_t m, int32_t n, int32_t k) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const Int8GemmPlan plan = int8_gemm_plan(m, n, k, device_cu_count());
  return plan.ksplit > 1 ? static_cast<size_t>(plan.ksplit) * m * n * sizeof(int32_t) : 0;
}

extern "C" int pi05w4a4_int8_gemm(const void* q, int64_t ldq, const float* sq, int64_t m, int32_t k, const void* w,
                                  int64_t ldw, const float* sw, int32_t n, const void* bias, const void* residual,
                                  int64_t ldr, int32_t elem, void* y, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (int rc = check_elem(elem)) return rc;
  if (m < 0 || m > 0x7fffffffLL) return capi_fail(PI05W4A4_EINVAL, "M must be in [0, 2^31), got %lld", (long long)m);
  if (n < 0 || n > (1 << 28)) return capi_fail(PI05W4A4_EINVAL, "N must be in [0, 2^28], got %d", n);
  // int32 sums: 2^14 (codes down to -128) * 65536 = 2^30.
  if (k <= 0 || k % 16 != 0 || k > 65536)
    return capi_fail(PI05W4A4_EINVAL, "K must be a multiple of 16 of at most 65536, got %d", k);
  if (m == 0 || n == 0) return capi_ok();
  if (q == nullptr || sq == nullptr || w == nullptr || sw == nullptr || y == nullptr)
    return capi_fail(PI05W4A4_EINVAL, "null pointer argument");
  if (!aligned(q, 16) || !aligned(w, 16) || !aligned(y, 16) || !aligned(sq, 4) || !aligned(sw, 4) || !aligned(bias, 2) ||
      !aligned(residual, 2))
    return capi_fail(PI05W4A4_EINVAL, "q, w and y must be 16-byte aligned");
  // Strides: 32-bit offsets within a tile of 256 rows.
  if (ldq < 0 || ldq % 16 != 0 || ldq > (1 << 23) || ldw < 0 || ldw % 16 != 0 || ldw > (1 << 23))
    return capi_fail(PI05W4A4_EINVAL, "row strides of q and w must be multiples of 16 bytes of at most 2^23, got %lld and %lld",
                     (long long)ldq, (long long)ldw);
  if (residual != nullptr && ldr < 0) return capi_fail(PI05W4A4_EINVAL, "the residual's row stride must be >= 0");
  if (((m + 63) / 64) * ((n + 31LL) / 32) > 0x7fffffffLL / 16)
    return capi_fail(PI05W4A4_EINVAL, "M=%lld N=%d is more tiles than one launch holds", (long long)m, n);
  const Int8GemmPlan plan = int8_gemm_plan(m, n, k, device_cu_count());
  const size_t need = plan.ksplit > 1 ? static_cast<size_t>(plan.ksplit) * m * n * sizeof(int32_t) : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return capi_fail(PI05W4A4_EWORKSPACE, "int8_gemm needs a 16-byte aligned workspace of %zu bytes, got %zu", need, workspace_bytes);
  Int8GemmParams p{};
  p.q = static_cast<const int8_t*>(q);
  p.w = static_cast<const int8_t*>(w);
  p.sq = sq;
  p.sw = sw;
  p.bias = bias;
  p.res = residual;
  p.y = y;
  p.m = m;
  p.ldq = ldq;
  p.ldw = ldw;
  p.ldr = ldr;
  p.n = n;
  p.k = k;
  p.partial = static_cast<int32_t*>(workspace);
  return capi_hip(launch_int8_gemm(p, plan, elem, static_cast<hipStream_t>(stream)), "int8_gemm launch");
}

extern "C" int pi05w4a4_int8_kv_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                       int32_t elem, int32_t b, int32_t t, int32_t kvh, int32_t d, void* k_cache,
                                       void* v_cache, float* k_scale, float* v_scale, int32_t pages,
                                       const int32_t* table, int64_t table_stride, int32_t table_pages,
                                       const int32_t* lens, const int32_t* counts, void* stream) {
  if (int rc = check_elem(elem)) return rc;
  KvAppendParams p{};
  p.c = {static_cast<int8_t*>(k_cache), static_cast<int8_t*>(v_cache), k_scale, v_scale, table, lens, table_stride, pages, table_pages, kvh, d};
  if (int rc = check_cache(p.c, b, t)) return rc;
  if (b == 0 || t == 0) return capi_ok();
  if (int rc = check_cache_pointers(p.c)) return rc;
  if (int rc = check_strides(k, k_strides, "k")) return rc;
  if (int rc = check_strides(v, v_strides, "v")) return rc;
  if (!aligned(counts, 4)) return capi_fail(PI05W4A4_EINVAL, "counts must be 4-byte aligned");
  p.k = k;
  p.v = v;
  for (int i = 0; i < 3; ++i) {
    p.k_stride[i] = k_strides[i];
    p.v_stride[i] = v_strides[i];
  }
  p.counts = counts;
  p.b = b;
  p.t = t;
  return capi_hip(launch_kv_append(p, elem, static_cast<hipStream_t>(stream)), "int8_kv_append launch");
}

extern "C" size_t pi05w4a4_int8_kv_attention_workspace_bytes(int32_t b, int32_t t, int32_t h, int32_t kvh, int32_t d,
                                                             int32_t table_pages) {
  if (b <= 0 || t <= 0 || kvh <= 0 || h < kvh || table_pages <= 0) return 0;
  return kv_attn_workspace(b, t, h, d, kv_attn_plan(b, t, h, kvh, d, table_pages, device_cu_count()).nsplit);
}

extern "C" int pi05w4a4_int8_kv_attention(const void* q, const int64_t* q_strides, int32_t elem, int32_t b, int32_t t,
                                          int32_t h, int32_t kvh, int32_t d, const void* k_cache, const void* v_cache,
                                          const float* k_scale, const float* v_scale, int32_t pages,
                                          const int32_t* table, int64_t table_stride, int32_t table_pages,
                                          const int32_t* lens, const int32_t* q_lens, float scaling, int32_t causal,
                                          void* out, float* lse, void* workspace, size_t workspace_bytes,
                                          void* stream) {
  if (int rc = check_elem(elem)) return rc;
  KvAttnParams p{};
  p.c = {const_cast<int8_t*>(static_cast<const int8_t*>(k_cache)), const_cast<int8_t*>(static_cast<const int8_t*>(v_cache)),
         const_cast<float*>(k_scale), const_cast<float*>(v_scale), table, lens, table_stride, pages, table_pages, kvh, d};
  if (int rc = check_cache(p.c, b, t)) return rc;
  if (h <= 0 || h % kvh != 0 || h > 65535)
    return capi_fail(PI05W4A4_EINVAL, "query heads must be a multiple of the KV heads, got %d and %d", h, kvh);
  if (static_cast<int64_t>(t) * (h / kvh) > (1 << 26))
    return capi_fail(PI05W4A4_EINVAL, "T * H / KVH must be at most 2^26, got T=%d H=%d KVH=%d", t, h, kvh);
  if (!std::isfinite(scaling)) return capi_fail(PI05W4A4_EINVAL, "scaling must be finite");
  if (b == 0 || t == 0) return capi_ok();
  if (int rc = check_cache_pointers(p.c)) return rc;
  if (int rc = check_strides(q, q_strides, "q")) return rc;
  if (out == nullptr || !aligned(out, 16) || !aligned(lse, 4) || !aligned(q_lens, 4))
    return capi_fail(PI05W4A4_EINVAL, "out must be 16-byte aligned");
  const KvAttnPlan plan = kv_attn_plan(b, t, h, kvh, d, table_pages, device_cu_count());
  p.nsplit = plan.nsplit;
  p.wide = plan.wide;
  const size_t need = kv_attn_workspace(b, t, h, d, p.nsplit);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return capi_fail(PI05W4A4_EWORKSPACE, "int8_kv_attention needs a 16-byte aligned workspace of %zu bytes, got %zu", need, workspace_bytes);
  p.q = q;
  for (int i = 0; i < 3; ++i) p.q_stride[i] = q_strides[i];
  p.q_lens = q_lens;
  p.out = out;
  p.lse = lse;
  p.ws = static_cast<float*>(workspace);
  p.scaling = scaling;
  p.causal = causal != 0;
  p.b = b;
  p.t = t;
  p.h = h;
  return capi_hip(launch_kv_attention(p, elem, static_cast<hipStream_t>(stream)), "int8_kv_attention launch");
}
