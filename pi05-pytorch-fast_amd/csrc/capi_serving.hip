// extern "C" entry points of the 16-bit serving operators (declared in include/pi05_w4a4.h): every
// bound that the kernels and their grids rely on is checked here, before anything is launched.

#include <cmath>

#include "../../include/pi05_w4a4.h"
#include "serving_internal.h"

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

int check_cache(const KvCache16& c, int32_t b, int32_t t) {
  if (c.d != 64 && c.d != 128 && c.d != 256)
    return capi_fail(PI05W4A4_EINVAL, "the KV cache takes head_dim 64, 128 or 256, got %d", c.d);
  if (b < 0 || t < 0 || b > 65535 || c.kvh <= 0 || c.kvh > 32767)
    return capi_fail(PI05W4A4_EINVAL, "batch %d (at most 65535), tokens %d or KV heads %d out of range", b, t, c.kvh);
  if (c.pages < 0 || c.table_pages < 0 || c.table_stride < 0 || c.table_pages > (1 << 24))
    return capi_fail(PI05W4A4_EINVAL, "pages and table sizes must be >= 0, table rows at most 2^24 pages");
  if (t > (1 << 24)) return capi_fail(PI05W4A4_EINVAL, "at most 2^24 tokens a call, got %d", t);
  return PI05W4A4_OK;
}

int check_cache_pointers(const KvCache16& c) {
  if (c.lens == nullptr || (c.table_pages > 0 && c.table == nullptr)) return capi_fail(PI05W4A4_EINVAL, "null pointer argument");
  if (c.pages > 0 && (c.k == nullptr || c.v == nullptr)) return capi_fail(PI05W4A4_EINVAL, "null pointer argument");
  if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.table, 4) || !aligned(c.lens, 4))
    return capi_fail(PI05W4A4_EINVAL, "the KV cache must be 16-byte aligned");
  return PI05W4A4_OK;
}

// The parts of a call that concern the heads: sizes, strides, norm and rotation.
int check_heads(const HeadRopeParams& p) {
  for (int i = 0; i < 3; ++i)
    if (p.heads[i] < 0 || p.heads[i] > 32767) return capi_fail(PI05W4A4_EINVAL, "heads must be in [0, 32767], got %d", p.heads[i]);
  if (p.b < 0 || p.t < 0 || static_cast<int64_t>(p.b) * p.t > (1 << 24))
    return capi_fail(PI05W4A4_EINVAL, "at most 2^24 tokens a call, got %d x %d", p.b, p.t);
  return PI05W4A4_OK;
}

void set_strides(int64_t* to, const int64_t* from) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

}  // namespace

// Whether `bytes` bytes from a and `more` from b share some.
static bool ranges_overlap(const void* a, int64_t bytes, const void* b, int64_t more) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return bytes > 0 && more > 0 && x < y + more && y < x + bytes;
}

// A call that reads rows of the cache while it writes others would depend on the order of its waves.
static int check_apart(const HeadRopeParams& p) {
  const int64_t cache = static_cast<int64_t>(p.c.pages) * p.c.kvh * kKvPage * p.d * 2;
  if (ranges_overlap(p.c.k, cache, p.c.v, cache)) return capi_fail(PI05W4A4_EINVAL, "k_cache and v_cache must not overlap");
  for (int i = 0; i < 3; ++i) {
    if (p.x[i] == nullptr) continue;
    const int64_t* const st = p.stride[i];
    const int64_t bytes = 2 * ((p.b - 1) * st[0] + (p.t - 1) * st[1] + (p.heads[i] - 1) * st[2] + p.d);
    if (ranges_overlap(p.x[i], bytes, p.c.k, cache) || ranges_overlap(p.x[i], bytes, p.c.v, cache))
      return capi_fail(PI05W4A4_EINVAL, "the new tokens must not lie in the cache");
  }
  return PI05W4A4_OK;
}

static int run_head_rope(HeadRopeParams& p, int32_t elem, void* stream, const char* what) {
  p.parts = head_rope_parts(p, device_cu_count());
  // A launch holds fewer than 2^32 threads: a wave for each part of a token, four a workgroup.
  if (static_cast<int64_t>(p.b) * p.t * p.parts > (1 << 26) - 4)
    return capi_fail(PI05W4A4_EINVAL, "%d x %d tokens of %d heads are more than one launch holds", p.b, p.t,
                     p.heads[0] + p.heads[1] + p.heads[2]);
  if (p.c.lens != nullptr)
    if (int rc = check_apart(p)) return rc;
  return capi_hip(launch_head_rope(p, elem, static_cast<hipStream_t>(stream)), what);
}

// Everything of pi05w4a4_qk_norm_rope and its append form but the destination of the keys.
static int rope_params(HeadRopeParams& p, const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                       int32_t elem, int32_t b, int32_t t, int32_t h, int32_t kvh, int32_t d, const void* q_weight,
                       const void* k_weight, float eps, int32_t unit_offset, const void* positions,
                       const int64_t* pos_strides, int32_t pos_bytes, int32_t axes, const uint8_t* axis_of_pair,
                       const float* inv_freq, int32_t rot, int32_t interleaved, void* q_out) {
  if (int rc = check_elem(elem)) return rc;
  if (d <= 0 || d % 16 != 0 || d > kMaxHeadDim)
    return capi_fail(PI05W4A4_EINVAL, "head_dim must be a multiple of 16 of at most %d, got %d", kMaxHeadDim, d);
  if (h <= 0 || kvh <= 0) return capi_fail(PI05W4A4_EINVAL, "query and KV heads must be positive, got %d and %d", h, kvh);
  if (rot < 0 || rot % 16 != 0 || rot > d)
    return capi_fail(PI05W4A4_EINVAL, "the rotated dimensions must be a multiple of 16 of at most head_dim, got %d", rot);
  if (axes < 1 || axes > kRopeAxes) return capi_fail(PI05W4A4_EINVAL, "axes must be in [1, %d], got %d", kRopeAxes, axes);
  if (pos_bytes != 4 && pos_bytes != 8) return capi_fail(PI05W4A4_EINVAL, "positions have 4 or 8 bytes, got %d", pos_bytes);
  if (!(eps >= 0.0f) || !std::isfinite(eps)) return capi_fail(PI05W4A4_EINVAL, "eps must be finite and not negative");
  p.heads[0] = h;
  p.heads[1] = kvh;
  p.b = b;
  p.t = t;
  p.d = d;
  if (int rc = check_heads(p)) return rc;
  for (int j = 0; j < rot / 2; ++j) {
    const int a = axis_of_pair != nullptr ? axis_of_pair[j] : 0;
    if (a >= axes) return capi_fail(PI05W4A4_EINVAL, "pair %d is on axis %d of %d", j, a, axes);
    p.axis[j / 16] |= static_cast<uint32_t>(a) << (2 * (j % 16));
  }
  p.rot = rot;
  p.axes = axes;
  p.pos64 = pos_bytes == 8;
  p.interleaved = interleaved != 0;
  p.unit_offset = unit_offset != 0;
  p.eps = eps;
  if (b == 0 || t == 0) return PI05W4A4_OK;
  if (int rc = check_strides(q, q_strides, "q")) return rc;
  if (int rc = check_strides(k, k_strides, "k")) return rc;
  if (q_out == nullptr || !aligned(q_out, 16)) return capi_fail(PI05W4A4_EINVAL, "the outputs must be 16-byte aligned");
  if (!aligned(q_weight, 16) || !aligned(k_weight, 16)) return capi_fail(PI05W4A4_EINVAL, "the norm weights must be 16-byte aligned");
  if (rot > 0) {
    if (positions == nullptr || pos_strides == nullptr || inv_freq == nullptr) return capi_fail(PI05W4A4_EINVAL, "null pointer argument");
    if (!aligned(positions, pos_bytes) || !aligned(inv_freq, 4))
      return capi_fail(PI05W4A4_EINVAL, "positions and frequencies must be aligned to their elements");
    for (int i = 0; i < 3; ++i)
      if (pos_strides[i] < 0) return capi_fail(PI05W4A4_EINVAL, "the strides of the positions must be >= 0");
    set_strides(p.pos_stride, pos_strides);
  }
  p.x[0] = q;
  p.x[1] = k;
  set_strides(p.stride[0], q_strides);
  set_strides(p.stride[1], k_strides);
  p.w[0] = q_weight;
  p.w[1] = k_weight;
  p.pos = positions;
  p.freq = inv_freq;
  p.q_out = q_out;
  return PI05W4A4_OK;
}

extern "C" int pi05w4a4_qk_norm_rope(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                     int32_t elem, int32_t b, int32_t t, int32_t h, int32_t kvh, int32_t d,
                                     const void* q_weight, const void* k_weight, float eps, int32_t unit_offset,
                                     const void* positions, const int64_t* pos_strides, int32_t pos_bytes, int32_t axes,
                                     const uint8_t* axis_of_pair, const float* inv_freq, int32_t rot,
                                     int32_t interleaved, void* q_out, void* k_out, void* stream) {
  HeadRopeParams p{};
  if (int rc = rope_params(p, q, q_strides, k, k_strides, elem, b, t, h, kvh, d, q_weight, k_weight, eps, unit_offset, positions,
                           pos_strides, pos_bytes, axes, axis_of_pair, inv_freq, rot, interleaved, q_out))
    return rc;
  if (b == 0 || t == 0) return capi_ok();
  if (k_out == nullptr || !aligned(k_out, 16)) return capi_fail(PI05W4A4_EINVAL, "the outputs must be 16-byte aligned");
  p.k_out = k_out;
  return run_head_rope(p, elem, stream, "qk_norm_rope launch");
}

extern "C" int pi05w4a4_qk_norm_rope_append(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                            const void* v, const int64_t* v_strides, int32_t elem, int32_t b, int32_t t,
                                            int32_t h, int32_t kvh, int32_t d, const void* q_weight, const void* k_weight,
                                            float eps, int32_t unit_offset, const void* positions,
                                            const int64_t* pos_strides, int32_t pos_bytes, int32_t axes,
                                            const uint8_t* axis_of_pair, const float* inv_freq, int32_t rot,
                                            int32_t interleaved, void* q_out, void* k_cache, void* v_cache, int32_t pages,
                                            const int32_t* table, int64_t table_stride, int32_t table_pages,
                                            const int32_t* lens, const int32_t* counts, void* stream) {
  HeadRopeParams p{};
  if (int rc = rope_params(p, q, q_strides, k, k_strides, elem, b, t, h, kvh, d, q_weight, k_weight, eps, unit_offset, positions,
                           pos_strides, pos_bytes, axes, axis_of_pair, inv_freq, rot, interleaved, q_out))
    return rc;
  p.c = {k_cache, v_cache, table, lens, table_stride, pages, table_pages, kvh, d};
  if (int rc = check_cache(p.c, b, t)) return rc;
  if (b == 0 || t == 0) return capi_ok();
  if (int rc = check_cache_pointers(p.c)) return rc;
  if (int rc = check_strides(v, v_strides, "v")) return rc;
  if (!aligned(counts, 4)) return capi_fail(PI05W4A4_EINVAL, "counts must be 4-byte aligned");
  p.x[2] = v;
  set_strides(p.stride[2], v_strides);
  p.heads[2] = kvh;
  p.counts = counts;
  return run_head_rope(p, elem, stream, "qk_norm_rope_append launch");
}

extern "C" int pi05w4a4_kv_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, int32_t elem,
                                  int32_t b, int32_t t, int32_t kvh, int32_t d, void* k_cache, void* v_cache, int32_t pages,
                                  const int32_t* table, int64_t table_stride, int32_t table_pages, const int32_t* lens,
                                  const int32_t* counts, void* stream) {
  if (int rc = check_elem(elem)) return rc;
  HeadRopeParams p{};
  p.c = {k_cache, v_cache, table, lens, table_stride, pages, table_pages, kvh, d};
  if (int rc = check_cache(p.c, b, t)) return rc;
  p.heads[1] = p.heads[2] = kvh;
  p.b = b;
  p.t = t;
  p.d = d;
  p.axes = 1;
  if (int rc = check_heads(p)) return rc;
  if (b == 0 || t == 0) return capi_ok();
  if (int rc = check_cache_pointers(p.c)) return rc;
  if (int rc = check_strides(k, k_strides, "k")) return rc;
  if (int rc = check_strides(v, v_strides, "v")) return rc;
  if (!aligned(counts, 4)) return capi_fail(PI05W4A4_EINVAL, "counts must be 4-byte aligned");
  p.x[1] = k;
  p.x[2] = v;
  set_strides(p.stride[1], k_strides);
  set_strides(p.stride[2], v_strides);
  p.counts = counts;
  return run_head_rope(p, elem, stream, "kv_append launch");
}

extern "C" size_t pi05w4a4_kv_attention_workspace_bytes(int32_t b, int32_t t, int32_t h, int32_t kvh, int32_t d,
                                                        int32_t table_pages) {
  if (b <= 0 || t <= 0 || kvh <= 0 || h < kvh || table_pages <= 0) return 0;
  return kv_attn16_workspace(b, t, h, d, kv_attn16_plan(b, t, h, kvh, d, table_pages, device_cu_count()).nsplit);
}

extern "C" int pi05w4a4_kv_attention(const void* q, const int64_t* q_strides, int32_t elem, int32_t b, int32_t t, int32_t h,
                                     int32_t kvh, int32_t d, const void* k_cache, const void* v_cache, int32_t pages,
                                     const int32_t* table, int64_t table_stride, int32_t table_pages, const int32_t* lens,
                                     const int32_t* q_lens, float scaling, int32_t causal, void* out, float* lse,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_elem(elem)) return rc;
  KvAttn16Params p{};
  p.c = {const_cast<void*>(k_cache), const_cast<void*>(v_cache), table, lens, table_stride, pages, table_pages, kvh, d};
  if (int rc = check_cache(p.c, b, t)) return rc;
  if (h <= 0 || h % kvh != 0 || h > 65535)
    return capi_fail(PI05W4A4_EINVAL, "query heads must be a multiple of the KV heads, got %d and %d", h, kvh);
  if (static_cast<int64_t>(t) * (h / kvh) > (1 << 26))
    return capi_fail(PI05W4A4_EINVAL, "T * H / KVH must be at most 2^26, got T=%d H=%d KVH=%d", t, h, kvh);
  if (static_cast<int64_t>(b) * t * h > (1 << 30))
    return capi_fail(PI05W4A4_EINVAL, "B * T * H must be at most 2^30, got %d x %d x %d", b, t, h);
  if (!std::isfinite(scaling)) return capi_fail(PI05W4A4_EINVAL, "scaling must be finite");
  if (b == 0 || t == 0) return capi_ok();
  if (int rc = check_cache_pointers(p.c)) return rc;
  if (int rc = check_strides(q, q_strides, "q")) return rc;
  if (out == nullptr || !aligned(out, 16) || !aligned(lse, 4) || !aligned(q_lens, 4))
    return capi_fail(PI05W4A4_EINVAL, "out must be 16-byte aligned");
  const KvAttn16Plan plan = kv_attn16_plan(b, t, h, kvh, d, table_pages, device_cu_count());
  p.nsplit = plan.nsplit;
  p.waves = plan.waves;
  p.wide = plan.wide;
  const size_t need = kv_attn16_workspace(b, t, h, d, p.nsplit);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return capi_fail(PI05W4A4_EWORKSPACE, "kv_attention needs a 16-byte aligned workspace of %zu bytes, got %zu", need, workspace_bytes);
  p.q = q;
  set_strides(p.q_stride, q_strides);
  p.q_lens = q_lens;
  p.out = out;
  p.lse = lse;
  p.ws = static_cast<float*>(workspace);
  p.scaling = scaling;
  p.down = kv_attn16_down(elem, table_pages);
  p.up = 1.0f / p.down;
  p.causal = causal != 0;
  p.b = b;
  p.t = t;
  p.h = h;
  return capi_hip(launch_kv_attn16(p, elem, static_cast<hipStream_t>(stream)), "kv_attention launch");
}

static int check_lora(int64_t m, int64_t per_id, int32_t k, int32_t n, int32_t r, int32_t slices, int32_t adapters) {
  if (m < 0 || m > (1 << 26)) return capi_fail(PI05W4A4_EINVAL, "M must be in [0, 2^26], got %lld", (long long)m);
  if (per_id < 1 || per_id > (1 << 26))
    return capi_fail(PI05W4A4_EINVAL, "rows of an id must be in [1, 2^26], got %lld", (long long)per_id);
  if (k <= 0 || k % 8 != 0 || k > (1 << 20))
    return capi_fail(PI05W4A4_EINVAL, "K must be a multiple of 8 of at most 2^20, got %d", k);
  if (n < 0 || n > (1 << 22)) return capi_fail(PI05W4A4_EINVAL, "N must be in [0, 2^22], got %d", n);
  if (r <= 0 || r % 8 != 0 || r > kLoraMaxRank)
    return capi_fail(PI05W4A4_EINVAL, "the rank must be a multiple of 8 of at most %d, got %d", kLoraMaxRank, r);
  if (slices < 1 || slices > kLoraSlices) return capi_fail(PI05W4A4_EINVAL, "slices must be in [1, %d], got %d", kLoraSlices, slices);
  if (adapters < 0) return capi_fail(PI05W4A4_EINVAL, "adapters must be >= 0, got %d", adapters);
  return PI05W4A4_OK;
}

// Whether rows of k elements at x and of n at out share bytes (2 bytes an element): rows beside each other in wider ones do not.
static bool rows_overlap(const void* x, int64_t ldx, int32_t k, const void* out, int64_t ldo, int32_t n, int64_t m) {
  const int64_t a = reinterpret_cast<intptr_t>(x), b = reinterpret_cast<intptr_t>(out);
  const int64_t a_end = a + 2 * ((m - 1) * ldx + k), b_end = b + 2 * ((m - 1) * ldo + n);
  if (a_end <= b || b_end <= a) return false;
  if (ldx != ldo || ldx < k + static_cast<int64_t>(n)) return true;
  const int64_t ld = 2 * ldo, off = ((a - b) % ld + ld) % ld;  // of x's rows behind out's
  return off < 2 * static_cast<int64_t>(n) || off + 2 * static_cast<int64_t>(k) > ld;
}

static size_t lora_workspace(int64_t m, int32_t r, int32_t slices, int ksplit) {
  return sizeof(float) * static_cast<size_t>(ksplit) * static_cast<size_t>(lora_h_floats(m, r, slices));
}

extern "C" size_t pi05w4a4_lora_workspace_bytes(int64_t m, int64_t per_id, int32_t k, int32_t n, int32_t r, int32_t slices,
                                                int32_t adapters) {
  if (check_lora(m, per_id, k, n, r, slices, adapters) != PI05W4A4_OK || m == 0 || n == 0 || adapters == 0) return 0;
  return lora_workspace(m, r, slices, lora_plan(m, per_id, k, n, r, slices, adapters, device_cu_count()).ksplit);
}

extern "C" int pi05w4a4_lora_add(const void* y, int64_t ldy, const void* x, int64_t ldx, int64_t m, int32_t k, const void* a,
                                 const void* b, const float* scale, int32_t adapters, int32_t r, const int32_t* ids,
                                 int64_t per_id, int32_t n, int32_t slices, const int32_t* widths, int32_t elem, void* out,
                                 int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_elem(elem)) return rc;
  if (int rc = check_lora(m, per_id, k, n, r, slices, adapters)) return rc;
  LoraParams p{};
  int64_t sum = 0;
  for (int s = 0; s < slices; ++s) {
    p.width[s] = widths != nullptr ? widths[s] : n;
    if (p.width[s] <= 0 && n > 0) return capi_fail(PI05W4A4_EINVAL, "slice %d has %d columns", s, p.width[s]);
    sum += p.width[s];
  }
  if (sum != n) return capi_fail(PI05W4A4_EINVAL, "the slices have %lld columns, the outputs %d", (long long)sum, n);
  if (m == 0 || n == 0) return capi_ok();
  if (y == nullptr || x == nullptr || ids == nullptr || out == nullptr) return capi_fail(PI05W4A4_EINVAL, "null pointer argument");
  if (adapters > 0 && (a == nullptr || b == nullptr)) return capi_fail(PI05W4A4_EINVAL, "null pointer argument");
  if (!aligned(x, 16) || !aligned(a, 16) || !aligned(b, 16) || !aligned(scale, 4) || !aligned(ids, 4) || !aligned(y, 2) || !aligned(out, 2))
    return capi_fail(PI05W4A4_EINVAL, "x, a and b must be 16-byte aligned");
  if (ldx < 0 || ldx % 8 != 0) return capi_fail(PI05W4A4_EINVAL, "the row stride of x must be a multiple of 8 elements, got %lld", (long long)ldx);
  if (ldy < 0 || ldo < n) return capi_fail(PI05W4A4_EINVAL, "row strides must be >= 0, and those of the output >= N");
  if (rows_overlap(x, ldx, k, out, ldo, n, m)) return capi_fail(PI05W4A4_EINVAL, "x must not overlap the output");
  if (!(y == out && (ldy == ldo || m == 1)) && rows_overlap(y, ldy, n, out, ldo, n, m))
    return capi_fail(PI05W4A4_EINVAL, "y must be the output or not overlap it");
  const LoraPlan plan = lora_plan(m, per_id, k, n, r, slices, adapters, device_cu_count());
  p.m = m;
  p.r = r;
  p.slices = slices;
  p.per_id = per_id;
  if (!lora_grid(p, plan)) return capi_fail(PI05W4A4_EINVAL, "tiles of %lld rows by %d columns are more waves than one launch holds", (long long)m, n);
  const size_t need = adapters > 0 ? lora_workspace(m, r, slices, plan.ksplit) : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return capi_fail(PI05W4A4_EWORKSPACE, "lora_add needs a 16-byte aligned workspace of %zu bytes, got %zu", need, workspace_bytes);
  p.x = x;
  p.a = a;
  p.b = b;
  p.scale = scale;
  p.ids = ids;
  p.y = y;
  p.out = out;
  p.h = static_cast<float*>(workspace);
  p.ldx = ldx;
  p.ldy = ldy;
  p.ldo = ldo;
  p.k = k;
  p.n = n;
  p.adapters = adapters;
  return capi_hip(launch_lora(p, elem, static_cast<hipStream_t>(stream)), "lora_add launch");
}
