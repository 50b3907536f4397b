// Shared by the 8-bit operators' translation units (int8_rows, int8_gemm, kv_int8; not part of
// the ABI): their parameter blocks, launch functions and the two 16-bit element types.
#pragma once

#include "w4a4_internal.h"

namespace w4a4 {

// fp16 and bf16 elements: PI05W4A4_FP16 / PI05W4A4_BF16 of the ABI.
enum ElemType : int { kFp16 = 0, kBf16 = 1 };

struct Int8RowsParams {
  const void* x;      // [M, K] elements, row stride ldx
  const void* res;    // residual [M, K], row stride ldr (add form) or null
  const void* w;      // norm weight [K] or null (no norm)
  int64_t ldx, ldr;
  int64_t m;
  int32_t k;
  float eps;
  int32_t unit_offset;
  int8_t* q;          // [M, K]
  float* scale;       // [M]
  void* h;            // [M, K] x + residual (add form)
};
hipError_t launch_int8_rows(const Int8RowsParams& p, int elem, hipStream_t stream);

struct Int8GemmParams {
  const int8_t* q;   // [M, K], row stride ldq
  const int8_t* w;   // [N, K], row stride ldw
  const float* sq;   // [M]
  const float* sw;   // [N]
  const void* bias;  // [N] or null
  const void* res;   // [M, N], row stride ldr, or null
  void* y;           // [M, N]
  int64_t m, ldq, ldw, ldr;
  int32_t n, k;
  int32_t mtiles, ntiles;
  int32_t ksplit;    // K slices, each to its own partial sums (1: none)
  int32_t* partial;  // int32 [ksplit, M, N]
};
// Tile and K split of a call: a rule on M, N, K and the CU count.
struct Int8GemmPlan {
  int tile;    // kernel variant
  int ksplit;
};
Int8GemmPlan int8_gemm_plan(int64_t m, int32_t n, int32_t k, int cus);
hipError_t launch_int8_gemm(Int8GemmParams p, const Int8GemmPlan& plan, int elem, hipStream_t stream);

// An 8-bit KV cache: pages of 64 tokens, codes and one scale for each page and KV head.
constexpr int kKvPage = 64;
struct KvCache8 {
  int8_t* k;           // [pages, KVH, 64, D]
  int8_t* v;           // [pages, KVH, D, 64]
  float* ks;           // [pages, KVH]
  float* vs;           // [pages, KVH]
  const int32_t* table;  // [B, table_pages], row stride table_stride
  const int32_t* lens;   // [B]
  int64_t table_stride;
  int32_t pages;
  int32_t table_pages;
  int32_t kvh, d;
};
struct KvAppendParams {
  KvCache8 c;
  const void* k;
  const void* v;
  int64_t k_stride[3], v_stride[3];  // batch, token, head (elements)
  const int32_t* counts;  // [B] or null: all T
  int32_t b, t;
};
hipError_t launch_kv_append(const KvAppendParams& p, int elem, hipStream_t stream);

struct KvAttnParams {
  KvCache8 c;
  const void* q;
  int64_t q_stride[3];    // batch, token, head (elements)
  const int32_t* q_lens;  // [B] or null: all T
  void* out;              // [B, T, H, D]
  float* lse;             // [B, T, H] or null
  float* ws;              // partial results when nsplit > 1
  float scaling;
  int32_t causal;
  int32_t b, t, h;
  int32_t nsplit;
  bool wide;  // 128 rows a workgroup, else 16
};
struct KvAttnPlan {
  bool wide;
  int nsplit;
};
KvAttnPlan kv_attn_plan(int64_t b, int64_t t, int32_t h, int32_t kvh, int32_t d, int64_t table_pages, int cus);
size_t kv_attn_workspace(int64_t b, int64_t t, int32_t h, int32_t d, int nsplit);
hipError_t launch_kv_attention(const KvAttnParams& p, int elem, hipStream_t stream);

// Error text and status shared with the other entry points (capi.hip).
int capi_fail(int code, const char* fmt, ...);
int capi_ok();
int capi_hip(hipError_t e, const char* what);

}  // namespace w4a4
