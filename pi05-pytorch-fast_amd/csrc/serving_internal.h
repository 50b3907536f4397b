// Shared by the 16-bit serving operators' translation units (head_rope, kv_attn, lora; not part of the
// ABI): their parameter blocks and launch functions.
#pragma once

#include "int8_internal.h"

namespace w4a4 {

// A 16-bit KV cache: pages of 64 tokens, keys and values [pages, KVH, 64, D].
struct KvCache16 {
  void* k;
  void* v;
  const int32_t* table;  // [B, table_pages], row stride table_stride
  const int32_t* lens;   // [B]
  int64_t table_stride;
  int32_t pages;
  int32_t table_pages;
  int32_t kvh, d;
};

// Query and key heads behind their norm and rotation, keys and values into a cache: any of the parts
// may be missing.
constexpr int kRopeAxes = 4;
constexpr int kMaxHeadDim = 512;
struct HeadRopeParams {
  const void* x[3];       // q, k, v [B, T, heads, D] (null: none)
  int64_t stride[3][3];   // batch, token, head (elements)
  int32_t heads[3];
  const void* w[2];       // norm weights [D] of q and k, or null
  const void* pos;        // positions [axes, B, T], int32 or int64
  int64_t pos_stride[3];  // axis, batch, token
  const float* freq;      // [rot / 2]
  uint32_t axis[kMaxHeadDim / 32];  // axis of each pair, two bits each
  int32_t pos64, axes;
  int32_t rot;            // rotated dimensions (0: none)
  int32_t interleaved;
  int32_t unit_offset;
  float eps;
  int32_t b, t, d;
  int32_t parts;          // waves that share a token's heads
  void* q_out;            // [B, T, H, D]
  void* k_out;            // [B, T, KVH, D], or null: into the cache
  KvCache16 c;            // c.lens null: no cache
  const int32_t* counts;  // [B] or null: all T
};
int32_t head_rope_parts(const HeadRopeParams& p, int cus);
hipError_t launch_head_rope(const HeadRopeParams& p, int elem, hipStream_t stream);

struct KvAttn16Params {
  KvCache16 c;
  const void* q;
  int64_t q_stride[3];    // batch, token, head (elements)
  const int32_t* q_lens;  // [B] or null: all T
  void* out;              // [B, T, H, D]
  float* lse;             // [B, T, H] or null
  float* ws;              // partial results when nsplit > 1
  float scaling;
  float down, up;         // factor of the softmax weights and its inverse, powers of two (fp16: 1)
  int32_t causal;
  int32_t b, t, h;
  int32_t nsplit;         // runs of pages of a sequence
  int32_t waves;          // of a workgroup
  int32_t wide;           // 64 rows a workgroup, not 16
};
struct KvAttn16Plan {
  int nsplit;
  int waves;
  bool wide;
};
KvAttn16Plan kv_attn16_plan(int64_t b, int64_t t, int32_t h, int32_t kvh, int32_t d, int64_t table_pages, int cus);
float kv_attn16_down(int elem, int64_t table_pages);
size_t kv_attn16_workspace(int64_t b, int64_t t, int32_t h, int32_t d, int nsplit);
hipError_t launch_kv_attn16(const KvAttn16Params& p, int elem, hipStream_t stream);

// out = y + scale[id] (x A[id]^T) B[id]^T, the id of each row.
constexpr int kLoraSlices = 4;
constexpr int kLoraMaxRank = 128;
struct LoraParams {
  const void* x;       // [M, K], row stride ldx
  const void* a;       // [adapters, slices * R, K]
  const void* b;       // [adapters, N, R]
  const float* scale;  // [adapters] or null
  const int32_t* ids;  // [M / per_id]
  const void* y;       // [M, N], row stride ldy
  void* out;           // [M, N], row stride ldo (may be y)
  float* h;            // [ksplit, h_plane]
  int64_t m, per_id, ldx, ldy, ldo;
  int32_t k, n, r, adapters, slices;
  int32_t width[kLoraSlices];  // columns of each slice
  int32_t ksplit;      // K slices of the first launch; 0: both products in one
  int32_t units;       // 16-row tiles of requests, or windows of rows
  int32_t unit0;       // the first one of a launch
  int32_t groups;      // workgroups of a window: its tiles at most
  int32_t tiles;       // of a request
  int32_t gather;      // windows
  int32_t leaders;     // a workgroup for each row of a window
  int32_t runs;        // of a workgroup's columns, over the slices
  int64_t h_plane;     // floats of a K slice in h
};
struct LoraPlan {
  int32_t ksplit, units, groups, tiles;
  bool gather, leaders;
};
LoraPlan lora_plan(int64_t m, int64_t per_id, int32_t k, int32_t n, int32_t r, int32_t slices, int32_t adapters, int cus);
int64_t lora_h_floats(int64_t m, int32_t r, int32_t slices);
// What of a call follows from its plan; false: whole tiles of its rows are more waves than one launch holds.
bool lora_grid(LoraParams& p, const LoraPlan& plan);
hipError_t launch_lora(const LoraParams& p, int elem, hipStream_t stream);

}  // namespace w4a4
