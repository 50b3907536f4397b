// An 8-bit KV cache of 64-token pages with one scale for each page and KV head (keys and values
// have their own), the append that writes it and the attention that reads it.
//
// Layout: K codes [pages, KVH, 64, D]; V codes transposed within the page, [pages, KVH, D, 64].  The
// attention computes S^T = K Q^T and O^T = V^T P^T on matrix instructions whose operands are 16-byte
// loads of consecutive codes of either array: no transposes.

#include "direct_load.h"
#include <algorithm>

#include "int8_internal.h"

namespace w4a4 {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

constexpr float kRintMagic = 12582912.0f;  // 1.5 * 2^23: the low byte of x + magic is rint(x)
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x0c0c0400u),
                               __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x0c0c0400u), 0x05040100u);
}

// ------------------------------------------------------------------ append
// One workgroup for each (sequence, touched page, KV head, side): it finds the largest new value,
// settles the page's scale
//   s = max(s0, max|new| / 127 + 1e-12),  s0 the scale of the tokens that are there (0: none),
// brings the old codes to it where it grew, c' = rint(c (s0 / s)), and writes the new ones,
// c = rint(x (1 / s)).  A page whose first token is new is written whole, zeros behind the last
// token, so that nothing of the page's earlier owner is left.  Its time is a chain of loads, lens -> table ->
// values and scale -> old codes, of which only the first link has to be one: 16 x 1 tokens 6.5 us, 8 x 776
// tokens 6.3 (9.5 MB, 1.5 TB/s; 69% of a wave's clocks are waits).
template <typename T, int D>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendParams p) {
  // A thread holds kRows consecutive page rows of eight consecutive dimensions, so that a V row (one
  // dimension) takes its kRows codes in one LDS write.
  constexpr int kRows = kKvPage * D / 8 / 256, kRowChunks = D / 8;
  constexpr int kStride = kKvPage + 8;            // staged V row, bytes
  constexpr int kGroups = D * 4 / 256;            // 16-token groups of V rows that a thread writes
  __shared__ uint32_t red[4];
  __shared__ __align__(16) char vt[D * kStride];
  const int tid = threadIdx.x;
  const int b = blockIdx.z;
  const int head = blockIdx.y >> 1;
  const bool is_v = (blockIdx.y & 1) != 0;
  const int64_t len = max(p.c.lens[b], 0);
  const int64_t count = min(max(p.counts != nullptr ? p.counts[b] : p.t, 0), p.t);
  const int64_t slot = len / kKvPage + blockIdx.x;
  const int64_t tok0 = slot * kKvPage - len;  // token of page row 0
  if (tok0 >= count || slot >= p.c.table_pages) return;
  const int first = static_cast<int>(max(-tok0, static_cast<int64_t>(0)));  // new tokens: page rows first .. last - 1
  const int last = static_cast<int>(min(count - tok0, static_cast<int64_t>(kKvPage)));
  if (last <= first) return;
  const int page = p.c.table[b * p.c.table_stride + slot];
  if (page < 0 || page >= p.c.pages) return;
  const int64_t ph = static_cast<int64_t>(page) * p.c.kvh + head;
  const int64_t* const st = is_v ? p.v_stride : p.k_stride;
  const T* const src = static_cast<const T*>(is_v ? p.v : p.k) + b * st[0] + head * st[2];
  const int row0 = tid / kRowChunks * kRows, d0 = (tid % kRowChunks) * 8;

  vec8<T> x[kRows];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int row = row0 + j;
    x[j] = vec8<T>{};
    if (row >= first && row < last) x[j] = *reinterpret_cast<const vec8<T>*>(src + (tok0 + row) * st[1] + d0);
  }
  float* const scale = (is_v ? p.c.vs : p.c.ks) + ph;
  const float s0 = first > 0 ? *scale : 0.0f;
#pragma unroll
  for (int j = 0; j < kRows; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(static_cast<float>(x[j][e])) & 0x7fffffffu);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o, 64)));
  if ((tid & 63) == 0) red[tid >> 6] = top;
  __syncthreads();  // also: every thread has read the old scale
  top = max(max(red[0], red[1]), max(red[2], red[3]));
  const float amax = __uint_as_float(top);
  const float need = amax / 127.0f + 1e-12f;
  // A NaN or infinity among the new values, or a scale that is NaN already, makes the page's scale NaN.
  const bool finite = amax <= 3.4028235e38f && s0 <= 3.4028235e38f;
  const bool grow = !finite || need > s0;
  const float s = !finite ? __builtin_nanf("") : grow ? need : s0;
  if (tid == 0 && grow) *scale = s;
  const float inv = finite ? 1.0f / s : 0.0f;
  const float ratio = finite && first > 0 ? s0 / s : 0.0f;

  uint32_t code[kRows][2];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = finite ? fmaf(static_cast<float>(x[j][e]), inv, kRintMagic) : kRintMagic;
    code[j][0] = pack4(f[0], f[1], f[2], f[3]);
    code[j][1] = pack4(f[4], f[5], f[6], f[7]);
  }
  auto rescaled = [&](uint32_t w) {  // the four old codes of w at the new scale
    float f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = fmaf(static_cast<float>(static_cast<int8_t>(w >> (8 * e))), ratio, kRintMagic);
    return pack4(f[0], f[1], f[2], f[3]);
  };
  const bool keep = first > 0;  // the page has tokens of before
  if (!is_v) {
    char* const dst = reinterpret_cast<char*>(p.c.k) + ph * (kKvPage * D) + row0 * D + d0;
    uint2 old[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const bool fresh = row0 + j >= first && row0 + j < last;
      old[j] = uint2{0u, 0u};
      if (!fresh && keep && grow) old[j] = *reinterpret_cast<const uint2*>(dst + j * D);
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const bool fresh = row0 + j >= first && row0 + j < last;
      if (fresh)
        *reinterpret_cast<uint2*>(dst + j * D) = uint2{code[j][0], code[j][1]};
      else if (!keep || grow)
        *reinterpret_cast<uint2*>(dst + j * D) = keep ? uint2{rescaled(old[j].x), rescaled(old[j].y)} : uint2{0u, 0u};
    }
    return;
  }
  // V: the new codes are turned in LDS; each thread then writes 16 tokens of one dimension at a time.
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < kRows; ++j) w[j >> 2] |= ((code[j][e >> 2] >> (8 * (e & 3))) & 0xffu) << (8 * (j & 3));
    char* const o = vt + (d0 + e) * kStride + row0;
    if constexpr (kRows == 8) *reinterpret_cast<uint2*>(o) = uint2{w[0], w[1]};
    else if constexpr (kRows == 4) *reinterpret_cast<uint32_t*>(o) = w[0];
    else *reinterpret_cast<uint16_t*>(o) = static_cast<uint16_t>(w[0]);
  }
  __syncthreads();
  char* const dst = reinterpret_cast<char*>(p.c.v) + ph * (kKvPage * D);
  v4i old[kGroups];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int at = i * 256 + tid, t0 = (at & 3) * 16;
    old[i] = v4i{0, 0, 0, 0};
    if (keep && (grow || (t0 + 16 > first && t0 < last))) old[i] = *reinterpret_cast<const v4i*>(dst + at * 16);
  }
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int at = i * 256 + tid, d = at >> 2, t0 = (at & 3) * 16;
    if (!grow && (t0 + 16 <= first || t0 >= last)) continue;
    v4i out;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t fresh = *reinterpret_cast<const uint32_t*>(vt + d * kStride + t0 + 4 * q);
      const uint32_t was = grow && keep ? rescaled(static_cast<uint32_t>(old[i][q])) : static_cast<uint32_t>(old[i][q]);
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (t0 + 4 * q + e >= first && t0 + 4 * q + e < last) m |= 0xffu << (8 * e);
      out[q] = static_cast<int>((fresh & m) | (was & ~m));
    }
    *reinterpret_cast<v4i*>(dst + at * 16) = out;
  }
}

// ------------------------------------------------------------------ attention
// Two kernels.  kv_attn_kernel: 16 query rows of one KV head (row = token * (H / KVH) + query
// head) and a run of the sequence's pages a workgroup, whose W waves take every W-th page, each with a
// softmax of its own (running maximum and sum), and meet in LDS at the end: decoded tokens, where
// the cache is read once and its bytes bound, and as many more rows as one round of the CUs holds.
// kv_attn_wide_kernel: 128 rows, 32 a wave, over pages that the waves share in LDS: chunks of tokens.
//
// Q K^T in int8: a query row is held as 16-bit integers v = rint(q / sq), |v| <= 32512, split
// v = 256 hi + lo into two int8 operands, so that S = sq ks (256 K hi + K lo) is exact but for
// the rounding of q, 2^-16 of the row's maximum: finer than fp16 there, and no conversion of K.
// P V in fp16: the codes are exact in fp16.  The page's V scale is folded into the exponent,
// w = 2^(S log2e + log2 vs - m) with m a reference that follows the running maximum of that sum from
// below, so that the weights of all pages share one accumulator; the sum of the probabilities is
// that of w / vs.  Sums, references and accumulators are fp32; w is rounded to fp16 (2^-11) for the product.
template <typename T, int D, int STEP>
__device__ __forceinline__ void load_query(const T* row, float& sq, v4i (&hi)[D / STEP], v4i (&lo)[D / STEP], int g) {
  // The lane's 16 elements at 16 g of every STEP; the row's lanes are those with the same lane % (1024 / STEP).
  float f[D / STEP][16];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < D / STEP; ++i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const vec8<T> v = *reinterpret_cast<const vec8<T>*>(row + STEP * i + 16 * g + 8 * h);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[i][8 * h + e] = static_cast<float>(v[e]);
        top = max(top, __float_as_uint(f[i][8 * h + e]) & 0x7fffffffu);
      }
    }
  }
  if constexpr (STEP == 64) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
  const float amax = __uint_as_float(top);
  const bool finite = amax <= 3.4028235e38f;
  sq = finite ? amax / 32512.0f : __builtin_nanf("");
  const float inv = finite && amax >= 1e-30f ? 32512.0f / amax : 0.0f;
  // v + 1.5 * 2^23 holds v in its low 16 bits: lo is the low byte as it is, hi the next one after adding 128.
#pragma unroll
  for (int i = 0; i < D / STEP; ++i) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __float_as_uint(finite ? fmaf(f[i][4 * w + e], inv, kRintMagic) : kRintMagic);
      lo[i][w] = static_cast<int>(__builtin_amdgcn_perm(__builtin_amdgcn_perm(v[3], v[2], 0x0c0c0400u),
                                                        __builtin_amdgcn_perm(v[1], v[0], 0x0c0c0400u), 0x05040100u));
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += 128u;
      hi[i][w] = static_cast<int>(__builtin_amdgcn_perm(__builtin_amdgcn_perm(v[3], v[2], 0x0c0c0501u),
                                                        __builtin_amdgcn_perm(v[1], v[0], 0x0c0c0501u), 0x05040100u));
    }
  }
}

// Eight codes as fp16: byte + 128 under the exponent of 1024, less 1152.
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ half8 codes_to_half(int w0, int w1) {
  const uint32_t u0 = static_cast<uint32_t>(w0) ^ 0x80808080u, u1 = static_cast<uint32_t>(w1) ^ 0x80808080u;
  const half2 bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
  half2 h[4];
  h[0] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, u0, 0x04010400u)) - bias;
  h[1] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, u0, 0x04030402u)) - bias;
  h[2] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, u1, 0x04010400u)) - bias;
  h[3] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, u1, 0x04030402u)) - bias;
  half8 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[2 * i] = h[i][0];
    o[2 * i + 1] = h[i][1];
  }
  return o;
}

constexpr float kNone = -1e30f;  // reference before the first visible key
// The reference is kLift below the largest exponent when it is set, and is set again only when an exponent
// is kTop above it: the largest weight of a row is between 2^kLift and 2^kTop, at the upper end of fp16, so
// that weights down to 2^-21 of it are rounded to 2^-11 and smaller ones to 2^-32 of it (many keys of
// little mass behind one that takes nearly all of it), and the accumulators are rescaled once or twice a run
// (a lift of 11 keeps four more bits and rescales more often: 2 x 776 tokens over 4096 keys 101.2 -> 103.6 us;
// without a lift 100.7).
constexpr float kLift = 7.0f, kTop = 15.0f;

// A load at a uniform address that nothing in the kernel writes: through the scalar cache, so that
// no wait for vector loads stands before its use.
template <typename U>
__device__ __forceinline__ U scalar_load(const U* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) U*>(reinterpret_cast<uintptr_t>(p));
}

// Partial results of a run: O (unnormalised, fp32), the maximum and the sum of each row; whole 16 bytes.
__host__ __device__ inline int64_t split_floats(int64_t rows, int d) { return (rows * (d + 2) + 3) & ~int64_t{3}; }

// What a workgroup's rows see.  ROWS query rows of a KV head from row0 on; a lane's row is given.
struct Span {
  int64_t q_len, len;
  int causal;
  __device__ __forceinline__ Span(const KvAttnParams& p, int b) {
    const int64_t cap = static_cast<int64_t>(p.c.table_pages) * kKvPage;
    len = p.c.pages > 0 ? min(static_cast<int64_t>(max(p.c.lens[b], 0)), cap) : 0;
    q_len = min(max(p.q_lens != nullptr ? p.q_lens[b] : p.t, 0), p.t);
    causal = p.causal;
  }
  // Tokens that query `token` sees: none past q_len.
  __device__ __forceinline__ int64_t seen(int64_t token) const {
    return token >= q_len ? static_cast<int64_t>(0) : causal ? max(len - q_len + token + 1, static_cast<int64_t>(0)) : len;
  }
  // The most that any of the tokens first .. last sees, and what all of them do.
  __device__ __forceinline__ int64_t most(int64_t first, int64_t last) const { return seen(min(last, max(q_len - 1, first))); }
  __device__ __forceinline__ int64_t least(int64_t first, int64_t last) const { return last < q_len ? seen(first) : 0; }
};

// The end of a row: its output, or its part of a run's partial results.  v: columns 4 consecutive from c.
template <typename T>
__device__ __forceinline__ void store_quad(const KvAttnParams& p, const v4f v, float inv, int split, int64_t orow, int d, int c) {
  if (p.nsplit > 1) {
    const int64_t all_rows = static_cast<int64_t>(p.b) * p.t * p.h;
    *reinterpret_cast<v4f*>(p.ws + split * split_floats(all_rows, d) + orow * d + c) = v;
  } else {
    typedef T tv4 __attribute__((ext_vector_type(4)));
    tv4 y;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = static_cast<T>(inv == 0.0f ? 0.0f : v[r] * inv);
    *reinterpret_cast<tv4*>(static_cast<T*>(p.out) + orow * d + c) = y;
  }
}
__device__ __forceinline__ void store_sums(const KvAttnParams& p, float m, float l, int split, int64_t orow, int d) {
  if (p.nsplit > 1) {
    const int64_t all_rows = static_cast<int64_t>(p.b) * p.t * p.h;
    float* const ml = p.ws + split * split_floats(all_rows, d) + all_rows * d + orow * 2;
    ml[0] = m;
    ml[1] = l;
  } else if (p.lse != nullptr) {
    p.lse[orow] = l == 0.0f ? -__builtin_inff() : m / kLog2e + __builtin_logf(l);
  }
}

// Lane L of a 16 x 16 S^T tile holds row L % 16 and four consecutive tile rows 4 (L / 16) ..  Tile
// t's row 4 a + r is key 16 a + 4 t + r, so that over the four tiles of a page the lane holds
// keys 16 (L / 16) .. + 15: the 16 bytes that it loads of a V row.
// A page's values are requested before its scores, the next page's keys as the values are used up.
// Bound by the cache's bytes: 64 sequences of up to 8192 keys, 8 heads on one of D = 256, 45 us for 202
// MB, 4.5 TB/s where plain reads reach 6.3; a single sequence by the chain length, table entry, scales
// and keys, queries (776 keys: 6.8 us, and 3.2 of the join).
template <typename T, int D, int W>
__global__ __launch_bounds__(64 * W, 2) void kv_attn_kernel(KvAttnParams p) {
  constexpr int F = D / 64, DT = D / 16;
  static_assert(DT == 4 * F, "a key load for each tile of values");
  extern __shared__ __align__(16) v4f obuf[];  // [W][DT][64]
  __shared__ float mbuf[W][16], lbuf[W][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int group = p.h / p.c.kvh;
  const int rows = p.t * group;
  const int tiles = (rows + 15) >> 4;
  const int tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
  const int head = blockIdx.y, b = blockIdx.z;
  const Span span(p, b);

  // This lane's row; rows past the last one, and tokens past q_len, see nothing.
  const int row = tile * 16 + col;
  const int tok = min(row / group, p.t - 1), qh = head * group + row % group;
  const int64_t seen = row < rows ? span.seen(row / group) : 0;
  const int64_t tok_first = tile * 16 / group, tok_last = min(tile * 16 + 15, rows - 1) / group;
  const int64_t least = tile * 16 + 15 < rows ? span.least(tok_first, tok_last) : 0;
  const int pages = static_cast<int>((span.most(tok_first, tok_last) + kKvPage - 1) / kKvPage);
  const int per = (pages + p.nsplit - 1) / p.nsplit;
  const int begin = split * per, end = min(begin + per, pages);

  float sq;
  v4i qhi[F], qlo[F];
  const T* const qrow = static_cast<const T*>(p.q) + b * p.q_stride[0] + tok * p.q_stride[1] + qh * p.q_stride[2];
  load_query<T, D, 64>(qrow, sq, qhi, qlo, g);
  const float qfac = sq * p.scaling * kLog2e;

  float m = kNone, l = 0.0f;
  v4f o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  // Entries that name no page are read as page 0, whose keys then count as not there.
  const int32_t* const table = p.c.table + b * p.c.table_stride;
  const int64_t koff = (16 * (col >> 2) + (col & 3)) * D + 16 * g, voff = col * kKvPage + 16 * g;
  auto page_at = [&](int pg) { return pg < end ? scalar_load(table + __builtin_amdgcn_readfirstlane(pg)) : -1; };
  auto place = [&](int page) {
    return static_cast<int64_t>(__builtin_amdgcn_readfirstlane(page >= 0 && page < p.c.pages ? page : 0)) * p.c.kvh + head;
  };
  v4i kc[4][F];
  auto load_key = [&](const int8_t* kp, int i) { kc[i / F][i % F] = *reinterpret_cast<const v4i*>(kp + 4 * (i / F) * D + 64 * (i % F)); };
  int page = page_at(begin + wave);
  if (begin + wave < end) {
#pragma unroll
    for (int i = 0; i < 4 * F; ++i) load_key(p.c.k + place(page) * (kKvPage * D) + koff, i);
  }
  for (int pg = begin + wave; pg < end; pg += W) {
    const int64_t ph = place(page);
    const bool there = page >= 0 && page < p.c.pages;
    const int next = page_at(pg + W);
    const int8_t* const vp = p.c.v + ph * (kKvPage * D) + voff;
    const float ks = scalar_load(p.c.ks + ph);
    float vs = scalar_load(p.c.vs + ph);
    if (vs == 0.0f) vs = 1e-20f;  // zeros, whatever the codes: the page still counts in the sum
    v4i vc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) vc[i] = *reinterpret_cast<const v4i*>(vp + 16 * i * kKvPage);

    const float fac = qfac * ks, lvs = __builtin_log2f(vs);
    float s[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      v4i ah{0, 0, 0, 0}, al{0, 0, 0, 0};
#pragma unroll
      for (int f = 0; f < F; ++f) {
        ah = __builtin_amdgcn_mfma_i32_16x16x64_i8(kc[t][f], qhi[f], ah, 0, 0, 0);
        al = __builtin_amdgcn_mfma_i32_16x16x64_i8(kc[t][f], qlo[f], al, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) s[t][r] = fmaf(static_cast<float>(256 * ah[r] + al[r]), fac, lvs);
    }
    const int64_t key0 = static_cast<int64_t>(pg) * kKvPage;
    const int64_t limit = there ? seen : 0;
    if (!there || key0 + kKvPage > least) {  // some row does not see the whole page
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + 16 * g + 4 * t + r >= limit) s[t][r] = -__builtin_inff();
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[t][r]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > m + kTop)) {
      const float m1 = fmaxf(m, top - kLift);
      const float alpha = __builtin_amdgcn_exp2f(m - m1);
      m = m1;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < DT; ++i) o[i] *= alpha;
    }
    float sum = 0.0f;
    half8 w[2];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f(s[t][r] - m);
        sum += e;
        w[t >> 1][4 * (t & 1) + r] = static_cast<_Float16>(e);
      }
    // A row that sees nothing of the page takes nothing from its scale either (it may be NaN).
    l += sum != 0.0f ? sum / vs : 0.0f;
    // The next page's keys take the registers of the values as these are used (past the last page:
    // this one's again, not used).
    const int8_t* const kn = p.c.k + (pg + W < end ? place(next) : ph) * (kKvPage * D) + koff;
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_half(vc[i][0], vc[i][1]), w[0], o[i], 0, 0, 0);
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_half(vc[i][2], vc[i][3]), w[1], o[i], 0, 0, 0);
      load_key(kn, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    page = next;
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  const int64_t orow = (static_cast<int64_t>(b) * p.t + tok) * p.h + qh;
  if constexpr (W == 1) {
    if (row >= rows) return;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < DT; ++i) store_quad<T>(p, o[i], inv, split, orow, D, 16 * i + 4 * g);
    if (g == 0) store_sums(p, m, l, split, orow, D);
    return;
  }
  // The waves' parts meet in LDS, scaled to a common maximum; each wave sums and finishes DT / W tiles
  // of dimensions.
  if (g == 0) {
    mbuf[wave][col] = m;
    lbuf[wave][col] = l;
  }
  __syncthreads();
  float mall = mbuf[0][col];
#pragma unroll
  for (int w = 1; w < W; ++w) mall = fmaxf(mall, mbuf[w][col]);
  const float mine = __builtin_amdgcn_exp2f(m - mall);
#pragma unroll
  for (int i = 0; i < DT; ++i) obuf[(wave * DT + i) * 64 + lane] = o[i] * mine;
  float lall = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) lall += lbuf[w][col] * __builtin_amdgcn_exp2f(mbuf[w][col] - mall);
  __syncthreads();
  if (row >= rows) return;
  const float inv = lall != 0.0f ? 1.0f / lall : 0.0f;  // 0: no visible key (NaN stays NaN)
  for (int i = wave; i < DT; i += W) {
    v4f v = obuf[i * 64 + lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += obuf[(w * DT + i) * 64 + lane];
    store_quad<T>(p, v, inv, split, orow, D, 16 * i + 4 * g);
  }
  if (wave == 0 && g == 0) store_sums(p, mall, lall, split, orow, D);
}

// ------------------------------------------------------------------ attention of many rows
// Four waves of 32 query rows; the pages of the run come through an LDS ring of three by direct
// loads, each read once for 128 rows.  32 x 32 matrix instructions, which one wave a SIMD feeds at
// their rate; at D = 256 accumulators (128 registers) and queries (64) leave no room for a second one,
// below that two workgroups share a CU (D = 128: 8 x 50 tokens of 32 heads on 8 over 826 keys 30 -> 28 us,
// 1 x 776 tokens 32.6 -> 29.5).
//
// Lane L holds query row L % 32 and, of a 32-key S^T tile, the tile rows 8 a + 4 (L / 32) + r.  Tile
// t's row 8 a + 4 h + r is key 32 h + 16 t + 4 a + r, so that the lane holds keys 32 (L / 32) .. + 31,
// and eight consecutive of them are what it gives to one 16-deep step of P V: 32 bytes of a V row.
// LDS: 16-byte chunk c of key row k is kept at c ^ swizzle(k), and of a V row likewise, so that
// eight lanes that read one chunk of their rows meet eight different bank groups.
// 2 x 776 tokens of 8 heads on one over 4096 keys, D = 256: 97 us, 400 TFLOP/s where a large fp16 product
// reaches 1154.  Bound by a wave's own instructions: of the 5700 clocks of a page half are vector
// instructions (softmax, value codes to fp16), a quarter MFMAs, a fifth waits, one after the other.  The
// next page's scores issued beside the softmax (107 us) and values converted once for the four waves
// (109) gain nothing: the waves walk in step.
typedef int v16i __attribute__((ext_vector_type(16)));
typedef float v16f __attribute__((ext_vector_type(16)));

template <int D>
struct WideAttn {
  static constexpr int kWaves = 4, kRows = 32 * kWaves, kSlots = 3;
  static constexpr int kSide = kKvPage * D;                   // bytes of a page's keys (or values)
  static constexpr int kPieces = kSide / 1024 / kWaves;       // 1 KB pieces of a wave and side
  static constexpr int kLds = kSlots * 2 * kSide;
  static constexpr int kChunks = D / 16;                      // 16-byte chunks of a key row
  static constexpr int kPieceRows = 1024 / D;                 // key rows of a piece
  __device__ static int key_swizzle(int k) {
    return D >= 128 ? (k & 3) | ((k >> 5) & 1) << 2 : ((k >> 1) & 1) | ((k >> 5) & 1) << 1;
  }
  __device__ static int value_swizzle(int d) { return (d >> 1) & 3; }
};

template <typename T, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void kv_attn_wide_kernel(KvAttnParams p) {
  using C = WideAttn<D>;
  constexpr int F = D / 32;  // 32-deep steps of Q K^T, and 32-row tiles of O^T
  extern __shared__ __align__(1024) char lds[];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5, col = lane & 31;
  const int group = p.h / p.c.kvh;
  const int rows = p.t * group;
  const int tiles = (rows + C::kRows - 1) / C::kRows;
  const int tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
  const int head = blockIdx.y, b = blockIdx.z;
  const Span span(p, b);

  const int row = tile * C::kRows + wave * 32 + col;
  const int tok = min(row / group, p.t - 1), qh = head * group + row % group;
  const int64_t seen = row < rows ? span.seen(row / group) : 0;
  // The pages of the workgroup's rows, and those of this wave's.
  const int first = tile * C::kRows, last = min(first + C::kRows - 1, rows - 1);
  const int wfirst = first + wave * 32, wlast = min(wfirst + 31, rows - 1);
  const int64_t least = wfirst + 31 < rows ? span.least(wfirst / group, wlast / group) : 0;
  const int64_t wmost = wfirst < rows ? span.most(wfirst / group, wlast / group) : 0;
  const int pages = static_cast<int>((span.most(first / group, last / group) + kKvPage - 1) / kKvPage);
  const int per = (pages + p.nsplit - 1) / p.nsplit;
  const int begin = __builtin_amdgcn_readfirstlane(split * per);
  const int end = __builtin_amdgcn_readfirstlane(min(begin + per, pages));

  float sq;
  v4i qhi[F], qlo[F];
  const T* const qrow = static_cast<const T*>(p.q) + b * p.q_stride[0] + tok * p.q_stride[1] + qh * p.q_stride[2];
  load_query<T, D, 32>(qrow, sq, qhi, qlo, h);
  const float qfac = sq * p.scaling * kLog2e;

  // Loader: the wave's pieces of either side (a piece of values is 16 rows of 64 bytes).
  uint32_t ko[C::kPieces], vo[C::kPieces];
#pragma unroll
  for (int j = 0; j < C::kPieces; ++j) {
    const int pc = wave * C::kPieces + j;
    const int key = pc * C::kPieceRows + lane / C::kChunks;
    ko[j] = static_cast<uint32_t>(key * D + ((lane % C::kChunks) ^ C::key_swizzle(key)) * 16);
    const int d = pc * 16 + (lane >> 2);
    vo[j] = static_cast<uint32_t>(d * kKvPage + ((lane & 3) ^ C::value_swizzle(d)) * 16);
  }
  const int32_t* const table = p.c.table + b * p.c.table_stride;
  auto place = [&](int page) {  // entries that name no page are read as page 0
    const int id = __builtin_amdgcn_readfirstlane(page);
    return static_cast<int64_t>(id >= 0 && id < p.c.pages ? id : 0) * p.c.kvh + head;
  };
  auto request = [&](int page, int slot) {
    const int64_t ph = place(page);
    const char* const kb = reinterpret_cast<const char*>(p.c.k) + ph * C::kSide;
    const char* const vb = reinterpret_cast<const char*>(p.c.v) + ph * C::kSide;
    const uint32_t dst = lds0 + slot * 2 * C::kSide + wave * C::kPieces * 1024;
#pragma unroll
    for (int j = 0; j < C::kPieces; ++j) load_lds_1k(kb, ko[j], dst + j * 1024);
#pragma unroll
    for (int j = 0; j < C::kPieces; ++j) load_lds_1k(vb, vo[j], dst + C::kSide + j * 1024);
  };

  float m = kNone, l = 0.0f;
  v16f o[F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.0f;

  // This lane's key of the first tile (row col of it), and its reads' offsets.
  const int key = 32 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3);  // + 16 for the second: the same swizzle
  const int kswz = C::key_swizzle(key), vswz = C::value_swizzle(col);

  // Table entries two pages ahead of their use.
  auto entry = [&](int pg) { return pg < end ? scalar_load(table + pg) : -1; };
  int page = entry(begin), page1 = entry(begin + 1), page2 = entry(begin + 2);
  if (begin < end) request(page, 0);
  if (begin + 1 < end) request(page1, 1);
  int slot = 0;
  for (int pg = begin; pg < end; ++pg) {
    const int64_t ph = place(page);
    const float ks = scalar_load(p.c.ks + ph);
    float vs = scalar_load(p.c.vs + ph);
    if (vs == 0.0f) vs = 1e-20f;  // zeros, whatever the codes: the page still counts in the sum
    const int page3 = entry(pg + 3);
    // Younger than this page's loads: the next page's.
    if (pg + 1 < end) wait_vm<2 * C::kPieces>();
    else wait_vm<0>();
    lds_done_barrier();  // every wave's pieces are there, and the slot of the page before is free
    if (pg + 2 < end) request(page2, slot == 0 ? 2 : slot - 1);
    const char* const kst = lds + slot * 2 * C::kSide;
    const char* const vst = kst + C::kSide;
    const int64_t key0 = static_cast<int64_t>(pg) * kKvPage;
    if (page >= 0 && page < p.c.pages && key0 < wmost) {  // uniform over the wave
      const float fac = qfac * ks, lvs = __builtin_log2f(vs);
      v4i kf[2][F];
      auto read_keys = [&](int t) {
#pragma unroll
        for (int f = 0; f < F; ++f)
          kf[t][f] = *reinterpret_cast<const v4i*>(kst + (key + 16 * t) * D + (((2 * f + h) ^ kswz) * 16));
      };
      read_keys(0);
      float s[2][16];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (t == 0) read_keys(1);
        __builtin_amdgcn_sched_barrier(0);
        v16i ah, al;
#pragma unroll
        for (int r = 0; r < 16; ++r) ah[r] = al[r] = 0;
#pragma unroll
        for (int f = 0; f < F; ++f) {
          ah = __builtin_amdgcn_mfma_i32_32x32x32_i8(kf[t][f], qhi[f], ah, 0, 0, 0);
          al = __builtin_amdgcn_mfma_i32_32x32x32_i8(kf[t][f], qlo[f], al, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = fmaf(static_cast<float>(256 * ah[r] + al[r]), fac, lvs);
      }
      // The values' first reads pass under the softmax.
      v4i vf[F][2];
      auto read_values = [&](int i) {
        const char* const vrow = vst + (32 * i + col) * kKvPage;  // 32 i: the same swizzle
        vf[i][0] = *reinterpret_cast<const v4i*>(vrow + (((2 * h) ^ vswz) * 16));
        vf[i][1] = *reinterpret_cast<const v4i*>(vrow + (((2 * h + 1) ^ vswz) * 16));
      };
      read_values(0);
      read_values(1);
      if (key0 + kKvPage > least) {  // some row does not see the whole page
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (key0 + 32 * h + 16 * t + r >= seen) s[t][r] = -__builtin_inff();
      }
      float top = s[0][0];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[t][r]);
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__any(top > m + kTop)) {
        const float m1 = fmaxf(m, top - kLift);
        const float alpha = __builtin_amdgcn_exp2f(m - m1);
        m = m1;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < F; ++i) o[i] *= alpha;
      }
      float sum = 0.0f;
      half8 w[4];  // 16-deep steps of P V: keys 32 h + 8 step .. + 7
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = __builtin_amdgcn_exp2f(s[t][r] - m);
          sum += e;
          w[2 * t + (r >> 3)][r & 7] = static_cast<_Float16>(e);
        }
      l += sum != 0.0f ? sum / vs : 0.0f;
#pragma unroll
      for (int i = 0; i < F; ++i) {
        if (i + 2 < F) read_values(i + 2);
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_to_half(vf[i][0][0], vf[i][0][1]), w[0], o[i], 0, 0, 0);
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_to_half(vf[i][0][2], vf[i][0][3]), w[1], o[i], 0, 0, 0);
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_to_half(vf[i][1][0], vf[i][1][1]), w[2], o[i], 0, 0, 0);
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_to_half(vf[i][1][2], vf[i][1][3]), w[3], o[i], 0, 0, 0);
      }
    }
    slot = slot == 2 ? 0 : slot + 1;
    page = page1;
    page1 = page2;
    page2 = page3;
  }
  wait_vm<0>();
  l += __shfl_xor(l, 32, 64);
  if (row >= rows) return;
  const int64_t orow = (static_cast<int64_t>(b) * p.t + tok) * p.h + qh;
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;  // 0: no visible key (NaN stays NaN)
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      store_quad<T>(p, v4f{o[i][4 * a], o[i][4 * a + 1], o[i][4 * a + 2], o[i][4 * a + 3]}, inv, split, orow, D, 32 * i + 8 * a + 4 * h);
  if (h == 0) store_sums(p, m, l, split, orow, D);
}

// Joins the runs of a row, at most 64 of them: one wave a row, lane s with the maximum and sum of run s.
constexpr int kMaxRuns = 64;

// The first kAhead runs' parts are under way before their maxima meet (13 runs of 8 rows with 4 / 16 ahead
// 5.2 / 3.2 us; 2 runs of 12416 rows, where the registers cost waves, 8.0 / 9.1).
template <typename T, int D, int kAhead>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(KvAttnParams p) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t rows = static_cast<int64_t>(p.b) * p.t * p.h;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int64_t plane = split_floats(rows, D);
  struct alignas(4 * E) Vec { float v[E]; };
  struct alignas(2 * E) Out { T v[E]; };
  const float* const src = p.ws + row * D + lane * E;
  Vec x[kAhead];
#pragma unroll
  for (int s = 0; s < kAhead; ++s)
    if (s < p.nsplit) x[s] = *reinterpret_cast<const Vec*>(src + s * plane);
  float ms = kNone, ls = 0.0f;
  if (lane < p.nsplit) {
    const float2 ml = *reinterpret_cast<const float2*>(p.ws + lane * plane + rows * D + row * 2);
    ms = ml.x;
    ls = ml.y;
  }
  float m = ms;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float a = __builtin_amdgcn_exp2f(ms - m);
  float l = ls * a;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
  Vec sum{};
  auto add = [&](const Vec& part, int s) {
    const float as = __shfl(a, s, 64);
#pragma unroll
    for (int e = 0; e < E; ++e) sum.v[e] += part.v[e] * as;
  };
#pragma unroll
  for (int s = 0; s < kAhead; ++s)
    if (s < p.nsplit) add(x[s], s);
#pragma unroll 8
  for (int s = kAhead; s < p.nsplit; ++s) add(*reinterpret_cast<const Vec*>(src + s * plane), s);
  const bool empty = l == 0.0f;  // no visible key
  const float inv = 1.0f / l;
  Out y;
#pragma unroll
  for (int e = 0; e < E; ++e) y.v[e] = static_cast<T>(empty ? 0.0f : sum.v[e] * inv);
  *reinterpret_cast<Out*>(static_cast<T*>(p.out) + row * D + lane * E) = y;
  if (p.lse != nullptr && lane == 0) p.lse[row] = empty ? -__builtin_inff() : m / kLog2e + __builtin_logf(l);
}

template <typename T, int D>
void launch_append(const KvAppendParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.t + 62) / kKvPage + 1), static_cast<unsigned>(2 * p.c.kvh), static_cast<unsigned>(p.b));
  kv_append_kernel<T, D><<<grid, 256, 0, stream>>>(p);
}

template <typename T, int D>
void launch_attn(const KvAttnParams& p, hipStream_t stream) {
  const int rows = p.t * (p.h / p.c.kvh);
  const int tile = p.wide ? WideAttn<D>::kRows : 16;
  const dim3 grid(static_cast<unsigned>((rows + tile - 1) / tile * p.nsplit), static_cast<unsigned>(p.c.kvh), static_cast<unsigned>(p.b));
  if (p.wide) {
    kv_attn_wide_kernel<T, D><<<grid, 256, WideAttn<D>::kLds, stream>>>(p);
  } else {
    // Four waves from six pages of a run on, two from two pages on (D = 256, us with 8 / 4 / 2 / 1 waves: 13
    // pages 20.5 / 18.3 / 18.9 / 27.2, 4 pages 15.7 / 15.3 / 15.2 / 16.6, 1 page - / - / 10.5 / 9.9; D = 128, 32
    // pages 18.7 / 17.8 / 24.6 / 42).
    const int run = (p.c.table_pages + p.nsplit - 1) / p.nsplit;
    if (run >= 6) kv_attn_kernel<T, D, 4><<<grid, 64 * 4, 4 * D * 64, stream>>>(p);
    else if (run >= 2) kv_attn_kernel<T, D, 2><<<grid, 64 * 2, 2 * D * 64, stream>>>(p);
    else kv_attn_kernel<T, D, 1><<<grid, 64, 0, stream>>>(p);
  }
  if (p.nsplit > 1) {
    const int64_t all = static_cast<int64_t>(p.b) * p.t * p.h;
    const dim3 joins(static_cast<unsigned>((all + 3) / 4));
    if (p.nsplit <= 4) kv_attn_join_kernel<T, D, 4><<<joins, 256, 0, stream>>>(p);
    else kv_attn_join_kernel<T, D, 16><<<joins, 256, 0, stream>>>(p);
  }
}

}  // namespace

hipError_t launch_kv_append(const KvAppendParams& p, int elem, hipStream_t stream) {
  if (p.b <= 0 || p.t <= 0) return hipSuccess;
#define APPEND(T)                                                         \
  switch (p.c.d) {                                                        \
    case 64: launch_append<T, 64>(p, stream); break;                      \
    case 128: launch_append<T, 128>(p, stream); break;                    \
    default: launch_append<T, 256>(p, stream); break;                     \
  }
  if (elem == kFp16) {
    APPEND(_Float16)
  } else {
    APPEND(__bf16)
  }
#undef APPEND
  return hipGetLastError();
}

// No call asks for more partial results than the Infinity Cache holds.
constexpr size_t kMaxPartial = size_t{1} << 28;

// The kernel and its runs of pages: the least of the times (us, beside a launch) that these measurements
// give: for each round of the CUs the pages of a run, and the start of a workgroup where it does not run
// beside another (the wide kernel at D <= 128: two on a CU); for more than one run the join, partial
// results at 10 TB/s.
// Narrow, D = 256, 16 rows over 8192 keys in 1 / 2 / 3 / 4 / 8 runs: 64 sequences 104 / 65 / 54 / 54 / 57,
// 96 121 / 77 / 104 / 87 / 83, 150 130 / 150 / 120 / 130 / 129, 300 290 / 245 / 238 / 234 / 249.  Wide, D = 128, 2 x 6208
// rows over 4096 keys in 1 / 2 / 3 / 5 / 8 runs: 109 / 69 / 69 / 54 / 63.
// Narrow / wide: D = 256, 8 x 400 rows over 826 keys 18 / 28, 1 x 2400 over 4096 52 / 38, 32 x 400 over
// 826 71 / 44; D = 128, 16 x 200 over 2000 18 / 23, 64 x 200 over 826 41 / 28; D = 64, 2 x 6208 over 4096
// 37 / 42, 32 x 1600 over 826 42 / 30.
KvAttnPlan kv_attn_plan(int64_t b, int64_t t, int32_t h, int32_t kvh, int32_t d, int64_t table_pages, int cus) {
  KvAttnPlan plan{false, 1};
  const int64_t rows = t * (h / kvh);
  if (rows <= 0 || b <= 0 || table_pages <= 0) return plan;
  struct Cost {
    double start, page;
  };
  const Cost narrow = d == 64 ? Cost{2.5, 0.12} : d == 128 ? Cost{8, 0.3} : Cost{10, 0.62};
  const Cost wide = d == 64 ? Cost{4, 1.3} : d == 128 ? Cost{6, 1.65} : Cost{10, 2.9};
  const double partial = static_cast<double>(rows) * b * kvh * d * 8 / 1e7;  // of a run, written and read
  const int64_t few = (rows + 15) / 16 * b * kvh, many = (rows + 127) / 128 * b * kvh;
  double best = 1e300;
  auto consider = [&](bool is_wide, const Cost& c, int64_t groups, int n, int beside) {
    const int64_t rounds = (groups * n + cus - 1) / cus;
    const double us = static_cast<double>((rounds + beside - 1) / beside) * c.start +
                      static_cast<double>(rounds * ((table_pages + n - 1) / n)) * c.page + (n > 1 ? 4 + partial * n : 0);
    if (us < best) {
      best = us;
      plan = {is_wide, n};
    }
  };
  for (int n = 1; n <= kMaxRuns && n <= table_pages; ++n) {
    if (n > 1 && kv_attn_workspace(b, t, h, d, n) > kMaxPartial) break;
    consider(false, narrow, few, n, 1);
    if (n == 1 || 2 * (n - 1) < table_pages) consider(true, wide, many, n, d == 256 ? 1 : 2);  // two pages at least
  }
  return plan;
}

size_t kv_attn_workspace(int64_t b, int64_t t, int32_t h, int32_t d, int nsplit) {
  return nsplit > 1 ? sizeof(float) * static_cast<size_t>(nsplit) * static_cast<size_t>(split_floats(b * t * h, d)) : 0;
}

hipError_t launch_kv_attention(const KvAttnParams& p, int elem, hipStream_t stream) {
  if (p.b <= 0 || p.t <= 0) return hipSuccess;
#define ATTEND(T)                                                       \
  switch (p.c.d) {                                                      \
    case 64: launch_attn<T, 64>(p, stream); break;                      \
    case 128: launch_attn<T, 128>(p, stream); break;                    \
    default: launch_attn<T, 256>(p, stream); break;                     \
  }
  if (elem == kFp16) {
    ATTEND(_Float16)
  } else {
    ATTEND(__bf16)
  }
#undef ATTEND
  return hipGetLastError();
}

}  // namespace w4a4
