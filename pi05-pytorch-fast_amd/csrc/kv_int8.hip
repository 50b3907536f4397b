// An 8-bit KV cache of 64-token pages with one scale for each page and KV head (keys and values
// have their own), the append that writes it and the attention that reads it.
//
// Layout: K codes [pages, KVH, 64, D]; V codes transposed within the page, [pages, KVH, D, 64].  The
// attention computes S^T = K Q^T and O^T = V^T P^T on 16-row matrix instructions whose operands
// are 16-byte loads of consecutive codes of either array: no transposes, no LDS for the cache.

#include "int8_internal.h"
#include "quant_row.h"

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
// token, so that nothing of the page's earlier owner is left.  Bound by latency for single
// tokens (lens -> table -> scale, one after the other) and by HBM for prefixes.
template <typename T, int D>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendParams p) {
  constexpr int kChunks = kKvPage * D / 8 / 256;  // 8-element chunks of a thread
  constexpr int kRowChunks = D / 8;
  constexpr int kStride = kKvPage + 4;            // staged V row (one d), bytes
  __shared__ uint32_t red[4];
  __shared__ __align__(16) char vt[D * kStride];
  const int tid = threadIdx.x;
  const int b = blockIdx.z;
  const int head = blockIdx.y >> 1;
  const bool is_v = (blockIdx.y & 1) != 0;
  const int64_t len = max(p.c.lens[b], 0);
  const int64_t count = min(max(p.counts != nullptr ? p.counts[b] : p.t, 0), p.t);
  const int64_t slot = len / kKvPage + blockIdx.x;
  const int64_t first = max(len - slot * kKvPage, static_cast<int64_t>(0));  // new tokens: page rows first .. last - 1
  const int64_t last = min(len + count - slot * kKvPage, static_cast<int64_t>(kKvPage));
  if (last <= first || slot >= p.c.table_pages) return;
  const int page = p.c.table[b * p.c.table_stride + slot];
  if (page < 0 || page >= p.c.pages) return;
  const int64_t ph = static_cast<int64_t>(page) * p.c.kvh + head;
  const int64_t* const st = is_v ? p.v_stride : p.k_stride;
  const T* const src = static_cast<const T*>(is_v ? p.v : p.k) + b * st[0] + head * st[2];
  const int64_t tok0 = slot * kKvPage - len;  // token of page row 0

  vec8<T> x[kChunks];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int c = j * 256 + tid, row = c / kRowChunks;
    x[j] = vec8<T>{};
    if (row >= first && row < last) x[j] = *reinterpret_cast<const vec8<T>*>(src + (tok0 + row) * st[1] + (c % kRowChunks) * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(static_cast<float>(x[j][e])) & 0x7fffffffu);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o, 64)));
  if ((tid & 63) == 0) red[tid >> 6] = top;
  float* const scale = (is_v ? p.c.vs : p.c.ks) + ph;
  const float s0 = first > 0 ? *scale : 0.0f;
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

  uint32_t code[kChunks][2];
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
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
  if (!is_v) {
    char* const dst = reinterpret_cast<char*>(p.c.k) + ph * (kKvPage * D);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const int c = j * 256 + tid, row = c / kRowChunks;
      uint2* const d = reinterpret_cast<uint2*>(dst + c * 8);
      if (row >= first && row < last)
        *d = uint2{code[j][0], code[j][1]};
      else if (first == 0)
        *d = uint2{0u, 0u};
      else if (grow) {
        const uint2 o = *d;
        *d = uint2{rescaled(o.x), rescaled(o.y)};
      }
    }
    return;
  }
  // V: the new codes are turned in LDS; each thread then owns 16 tokens of one d at a time.
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int c = j * 256 + tid, row = c / kRowChunks, d0 = (c % kRowChunks) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) vt[(d0 + e) * kStride + row] = static_cast<char>(code[j][e >> 2] >> (8 * (e & 3)));
  }
  __syncthreads();
  char* const dst = reinterpret_cast<char*>(p.c.v) + ph * (kKvPage * D);
  for (int i = tid; i < D * (kKvPage / 4); i += 256) {
    const int d = i / (kKvPage / 4), t0 = (i % (kKvPage / 4)) * 4;
    if (!grow && (t0 + 4 <= first || t0 >= last)) continue;
    uint32_t* const o = reinterpret_cast<uint32_t*>(dst + d * kKvPage + t0);
    const uint32_t fresh = *reinterpret_cast<const uint32_t*>(vt + d * kStride + t0);
    uint32_t old = 0;
    if (first > 0 && (t0 < first || t0 + 4 > last)) old = grow ? rescaled(*o) : *o;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t m = 0xffu << (8 * e);
      w |= (t0 + e >= first && t0 + e < last ? fresh : old) & m;
    }
    *o = w;
  }
}

// ------------------------------------------------------------------ attention
// A workgroup holds 16 query rows of one KV head (row = token * (H / KVH) + query head) and a run
// of the sequence's pages; its four waves take every fourth page of the run, each with a softmax
// of its own (running maximum and sum), and meet in LDS at the end.
//
// Q K^T in int8: a query row is held as 16-bit integers v = rint(q / sq), |v| <= 32512, split
// v = 256 hi + lo into two int8 operands, so that S = sq ks (256 K hi + K lo) is exact but for
// the rounding of q, 2^-16 of the row's maximum: finer than fp16 there, and no conversion of K.
// P V in fp16: the codes are exact in fp16.  The page's V scale is folded into the exponent,
// w = 2^(S log2e + log2 vs - m) with m the running maximum of that sum, so that the weights of
// all pages share one accumulator and stay at most 1; the sum of the probabilities is that of
// w / vs.  Sums, maxima and accumulators are fp32; w is rounded to fp16 (2^-11) for the product.
//
// Lane L of a 16 x 16 S^T tile holds row L % 16 and four consecutive tile rows 4 (L / 16) ..  Tile
// t's row 4 a + r is key 16 a + 4 t + r, so that over the four tiles of a page the lane holds
// keys 16 (L / 16) .. + 15: the 16 bytes that it loads of a V row.
template <typename T, int D>
__device__ __forceinline__ void load_query(const T* row, float& sq, v4i (&hi)[D / 64], v4i (&lo)[D / 64], int g) {
  float f[D / 64][16];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const vec8<T> v = *reinterpret_cast<const vec8<T>*>(row + 64 * i + 16 * g + 8 * h);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[i][8 * h + e] = static_cast<float>(v[e]);
        top = max(top, __float_as_uint(f[i][8 * h + e]) & 0x7fffffffu);
      }
    }
  }
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
  const float amax = __uint_as_float(top);
  const bool finite = amax <= 3.4028235e38f;
  sq = finite ? amax / 32512.0f : __builtin_nanf("");
  const float inv = finite && amax >= 1e-30f ? 32512.0f / amax : 0.0f;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t ph = 0, pl = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = finite ? static_cast<int>(__builtin_rintf(f[i][4 * w + e] * inv)) : 0;
        const int h = (v + 128) >> 8;
        ph |= static_cast<uint32_t>(h & 0xff) << (8 * e);
        pl |= static_cast<uint32_t>((v - 256 * h) & 0xff) << (8 * e);
      }
      hi[i][w] = static_cast<int>(ph);
      lo[i][w] = static_cast<int>(pl);
    }
  }
}

// Four codes as fp16: byte + 128 under the exponent of 1024, less 1152.
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

constexpr float kNone = -1e30f;  // running maximum before the first visible key

// Partial results of a run: O (unnormalised, fp32), the maximum and the sum of each row.
__host__ __device__ inline int64_t split_floats(int64_t rows, int d) { return rows * (d + 2); }

template <typename T, int D>
__global__ __launch_bounds__(256) void kv_attn_kernel(KvAttnParams p) {
  constexpr int F = D / 64, DT = D / 16;
  __shared__ v4f obuf[3][DT * 64];
  __shared__ float mbuf[4][16], lbuf[4][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int group = p.h / p.c.kvh;
  const int rows = p.t * group;
  const int tiles = (rows + 15) >> 4;
  const int tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
  const int head = blockIdx.y, b = blockIdx.z;
  const int64_t cap = static_cast<int64_t>(p.c.table_pages) * kKvPage;
  const int64_t len = min(static_cast<int64_t>(max(p.c.lens[b], 0)), cap);
  const int64_t q_len = min(max(p.q_lens != nullptr ? p.q_lens[b] : p.t, 0), p.t);

  // This lane's row; rows past the last one, and tokens past q_len, see nothing.
  const int row = tile * 16 + col;
  const int tok = min(row / group, p.t - 1), qh = head * group + row % group;
  auto visible = [&](int64_t token) {
    return token >= q_len ? static_cast<int64_t>(0) : p.causal ? max(len - q_len + token + 1, static_cast<int64_t>(0)) : len;
  };
  const int64_t seen = row < rows ? visible(row / group) : 0;
  // Keys that the tile's rows see: those of its last token (of none, if that is past q_len and
  // so are all the others').
  const int64_t tok_first = tile * 16 / group, tok_last = min(tile * 16 + 15, rows - 1) / group;
  const int64_t most = visible(min(tok_last, max(q_len - 1, tok_first)));
  const int64_t least = tile * 16 + 15 < rows && tok_last < q_len ? visible(tok_first) : 0;
  const int pages = static_cast<int>((most + kKvPage - 1) / kKvPage);
  const int per = (pages + p.nsplit - 1) / p.nsplit;
  const int begin = split * per, end = min(begin + per, pages);

  float sq;
  v4i qhi[F], qlo[F];
  const T* const qrow = static_cast<const T*>(p.q) + b * p.q_stride[0] + tok * p.q_stride[1] + qh * p.q_stride[2];
  load_query<T, D>(qrow, sq, qhi, qlo, g);
  const float qfac = sq * p.scaling * kLog2e;

  float m = kNone, l = 0.0f;
  v4f o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  const int32_t* const table = p.c.table + b * p.c.table_stride;
  for (int pg = begin + wave; pg < end; pg += 4) {
    const int page = table[pg];
    if (page < 0 || page >= p.c.pages) continue;  // no such page: its keys are not there
    const int64_t ph = static_cast<int64_t>(page) * p.c.kvh + head;
    const int8_t* const kp = p.c.k + ph * (kKvPage * D) + (16 * (col >> 2) + (col & 3)) * D + 16 * g;
    const int8_t* const vp = p.c.v + ph * (kKvPage * D) + col * kKvPage + 16 * g;
    const float ks = p.c.ks[ph];
    float vs = p.c.vs[ph];
    if (vs == 0.0f) vs = 1e-30f;  // zeros, whatever the codes: the page still counts in the sum
    v4i kc[4][F], vc[DT];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int f = 0; f < F; ++f) kc[t][f] = *reinterpret_cast<const v4i*>(kp + 4 * t * D + 64 * f);
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
      for (int r = 0; r < 4; ++r) s[t][r] = static_cast<float>(256 * ah[r] + al[r]) * fac + lvs;
    }
    const int64_t key0 = static_cast<int64_t>(pg) * kKvPage;
    if (key0 + kKvPage > least) {  // some row does not see the whole page
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + 16 * g + 4 * t + r >= seen) s[t][r] = -__builtin_inff();
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[t][r]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float m1 = fmaxf(m, top);
    const float alpha = __builtin_amdgcn_exp2f(m - m1);
    m = m1;
    float sum = 0.0f;
    half8 w[2];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f(s[t][r] - m1);
        sum += e;
        w[t >> 1][4 * (t & 1) + r] = static_cast<_Float16>(e);
      }
    // A row that sees nothing of the page takes nothing from its scale either (it may be NaN).
    l = l * alpha + (sum != 0.0f ? sum / vs : 0.0f);
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      o[i] *= alpha;
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_half(vc[i][0], vc[i][1]), w[0], o[i], 0, 0, 0);
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_half(vc[i][2], vc[i][3]), w[1], o[i], 0, 0, 0);
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // The four waves' parts: a common maximum, then the sums of the scaled parts.
  if (g == 0) {
    mbuf[wave][col] = m;
    lbuf[wave][col] = l;
  }
  __syncthreads();
  const float mall = fmaxf(fmaxf(mbuf[0][col], mbuf[1][col]), fmaxf(mbuf[2][col], mbuf[3][col]));
  const float mine = __builtin_amdgcn_exp2f(m - mall);
#pragma unroll
  for (int i = 0; i < DT; ++i) {
    o[i] *= mine;
    if (wave > 0) obuf[wave - 1][i * 64 + lane] = o[i];
  }
  __syncthreads();
  if (wave != 0) return;
  float lall = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) lall += lbuf[w][col] * __builtin_amdgcn_exp2f(mbuf[w][col] - mall);
  const int64_t all_rows = static_cast<int64_t>(p.b) * p.t * p.h;
  const int64_t orow = (static_cast<int64_t>(b) * p.t + tok) * p.h + qh;
  const float inv = lall != 0.0f ? 1.0f / lall : 0.0f;
  const bool empty = lall == 0.0f;  // no visible key (false for NaN)
  if (row >= rows) return;
#pragma unroll
  for (int i = 0; i < DT; ++i) {
    v4f v = o[i];
#pragma unroll
    for (int w = 0; w < 3; ++w) v += obuf[w][i * 64 + lane];
    if (p.nsplit > 1) {
      *reinterpret_cast<v4f*>(p.ws + split * split_floats(all_rows, D) + orow * D + 16 * i + 4 * g) = v;
    } else {
      typedef T tv4 __attribute__((ext_vector_type(4)));
      tv4 y;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = static_cast<T>(empty ? 0.0f : v[r] * inv);
      *reinterpret_cast<tv4*>(static_cast<T*>(p.out) + orow * D + 16 * i + 4 * g) = y;
    }
  }
  if (g == 0) {
    if (p.nsplit > 1) {
      float* const ml = p.ws + split * split_floats(all_rows, D) + all_rows * D + orow * 2;
      ml[0] = mall;
      ml[1] = lall;
    } else if (p.lse != nullptr) {
      p.lse[orow] = empty ? -__builtin_inff() : mall / kLog2e + __builtin_logf(lall);
    }
  }
}

// Joins the runs of a row: one wave a row.
template <typename T, int D>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(KvAttnParams p) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t rows = static_cast<int64_t>(p.b) * p.t * p.h;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int64_t plane = split_floats(rows, D);
  float m = kNone, l = 0.0f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
  for (int s = 0; s < p.nsplit; ++s) m = fmaxf(m, p.ws[s * plane + rows * D + row * 2]);
  for (int s = 0; s < p.nsplit; ++s) {
    const float* const ml = p.ws + s * plane + rows * D + row * 2;
    const float a = __builtin_amdgcn_exp2f(ml[0] - m);
    l += ml[1] * a;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += p.ws[s * plane + row * D + e * 64 + lane] * a;
  }
  const bool empty = l == 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) static_cast<T*>(p.out)[row * D + e * 64 + lane] = static_cast<T>(empty ? 0.0f : o[e] / l);
  if (p.lse != nullptr && lane == 0) p.lse[row] = empty ? -__builtin_inff() : m / kLog2e + __builtin_logf(l);
}

template <typename T, int D>
void launch_append(const KvAppendParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.t + 62) / kKvPage + 1), static_cast<unsigned>(2 * p.c.kvh), static_cast<unsigned>(p.b));
  kv_append_kernel<T, D><<<grid, 256, 0, stream>>>(p);
}

template <typename T, int D>
void launch_attn(const KvAttnParams& p, hipStream_t stream) {
  const int tiles = (p.t * (p.h / p.c.kvh) + 15) / 16;
  const dim3 grid(static_cast<unsigned>(tiles * p.nsplit), static_cast<unsigned>(p.c.kvh), static_cast<unsigned>(p.b));
  kv_attn_kernel<T, D><<<grid, 256, 0, stream>>>(p);
  if (p.nsplit > 1) {
    const int64_t rows = static_cast<int64_t>(p.b) * p.t * p.h;
    kv_attn_join_kernel<T, D><<<dim3(static_cast<unsigned>((rows + 3) / 4)), 256, 0, stream>>>(p);
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

// Runs of pages for each (sequence, KV head, 16-row tile): enough workgroups for two a CU, a run
// being at least four pages long (one for each wave).
int kv_attn_splits(int64_t b, int64_t t, int32_t h, int32_t kvh, int32_t d, int64_t table_pages, int cus) {
  (void)d;
  const int64_t tiles = (t * (h / kvh) + 15) / 16 * b * kvh;
  if (tiles <= 0) return 1;
  int64_t n = (2 * cus + tiles - 1) / tiles;
  n = n < (table_pages + 3) / 4 ? n : (table_pages + 3) / 4;
  return static_cast<int>(n < 1 ? 1 : n > 64 ? 64 : n);
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
