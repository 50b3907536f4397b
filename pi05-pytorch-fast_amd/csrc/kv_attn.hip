// Attention over a 16-bit paged KV cache: decoded tokens, and few tokens a sequence.
//
// A workgroup takes 16 query rows of one KV head (row = token * (H / KVH) + query head) and a run of the
// sequence's pages; its W waves take every W-th half page (32 keys), each with a softmax of its own
// (reference and sum), and meet in LDS at the end.  Runs are joined by a second launch.
//
// S^T = K Q^T and O^T = V^T P^T on 16 x 16 x 32 matrix instructions.  Row i of the key tile t is
// key 8 (i / 4) + 4 t + i % 4 of the half page, so that a lane's results, rows 4 (L / 16) + r of the
// two tiles, are the eight consecutive keys that it gives to P V.  Values are loaded as they lie, eight keys
// of VE consecutive dimensions a lane, and turned in registers (two byte permutes for four elements);
// tile e of a chunk of 16 VE dimensions then holds dimensions VE i + e, and a lane ends with 4 VE
// consecutive ones.
//
// Weights are rounded to 16 bits as a sum of two parts, w = hi + lo, each with its own product: the
// matrix pipe has the time (the cache's bytes bound), and the result is that of fp32 weights to 2^-16 (bf16,
// whose 8 bits alone would cost as much as the rounding of the output) or 2^-21 (fp16).

#include <algorithm>

#include "serving_internal.h"

namespace w4a4 {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kHalf = 32;  // keys of a step

__device__ __forceinline__ v4f mfma(const vec8<_Float16> a, const vec8<_Float16> b, const v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma(const vec8<__bf16> a, const vec8<__bf16> b, const v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The reference of a row's exponents is kLift below the largest one when it is set, and is set again only
// when an exponent is kTop above it.  fp16: the largest weight is between 2^7 and 2^15, at the upper end of
// the type, so that small weights beside a large one keep their bits; bf16 has fp32's range.
constexpr float kLift = 7.0f, kTop = 15.0f;

// A load at a uniform address that nothing in the kernel writes: through the scalar cache, so that
// no wait for vector loads stands before its use.
template <typename U>
__device__ __forceinline__ U scalar_load(const U* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) U*>(reinterpret_cast<uintptr_t>(p));
}

// Partial results of a run: O (unnormalised, fp32), the reference and the sum of each row; whole 16 bytes.
__host__ __device__ inline int64_t split_floats(int64_t rows, int d) { return (rows * (d + 2) + 3) & ~int64_t{3}; }

// What the rows of a sequence see.
struct Span {
  int64_t q_len, len;
  int causal;
  __device__ __forceinline__ Span(const KvAttn16Params& p, int b) {
    const int64_t cap = static_cast<int64_t>(p.c.table_pages) * kKvPage;
    len = p.c.pages > 0 ? min(static_cast<int64_t>(max(scalar_load(p.c.lens + b), 0)), cap) : 0;
    q_len = min(max(p.q_lens != nullptr ? scalar_load(p.q_lens + b) : p.t, 0), p.t);
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

// The four consecutive columns from c of a row: its output, or its part of a run's partial results.
template <typename T>
__device__ __forceinline__ void store_quad(const KvAttn16Params& p, const v4f v, float inv, int split, int64_t orow, int d, int c) {
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
__device__ __forceinline__ void store_sums(const KvAttn16Params& p, float m, float l, int split, int64_t orow, int d) {
  if (p.nsplit > 1) {
    const int64_t all_rows = static_cast<int64_t>(p.b) * p.t * p.h;
    float* const ml = p.ws + split * split_floats(all_rows, d) + all_rows * d + orow * 2;
    ml[0] = m;
    ml[1] = l;
  } else if (p.lse != nullptr) {
    p.lse[orow] = l == 0.0f ? -__builtin_inff() : m / kLog2e + __builtin_logf(l);
  }
}

// exp2(m - to), 0 for a part without a key (m = -inf).
__device__ __forceinline__ float weight_of(float m, float to) {
  return m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - to);
}

// Two elements of a word: whether one is NaN or infinite, and the word with zeros in such places.
template <typename T>
constexpr uint32_t kExponent = static_cast<float>(static_cast<T>(65536.0f)) > 1e30f ? 0x7c00u : 0x7f80u;  // fp16, bf16
template <typename T>
__device__ __forceinline__ bool any_nonfinite(uint32_t w) {
  constexpr uint32_t kLow = kExponent<T>, kHigh = kLow << 16;
  return (w & kLow) == kLow || (w & kHigh) == kHigh;
}
template <typename T>
__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  constexpr uint32_t kLow = kExponent<T>, kHigh = kLow << 16;
  return ((w & kLow) == kLow ? 0u : w & 0xffffu) | ((w & kHigh) == kHigh ? 0u : w & 0xffff0000u);
}

// MIXED: rows of a tile may be of several tokens, which see different keys.
template <typename T, int D, int W, bool MIXED>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void kv_attn16_kernel(KvAttn16Params p) {
  constexpr int F = D / 32, DT = D / 16;
  constexpr int VE = D >= 128 ? 8 : 4, CH = D / (16 * VE), VW = VE / 2;  // a value chunk: elements, chunks, words
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

  // This lane's row; tokens past q_len see nothing.
  const int row = tile * 16 + col;
  const int tok = min(row / group, p.t - 1), qh = head * group + row % group;
  const int64_t seen = row < rows ? span.seen(row / group) : 0;
  const int64_t tok_first = tile * 16 / group, tok_last = min(tile * 16 + 15, rows - 1) / group;
  const int64_t most = span.most(tok_first, tok_last);
  const int64_t least = span.least(tok_first, tok_last);  // rows past the last one are computed as they come, and not stored
  const int pages = static_cast<int>((most + kKvPage - 1) / kKvPage);
  // The run's pages are split, split + nsplit, ..: the first is known without the length.  Its steps are
  // the halves of 32 keys; a last half that no row sees is left out.
  const int mine = pages > split ? (pages - split - 1) / p.nsplit + 1 : 0;
  const bool half = mine > 0 && split + (mine - 1) * p.nsplit == pages - 1 && most <= static_cast<int64_t>(pages) * kKvPage - kHalf;
  const int end = 2 * mine - (half ? 1 : 0);

  vec8<T> q[F];
  const T* const qrow = static_cast<const T*>(p.q) + b * p.q_stride[0] + tok * p.q_stride[1] + qh * p.q_stride[2];
#pragma unroll
  for (int f = 0; f < F; ++f) q[f] = *reinterpret_cast<const vec8<T>*>(qrow + 32 * f + 8 * g);
  const float qfac = p.scaling * kLog2e;

  float m = -__builtin_inff(), l = 0.0f;
  v4f o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  // Entries that name no page are read as page 0, whose keys then count as not there.
  const int32_t* const table = p.c.table + b * p.c.table_stride;
  auto page_of = [&](int step) { return __builtin_amdgcn_readfirstlane(split + (step >> 1) * p.nsplit); };
  auto page_at = [&](int step) { return page_of(step) < p.c.table_pages ? scalar_load(table + page_of(step)) : -1; };
  auto place = [&](int page, int step) {  // first element of the step's keys
    const int64_t id = __builtin_amdgcn_readfirstlane(page >= 0 && page < p.c.pages ? page : 0);
    return ((id * p.c.kvh + head) * kKvPage + (step & 1) * kHalf) * D;
  };
  // Four neighbouring lanes load 64 consecutive bytes of a key (16 lanes 16 keys, as the operand has them, are 16
  // bytes of as many lines: a quarter of the rate); the fragment's chunk is lane 4 row + chunk's.
  const int kr = lane >> 2, from = (4 * col + g) * 4;
  const int koff = (8 * (kr >> 2) + (kr & 3)) * D + 8 * (lane & 3), voff = 8 * g * D + col * VE;
  vec8<T> kc[2][F];
  auto load_keys = [&](int64_t at) {
    const T* const kp = static_cast<const T*>(p.c.k) + at + koff;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int f = 0; f < F; ++f) kc[t][f] = *reinterpret_cast<const vec8<T>*>(kp + 4 * t * D + 32 * f);
  };
  int step = wave;
  int page = page_at(step);
  if (p.c.pages > 0) load_keys(place(page, step));  // before the length is known
  for (; step < end; step += W) {
    const int64_t at = place(page, step);
    const bool there = page >= 0 && page < p.c.pages;
    const int next = page_at(step + W);
    const T* const vp = static_cast<const T*>(p.c.v) + at + voff;
    typedef uint32_t vword __attribute__((ext_vector_type(VW)));
    vword v[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] = *reinterpret_cast<const vword*>(vp + j * D + c * 16 * VE);

    float s[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      v4f a{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int f = 0; f < F; ++f) {
        v4u x = __builtin_bit_cast(v4u, kc[t][f]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_ds_bpermute(from, x[i]);
        a = mfma(__builtin_bit_cast(vec8<T>, x), q[f], a);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) s[t][r] = a[r] * qfac;
    }
    // The next step's keys (past the last one: this one's again, not used).
    load_keys(step + W < end ? place(next, step + W) : at);
    page = next;
    const int64_t key0 = static_cast<int64_t>(page_of(step)) * kKvPage + (step & 1) * kHalf;
    if (!there) continue;  // uniform
    const bool edge = key0 + kHalf > least;  // some row does not see all of the step
    uint32_t poison = 0;  // bit j: key 8 g + j's value holds a NaN or infinity somewhere in this lane's part
    if (edge) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + 8 * g + 4 * t + r >= seen) s[t][r] = -__builtin_inff();
      // What no row sees may hold anything: zeros, as 0 * NaN is not 0.
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool hidden = key0 + 8 * g + j >= most;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            if (hidden) v[c][j][w] = 0u;
            if (MIXED && any_nonfinite<T>(v[c][j][w])) poison |= 1u << j;
          }
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[t][r]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const bool up = top > m + kTop;
    if (__any(up)) {  // each row by itself: what it gets does not depend on the rows beside it
      const float m1 = up ? top - kLift : m;
      const float alpha = up ? weight_of(m, m1) : 1.0f;
      m = m1;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < DT; ++i) o[i] *= alpha;
    }
    const float ref = m == -__builtin_inff() ? 0.0f : m;
    float sum = 0.0f;
    vec8<T> hi, lo;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f(s[t][r] - ref);
        sum += e;
        hi[4 * t + r] = static_cast<T>(e);
        lo[4 * t + r] = static_cast<T>(e - static_cast<float>(hi[4 * t + r]));
      }
    l += sum;
    // Element 2 w + k of eight keys: word w's halves, two keys a permute.
    auto turned = [&](int c, int e) {
      v4u x;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[i] = __builtin_amdgcn_perm(v[c][2 * i + 1][e >> 1], v[c][2 * i][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
      return __builtin_bit_cast(vec8<T>, x);
    };
    if (MIXED && edge && __any(poison != 0)) {
      // A value that some rows see and others do not is NaN or infinite: it makes NaN of the rows that
      // see it, and is zero for the product.  Rare.
      vec8<T> sees;
#pragma unroll
      for (int j = 0; j < 8; ++j) sees[j] = static_cast<T>(key0 + 8 * g + j < seen ? 1.0f : 0.0f);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const vec8<T> x = turned(c, e);
          vec8<T> bad{};
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!(__builtin_fabsf(static_cast<float>(x[j])) <= 3.4028235e38f)) bad[j] = static_cast<T>(1.0f);
          const v4f count = mfma(bad, sees, v4f{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (count[r] > 0.0f) o[c * VE + e][r] = __builtin_nanf("");
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int w = 0; w < VW; ++w) v[c][j][w] = finite_halves<T>(v[c][j][w]);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const vec8<T> x = turned(c, e);
        o[c * VE + e] = mfma(x, hi, o[c * VE + e]);
        o[c * VE + e] = mfma(x, lo, o[c * VE + e]);
      }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // Quad i = (c, r, w): dimensions 16 VE c + (4 g + r) VE + 4 w .. + 3.
  const int64_t orow = (static_cast<int64_t>(b) * p.t + tok) * p.h + qh;
  auto quad = [&](int i) {
    const int w = i % (VE / 4), r = i / (VE / 4) % 4, c = i / VE;
    v4f x;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = o[c * VE + 4 * w + k][r];
    return x;
  };
  auto column = [&](int i) { return i / VE * 16 * VE + (4 * g + i / (VE / 4) % 4) * VE + i % (VE / 4) * 4; };
  if constexpr (W == 1) {
    if (row >= rows) return;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < DT; ++i) store_quad<T>(p, quad(i), inv, split, orow, D, column(i));
    if (g == 0) store_sums(p, m, l, split, orow, D);
    return;
  }
  // The waves' parts meet in LDS, scaled to a common reference; each wave sums and finishes DT / W quads.
  if (g == 0) {
    mbuf[wave][col] = m;
    lbuf[wave][col] = l;
  }
  __syncthreads();
  float mall = mbuf[0][col];
#pragma unroll
  for (int w = 1; w < W; ++w) mall = fmaxf(mall, mbuf[w][col]);
  const float share = weight_of(m, mall);
#pragma unroll
  for (int i = 0; i < DT; ++i) obuf[(wave * DT + i) * 64 + lane] = quad(i) * share;
  float lall = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) lall += lbuf[w][col] * weight_of(mbuf[w][col], mall);
  __syncthreads();
  if (row >= rows) return;
  const float inv = lall != 0.0f ? 1.0f / lall : 0.0f;  // 0: no visible key (NaN stays NaN)
  for (int i = wave; i < DT; i += W) {
    v4f v = obuf[i * 64 + lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += obuf[(w * DT + i) * 64 + lane];
    store_quad<T>(p, v, inv, split, orow, D, column(i));
  }
  if (wave == 0 && g == 0) store_sums(p, mall, lall, split, orow, D);
}

// Joins the runs of a row, at most 64 of them: one wave a row, lane s with the reference and sum of run s.
constexpr int kMaxRuns = 64;

template <typename T, int D, int kAhead>
__global__ __launch_bounds__(256) void kv_attn16_join_kernel(KvAttn16Params p) {
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
  float ms = -__builtin_inff(), ls = 0.0f;
  if (lane < p.nsplit) {
    const float2 ml = *reinterpret_cast<const float2*>(p.ws + lane * plane + rows * D + row * 2);
    ms = ml.x;
    ls = ml.y;
  }
  float m = ms;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float a = weight_of(ms, m);
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
void launch_attn(const KvAttn16Params& p, hipStream_t stream) {
  const int rows = p.t * (p.h / p.c.kvh);
  const dim3 grid(static_cast<unsigned>((rows + 15) / 16 * p.nsplit), static_cast<unsigned>(p.c.kvh), static_cast<unsigned>(p.b));
  auto launch = [&](auto kernel, int waves) { kernel<<<grid, 64 * waves, waves > 1 ? waves * D * 64 : 0, stream>>>(p); };
  if (p.t > 1) {
    if (p.waves == 4) launch(kv_attn16_kernel<T, D, 4, true>, 4);
    else if (p.waves == 2) launch(kv_attn16_kernel<T, D, 2, true>, 2);
    else launch(kv_attn16_kernel<T, D, 1, true>, 1);
  } else {
    if (p.waves == 4) launch(kv_attn16_kernel<T, D, 4, false>, 4);
    else if (p.waves == 2) launch(kv_attn16_kernel<T, D, 2, false>, 2);
    else launch(kv_attn16_kernel<T, D, 1, false>, 1);
  }
  if (p.nsplit > 1) {
    const int64_t all = static_cast<int64_t>(p.b) * p.t * p.h;
    const dim3 joins(static_cast<unsigned>((all + 3) / 4));
    if (p.nsplit <= 4) kv_attn16_join_kernel<T, D, 4><<<joins, 256, 0, stream>>>(p);
    else kv_attn16_join_kernel<T, D, 16><<<joins, 256, 0, stream>>>(p);
  }
}

}  // namespace

// No call asks for more partial results than the Infinity Cache holds.
constexpr size_t kMaxPartial = size_t{1} << 28;

// The runs of pages: the least of the times (us) that these measurements give.  A workgroup's start, and a step of
// its four waves, for each round of the CUs (two workgroups beside each other at D <= 128); not less than the cache's
// bytes at 5.5 TB/s, which fewer workgroups than CUs do not reach; for more than one run the join, whose loads past
// the sixteenth run follow one another, and partial results at 10 TB/s.
// us in 1 / 2 / 4 / 8 / 16 / 32 runs: D = 256, one sequence of 8192 keys 109 / - / - / - / 16.3 / 17.0, 16 of 2048
// 32.5 / 23.1 / 17.3 / 14.6 / 15.0 (12) / -, 64 of 8192 - / 108 / 83 / 85 / 94 / -, 8 x 50 tokens over 826 18.2 / 26; D = 128, 8
// KV heads, 8 of 1024 13.3 / 12.3 / 11.5 / 12.8 / - / -; D = 64, 8 KV heads, 4 of 4096 25.4 / 18.3 / 13.3 / 11.8 / 13.1 / 17.4.
// Runs of one page take two waves (one sequence of 776 keys, 13 runs, 1 / 2 / 4 waves: 9.6 / 9.8 / 11.2).
KvAttn16Plan kv_attn16_plan(int64_t b, int64_t t, int32_t h, int32_t kvh, int32_t d, int64_t table_pages, int cus) {
  KvAttn16Plan plan{1, 4};
  const int64_t rows = t * (h / kvh);
  if (rows <= 0 || b <= 0 || table_pages <= 0) return plan;
  const double start = d == 256 ? 5.5 : 4.0, step = d == 256 ? 1.6 : d == 128 ? 1.1 : 0.67;
  const int64_t groups = (rows + 15) / 16 * b * kvh, slots = static_cast<int64_t>(cus) * (d == 256 ? 1 : 2);
  const double bytes = static_cast<double>(b) * kvh * table_pages * kKvPage * d * 4;
  const double partial = static_cast<double>(rows) * b * kvh * d * 8 / 1e7;
  double best = 1e300;
  for (int n = 1; n <= kMaxRuns && n <= table_pages; ++n) {
    if (n > 1 && kv_attn16_workspace(b, t, h, d, n) > kMaxPartial) break;
    const int64_t steps = (2 * ((table_pages + n - 1) / n) + 3) / 4, rounds = (groups * n + slots - 1) / slots;
    const double filled = std::min(1.0, 0.7 + 0.3 * static_cast<double>(groups * n) / static_cast<double>(cus));
    const double each = table_pages > n ? step : step / 2;  // two waves
    const double us = std::max(static_cast<double>(rounds) * (start + static_cast<double>(steps) * each), start + bytes / (5.5e6 * filled)) +
                      (n > 1 ? 3.5 + 0.05 * n + 0.2 * std::max(0, n - 16) + partial * n : 0.0);
    if (us < best) {
      best = us;
      plan.nsplit = n;
    }
  }
  plan.waves = table_pages > plan.nsplit ? 4 : 2;
  return plan;
}

size_t kv_attn16_workspace(int64_t b, int64_t t, int32_t h, int32_t d, int nsplit) {
  return nsplit > 1 ? sizeof(float) * static_cast<size_t>(nsplit) * static_cast<size_t>(split_floats(b * t * h, d)) : 0;
}

hipError_t launch_kv_attn16(const KvAttn16Params& p, int elem, hipStream_t stream) {
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
