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
// Few rows are bound by the cache's bytes: 64 sequences of up to 8192 tokens, D = 256, 400 MB, 81.8 us, 4.9 TB/s, where a
// copy reaches 5.2; one sequence of 776 tokens by the latency of its loads one behind the other (lengths and
// table, keys and values, the join), 9.2 us.  Many rows have a kernel of their own below.
//
// Weights go into the products as a sum of 16-bit parts, each with its own product: the matrix pipe has the
// time (the cache's bytes bound).  Three parts of bf16 hold all 24 bits of an fp32 weight, two of fp16 hold
// it to 2^-22 and 2^-32 of the row's largest.  bf16 in two / three parts, us: 64 sequences of up to 8192 tokens 82.0 / 82.2,
// 8 x 50 tokens over 826 17.3 / 17.9, 64 x 64 53.2 / 58.9; rounded outputs that differ from the exact ones' rounding, 64 x 8192:
// 0.24% / 0.05%.

#include <algorithm>
#include <cmath>

#include "direct_load.h"
#include "serving_internal.h"

namespace w4a4 {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
// 16-bit parts of a softmax weight.
template <typename T>
constexpr int kParts = 2;
template <>
constexpr int kParts<__bf16> = 3;
constexpr int kHalf = 32;  // keys of a step

__device__ __forceinline__ v4f mfma(const vec8<_Float16> a, const vec8<_Float16> b, const v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma(const vec8<__bf16> a, const vec8<__bf16> b, const v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The reference of a row's exponents is kLift below the largest one when it is set, and is set again only
// when an exponent is kTop above it.  fp16: the largest weight is between 2^7 and 2^15, at the upper end of
// the type, so that small weights beside a large one keep their bits.  bf16 has fp32's range, its values too: weights
// are scaled by KvAttn16Params::down, so that a table of them adds up to one at most, and sums of any finite values stay
// finite (up to 2^15 they were infinite from values of 2^112 on); in exchange values below 2^-84, over a thousand keys,
// lose low bits.  8 x 50 tokens over 826 18.0 -> 18.3 us, 64 x 64 58.9 -> 60.2.
constexpr float kLift = 7.0f, kTop = 15.0f;

// A load at a uniform address that nothing in the kernel writes: through the scalar cache, so that
// no wait for vector loads stands before its use.
template <typename U>
__device__ __forceinline__ U scalar_load(const U* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) U*>(reinterpret_cast<uintptr_t>(p));
}

// Partial results of a run: O (unnormalised, fp32), the reference and the sum of each row; whole 16 bytes.
__host__ __device__ inline int64_t split_floats(int64_t rows, int d) { return (rows * (d + 2) + 3) & ~int64_t{3}; }

// What the rows of a sequence see; lengths and counts fit 31 bits, places of keys 32.
struct Span {
  int q_len, len, causal;
  __device__ __forceinline__ Span(const KvAttn16Params& p, int b) {
    const int64_t cap = static_cast<int64_t>(p.c.table_pages) * kKvPage;
    len = p.c.pages > 0 ? static_cast<int>(min(static_cast<int64_t>(max(scalar_load(p.c.lens + b), 0)), cap)) : 0;
    q_len = min(max(p.q_lens != nullptr ? scalar_load(p.q_lens + b) : p.t, 0), p.t);
    causal = p.causal;
  }
  // Tokens that query `token` sees: none past q_len.
  __device__ __forceinline__ uint32_t seen(int token) const {
    return static_cast<uint32_t>(token >= q_len ? 0 : causal ? max(len - q_len + token + 1, 0) : len);
  }
  // The most that any of the tokens first .. last sees, and what all of them do.
  __device__ __forceinline__ uint32_t most(int first, int last) const { return seen(min(last, max(q_len - 1, first))); }
  __device__ __forceinline__ uint32_t least(int first, int last) const { return last < q_len ? seen(first) : 0; }
};

// The four consecutive columns from c of a row: its output, or its part of a run's partial results.
template <typename T>
__device__ __forceinline__ void store_quad(const KvAttn16Params& p, const v4f v, int split, int64_t orow, int d, int c) {
  if (p.nsplit > 1) {
    const int64_t all_rows = static_cast<int64_t>(p.b) * p.t * p.h;
    *reinterpret_cast<v4f*>(p.ws + split * split_floats(all_rows, d) + orow * d + c) = v;
  } else {
    typedef T tv4 __attribute__((ext_vector_type(4)));
    tv4 y;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = static_cast<T>(v[r]);
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
    p.lse[orow] = l == 0.0f ? -__builtin_inff() : m / kLog2e + __builtin_logf(l * p.up);
  }
}

// exp2(m - to), 0 for a part without a key (m = -inf).
__device__ __forceinline__ float weight_of(float m, float to) {
  return m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - to);
}

// The largest of the four lanes of a row (16 apart), without LDS.
__device__ __forceinline__ float most_of_row(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The weights of a row's eight keys of a step, from their scores: exponents over the row's reference m, in parts.
template <typename T, int DT>
__device__ __forceinline__ void weigh(const float (&s)[2][4], float down, float& m, float& l, v4f (&o)[DT], vec8<T> (&w)[kParts<T>]) {
  float top = s[0][0];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) top = fmaxf(top, s[t][r]);
  top = most_of_row(top);
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
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float e = __builtin_amdgcn_exp2f(s[t][r] - ref);
      if constexpr (kParts<T> == 3) e *= down;  // bf16
      sum += e;
#pragma unroll
      for (int i = 0; i < kParts<T>; ++i) {
        w[i][4 * t + r] = static_cast<T>(e);
        e -= static_cast<float>(w[i][4 * t + r]);
      }
    }
  l += sum;
}

// Adds the N tiles of values that tile(e) gives (eight keys from `key` of a dimension, a lane) to their sums.  MIXED:
// rows may be of several tokens, which see different keys; edge: some row does not see all of the step.
template <typename T, int N, bool MIXED, typename Tile>
__device__ __forceinline__ void add_values(Tile tile, const vec8<T> (&w)[kParts<T>], v4f* o, bool edge, uint32_t key, uint32_t seen,
                                           uint32_t most) {
  vec8<T> x[N];
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = tile(e);
  if (edge) {
    // What no row sees may hold anything: zeros, as 0 * NaN is not 0.
    v4u keep;
#pragma unroll
    for (int i = 0; i < 4; ++i) keep[i] = (key + 2 * i < most ? 0xffffu : 0u) | (key + 2 * i + 1 < most ? 0xffff0000u : 0u);
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = __builtin_bit_cast(vec8<T>, __builtin_bit_cast(v4u, x[e]) & keep);
    if constexpr (MIXED) {
      // Zeros times the values: NaN where one is NaN or infinite.
      v4f probe[2]{};
#pragma unroll
      for (int e = 0; e < N; ++e) probe[e & 1] = mfma(x[e], vec8<T>{}, probe[e & 1]);
      bool poison = false;
#pragma unroll
      for (int r = 0; r < 4; ++r) poison = poison || __builtin_isnan(probe[0][r]) || __builtin_isnan(probe[1][r]);
      if (__any(poison)) {
        // A value that some rows see and others do not is NaN or infinite: it makes NaN of the rows that
        // see it, and is zero for the product.  Rare.
        const uint32_t here = static_cast<uint32_t>(opaque_copy(static_cast<int>(key)));  // not computed before the branch
        vec8<T> sees;
#pragma unroll
        for (int j = 0; j < 8; ++j) sees[j] = static_cast<T>(here + j < seen ? 1.0f : 0.0f);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          vec8<T> bad{};
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!(__builtin_fabsf(static_cast<float>(x[e][j])) <= 3.4028235e38f)) {
              bad[j] = static_cast<T>(1.0f);
              x[e][j] = static_cast<T>(0.0f);
            }
          const v4f count = mfma(bad, sees, v4f{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (count[r] > 0.0f) o[e][r] = __builtin_nanf("");
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  // A product does not wait for the one before it.
#pragma unroll
  for (int i = 0; i < kParts<T>; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = mfma(x[e], w[i], o[e]);
}

// The results of a tile's 16 rows from its P waves, each with some of the keys: parts meet in LDS as rows of columns (the
// quads of row r in the order quad ^ r, so that no bank is met more often than others), scaled to a common
// reference, and each wave sums and stores 16 / P whole rows.
//   buf [P][16][D / 4], mbuf and lbuf [P][16]: the tile's; all waves of the workgroup come here.
template <typename T, int D, int P, int VE>
__device__ __forceinline__ void finish_rows(const KvAttn16Params& p, v4f* buf, float (*mbuf)[16], float (*lbuf)[16], int part, int lane,
                                            const v4f (&o)[D / 16], float m, float l, int split, int b, int head, int row0, int rows) {
  constexpr int kQuads = D / 4, kRows = 64 / kQuads;
  const int g = lane >> 4, col = lane & 15;
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) {
    mbuf[part][col] = m;
    lbuf[part][col] = l;
  }
  __syncthreads();
  float mall = mbuf[0][col];
#pragma unroll
  for (int w = 1; w < P; ++w) mall = fmaxf(mall, mbuf[w][col]);
  float lall = 0.0f;
#pragma unroll
  for (int w = 0; w < P; ++w) lall += lbuf[w][col] * weight_of(mbuf[w][col], mall);
  const float inv = p.nsplit > 1 ? 1.0f : lall != 0.0f ? 1.0f / lall : 0.0f;  // 0: no visible key (NaN stays NaN)
  const float share = weight_of(m, mall) * inv;
  const int group = p.h / p.c.kvh, row = row0 + col;
  const int orow = static_cast<int>((static_cast<int64_t>(b) * p.t + row / group) * p.h + head * group + row % group);
  if (part == 0 && g == 0 && row < rows) store_sums(p, mall, lall, split, orow, D);
  // Tile c VE + e holds dimensions 16 VE c + (4 g + r) VE + e.
  v4f* const mine = buf + (part * 16 + col) * kQuads;
#pragma unroll
  for (int c = 0; c < D / (16 * VE); ++c) {
    if constexpr (VE == 1) {
      mine[(4 * c + g) ^ col] = o[c] * share;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int w = 0; w < VE / 4; ++w) {
          v4f x;
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = o[c * VE + 4 * w + k][r] * share;
          mine[(c * 4 * VE + (4 * g + r) * (VE / 4) + w) ^ col] = x;
        }
    }
  }
  __syncthreads();
  // Few rows are shared by the waves too.
#pragma unroll
  for (int n = 0; n < 16; n += P * kRows) {
    if (row0 + n >= rows) break;
    const int r = n + part * kRows + lane / kQuads, quad = lane % kQuads;
    v4f v = buf[r * kQuads + (quad ^ r)];
#pragma unroll
    for (int w = 1; w < P; ++w) v += buf[(w * 16 + r) * kQuads + (quad ^ r)];
    const int to = __shfl(orow, r, 64);
    if (row0 + r < rows) store_quad<T>(p, v, split, to, D, 4 * quad);
  }
}

// What a workgroup does: a tile of the rows of (sequence, KV head), and a run of its pages.
struct Place {
  int tile, split, head, b;
};
__host__ __device__ inline uint32_t places(const KvAttn16Params& p, int tiles) {
  return static_cast<uint32_t>(p.b) * p.c.kvh * p.nsplit * tiles;
}
// Workgroups whose numbers are equal mod 8 share an XCD and its L2: each XCD gets a block of consecutive places, so that the
// tiles of a run meet there (16 x 16 tokens over 2048, 32 heads on 8 KV heads of 128: 34 us, 65 with them spread).  Few
// runs are spread, for their tiles see different numbers of keys.
__device__ __forceinline__ bool place_of(const KvAttn16Params& p, int tiles, Place& at) {
  const uint32_t all = places(p, tiles), id = blockIdx.y * gridDim.x + blockIdx.x;
  uint32_t item = id;
  if (all >= 8u * tiles) {
    const uint32_t each = (all + 7) / 8;
    if ((id >> 3) >= each) return false;
    item = (id & 7) * each + (id >> 3);
  }
  if (item >= all) return false;
  const uint32_t run = item / tiles, side = run / p.nsplit;
  at = {static_cast<int>(item - run * tiles), static_cast<int>(run - side * p.nsplit), static_cast<int>(side % p.c.kvh),
        static_cast<int>(side / p.c.kvh)};
  return true;
}
// The grid: eight equal blocks at least, in rows of 2^16.
inline dim3 place_grid(const KvAttn16Params& p, int tiles) {
  const uint32_t all = (places(p, tiles) + 7) / 8 * 8, x = std::min(all, 1u << 16);
  return dim3(x, (all + x - 1) / x);
}

template <typename T, int D, int W, bool MIXED>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void kv_attn16_kernel(KvAttn16Params p) {
  constexpr int F = D / 32, DT = D / 16;
  constexpr int VE = D >= 128 ? 8 : 4, CH = D / (16 * VE), VW = VE / 2;  // a value chunk: elements, chunks, words
  extern __shared__ __align__(16) v4f obuf[];  // [W][16][D / 4]
  __shared__ float mbuf[W][16], lbuf[W][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int group = p.h / p.c.kvh;
  const int rows = p.t * group;
  const int tiles = (rows + 15) >> 4;
  Place at{static_cast<int>(blockIdx.x % tiles), static_cast<int>(blockIdx.x / tiles), static_cast<int>(blockIdx.y), static_cast<int>(blockIdx.z)};
  if (MIXED && !place_of(p, tiles, at)) return;
  const int tile = at.tile, split = at.split, head = at.head, b = at.b;
  const Span span(p, b);

  // This lane's row; tokens past q_len see nothing.
  const int row = tile * 16 + col;
  const int tok = min(row / group, p.t - 1), qh = head * group + row % group;
  const uint32_t seen = row < rows ? span.seen(row / group) : 0;
  const int tok_first = tile * 16 / group, tok_last = min(tile * 16 + 15, rows - 1) / group;
  const uint32_t most = span.most(tok_first, tok_last);
  const uint32_t least = span.least(tok_first, tok_last);  // rows past the last one are computed as they come, and not stored
  const int pages = static_cast<int>((most + kKvPage - 1) / kKvPage);
  // The run's pages are split, split + nsplit, ..: the first is known without the length.  Its steps are
  // the halves of 32 keys; a last half that no row sees is left out.
  const int mine = pages > split ? (pages - split - 1) / p.nsplit + 1 : 0;
  const bool half = mine > 0 && split + (mine - 1) * p.nsplit == pages - 1 && most <= static_cast<uint32_t>(pages) * kKvPage - kHalf;
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
    const uint32_t key0 = static_cast<uint32_t>(page_of(step)) * kKvPage + (step & 1) * kHalf;
    if (!there) continue;  // uniform
    const bool edge = key0 + kHalf > least;  // some row does not see all of the step
    if (edge) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + 8 * g + 4 * t + r >= seen) s[t][r] = -__builtin_inff();
    }
    vec8<T> w[kParts<T>];
    weigh<T>(s, p.down, m, l, o, w);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      // Element 2 w + k of eight keys: word w's halves, two keys a permute.
      auto turned = [&](int e) {
        v4u x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = __builtin_amdgcn_perm(v[c][2 * i + 1][e >> 1], v[c][2 * i][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
        return __builtin_bit_cast(vec8<T>, x);
      };
      add_values<T, VE, MIXED>(turned, w, o + c * VE, edge, key0 + 8 * g, seen, most);
    }
  }
  finish_rows<T, D, W, VE>(p, obuf, mbuf, lbuf, wave, lane, o, m, l, split, b, head, tile * 16, rows);
}

// The same for many rows: a workgroup takes 64 of a KV head, and a run of pages that reach LDS by direct loads, one
// ahead.  Waves w and w + 4 take rows 16 w .. of it, and the page's first and second half.  Where 16 rows a workgroup
// read every key for themselves, at the rate of the L2, this is bound by LDS (64 KB in and 256 KB out a page of
// D = 256: 1.1 of its 1.6 us) and by the matrix products beside it: 32 x 50 tokens of 8 heads of 256 over 826 29.8 us
// (16 rows a workgroup: 54), 64 x 64 54 (110), 8 x 776 over 776 69 (135), 430 TFLOP/s; bf16, whose weights take a third
// product, 32.8 (58), 60 (118), 75 (143).
//
// Values are read from LDS a dimension a lane, so that they need no turning.  A key's 16-byte chunks stand in the order
// chunk ^ f(key), f by the bits of the key that differ among the rows of a read, so that it meets every bank alike
// (without it for the values alone: a third of the LDS cycles are conflicts).
template <typename T, int D>
__global__ __launch_bounds__(512, 2) void kv_attn16_wide_kernel(KvAttn16Params p) {
  constexpr int F = D / 32, DT = D / 16;
  constexpr int kSide = kKvPage * D * 2, kPieces = kSide / 8192;  // bytes of a page's keys or values; KB a wave of each
  extern __shared__ __align__(16) char stage[];                  // [2][keys, values]; then [4][2][16][D / 4] results
  __shared__ float mbuf[4][2][16], lbuf[4][2][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = wave >> 2;
  const int g = lane >> 4, col = lane & 15;
  const int group = p.h / p.c.kvh;
  const int rows = p.t * group;
  Place at;
  if (!place_of(p, (rows + 63) >> 6, at)) return;
  const int split = at.split, head = at.head, b = at.b;
  const Span span(p, b);

  // This lane's row; the wave's rows, and the workgroup's.  Rows past the last one see nothing.
  const int first = at.tile * 64, row0 = first + 16 * (wave & 3);
  const int row = row0 + col;
  const int tok = min(row / group, p.t - 1), qh = head * group + row % group;
  const uint32_t seen = row < rows ? span.seen(row / group) : 0;
  const int tok_first = min(row0, rows - 1) / group, tok_last = min(row0 + 15, rows - 1) / group;
  const uint32_t most = row0 < rows ? span.most(tok_first, tok_last) : 0;
  const uint32_t least = span.least(tok_first, tok_last);
  const int pages = static_cast<int>((span.most(first / group, min(first + 63, rows - 1) / group) + kKvPage - 1) / kKvPage);
  const int end = pages > split ? (pages - split - 1) / p.nsplit + 1 : 0;  // pages split, split + nsplit, ..

  vec8<T> q[F];
  const T* const qrow = static_cast<const T*>(p.q) + b * p.q_stride[0] + tok * p.q_stride[1] + qh * p.q_stride[2];
#pragma unroll
  for (int f = 0; f < F; ++f) q[f] = *reinterpret_cast<const vec8<T>*>(qrow + 32 * f + 8 * g);
  const float qfac = p.scaling * kLog2e;

  float m = -__builtin_inff(), l = 0.0f;
  v4f o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  const int32_t* const table = p.c.table + b * p.c.table_stride;
  auto page_of = [&](int step) { return __builtin_amdgcn_readfirstlane(split + step * p.nsplit); };
  auto page_at = [&](int step) { return page_of(step) < p.c.table_pages ? scalar_load(table + page_of(step)) : -1; };
  // D = 64: two keys a 256 bytes, so the key's lowest bit is in the place already.
  auto k_order = [](int key) { return D == 64 ? ((key >> 1) & 1) | ((key >> 3) & 3) << 1 : (key & 3) | ((key >> 3) & 3) << 2; };
  auto v_order = [](int key) { return D == 64 ? (key & 2) | ((key >> 3) & 1) << 2 : (key & 3) << 1 | ((key >> 3) & 1) << 3; };
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)stage));
  uint32_t k_off[kPieces], v_off[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int at = (wave * kPieces + i) * 64 + lane, key = at / (D / 8), chunk = at % (D / 8);
    k_off[i] = (key * (D / 8) + (chunk ^ k_order(key))) * 16;
    v_off[i] = (key * (D / 8) + (chunk ^ v_order(key))) * 16;
  }
  // Entries that name no page are read as page 0, whose keys then count as not there.
  auto load = [&](int page, int slot) {
    const int64_t id = __builtin_amdgcn_readfirstlane(page >= 0 && page < p.c.pages ? page : 0);
    const int64_t at = (id * p.c.kvh + head) * kSide;
    const uint32_t dst = lds0 + slot * 2 * kSide + wave * kPieces * 1024;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) load_lds_1k(static_cast<const char*>(p.c.k) + at, k_off[i], dst + i * 1024);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) load_lds_1k(static_cast<const char*>(p.c.v) + at, v_off[i], dst + kSide + i * 1024);
  };
  int next = page_at(0);
  if (end > 0) load(next, 0);
  // The queries are here before the loop: a wait for them inside would wait for the pages under way as well.
#pragma unroll
  for (int f = 0; f < F; ++f) asm volatile("" : "+v"(q[f]));
  for (int step = 0; step < end; ++step) {
    wait_vm<0>();
    lds_done_barrier();  // the page is whole, and the one before it read by all
    const int page = next;
    next = page_at(step + 1);
    if (step + 1 < end) load(next, (step + 1) & 1);
    const char* const ks = stage + (step & 1) * 2 * kSide + half * kHalf * D * 2;
    const char* const vs = ks + kSide;
    const uint32_t key0 = static_cast<uint32_t>(page_of(step)) * kKvPage + half * kHalf;
    if (page < 0 || page >= p.c.pages || key0 >= most) continue;  // uniform

    vec8<T> k[2][F];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key = 8 * (col >> 2) + 4 * t + (col & 3);
        k[t][f] = *reinterpret_cast<const vec8<T>*>(ks + (key * (D / 8) + ((4 * f + g) ^ k_order(key))) * 16);
      }
    __builtin_amdgcn_sched_barrier(0);  // all reads under way before the first product waits
    v4f a[2]{};
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int t = 0; t < 2; ++t) a[t] = mfma(k[t][f], q[f], a[t]);
    float s[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[t][r] = a[t][r] * qfac;
    const bool edge = key0 + kHalf > least;
    if (edge) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + 8 * g + 4 * t + r >= seen) s[t][r] = -__builtin_inff();
    }
    vec8<T> w[kParts<T>];
    weigh<T>(s, p.down, m, l, o, w);
    // Each group of 16 lanes reads four keys of 16 dimensions, and gets them a dimension a lane.
#pragma unroll
    for (int c = 0; c < DT; c += 8 < DT ? 8 : DT)
      add_values<T, (8 < DT ? 8 : DT), true>(
          [&](int e) {
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef short s8 __attribute__((ext_vector_type(8)));
            s4 part[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int key = 8 * g + 4 * h + (col >> 2), chunk = 2 * (c + e) + ((col & 3) >> 1);
              const char* const at = vs + (key * (D / 8) + (chunk ^ v_order(key))) * 16 + (col & 1) * 8;
              part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)at);
            }
            return __builtin_bit_cast(vec8<T>, s8(__builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7)));
          },
          w, o + c, edge, key0 + 8 * g, seen, most);
  }
  finish_rows<T, D, 2, 1>(p, reinterpret_cast<v4f*>(stage) + (wave & 3) * 2 * 16 * (D / 4), mbuf[wave & 3], lbuf[wave & 3], half, lane,
                           o, m, l, split, b, head, row0, rows);
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
  if (p.lse != nullptr && lane == 0) p.lse[row] = empty ? -__builtin_inff() : m / kLog2e + __builtin_logf(l * p.up);
}

template <typename T, int D>
void launch_attn(const KvAttn16Params& p, hipStream_t stream) {
  const int rows = p.t * (p.h / p.c.kvh);
  if (p.wide) {
    kv_attn16_wide_kernel<T, D><<<place_grid(p, (rows + 63) / 64), 512, 2 * 2 * kKvPage * D * 2, stream>>>(p);
  } else {
    const int tiles = (rows + 15) / 16;
    auto launch = [&](auto kernel, dim3 grid, int waves) { kernel<<<grid, 64 * waves, waves * D * 64, stream>>>(p); };
    if (p.t > 1) {
      const dim3 grid = place_grid(p, tiles);
      if (p.waves == 4) launch(kv_attn16_kernel<T, D, 4, true>, grid, 4);
      else launch(kv_attn16_kernel<T, D, 2, true>, grid, 2);
    } else {
      const dim3 grid(static_cast<unsigned>(tiles * p.nsplit), static_cast<unsigned>(p.c.kvh), static_cast<unsigned>(p.b));
      if (p.waves == 4) launch(kv_attn16_kernel<T, D, 4, false>, grid, 4);
      else launch(kv_attn16_kernel<T, D, 2, false>, grid, 2);
    }
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

// The kernel and its runs of pages: the least of the times (us) that these measurements give.  A workgroup's start and its
// pages, for each round of the CUs (two workgroups beside each other where they fit); not less than the cache's
// bytes at 5.5 TB/s, which fewer workgroups than CUs do not reach; for more than one run the join, whose loads past
// the sixteenth run follow one another, and partial results at 3.5 TB/s.
// 16 rows a workgroup, us in 1 / 2 / 4 / 8 / 16 / 32 runs: D = 256, one sequence of 8192 keys 109 / - / - / - / 16.3 / 17.0, 16 of
// 2048 32.5 / 23.1 / 17.3 / 14.6 / 15.0 (12) / -, 64 of 8192 - / 108 / 82 / 85 / 94 / -, 8 x 50 tokens over 826 18.9 / 28.7; D = 128, 8
// KV heads, 8 of 1024 13.3 / 12.3 / 11.5 / 12.8 / - / -; D = 64, 8 KV heads, 4 of 4096 25.4 / 18.3 / 13.3 / 11.8 / 13.1 / 17.4.
// 64 rows, us in 1 / 2 / 3 / 4 / 6 runs: D = 256, 8 x 50 tokens over 826 31.2 / 27.0 / 25.9 / 26.0 / 32.3; 8 KV heads of 128 with
// 64 rows, 16 of 2048 37.4 / 31.5 / 39.0 / 38.0 / 44.8, of 64 26.7 / 21.7 / 22.9 / 22.1 / 25.0.
// Runs of one page take two waves (one sequence of 776 keys, 13 runs, 1 / 2 / 4 waves: 9.6 / 9.8 / 11.2).
KvAttn16Plan kv_attn16_plan(int64_t b, int64_t t, int32_t h, int32_t kvh, int32_t d, int64_t table_pages, int cus) {
  KvAttn16Plan plan{1, 4, false};
  const int64_t rows = t * (h / kvh);
  if (rows <= 0 || b <= 0 || table_pages <= 0) return plan;
  const double bytes = static_cast<double>(b) * kvh * table_pages * kKvPage * d * 4;
  const double partial = static_cast<double>(rows) * b * kvh * d * 8 / 3.5e6;
  double best = 1e300;
  for (int wide = 0; wide <= (rows > 16 ? 1 : 0); ++wide) {
    const double start = d == 256 || wide ? 5.5 : 4.0;
    const double page = wide ? (d == 256 ? 1.6 : d == 128 ? 1.0 : 0.7) : (d == 256 ? 0.8 : d == 128 ? 0.55 : 0.33);
    const int64_t groups = (wide ? (rows + 63) / 64 : (rows + 15) / 16) * b * kvh;
    const int64_t slots = static_cast<int64_t>(cus) * (d == 256 || (wide && d == 128) ? 1 : 2);
    for (int n = 1; n <= kMaxRuns && n <= table_pages; ++n) {
      if (n > 1 && kv_attn16_workspace(b, t, h, d, n) > kMaxPartial) break;
      const int64_t rounds = (groups * n + slots - 1) / slots, most = (table_pages + n - 1) / n;
      const int64_t pages = wide || most == 1 ? most : (most + 1) & ~int64_t{1};  // four waves take two at a time
      const double filled = std::min(1.0, 0.7 + 0.3 * static_cast<double>(groups * n) / static_cast<double>(cus));
      const double us = std::max(static_cast<double>(rounds) * (start + static_cast<double>(pages) * page),
                                 start + bytes / (5.5e6 * filled)) +
                        (n > 1 ? 3.5 + 0.05 * n + 0.2 * std::max(0, n - 16) + partial * n : 0.0);
      if (us < best) {
        best = us;
        plan.nsplit = n;
        plan.wide = wide != 0;
      }
    }
  }
  plan.waves = table_pages > plan.nsplit ? 4 : 2;
  return plan;
}

float kv_attn16_down(int elem, int64_t table_pages) {
  int exponent = 0;
  if (elem != kFp16)
    for (exponent = 15; (int64_t{1} << (exponent - 15)) < table_pages * kKvPage;) ++exponent;
  return std::ldexp(1.0f, -exponent);
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
