// Low-rank adapters of many requests beside a shared projection.
//
//   h[m] = A[id(m)] x[m];   out[m, n] = y[m, n] + scale[id(m)] * sum_r h[m, g(n) R + r] B[id(m), n, r]
//
// g(n) is the slice of column n (the parts of a joined projection have first factors of their own, one
// below the other in A).  Two launches on 16 x 16 x 32 matrix instructions:
//
// lora_down_kernel: 16 rows x up to 64 rows of A, the K slice of a workgroup over its eight waves, joined
// in LDS; fp32 sums of each K slice to the workspace.
// lora_up_kernel: 16 rows x 128 columns a wave.  h is the sum of the K slices in fp32, split into 16-bit parts
// whose products with B are summed: three of bf16, which hold all of it, or two of fp16, which hold it to 2^-22 and
// 2^-38 of its row's largest (after a shift that brings that one into the upper range, so that no h overflows).  bf16 in
// two / three parts, us: 6208 x 32768 of rank 32 159.4 / 160.1, of rank 64 198 / 209, 6208 x 2560 of rank 128 72.6 / 74.0.
//
// Rows need no order.  A tile is up to 16 rows of one adapter: 16 consecutive ones of a request of 64 or more, else those
// of an adapter among 64 consecutive rows, which each workgroup finds by itself (191 rows of 14 adapters, 2048 x 3509: 9.6 us;
// 17.2 with tiles of 16 consecutive rows, taken once for each of their adapters).  Rows without an adapter keep y.
//
// Operands are loaded with four neighbouring lanes on 64 consecutive bytes of a row and then handed to the
// lanes that the matrix instruction wants them in: as it has them, 16 neighbouring lanes are 16 bytes of as many rows,
// which arrive at a quarter of the rate (first launch, 6208 x 2048 with 64 rows of A: 26 -> 17 us).

#include <algorithm>

#include "serving_internal.h"

namespace w4a4 {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

__device__ __forceinline__ v4f mfma(const vec8<_Float16> a, const vec8<_Float16> b, const v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma(const vec8<__bf16> a, const vec8<__bf16> b, const v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// From lanes 4 row + chunk to lanes 16 chunk + row.
template <typename T>
__device__ __forceinline__ vec8<T> to_operand(const vec8<T> v) {
  const int from = ((threadIdx.x & 15) * 4 + ((threadIdx.x & 63) >> 4)) * 4;
  v4u x = __builtin_bit_cast(v4u, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_ds_bpermute(from, x[i]);
  return __builtin_bit_cast(vec8<T>, x);
}

// h between the launches: blocks of 16 rows x 32 ranks of a slice, [K slice, rows / 16, slice, ranks / 32]; a block has
// ranks 8 g .. + 7 of its row i at 128 g + 8 i, as the lanes of the second launch take them.  Of a row and its block 0:
__device__ __forceinline__ int64_t lora_h_row(const LoraParams& p, int row, int slice) {
  return (static_cast<int64_t>(row >> 4) * p.slices + slice) * ((p.r + 31) / 32) * 512 + (row & 15) * 8;
}

constexpr int kWindow = 64;

// The rows of a tile and their adapter (-1: none).
template <bool GATHER>
struct Tile {
  int id;      // not GATHER: as it stands in ids, until known()
  int n;       // rows
  int row0;    // the first; GATHER: of the window
  int place;   // GATHER: lane i < 16: row i, from row0
  // The first use of the id that was loaded: false where the tile has nothing to do.
  __device__ __forceinline__ bool known(const LoraParams& p, bool none) {
    if constexpr (!GATHER) id = __builtin_amdgcn_readfirstlane(id < 0 || id >= p.adapters ? -1 : id);
    return none || id >= 0;
  }
  // Row i of the tile, from row0; past the last one the last one again.
  __device__ __forceinline__ int row(int i) const {
    const int at = min(i, n - 1);
    return GATHER ? __shfl(place, at, 64) : at;
  }
};

// The which-th tile of unit (16 rows of a request, or a window); false: there is none.  Uniform over the workgroup.  none: rows
// without an adapter have tiles too.  Rows of a request are known without their id, which nothing waits for here.
template <bool GATHER>
__device__ __forceinline__ bool find_tile(const LoraParams& p, int unit, int which, bool none, Tile<GATHER>& t) {
  const int m = static_cast<int>(p.m), per_id = static_cast<int>(p.per_id);  // at most 2^26
  if constexpr (!GATHER) {
    const int request = unit / p.tiles, at = 16 * (unit - request * p.tiles);
    t.row0 = request * per_id + at;
    t.n = min(min(per_id - at, m - t.row0), 16);
    if (t.n <= 0) return false;
    t.id = p.ids[request];
    return true;
  } else {
    const int lane = threadIdx.x & 63;
    t.row0 = unit * kWindow;
    const int raw = p.ids[min(t.row0 + lane, m - 1) / per_id];
    const int id = t.row0 + lane >= m ? -2 : raw < 0 || raw >= p.adapters ? -1 : raw;
    const int least = none ? -1 : 0;
    uint64_t same;
    int at;  // of the tile among the adapter's
    if (p.leaders) {  // the one whose first row is row `which`
      t.id = __builtin_amdgcn_readlane(id, which);
      same = __ballot(id == t.id);
      at = __builtin_popcountll(same & ((uint64_t{1} << which) - 1));
      if (t.id < least || at % 16 != 0) return false;
      at /= 16;
    } else {  // counted over the adapters in the order of their first rows
      uint64_t left = __ballot(id >= least);
      for (at = which;; at -= (__builtin_popcountll(same) + 15) / 16) {
        if (left == 0) return false;
        t.id = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        same = __ballot(id == t.id);
        if (16 * at < __builtin_popcountll(same)) break;
        left &= ~same;
      }
    }
    t.n = min(__builtin_popcountll(same) - 16 * at, 16);
    // Each row goes to the lane of its place in the tile; the others' to lane 63, where nobody looks.
    const int rank = __builtin_popcountll(same & ((uint64_t{1} << lane) - 1)) - 16 * at;
    const bool mine = id == t.id && rank >= 0 && rank < 16;
    t.place = __builtin_amdgcn_ds_permute(4 * (mine ? rank : 63), lane);
    return true;
  }
}

// Rows 16 NR y .. of A, K slice z; the slice's chunks of 32 elements are dealt to the waves in runs.
// Bound by the arrival of x and A (A from the L2 for all tiles of an adapter but the first): kAhead chunks of both are
// under way at once.  6208 x 2048 with 64 rows of A: 17 us.
template <typename T, int NR, bool GATHER>
__global__ __launch_bounds__(512) void lora_down_kernel(LoraParams p) {
  constexpr int W = 8, kAhead = 4;
  __shared__ __align__(16) v4f part[W][NR][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int lr = lane >> 2, lc = lane & 3;  // row and chunk that the lane loads
  Tile<GATHER> tile;
  // The K slices are the fastest: workgroups whose numbers are equal mod 8 share an XCD, whose L2 then holds its slices of A.
  const int place = blockIdx.x / p.ksplit, kslice = blockIdx.x - place * p.ksplit;
  if (!find_tile(p, p.unit0 + place / p.groups, place % p.groups, false, tile) || !tile.known(p, false)) return;
  const int total = p.slices * p.r;  // rows of an adapter's A
  const int rank0 = blockIdx.y * 16 * NR;
  const int chunks = (p.k + 31) / 32;
  const int per_slice = (chunks + p.ksplit - 1) / p.ksplit;
  const int c0 = kslice * per_slice, c1 = min(c0 + per_slice, chunks);
  const int per_wave = (per_slice + W - 1) / W;
  const int w0 = min(c0 + wave * per_wave, c1), w1 = min(w0 + per_wave, c1);
  const int whole = min(w1, p.k / 32);  // chunks that K fills

  const T* const xp = static_cast<const T*>(p.x) + tile.row0 * p.ldx + tile.row(lr) * p.ldx + 8 * lc;
  const T* ap[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i)  // rows past the last one: the last one again, not stored
    ap[i] = static_cast<const T*>(p.a) + (static_cast<int64_t>(tile.id) * total + min(rank0 + 16 * i + lr, total - 1)) * p.k + 8 * lc;
  v4f acc[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](const vec8<T> x, const vec8<T> (&a)[NR]) {
    const vec8<T> u = to_operand<T>(x);
#pragma unroll
    for (int i = 0; i < NR; ++i) acc[i] = mfma(u, to_operand<T>(a[i]), acc[i]);
  };
  auto load = [&](vec8<T>& x, vec8<T> (&a)[NR], int k) {
    x = *reinterpret_cast<const vec8<T>*>(xp + k);
#pragma unroll
    for (int i = 0; i < NR; ++i) a[i] = *reinterpret_cast<const vec8<T>*>(ap[i] + k);
  };
  int c = w0;
  for (; c + kAhead <= whole; c += kAhead) {
    vec8<T> x[kAhead], a[kAhead][NR];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) load(x[j], a[j], 32 * (c + j));
#pragma unroll
    for (int j = 0; j < kAhead; ++j) add(x[j], a[j]);
  }
  for (; c < w1; ++c) {  // the last ones, and one that K does not fill
    vec8<T> x, a[NR];
    const bool in = 32 * c + 8 * lc < p.k;
    load(x, a, in ? 32 * c : -8 * lc);  // elsewhere the row's first elements
    if (!in) {
      x = vec8<T>{};
#pragma unroll
      for (int i = 0; i < NR; ++i) a[i] = vec8<T>{};
    }
    add(x, a);
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) part[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < NR; i += W) {
    v4f s = part[0][i][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) s += part[w][i][lane];
    const int rank = rank0 + 16 * i + col, slice = rank / p.r, of = rank % p.r;
    float* const hp = p.h + kslice * p.h_plane + of / 8 * 128 + of % 8;  // blocks of 32 ranks follow one another
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = tile.row0 + tile.row(4 * g + r);
      if (4 * g + r < tile.n && rank < total) hp[lora_h_row(p, row, slice)] = s[r];
    }
  }
}

// 16-bit parts of h.
template <typename T>
constexpr int kParts = 2;
template <>
constexpr int kParts<__bf16> = 3;

// Brings the lane's row of h, ranks 32 s + 8 g .. + 7, into the range of its parts; returns the factor that takes the products back.
template <typename T, int KS>
__device__ __forceinline__ float shift_h(float (&f)[KS][8]) {
  float unshift = 1.0f;
  if constexpr (static_cast<float>(static_cast<T>(65536.0f)) > 1e30f) {  // fp16
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(f[s][e]));
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    // The row's largest to 2^13 .. 2^14; nothing to do for rows of zeros, infinities or NaN.
    const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    float shift = 1.0f;
    if (top > 0.0f && e < 128) {
      const int by = max(min(13 - e, 126), -126);
      shift = __uint_as_float(static_cast<uint32_t>(127 + by) << 23);
      unshift = __uint_as_float(static_cast<uint32_t>(127 - by) << 23);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[s][e] *= shift;
  }
  return unshift;
}

// B of NT tiles of columns: as loaded (row n0 + NT * (lane / 4) + i, chunk lane % 4), rows past `end` the last one, ranks
// past the last one the last eight.
template <typename T, int NT, int KS>
__device__ __forceinline__ void load_b(const LoraParams& p, int id, int n0, int end, vec8<T> (&w)[NT][KS]) {
  const int lr = (threadIdx.x & 63) >> 2, lc = threadIdx.x & 3;
  const T* const bp = static_cast<const T*>(p.b) + static_cast<int64_t>(id) * p.n * p.r;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int s = 0; s < KS; ++s)
      w[i][s] = *reinterpret_cast<const vec8<T>*>(bp + static_cast<int64_t>(min(n0 + NT * lr + i, end - 1)) * p.r + min(32 * s + 8 * lc, p.r - 8));
}

template <typename T, int NT, int KS>
__device__ __forceinline__ void times_b(const LoraParams& p, const vec8<T> (&w)[NT][KS], const float (&f)[KS][8], v4f (&acc)[NT]) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    vec8<T> h[kParts<T>];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v = f[s][e];
#pragma unroll
      for (int j = 0; j < kParts<T>; ++j) {
        h[j][e] = static_cast<T>(v);
        v -= static_cast<float>(h[j][e]);
      }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      vec8<T> u = to_operand<T>(w[i][s]);
      if (32 * s + 8 * g >= p.r) u = vec8<T>{};
#pragma unroll
      for (int j = 0; j < kParts<T>; ++j) acc[i] = mfma(h[j], u, acc[i]);
    }
  }
}

// y of the lane: columns nc .. + NT - 1 of its four rows.
template <typename T, int NT>
using vecn = T __attribute__((ext_vector_type(NT)));
template <typename T, int NT>
using vecn_h = T __attribute__((ext_vector_type(NT), aligned(2)));  // at any element
template <typename T, int NT>
__device__ __forceinline__ void load_y(const LoraParams& p, int row0, const int (&row)[4], int nc, int end, bool whole, vecn<T, NT> (&y)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const T* const yp = static_cast<const T*>(p.y) + row0 * p.ldy + row[r] * p.ldy + nc;
    if (whole) {
      y[r] = *reinterpret_cast<const vecn_h<T, NT>*>(yp);
    } else {
#pragma unroll
      for (int e = 0; e < NT; ++e) y[r][e] = nc + e < end ? yp[e] : static_cast<T>(0.0f);
    }
  }
}

// The lane's first n rows (id -1: as they were).
template <typename T, int NT>
__device__ __forceinline__ void store_rows(const LoraParams& p, int row0, const int (&row)[4], int n, int nc, int end, bool whole, int id,
                                           const float (&back)[4], float scale, const v4f (&acc)[NT], const vecn<T, NT> (&y)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (r >= n) continue;
    vecn<T, NT> z = y[r];
    if (id >= 0) {
#pragma unroll
      for (int e = 0; e < NT; ++e) z[e] = static_cast<T>(fmaf(acc[e][r] * back[r], scale, static_cast<float>(z[e])));
    }
    T* const op = static_cast<T*>(p.out) + row0 * p.ldo + row[r] * p.ldo + nc;
    if (whole) {
      __builtin_nontemporal_store(z, reinterpret_cast<vecn_h<T, NT>*>(op));  // past the L2, which B and h need
    } else {
#pragma unroll
      for (int e = 0; e < NT; ++e)
        if (nc + e < end) op[e] = z[e];
    }
  }
}

// A wave takes 16 rows and kCols columns of a slice, h and y (and the ids, on which only B waits) under way at
// once; nothing is kept for a second row tile: more waves hide as much, with less code (B kept over a wave's row tiles and
// the next tile under way, in a form whose stores went through the L2: 191 us for 6208 x 32768 in place of 199, but 51
// for 2560 columns in place of 47).  Column j of tile i is column NT j + i of the block: a lane ends with NT (eight, or four for large ranks) consecutive columns of four
// rows, and 16 lanes read and write 256 or 128 consecutive bytes of a row.  Bound by y and out in HBM where rows are
// many: 6208 x 32768 with rank 32, both launches 161 us, 5.3 TB/s.
template <int KS>
constexpr int kCols = KS <= 2 ? 128 : 64;

// KS: ranks / 32.
template <typename T, int KS, bool GATHER>
__global__ __launch_bounds__(256, KS == 1 ? 4 : 3) void lora_up_kernel(LoraParams p) {
  constexpr int C = kCols<KS>, NT = C / 16;  // a lane's consecutive columns
  constexpr int ZA = 4 / KS;                 // K slices of h that are loaded at once
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  // The workgroup's four blocks within a slice, and its rows.
  int run = blockIdx.x % p.runs, slice = 0, n0 = 0;
  const int rest = blockIdx.x / p.runs;
  for (; slice < p.slices; ++slice) {
    const int runs = (p.width[slice] + 4 * C - 1) / (4 * C);
    if (run < runs) break;
    run -= runs;
    n0 += p.width[slice];
  }
  const int end = n0 + p.width[slice];
  n0 += (run * 4 + wave) * C;
  if (n0 >= end) return;  // no barrier below
  const int nc = n0 + NT * col;
  const bool whole = n0 + C <= end;  // uniform
  const bool in_place = p.out == p.y && p.ldo == p.ldy;

  Tile<GATHER> tile;
  if (!find_tile(p, p.unit0 + rest / p.groups, rest % p.groups, !in_place, tile)) return;
  int row[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) row[r] = tile.row(4 * g + r);
  float back[4]{};
  v4f acc[NT]{};
  vecn<T, NT> y[4];
  if (p.adapters == 0) {
    load_y<T, NT>(p, tile.row0, row, nc, end, whole, y);
    if (!in_place) store_rows<T, NT>(p, tile.row0, row, tile.n - 4 * g, nc, end, whole, -1, back, 0.0f, acc, y);
    return;
  }
  // Under way at once: h (ranks 32 s + 8 g .. + 7 of row `col`), y (columns nc .. + NT - 1 of rows 4 g + r), and B as soon as
  // the id is here.
  const int64_t h_row = lora_h_row(p, tile.row0 + tile.row(col), slice) + 128 * g;
  v4f part[ZA][KS][2];
  auto load_h = [&](int z0) {
#pragma unroll
    for (int z = 0; z < ZA; ++z)
      if (z0 + z < p.ksplit) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const float* const hp = p.h + h_row + min(s, (p.r + 31) / 32 - 1) * 512 + (z0 + z) * p.h_plane;
          part[z][s][0] = *reinterpret_cast<const v4f*>(hp);
          part[z][s][1] = *reinterpret_cast<const v4f*>(hp + 4);
        }
      }
  };
  load_h(0);
  load_y<T, NT>(p, tile.row0, row, nc, end, whole, y);
  if (!tile.known(p, !in_place)) return;
  const int id = max(tile.id, 0);  // of a tile without an adapter: not used
  const float scale = p.scale != nullptr ? p.scale[id] : 1.0f;
  vec8<T> w[NT][KS];
  load_b<T, NT, KS>(p, id, n0, end, w);

  float f[KS][8];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) f[s][e] = part[0][s][e >> 2][e & 3];
  for (int z0 = 0;; load_h(z0)) {
#pragma unroll
    for (int z = 0; z < ZA; ++z)
      if (z0 + z > 0 && z0 + z < p.ksplit) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e) f[s][e] += part[z][s][e >> 2][e & 3];
      }
    z0 += ZA;
    if (z0 >= p.ksplit) break;
  }
#pragma unroll
  for (int s = 0; s < KS; ++s)
    if (32 * s + 8 * g >= p.r) {  // past the last rank: anything
#pragma unroll
      for (int e = 0; e < 8; ++e) f[s][e] = 0.0f;
    }
  const float unshift = shift_h<T, KS>(f);
  // What the lane ends with are rows 4 g + r, whose factors are in other lanes.
#pragma unroll
  for (int r = 0; r < 4; ++r) back[r] = __shfl(unshift, 4 * g + r, 64);
  times_b<T, NT, KS>(p, w, f, acc);
  store_rows<T, NT>(p, tile.row0, row, tile.n - 4 * g, nc, end, whole, tile.id, back, scale, acc, y);
}

// Both products in one launch, for few rows: a workgroup computes h of its tile, adapter and slice itself (its eight
// waves each an eighth of K, joined in LDS) while B and y are under way, and its waves take a block of kCols columns each.
// Bound by the arrival of A at one CU.  One row into 2560 columns in three slices: 6.0 us, two launches 7.7; 64 rows of
// 64 adapters into 2048: 7.0.
template <typename T, int NR, bool GATHER>
__global__ __launch_bounds__(512) void lora_fused_kernel(LoraParams p) {
  constexpr int W = 8, KS = (NR + 1) / 2, C = kCols<KS>, NT = C / 16;
  constexpr int kAhead = NR <= 2 ? 8 : 16 / NR;
  __shared__ __align__(16) v4f part[W][NR][64];
  __shared__ __align__(16) float hs[KS * 512];  // as a block of h
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int lr = lane >> 2, lc = lane & 3;  // row and chunk that the lane loads
  int run = blockIdx.x % p.runs, slice = 0, n0 = 0;
  const int rest = blockIdx.x / p.runs;
  for (; slice < p.slices; ++slice) {
    const int runs = (p.width[slice] + W * C - 1) / (W * C);
    if (run < runs) break;
    run -= runs;
    n0 += p.width[slice];
  }
  const int end = n0 + p.width[slice];
  n0 += (run * W + wave) * C;
  const bool columns = n0 < end;  // a wave without columns has its part of h to do
  const int nc = n0 + NT * col;
  const bool whole = n0 + C <= end;  // uniform
  const bool in_place = p.out == p.y && p.ldo == p.ldy;
  Tile<GATHER> tile;
  if (!find_tile(p, p.unit0 + rest / p.groups, rest % p.groups, !in_place, tile)) return;
  int row[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) row[r] = tile.row(4 * g + r);
  vecn<T, NT> y[4];
  if (columns) load_y<T, NT>(p, tile.row0, row, nc, end, whole, y);

  const int chunks = (p.k + 31) / 32, per_wave = (chunks + W - 1) / W;
  const int w0 = min(wave * per_wave, chunks), w1 = min(w0 + per_wave, chunks);
  const int full = min(w1, p.k / 32);  // chunks that K fills
  const T* const xp = static_cast<const T*>(p.x) + tile.row0 * p.ldx + tile.row(lr) * p.ldx + 8 * lc;
  float scale = 0.0f, back[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  v4f out[NT]{};
  if (!tile.known(p, !in_place)) return;
  const int id = tile.id;
  if (id >= 0) {  // uniform
    scale = p.scale != nullptr ? p.scale[id] : 1.0f;
    vec8<T> w[NT][KS];
    if (columns) load_b<T, NT, KS>(p, id, n0, end, w);
    const T* ap[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i)  // ranks past the last one: the last one again, not used
      ap[i] = static_cast<const T*>(p.a) + ((static_cast<int64_t>(id) * p.slices + slice) * p.r + min(16 * i + lr, p.r - 1)) * p.k + 8 * lc;
    v4f acc[NR]{};
    auto add = [&](const vec8<T> x, const vec8<T> (&a)[NR]) {
      const vec8<T> u = to_operand<T>(x);
#pragma unroll
      for (int i = 0; i < NR; ++i) acc[i] = mfma(u, to_operand<T>(a[i]), acc[i]);
    };
    auto load = [&](vec8<T>& x, vec8<T> (&a)[NR], int k) {
      x = *reinterpret_cast<const vec8<T>*>(xp + k);
#pragma unroll
      for (int i = 0; i < NR; ++i) a[i] = *reinterpret_cast<const vec8<T>*>(ap[i] + k);
    };
    int c = w0;
    for (; c + kAhead <= full; c += kAhead) {
      vec8<T> x[kAhead], a[kAhead][NR];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) load(x[j], a[j], 32 * (c + j));
#pragma unroll
      for (int j = 0; j < kAhead; ++j) add(x[j], a[j]);
    }
    for (; c < w1; ++c) {  // the last ones, and one that K does not fill
      vec8<T> x, a[NR];
      const bool in = 32 * c + 8 * lc < p.k;
      load(x, a, in ? 32 * c : -8 * lc);  // elsewhere the row's first elements
      if (!in) {
        x = vec8<T>{};
#pragma unroll
        for (int i = 0; i < NR; ++i) a[i] = vec8<T>{};
      }
      add(x, a);
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave < NR) {
      v4f s = part[0][wave][lane];
#pragma unroll
      for (int j = 1; j < W; ++j) s += part[j][wave][lane];
      const int rank = 16 * wave + col;
#pragma unroll
      for (int r = 0; r < 4; ++r) hs[rank / 32 * 512 + rank % 32 / 8 * 128 + (4 * g + r) * 8 + rank % 8] = s[r];
    }
    __syncthreads();
    if (columns) {
      float f[KS][8];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const v4f a = *reinterpret_cast<const v4f*>(hs + s * 512 + lane * 8), b = *reinterpret_cast<const v4f*>(hs + s * 512 + lane * 8 + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[s][e] = 32 * s + 8 * g >= p.r ? 0.0f : e < 4 ? a[e & 3] : b[e & 3];
      }
      const float unshift = shift_h<T, KS>(f);
#pragma unroll
      for (int r = 0; r < 4; ++r) back[r] = __shfl(unshift, 4 * g + r, 64);
      times_b<T, NT, KS>(p, w, f, out);
    }
  }
  if (columns) store_rows<T, NT>(p, tile.row0, row, tile.n - 4 * g, nc, end, whole, id, back, scale, out, y);
}

template <typename T, bool GATHER>
void launch_down(const LoraParams& p, int units, hipStream_t stream) {
  const unsigned tiles = static_cast<unsigned>(units) * p.groups * p.ksplit;
  const int total = p.slices * p.r;
  if (total <= 16)
    lora_down_kernel<T, 1, GATHER><<<tiles, 512, 0, stream>>>(p);
  else if (total <= 32)
    lora_down_kernel<T, 2, GATHER><<<tiles, 512, 0, stream>>>(p);
  else
    lora_down_kernel<T, 4, GATHER><<<dim3(tiles, (total + 63) / 64), 512, 0, stream>>>(p);
}

template <typename T, bool GATHER>
void launch_units(const LoraParams& p, int units, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(units) * p.groups * p.runs);
  if (p.ksplit == 0) {
    if (p.r <= 16) lora_fused_kernel<T, 1, GATHER><<<grid, 512, 0, stream>>>(p);
    else if (p.r <= 32) lora_fused_kernel<T, 2, GATHER><<<grid, 512, 0, stream>>>(p);
    else if (p.r <= 64) lora_fused_kernel<T, 4, GATHER><<<grid, 512, 0, stream>>>(p);
    else lora_fused_kernel<T, 8, GATHER><<<grid, 512, 0, stream>>>(p);
    return;
  }
  if (p.adapters > 0) launch_down<T, GATHER>(p, units, stream);
  if (p.r <= 32) lora_up_kernel<T, 1, GATHER><<<grid, 256, 0, stream>>>(p);
  else if (p.r <= 64) lora_up_kernel<T, 2, GATHER><<<grid, 256, 0, stream>>>(p);
  else lora_up_kernel<T, 4, GATHER><<<grid, 256, 0, stream>>>(p);
}

// A launch holds fewer than 2^32 threads.
constexpr int64_t kMaxWaves = 1 << 26;

// As many units at a time as a launch holds: all of them, but for windows of many adapters over very many rows, whose
// workgroups are up to 16 times those of whole tiles (a window's are 2^21 waves at most).
template <typename T, bool GATHER>
void launch(LoraParams p, hipStream_t stream) {
  const int64_t waves = p.groups * std::max<int64_t>(p.runs * (p.ksplit == 0 ? 8 : 4), p.ksplit * 8);
  const int64_t fit = (kMaxWaves - 1) / waves;
  for (int64_t at = 0; at < p.units; at += fit) {
    p.unit0 = static_cast<int32_t>(at);
    launch_units<T, GATHER>(p, static_cast<int>(std::min<int64_t>(fit, p.units - at)), stream);
  }
}

}  // namespace

int64_t lora_h_floats(int64_t m, int32_t r, int32_t slices) { return (m + 15) / 16 * slices * ((r + 31) / 32) * 512; }

constexpr int64_t kMaxPartial = int64_t{1} << 28;

// Tiles of consecutive rows where requests have 64 or more (or there is one).  Else windows: as many workgroups as a window
// can have tiles, found by counting; past 32 one for each row, the first row of a tile its workgroup's, which costs
// nothing to find.  One launch (ksplit 0) where its workgroups have a CU each and the ranks that each reads again
// are at most 128 KB (one / two launches, us: 64 KB 6.0 / 7.7, 256 KB (K = 4096, rank 32) 9.7 / 8.6, 512 KB 15.7 / 9.0).
// Else K slices for two workgroups a CU (1963 x 4096 with 96 rows of A, 260 workgroups: 32.9 us, in two slices 26.4).  More where A
// is more than an L2 holds, so that each XCD has some of the slices (us in 1 / 2 / 4 / 8: 1197 x 16384 with 256 rows
// of three adapters 137 / 91 / 79 / 77, 3553 x 16384 with 96 of 14 206 / 183 / 173 / 150, 2920 x 16384 with 64 of five
// 181 / 150 / 132 / 138), else of a long K for six workgroups a CU (12139 x 16384 with 24 of one 164 / 131 / 130 / 132).  With
// K = 2048 they cost more than they give (6208 x 32768 columns, 64 rows of A: 163 / 160 / 172 / 195).  Where rows alone
// give four workgroups a CU, two at most, for every wave of the second launch reads all planes of h (16384 x 16384 with 64
// of five 277 / 246 / 259 / 272, 65536 x 16384 with 32 of eight 1301 / 1279 / 1377 / 1539, 4096 x 4096 with 384 of eight 95 / 89
// / 90 / 119), past eight those of a long K only (65536 x 4096 with 64 of 16 443 / 466 / 527 / 685); and no planes of more than
// kMaxPartial together.
LoraPlan lora_plan(int64_t m, int64_t per_id, int32_t k, int32_t n, int32_t r, int32_t slices, int32_t adapters, int cus) {
  LoraPlan plan{};
  plan.gather = per_id < kWindow && per_id < m;
  if (plan.gather) {
    const int64_t rows = std::min<int64_t>(m, kWindow);
    const int64_t kinds = std::min<int64_t>({rows, (rows - 1) / per_id + 2, static_cast<int64_t>(adapters) + 1});
    const int64_t tiles = std::min((rows + 15 * kinds) / 16, rows);
    plan.leaders = tiles > 32;
    plan.units = static_cast<int32_t>((m + kWindow - 1) / kWindow);
    plan.groups = static_cast<int32_t>(plan.leaders ? rows : tiles);
  } else {
    plan.tiles = static_cast<int32_t>((std::min(per_id, m) + 15) / 16);
    plan.units = static_cast<int32_t>((m + per_id - 1) / per_id * plan.tiles);
    plan.groups = 1;
  }
  const int64_t all = static_cast<int64_t>(plan.units) * plan.groups;
  int64_t ranks = 16;
  while (ranks < r) ranks *= 2;
  const int64_t run = ranks <= 64 ? 1024 : 512;  // columns of a workgroup
  if (ranks * k * 2 <= (128 << 10) && all * ((n + run - 1) / run + slices - 1) <= cus) return plan;
  const int64_t down = all * ((slices * r + 63) / 64);
  const int64_t fill = std::min<int64_t>({(2 * cus + down - 1) / down, (k + 511) / 512, 8});
  const int64_t far = down < 4 * cus ? std::min<int64_t>(k / 2048, 8) : std::min<int64_t>(k / (down < 8 * cus ? 2048 : 8192), 2);
  const int64_t more = static_cast<int64_t>(adapters) * slices * r * k * 2 > (4 << 20) ? far
                                                                                      : std::min<int64_t>(k / 8192, (6 * cus + down - 1) / down);
  const int64_t most = kMaxPartial / (4 * lora_h_floats(m, r, slices));
  plan.ksplit = static_cast<int32_t>(std::max<int64_t>(1, std::min(std::max(fill, more), most)));
  return plan;
}

bool lora_grid(LoraParams& p, const LoraPlan& plan) {
  p.ksplit = plan.ksplit;
  p.groups = plan.groups;
  p.units = plan.units;
  p.tiles = plan.tiles;
  p.gather = plan.gather;
  p.leaders = plan.leaders;
  const int64_t waves = p.ksplit == 0 ? 8 : 4, columns = waves * (p.r <= 64 ? kCols<1> : kCols<4>);
  int64_t runs = 0;
  for (int s = 0; s < p.slices; ++s) runs += (p.width[s] + columns - 1) / columns;
  p.runs = static_cast<int32_t>(runs);
  p.h_plane = lora_h_floats(p.m, p.r, p.slices);
  return (p.m + 15) / 16 * runs * waves < kMaxWaves;
}

hipError_t launch_lora(const LoraParams& p, int elem, hipStream_t stream) {
  if (p.m <= 0 || p.n <= 0) return hipSuccess;
  if (elem == kFp16)
    p.gather ? launch<_Float16, true>(p, stream) : launch<_Float16, false>(p, stream);
  else
    p.gather ? launch<__bf16, true>(p, stream) : launch<__bf16, false>(p, stream);
  return hipGetLastError();
}

}  // namespace w4a4
