// Low-rank adapters of many requests beside a shared projection.
//
//   h[m] = A[id(m)] x[m];   out[m, n] = y[m, n] + scale[id(m)] * sum_r h[m, g(n) R + r] B[id(m), n, r]
//
// g(n) is the slice of column n (the parts of a joined projection have first factors of their own, one
// below the other in A).  Two launches on 16 x 16 x 32 matrix instructions:
//
// lora_down_kernel: 16 rows x up to 64 rows of A, the K slice of a workgroup over its eight waves, joined
// in LDS; fp32 sums of each K slice to the workspace.
// lora_up_kernel: 16 rows x 128 columns a wave.  h is the sum of the K slices in fp32, split into two 16-bit
// parts whose products with B are summed (fp16: after a shift that brings a row's largest into the upper
// range, so that no h overflows), so that nothing of h is lost beside the rounding of out.
//
// Rows need no order.  The adapters that occur in a tile of 16 rows are taken one by one: each is applied to the
// whole tile and kept for its own rows, and the workgroups of a tile share them out.  A tile of one request
// has one; 16 decoded tokens of 16 adapters have 16, whose weights have to be read anyway.  Rows without an
// adapter keep y.
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

// h between the launches: blocks of 16 rows x 32 ranks of a slice, [K slice, row tile, slice, ranks / 32], as the lanes
// of the second launch take them: lane 16 g + row has ranks 8 g .. + 7.
__device__ __forceinline__ int64_t lora_h_index(const LoraParams& p, int64_t tile, int slice, int s) {
  return ((tile * p.slices + slice) * ((p.r + 31) / 32) + s) * 512;
}

__device__ __forceinline__ int lora_raw_id(const LoraParams& p, int64_t row) {
  return p.ids[static_cast<uint32_t>(row) / static_cast<uint32_t>(p.per_id)];  // M and per_id <= 2^26
}
// -1: no adapter, -2: behind the last row.
__device__ __forceinline__ int lora_id(const LoraParams& p, int raw, int64_t row) {
  return row >= p.m ? -2 : raw < 0 || raw >= p.adapters ? -1 : raw;
}

// Calls f(id) for every which-th of a tile's adapters, in the order of their first rows (-1 among them when `none`).
// `id` is that of the tile's row lane % 16.  Uniform over the workgroup.
template <typename F>
__device__ __forceinline__ void each_adapter(int id, bool none, int which, int groups, F f) {
  uint32_t left = static_cast<uint32_t>(__ballot(id >= (none ? -1 : 0))) & 0xffffu;
  for (int n = 0; left != 0; ++n) {
    const int now = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
    left &= ~static_cast<uint32_t>(__ballot(id == now));
    if (n % groups == which) f(now);
  }
}

// Rows 16 NR y .. of A, K slice z; the slice's chunks of 32 elements are dealt to the waves in runs.
// Bound by the arrival of x and A (A from the L2 for all row tiles but the first): kAhead chunks of both are
// under way at once.  6208 x 2048 with 64 rows of A: 17 us.
template <typename T, int NR>
__global__ __launch_bounds__(512) void lora_down_kernel(LoraParams p) {
  constexpr int W = 8, kAhead = 4;
  __shared__ __align__(16) v4f part[W][NR][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int lr = lane >> 2, lc = lane & 3;  // row and chunk that the lane loads
  const int tile = blockIdx.x / p.groups;
  const int64_t first = 16LL * tile;
  const int64_t row = first + col;
  const int my_id = lora_id(p, lora_raw_id(p, min(row, p.m - 1)), row);
  const int total = p.slices * p.r;  // rows of an adapter's A
  const int rank0 = blockIdx.y * 16 * NR;
  const int chunks = (p.k + 31) / 32;
  const int per_slice = (chunks + p.ksplit - 1) / p.ksplit;
  const int c0 = blockIdx.z * per_slice, c1 = min(c0 + per_slice, chunks);
  const int per_wave = (per_slice + W - 1) / W;
  const int w0 = min(c0 + wave * per_wave, c1), w1 = min(w0 + per_wave, c1);
  const int whole = min(w1, p.k / 32);  // chunks that K fills

  const T* const xp = static_cast<const T*>(p.x) + min(first + lr, p.m - 1) * p.ldx + 8 * lc;
  each_adapter(my_id, false, blockIdx.x % p.groups, p.groups, [&](int id) {
    const T* ap[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i)  // rows past the last one: the last one again, not stored
      ap[i] = static_cast<const T*>(p.a) + (static_cast<int64_t>(id) * total + min(rank0 + 16 * i + lr, total - 1)) * p.k + 8 * lc;
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
      const int rank = rank0 + 16 * i + col;
      float* const hp = p.h + blockIdx.z * p.h_plane + lora_h_index(p, tile, rank / p.r, rank % p.r / 32) +
                        (rank % p.r % 32 / 8) * 128 + rank % p.r % 8;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int of = __shfl(my_id, 4 * g + r, 64);  // row 4 g + r of the tile
        if (of == id && rank < total) hp[(4 * g + r) * 8] = s[r];
      }
    }
    __syncthreads();
  });
}

// The lane's row of h, ranks 32 s + 8 g .. + 7, as two 16-bit parts; returns the factor that takes the products back.
template <typename T, int KS>
__device__ __forceinline__ float split_h(const float (&f)[KS][8], vec8<T> (&hi)[KS], vec8<T> (&lo)[KS]) {
  float shift = 1.0f, unshift = 1.0f;
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
    if (top > 0.0f && e < 128) {
      const int by = max(min(13 - e, 126), -126);
      shift = __uint_as_float(static_cast<uint32_t>(127 + by) << 23);
      unshift = __uint_as_float(static_cast<uint32_t>(127 - by) << 23);
    }
  }
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = f[s][e] * shift;
      hi[s][e] = static_cast<T>(v);
      lo[s][e] = static_cast<T>(v - static_cast<float>(hi[s][e]));
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
__device__ __forceinline__ void times_b(const LoraParams& p, const vec8<T> (&w)[NT][KS], const vec8<T> (&hi)[KS],
                                        const vec8<T> (&lo)[KS], v4f (&acc)[NT]) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      vec8<T> u = to_operand<T>(w[i][s]);
      if (32 * s + 8 * g >= p.r) u = vec8<T>{};
      acc[i] = mfma(hi[s], u, acc[i]);
      acc[i] = mfma(lo[s], u, acc[i]);
    }
  }
}

// y of the lane: rows 4 g + r of the tile (past the last one: the last one again), columns nc .. + NT - 1.
template <typename T, int NT>
using vecn = T __attribute__((ext_vector_type(NT)));
template <typename T, int NT>
using vecn_h = T __attribute__((ext_vector_type(NT), aligned(2)));  // at any element
template <typename T, int NT>
__device__ __forceinline__ void load_y(const LoraParams& p, int64_t first, int nc, int end, bool whole, vecn<T, NT> (&y)[4]) {
  const int g = (threadIdx.x & 63) >> 4;
  const int last = static_cast<int>(min(p.m - 1 - first, static_cast<int64_t>(15)));
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const T* const yp = static_cast<const T*>(p.y) + first * p.ldy + min(4 * g + r, last) * p.ldy + nc;
    if (whole) {
      y[r] = *reinterpret_cast<const vecn_h<T, NT>*>(yp);
    } else {
#pragma unroll
      for (int e = 0; e < NT; ++e) y[r][e] = nc + e < end ? yp[e] : static_cast<T>(0.0f);
    }
  }
}

// The rows of adapter id (-1: as they were).
template <typename T, int NT>
__device__ __forceinline__ void store_rows(const LoraParams& p, int64_t first, int nc, int end, bool whole, int id, const int (&of)[4],
                                           const float (&back)[4], float scale, const v4f (&acc)[NT], const vecn<T, NT> (&y)[4]) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (of[r] != id) continue;
    vecn<T, NT> z = y[r];
    if (id >= 0) {
#pragma unroll
      for (int e = 0; e < NT; ++e) z[e] = static_cast<T>(fmaf(acc[e][r] * back[r], scale, static_cast<float>(z[e])));
    }
    T* const op = static_cast<T*>(p.out) + first * p.ldo + (4 * g + r) * p.ldo + nc;
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
// many: 6208 x 32768 with rank 32, both launches 165 us, 5.1 TB/s.
template <int KS>
constexpr int kCols = KS <= 2 ? 128 : 64;

// KS: ranks / 32.
template <typename T, int KS>
__global__ __launch_bounds__(256, KS == 1 ? 4 : 2) void lora_up_kernel(LoraParams p) {
  constexpr int C = kCols<KS>, NT = C / 16;  // a lane's consecutive columns
  constexpr int ZA = KS == 1 ? 4 : 1;        // K slices of h that are loaded at once
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  // The workgroup's four blocks within a slice, its rows, and its part of their adapters.
  int run = blockIdx.x % p.runs, slice = 0, n0 = 0;
  const int rest = blockIdx.x / p.runs;
  const int which = rest % p.groups, tile = rest / p.groups;
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

  // The ids, h (ranks 32 s + 8 g .. + 7 of row `col`) and y (columns nc .. + NT - 1 of rows 4 g + r).  Rows past the last
  // one are the last one again.
  const int64_t first = 16LL * tile;
  const int last = static_cast<int>(min(p.m - 1 - first, static_cast<int64_t>(15)));
  const int raw = lora_raw_id(p, first + min(col, last));
  v4f part[ZA][KS][2];
  if (p.adapters > 0) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float* const hp = p.h + lora_h_index(p, tile, slice, s) + lane * 8;
#pragma unroll
      for (int z = 0; z < ZA; ++z)
        if (z < p.ksplit) {
          part[z][s][0] = *reinterpret_cast<const v4f*>(hp + z * p.h_plane);
          part[z][s][1] = *reinterpret_cast<const v4f*>(hp + z * p.h_plane + 4);
        }
    }
  }
  vecn<T, NT> y[4];
  load_y<T, NT>(p, first, nc, end, whole, y);

  const int my_id = lora_id(p, raw, first + col);
  vec8<T> hi[KS], lo[KS];
  float unshift;
  {
    float f[KS][8];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[s][e] = p.adapters > 0 ? part[0][s][e >> 2][e & 3] : 0.0f;
#pragma unroll
      for (int z = 1; z < ZA; ++z)
        if (z < p.ksplit) {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[s][e] += part[z][s][e >> 2][e & 3];
        }
      for (int z = ZA; z < p.ksplit; ++z) {
        const float* const hp = p.h + lora_h_index(p, tile, slice, s) + lane * 8 + z * p.h_plane;
        const v4f a = *reinterpret_cast<const v4f*>(hp), b = *reinterpret_cast<const v4f*>(hp + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[s][e] += a[e];
          f[s][4 + e] += b[e];
        }
      }
      if (32 * s + 8 * g >= p.r) {  // past the last rank: anything
#pragma unroll
        for (int e = 0; e < 8; ++e) f[s][e] = 0.0f;
      }
    }
    unshift = split_h<T, KS>(f, hi, lo);
  }
  // What the lane ends with are rows 4 g + r, whose adapters and factors are in other lanes.
  float back[4];
  int of[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    back[r] = __shfl(unshift, 4 * g + r, 64);
    of[r] = __shfl(my_id, 4 * g + r, 64);
  }
  each_adapter(my_id, !in_place, which, p.groups, [&](int id) {
    float scale = 0.0f;
    v4f acc[NT]{};
    if (id >= 0) {
      scale = p.scale != nullptr ? p.scale[id] : 1.0f;
      vec8<T> w[NT][KS];
      load_b<T, NT, KS>(p, id, n0, end, w);
      times_b<T, NT, KS>(p, w, hi, lo, acc);
    }
    store_rows<T, NT>(p, first, nc, end, whole, id, of, back, scale, acc, y);
  });
}

// Both products in one launch, for few rows: a workgroup computes h of its tile, adapter and slice itself (its eight
// waves each an eighth of K, joined in LDS) while B and y are under way, and its waves take a block of kCols columns each.
// Bound by the arrival of A at one CU.  One row into 2560 columns in three slices: 6.0 us, two launches 7.7; 64 rows of
// 64 adapters into 2048: 8.3, 9.8.
template <typename T, int NR>
__global__ __launch_bounds__(512) void lora_fused_kernel(LoraParams p) {
  constexpr int W = 8, KS = (NR + 1) / 2, C = kCols<KS>, NT = C / 16;
  constexpr int kAhead = NR <= 2 ? 8 : 16 / NR;
  __shared__ __align__(16) v4f part[W][NR][64];
  __shared__ __align__(16) float hs[KS * 512];  // as lora_h_index has a tile's block
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int lr = lane >> 2, lc = lane & 3;  // row and chunk that the lane loads
  int run = blockIdx.x % p.runs, slice = 0, n0 = 0;
  const int rest = blockIdx.x / p.runs;
  const int which = rest % p.groups, tile = rest / p.groups;
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
  const int64_t first = 16LL * tile;
  const int my_id = lora_id(p, lora_raw_id(p, min(first + col, p.m - 1)), first + col);
  vecn<T, NT> y[4];
  if (columns) load_y<T, NT>(p, first, nc, end, whole, y);
  int of[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) of[r] = __shfl(my_id, 4 * g + r, 64);

  const int chunks = (p.k + 31) / 32, per_wave = (chunks + W - 1) / W;
  const int w0 = min(wave * per_wave, chunks), w1 = min(w0 + per_wave, chunks);
  const int full = min(w1, p.k / 32);  // chunks that K fills
  const T* const xp = static_cast<const T*>(p.x) + min(first + lr, p.m - 1) * p.ldx + 8 * lc;
  each_adapter(my_id, !in_place, which, p.groups, [&](int id) {
    float scale = 0.0f, back[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    v4f out[NT]{};
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
        vec8<T> hi[KS], lo[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const v4f a = *reinterpret_cast<const v4f*>(hs + s * 512 + lane * 8), b = *reinterpret_cast<const v4f*>(hs + s * 512 + lane * 8 + 4);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[s][e] = 32 * s + 8 * g >= p.r ? 0.0f : e < 4 ? a[e & 3] : b[e & 3];
        }
        const float unshift = split_h<T, KS>(f, hi, lo);
#pragma unroll
        for (int r = 0; r < 4; ++r) back[r] = __shfl(unshift, 4 * g + r, 64);
        times_b<T, NT, KS>(p, w, hi, lo, out);
      }
    }
    if (columns) store_rows<T, NT>(p, first, nc, end, whole, id, of, back, scale, out, y);
  });
}

template <typename T>
void launch_down(const LoraParams& p, hipStream_t stream) {
  const unsigned tiles = static_cast<unsigned>((p.m + 15) / 16 * p.groups);
  const int total = p.slices * p.r;
  if (total <= 16)
    lora_down_kernel<T, 1><<<dim3(tiles, 1, p.ksplit), 512, 0, stream>>>(p);
  else if (total <= 32)
    lora_down_kernel<T, 2><<<dim3(tiles, 1, p.ksplit), 512, 0, stream>>>(p);
  else
    lora_down_kernel<T, 4><<<dim3(tiles, (total + 63) / 64, p.ksplit), 512, 0, stream>>>(p);
}

template <typename T, int KS>
void launch_up(const LoraParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.m + 15) / 16 * p.groups * p.runs));
  lora_up_kernel<T, KS><<<grid, 256, 0, stream>>>(p);
}

template <typename T, int NR>
void launch_fused(const LoraParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.m + 15) / 16 * p.groups * p.runs));
  lora_fused_kernel<T, NR><<<grid, 512, 0, stream>>>(p);
}

template <typename T>
void launch(const LoraParams& p, hipStream_t stream) {
  if (p.ksplit == 0) {
    if (p.r <= 16) launch_fused<T, 1>(p, stream);
    else if (p.r <= 32) launch_fused<T, 2>(p, stream);
    else if (p.r <= 64) launch_fused<T, 4>(p, stream);
    else launch_fused<T, 8>(p, stream);
    return;
  }
  if (p.adapters > 0) launch_down<T>(p, stream);
  if (p.r <= 32) launch_up<T, 1>(p, stream);
  else if (p.r <= 64) launch_up<T, 2>(p, stream);
  else launch_up<T, 4>(p, stream);
}

}  // namespace

int64_t lora_h_floats(int64_t m, int32_t r, int32_t slices) { return (m + 15) / 16 * slices * ((r + 31) / 32) * 512; }

// A tile's adapters go to as many workgroups as it can have adapters, where tiles are few.  One launch (ksplit 0) where its
// workgroups have a CU each and the ranks that each reads again are at most 128 KB (one / two launches, us: 64 KB 6.0 / 7.7,
// 256 KB (K = 4096, rank 32) 9.7 / 8.6, 512 KB 15.7 / 9.0; 256 rows of 64 adapters, 1024 workgroups, 27.6 / 21.1).  Else K slices
// for as many workgroups as CUs.
LoraPlan lora_plan(int64_t m, int64_t per_id, int32_t k, int32_t n, int32_t r, int32_t slices, int32_t adapters, int cus) {
  LoraPlan plan;
  const int64_t tiles = (m + 15) / 16;
  const int64_t most = std::min<int64_t>({16, 15 / per_id + 2, adapters + 1});
  plan.groups = per_id >= 16 ? 1 : static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, 2 * cus / tiles)));
  int64_t ranks = 16;
  while (ranks < r) ranks *= 2;
  const int64_t run = ranks <= 64 ? 1024 : 512;  // columns of a workgroup
  if (ranks * k * 2 <= (128 << 10) && tiles * plan.groups * ((n + run - 1) / run + slices - 1) <= cus) {
    plan.ksplit = 0;
    return plan;
  }
  const int64_t down = tiles * plan.groups * ((slices * r + 63) / 64);
  plan.ksplit = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({cus / down, (k + 511) / 512, 8})));
  return plan;
}

bool lora_grid(LoraParams& p) {
  const int64_t waves = p.ksplit == 0 ? 8 : 4, columns = waves * (p.r <= 64 ? kCols<1> : kCols<4>);
  int64_t runs = 0;
  for (int s = 0; s < p.slices; ++s) runs += (p.width[s] + columns - 1) / columns;
  p.runs = static_cast<int32_t>(runs);
  p.h_plane = lora_h_floats(p.m, p.r, p.slices);
  return (p.m + 15) / 16 * p.groups * runs * waves < (1 << 26);
}

hipError_t launch_lora(const LoraParams& p, int elem, hipStream_t stream) {
  if (p.m <= 0 || p.n <= 0) return hipSuccess;
  if (elem == kFp16)
    launch<_Float16>(p, stream);
  else
    launch<__bf16>(p, stream);
  return hipGetLastError();
}

}  // namespace w4a4
