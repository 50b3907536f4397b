// Low-rank adapters of many requests beside a shared projection.
//
//   h[m] = A[id(m)] x[m];   out[m, n] = y[m, n] + scale[id(m)] * sum_r h[m, g(n) R + r] B[id(m), n, r]
//
// g(n) is the slice of column n (the parts of a joined projection have first factors of their own, one
// below the other in A).  Two launches on 16 x 16 x 32 matrix instructions:
//
// lora_down_kernel: 16 rows x up to 64 rows of A, the K slice of a workgroup over its four waves, joined
// in LDS; fp32 sums of each K slice to the workspace.
// lora_up_kernel: 16 rows x 64 columns a wave at a time.  h is the sum of the K slices in fp32, split into two
// 16-bit parts whose products with B are summed (fp16: after a shift that brings a row's largest into the
// upper range, so that no h overflows), so that nothing of h is lost beside the rounding of out.
//
// Rows need no order.  The adapters that occur in a tile of 16 rows are taken one by one: each is applied to the
// whole tile and kept for its own rows, and the workgroups of a tile share them out (the first row
// of each adapter in the tile stands for it).  A tile of one request has one; 16 decoded tokens of 16
// adapters have 16, whose weights have to be read anyway.  Rows without an adapter keep y.

#include <algorithm>

#include "serving_internal.h"

namespace w4a4 {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

__device__ __forceinline__ v4f mfma(const vec8<_Float16> a, const vec8<_Float16> b, const v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma(const vec8<__bf16> a, const vec8<__bf16> b, const v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The adapter of a lane's row (row = first + lane % 16; -1: none), and the rows that stand for one.
struct TileIds {
  int id;
  uint32_t leaders;  // bit i: row i is the first of its adapter in the tile (none counts as one when `none`)
  __device__ __forceinline__ TileIds(const LoraParams& p, int64_t first, bool none) {
    const int i = threadIdx.x & 15;
    const int64_t row = first + i;
    id = -2;  // behind the last row
    if (row < p.m) {
      id = p.ids[row / p.per_id];
      if (id < 0 || id >= p.adapters) id = -1;
    }
    bool lead = id >= (none ? -1 : 0);
#pragma unroll
    for (int j = 0; j < 15; ++j) {
      const int other = __builtin_amdgcn_readlane(id, j);
      if (j < i && other == id) lead = false;
    }
    leaders = static_cast<uint32_t>(__ballot(lead) & 0xffffu);
  }
};

// Rows 64 y .. of A (NR tiles of 16), K slice z.
template <typename T, int NR>
__global__ __launch_bounds__(256) void lora_down_kernel(LoraParams p) {
  constexpr int W = 4;
  __shared__ __align__(16) v4f part[W][NR][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int64_t first = static_cast<int64_t>(blockIdx.x / p.groups) * 16;
  const int which = blockIdx.x % p.groups;
  const TileIds ids(p, first, false);
  const int total = p.slices * p.r;  // rows of an adapter's A
  const int rank0 = blockIdx.y * 16 * NR;
  // Chunks of 32 elements: the slice's, dealt to the waves in runs.
  const int chunks = (p.k + 31) / 32;
  const int per_slice = (chunks + p.ksplit - 1) / p.ksplit;
  const int c0 = blockIdx.z * per_slice, c1 = min(c0 + per_slice, chunks);
  const int per_wave = (per_slice + W - 1) / W;
  const int w0 = min(c0 + wave * per_wave, c1), w1 = min(w0 + per_wave, c1);

  const int64_t xrow = min(first + col, p.m - 1);
  const T* const xp = static_cast<const T*>(p.x) + xrow * p.ldx + 8 * g;
  int n = 0;
  for (uint32_t left = ids.leaders; left != 0; left &= left - 1, ++n) {
    if (n % p.groups != which) continue;  // uniform
    const int id = __builtin_amdgcn_readlane(ids.id, __builtin_ctz(left));
    const T* ap[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i)  // rows past the last one: the last one again, not stored
      ap[i] = static_cast<const T*>(p.a) + (static_cast<int64_t>(id) * total + min(rank0 + 16 * i + col, total - 1)) * p.k + 8 * g;
    v4f acc[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int c = w0; c < w1; ++c) {
      const bool in = 32 * c + 8 * g < p.k;
      const vec8<T> x = in ? *reinterpret_cast<const vec8<T>*>(xp + 32 * c) : vec8<T>{};
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const vec8<T> a = in ? *reinterpret_cast<const vec8<T>*>(ap[i] + 32 * c) : vec8<T>{};
        acc[i] = mfma(x, a, acc[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    for (int i = wave; i < NR; i += W) {
      v4f s = part[0][i][lane];
#pragma unroll
      for (int w = 1; w < W; ++w) s += part[w][i][lane];
      const int rank = rank0 + 16 * i + col;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int of = __shfl(ids.id, 4 * g + r, 64);  // rows 4 g + r of the tile
        if (of == id && rank < total)
          p.h[(static_cast<int64_t>(blockIdx.z) * p.m + first + 4 * g + r) * total + rank] = s[r];
      }
    }
    __syncthreads();
  }
}

// Columns: blocks of 64 of each slice, one a wave.
template <typename T, int KS>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraParams p) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int64_t first = static_cast<int64_t>(blockIdx.x / p.groups) * 16;
  const int which = blockIdx.x % p.groups;
  int block = blockIdx.y * 4 + wave, slice = 0, n0 = 0;
  while (slice < p.slices && block >= (p.width[slice] + 63) / 64) {
    block -= (p.width[slice] + 63) / 64;
    n0 += p.width[slice];
    ++slice;
  }
  if (slice == p.slices) return;  // no barrier below
  const int end = n0 + p.width[slice];
  n0 += 64 * block;
  const bool in_place = p.out == p.y && p.ldo == p.ldy;
  const TileIds ids(p, first, !in_place);
  const int total = p.slices * p.r;
  const int64_t row = min(first + col, p.m - 1);
  // This lane's 16 columns of its row.
  const int nc = n0 + 16 * g;
  const T* const yp = static_cast<const T*>(p.y) + row * p.ldy + nc;
  T* const op = static_cast<T*>(p.out) + row * p.ldo + nc;
  const bool whole = nc + 16 <= end && p.ldy % 8 == 0 && p.ldo % 8 == 0 && nc % 8 == 0 &&
                     (reinterpret_cast<uintptr_t>(p.y) & 15) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;

  // h of the lane's row, ranks 32 s + 8 g .. + 7, as two parts.
  vec8<T> hi[KS], lo[KS];
  float back = 1.0f;
  {
    float f[KS][8];
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int r = 32 * s + 8 * g;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[s][e] = 0.0f;
      if (r < p.r && ids.id >= 0) {
        const float* hp = p.h + row * total + slice * p.r + r;
        for (int z = 0; z < p.ksplit; ++z, hp += p.m * total) {
          const v4f u = *reinterpret_cast<const v4f*>(hp), v = *reinterpret_cast<const v4f*>(hp + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[s][e] += u[e];
            f[s][4 + e] += v[e];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(f[s][e]));
    }
    float shift = 1.0f;
    if constexpr (static_cast<float>(static_cast<T>(65536.0f)) > 1e30f) {  // fp16
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      // The largest to 2^13 .. 2^14; nothing to do for rows of zeros, infinities or NaN.
      const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
      if (top > 0.0f && e < 128) {
        const int by = max(min(13 - e, 126), -126);
        shift = __uint_as_float(static_cast<uint32_t>(127 + by) << 23);
        back = __uint_as_float(static_cast<uint32_t>(127 - by) << 23);
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
  }

  int n = 0;
  for (uint32_t left = ids.leaders; left != 0; left &= left - 1, ++n) {
    if (n % p.groups != which) continue;
    const int id = __builtin_amdgcn_readlane(ids.id, __builtin_ctz(left));
    v4f acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (id >= 0) {
      const T* const bp = static_cast<const T*>(p.b) + static_cast<int64_t>(id) * p.n * p.r + 8 * g;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        // Row i of tile t is column 16 (i / 4) + 4 t + i % 4 of the block: a lane ends with 16 consecutive ones.
        const int nb = min(n0 + 16 * (col >> 2) + 4 * t + (col & 3), end - 1);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          vec8<T> w{};
          if (32 * s + 8 * g < p.r) w = *reinterpret_cast<const vec8<T>*>(bp + static_cast<int64_t>(nb) * p.r + 32 * s);
          acc[t] = mfma(w, hi[s], acc[t]);
          acc[t] = mfma(w, lo[s], acc[t]);
        }
      }
    }
    if (ids.id != id) continue;  // the rows of other adapters
    const float scale = id < 0 ? 0.0f : (p.scale != nullptr ? p.scale[id] : 1.0f);
    if (whole) {
      const vec8<T> y0 = *reinterpret_cast<const vec8<T>*>(yp), y1 = *reinterpret_cast<const vec8<T>*>(yp + 8);
      vec8<T> z0 = y0, z1 = y1;
      if (id >= 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          z0[e] = static_cast<T>(fmaf(acc[e >> 2][e & 3] * back, scale, static_cast<float>(y0[e])));
          z1[e] = static_cast<T>(fmaf(acc[2 + (e >> 2)][e & 3] * back, scale, static_cast<float>(y1[e])));
        }
      }
      *reinterpret_cast<vec8<T>*>(op) = z0;
      *reinterpret_cast<vec8<T>*>(op + 8) = z1;
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (nc + e >= end) continue;
        const T y = yp[e];
        op[e] = id >= 0 ? static_cast<T>(fmaf(acc[e >> 2][e & 3] * back, scale, static_cast<float>(y))) : y;
      }
    }
  }
}

template <typename T>
void launch(const LoraParams& p, hipStream_t stream) {
  const unsigned tiles = static_cast<unsigned>((p.m + 15) / 16 * p.groups);
  const int total = p.slices * p.r;
  if (p.adapters > 0) {
    if (total <= 16)
      lora_down_kernel<T, 1><<<dim3(tiles, 1, p.ksplit), 256, 0, stream>>>(p);
    else if (total <= 32)
      lora_down_kernel<T, 2><<<dim3(tiles, 1, p.ksplit), 256, 0, stream>>>(p);
    else
      lora_down_kernel<T, 4><<<dim3(tiles, (total + 63) / 64, p.ksplit), 256, 0, stream>>>(p);
  }
  int blocks = 0;
  for (int s = 0; s < p.slices; ++s) blocks += (p.width[s] + 63) / 64;
  const dim3 grid(tiles, (blocks + 3) / 4);
  if (p.r <= 32)
    lora_up_kernel<T, 1><<<grid, 256, 0, stream>>>(p);
  else if (p.r <= 64)
    lora_up_kernel<T, 2><<<grid, 256, 0, stream>>>(p);
  else
    lora_up_kernel<T, 4><<<grid, 256, 0, stream>>>(p);
}

}  // namespace

// K slices for as many workgroups as CUs where row tiles are few; a tile's adapters go to as many workgroups
// as it can have adapters, where tiles are few.
LoraPlan lora_plan(int64_t m, int64_t per_id, int32_t k, int32_t n, int32_t r, int32_t slices, int32_t adapters, int cus) {
  const int64_t tiles = (m + 15) / 16;
  const int64_t most = std::min<int64_t>({16, 15 / per_id + 2, adapters + 1});
  LoraPlan plan;
  plan.groups = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, 4 * cus / tiles)));
  const int64_t down = tiles * plan.groups * ((slices * r + 63) / 64);
  plan.ksplit = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({cus / down, (k + 511) / 512, 8})));
  return plan;
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
