// Rows of 16-bit elements to int8 codes with one scale each, as they are, behind an RMSNorm, or
// behind a residual add and an RMSNorm.
//
//   h = T(x + residual)                                   (written back: the residual stream)
//   y = h g r,  g = 1 + w or w,  r = 1 / sqrt(mean(h^2) + eps)
//   s = max|y| / 127 + 1e-12,  c = rint(y / s)
//
// One pass: max|y| = r max|h g|, so the sum of squares and the maximum are reduced together, and
// a code is rint(h g c) with c = r / s, one fused multiply-add onto 1.5 * 2^23, whose low byte is
// the rounded code in two's complement (round half to even, |code| <= 127).  The norm is held in
// fp32 throughout; nothing is rounded between the norm and the code.
// The maximum is taken of the bits of |h g| as integers, in which a NaN is larger than every
// number: a row that holds a NaN or an infinity gets the scale NaN and codes 0.
// bf16 rows can leave fp32's range in h^2 or h g where y does not.  Such a row is read again, its squares are
// taken of h 2^96 or h 2^-96, and it goes on as the rows y themselves with r = 1; only a y past fp32 makes the
// scale NaN.
//
// Bound by HBM: 7 bytes an element in the add form, 3 in the others; 6208 x 2048 with the add take 17.0
// us, 5.2 TB/s, where a copy reaches 4.96.  A row belongs to one wave (K <= 2048 and enough rows) or to
// a workgroup, 8 elements of a thread at a time; it is read once and stays in registers.  A single row
// takes 2.2 us, its loads' and stores' latency.

#include "int8_internal.h"
#include "quant_row.h"

namespace w4a4 {
namespace {

template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, static_cast<uint32_t>(lane_xor_i<0>(static_cast<int>(v))));
  v = max(v, static_cast<uint32_t>(lane_xor_i<1>(static_cast<int>(v))));
  v = max(v, static_cast<uint32_t>(lane_xor_i<2>(static_cast<int>(v))));
  v = max(v, static_cast<uint32_t>(lane_xor_i<3>(static_cast<int>(v))));
  auto r16 = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(r16[0], r16[1]);
  auto r32 = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(r32[0], r32[1]);
}

constexpr float kRintMagic = 12582912.0f;  // 1.5 * 2^23
constexpr float kMax = 3.4028235e38f;

// WPR waves share a row; a thread holds CPT chunks of 8 elements, chunk j * 64 WPR + its index.
template <typename T, bool NORM, bool ADD, int WPR, int CPT>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void int8_rows_kernel(Int8RowsParams p) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int64_t row = WPR == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + wave : blockIdx.x;
  if (WPR == 1 && row >= p.m) return;  // the wave owns its row: no barrier below
  const int t = WPR == 1 ? lane : threadIdx.x;
  const int chunks = p.k >> 3;
  const T* const x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* const res = static_cast<const T*>(p.res) + (ADD ? row * p.ldr : 0);
  const T* const wt = static_cast<const T*>(p.w);

  vec8<T> v[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    const int c = j * 64 * WPR + t;
    v[j] = c < chunks ? *reinterpret_cast<const vec8<T>*>(x + 8 * c) : vec8<T>{};
  }
  if constexpr (ADD) {
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      const int c = j * 64 * WPR + t;
      if (c >= chunks) continue;
      const vec8<T> r = *reinterpret_cast<const vec8<T>*>(res + 8 * c);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] = static_cast<T>(static_cast<float>(v[j][e]) + static_cast<float>(r[e]));
      *reinterpret_cast<vec8<T>*>(static_cast<T*>(p.h) + row * p.k + 8 * c) = v[j];
    }
  }
  float f[CPT][8];  // h g
  float ss = 0.0f;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    const int c = j * 64 * WPR + t;
    vec8<T> g{};
    if (NORM && c < chunks) g = *reinterpret_cast<const vec8<T>*>(wt + 8 * c);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float h = static_cast<float>(v[j][e]);
      f[j][e] = h;
      if constexpr (NORM) {
        ss = fmaf(h, h, ss);
        f[j][e] = h * (p.unit_offset ? 1.0f + static_cast<float>(g[e]) : static_cast<float>(g[e]));
      }
      if (c < chunks) top = max(top, __float_as_uint(f[j][e]) & 0x7fffffffu);
    }
  }
  // Over the waves of the row; every thread holds the results.
  __shared__ float red_ss[WPR];
  __shared__ uint32_t red_top[WPR];
  auto reduce = [&]() {
    top = wave_max_u32(top);
    if constexpr (NORM) ss = wave_sum_f(ss);
    if constexpr (WPR > 1) {
      if (lane == 0) {
        red_ss[wave] = ss;
        red_top[wave] = top;
      }
      __syncthreads();
      ss = red_ss[0];
      top = red_top[0];
#pragma unroll
      for (int i = 1; i < WPR; ++i) {
        ss += red_ss[i];
        top = max(top, red_top[i]);
      }
    }
  };
  reduce();
  float r = 1.0f;
  if constexpr (NORM) {
    const float mean = ss / static_cast<float>(p.k) + p.eps;
    r = 1.0f / __builtin_sqrtf(mean);
    // fp16 does not come here but for what is not finite: 2^32 * 32768 at most, 2^-48 at least.
    if (!(ss <= kMax) || mean < 1e-30f || !(__uint_as_float(top) <= kMax)) {  // uniform over the row
      const float c = !(ss <= kMax) ? 0x1p-96f : mean < 1e-30f ? 0x1p96f : 1.0f;
      const T* const again = ADD ? static_cast<const T*>(p.h) + row * p.k : x;  // h, as this thread wrote it
      if constexpr (WPR > 1) __syncthreads();  // the first sums have been read
      ss = 0.0f;
#pragma unroll 1
      for (int i = t; i < chunks; i += 64 * WPR) {
        const vec8<T> h = *reinterpret_cast<const vec8<T>*>(again + 8 * i);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float hc = static_cast<float>(h[e]) * c;
          ss = fmaf(hc, hc, ss);
        }
      }
      reduce();
      const float rc = 1.0f / __builtin_sqrtf(ss / static_cast<float>(p.k) + p.eps * c * c);
      top = 0;
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        const int i = j * 64 * WPR + t;
        if (i >= chunks) continue;
        const vec8<T> h = *reinterpret_cast<const vec8<T>*>(again + 8 * i);
        const vec8<T> g = *reinterpret_cast<const vec8<T>*>(wt + 8 * i);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f[j][e] = static_cast<float>(h[e]) * c * rc * (p.unit_offset ? 1.0f + static_cast<float>(g[e]) : static_cast<float>(g[e]));
          top = max(top, __float_as_uint(f[j][e]) & 0x7fffffffu);
        }
      }
      if constexpr (WPR > 1) __syncthreads();  // the second sums have been read
      reduce();
      r = 1.0f;
    }
  }
  const float amax = __uint_as_float(top) * r;
  const bool finite = amax <= kMax;  // false for NaN too
  const float s = amax / 127.0f + 1e-12f;
  const float cf = finite ? r * (1.0f / s) : 0.0f;
  if (t == 0) p.scale[row] = finite ? s : __builtin_nanf("");
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    const int c = j * 64 * WPR + t;
    if (c >= chunks) continue;
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = finite ? __float_as_uint(fmaf(f[j][e], cf, kRintMagic)) : 0u;
    uint2 o;
    o.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
    o.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[7], b[6], 0x0c0c0400u), __builtin_amdgcn_perm(b[5], b[4], 0x0c0c0400u), 0x05040100u);
    *reinterpret_cast<uint2*>(p.q + row * p.k + 8 * c) = o;
  }
}

template <typename T, bool NORM, bool ADD, int WPR>
void launch_cpt(const Int8RowsParams& p, int cpt, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(WPR == 1 ? (p.m + 3) / 4 : p.m));
  const int threads = WPR == 1 ? 256 : 64 * WPR;
  if (cpt <= 1)
    int8_rows_kernel<T, NORM, ADD, WPR, 1><<<grid, threads, 0, stream>>>(p);
  else if (cpt <= 2)
    int8_rows_kernel<T, NORM, ADD, WPR, 2><<<grid, threads, 0, stream>>>(p);
  else
    int8_rows_kernel<T, NORM, ADD, WPR, 4><<<grid, threads, 0, stream>>>(p);
}

template <typename T, bool NORM, bool ADD>
void launch_form(const Int8RowsParams& p, hipStream_t stream) {
  const int chunks = p.k / 8;
  // One wave a row where the rows give every SIMD one; else, and for longer rows, a workgroup (us, K = 2048,
  // with 1 / 4 / 16 waves: 64 rows 4.3 / 3.4 / 3.5, 512 rows 4.6 / 3.8 / 4.7, 1024 rows 5.3 / 5.2 / 7.4, 6208 rows
  // 17.4 / 17.2 / 30; K = 512, 6208 rows 7.3 / 10.0 / 28; K = 8192, 512 rows - / 8.0 / 8.7).
  if (chunks <= 4 * 64 && p.m >= 4 * device_cu_count())
    launch_cpt<T, NORM, ADD, 1>(p, (chunks + 63) / 64, stream);
  else if (chunks <= 4 * 256)
    launch_cpt<T, NORM, ADD, 4>(p, (chunks + 255) / 256, stream);
  else
    launch_cpt<T, NORM, ADD, 16>(p, (chunks + 1023) / 1024, stream);
}

template <typename T>
void launch_elem(const Int8RowsParams& p, hipStream_t stream) {
  if (p.res != nullptr)
    launch_form<T, true, true>(p, stream);
  else if (p.w != nullptr)
    launch_form<T, true, false>(p, stream);
  else
    launch_form<T, false, false>(p, stream);
}

}  // namespace

hipError_t launch_int8_rows(const Int8RowsParams& p, int elem, hipStream_t stream) {
  if (p.m <= 0) return hipSuccess;
  if (elem == kFp16)
    launch_elem<_Float16>(p, stream);
  else
    launch_elem<__bf16>(p, stream);
  return hipGetLastError();
}

}  // namespace w4a4
