// Product of int8 codes with scales for each token (row of q) and channel (row of w):
//
//   y[m, n] = T( float(sum_k q[m, k] w[n, k]) * sq[m] * sw[n] + bias[n] + residual[m, n] )
//
// on v_mfma_i32_16x16x64_i8: the int32 sums are exact (K <= 65536), so neither tile, nor K split, nor
// order changes a result; the epilogue runs in fp32 and rounds once.  Both operands are row-major
// with K contiguous, as the quantizer writes them: no layout of the weights' own.
//
// The weights are MFMA operand A, so that a lane ends with four consecutive columns of one row.
// In a 64-deep step lane L holds k = 16 (L / 16) .. + 15 of row L % 16 of either operand.
//
// Two kernels:
//   int8_tile_kernel    BM x BN tiles through LDS, for everything but few rows: bound by the MFMAs
//                       (many rows) or by latency (few tiles);
//   int8_stream_kernel  up to 64 rows: the weights stream from memory straight into registers,
//                       the waves of a workgroup split K.

#include "direct_load.h"
#include "int8_internal.h"

namespace w4a4 {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
template <typename T>
using vec4 = T __attribute__((ext_vector_type(4)));

// y[row, col .. col + 3] of one accumulator quad, with the bias and the residual: fp32, one
// rounding.  `whole`: four columns inside N whose loads are aligned.
template <typename T>
struct Epilogue {
  const Int8GemmParams& p;
  bool res_vec;  // residual quads can be read as one aligned load
  __device__ explicit Epilogue(const Int8GemmParams& q) : p(q) {
    res_vec = (q.n & 3) == 0 && (q.ldr & 3) == 0 && (reinterpret_cast<uintptr_t>(q.res) & 7) == 0;
  }
  __device__ __forceinline__ void scales(int64_t col, float (&sw)[4], float (&bias)[4]) const {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t c = min(col + r, static_cast<int64_t>(p.n) - 1);
      sw[r] = p.sw[c];
      bias[r] = p.bias != nullptr ? static_cast<float>(static_cast<const T*>(p.bias)[c]) : 0.0f;
    }
  }
  __device__ __forceinline__ vec4<T> operator()(const v4i acc, float sq, const float (&sw)[4], const float (&bias)[4],
                                                int64_t row, int64_t col) const {
    float res[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.res != nullptr && row < p.m) {
      const T* const rp = static_cast<const T*>(p.res) + row * p.ldr + col;
      if (res_vec) {
        if (col < p.n) {
          const vec4<T> v = *reinterpret_cast<const vec4<T>*>(rp);
#pragma unroll
          for (int r = 0; r < 4; ++r) res[r] = static_cast<float>(v[r]);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (col + r < p.n) res[r] = static_cast<float>(rp[r]);
      }
    }
    vec4<T> o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = static_cast<T>((static_cast<float>(acc[r]) * sq) * sw[r] + bias[r] + res[r]);
    return o;
  }
};

// ------------------------------------------------------------------ LDS tiles
// Stage: BM rows of q, then BN rows of w, 128 bytes of K each.  A 1 KB direct load brings 8 rows;
// 16-byte chunk c of row r is kept at chunk c ^ (r % 8), so that eight rows read at one chunk
// meet eight different bank groups.
template <int BM, int BN, int WM, int WN, int ST>
struct Int8Tile {
  static constexpr int kWaves = (BM / WM) * (BN / WN);
  static constexpr int MI = WM / 16, NI = WN / 16;
  static constexpr int kStage = (BM + BN) * 128;
  static constexpr int kPA = BM / 8 / kWaves, kPB = BN / 8 / kWaves;  // pieces of a wave
  static constexpr int kOutStride = WN + 8;                           // staged output row, elements
  static constexpr int kLds = ST * kStage;
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0, "pieces are dealt evenly");
  static_assert(kWaves * 16 * kOutStride * 2 <= kLds, "the output rows are staged in the ring");
};

template <typename T, int BM, int BN, int WM, int WN, int ST>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN)) void int8_tile_kernel(Int8GemmParams p) {
  using C = Int8Tile<BM, BN, WM, WN, ST>;
  constexpr int MI = C::MI, NI = C::NI;
  __shared__ __align__(1024) char lds[C::kLds];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / (BN / WN), wn = wave % (BN / WN);

  // XCD x = b % 8 owns a contiguous run of the tiles, which walk the m-tiles of a group of 8 under
  // each n-tile: the tiles that run together on an XCD share operands in its L2.
  int mt, nt;
  {
    const int total = p.mtiles * p.ntiles;
    const int xcd = blockIdx.x & 7, q8 = total >> 3, r8 = total & 7;
    const int t = xcd * q8 + min(xcd, r8) + (static_cast<int>(blockIdx.x) >> 3);
    const int full = 8 * p.ntiles;
    const int g = t / full, rem = t - g * full;
    const int size = min(8, p.mtiles - 8 * g);
    nt = rem / size;
    mt = 8 * g + (rem - nt * size);
  }
  const int64_t m0 = static_cast<int64_t>(mt) * BM;
  const int n0 = nt * BN;
  const int nkb = (p.k + 127) >> 7;
  const bool ragged = (p.k & 127) != 0;

  // Rows past the matrix are clamped to its last one (their results are not stored).
  const int rchunk = (lane & 7) ^ (lane >> 3);
  uint32_t va[C::kPA], vb[C::kPB];
#pragma unroll
  for (int j = 0; j < C::kPA; ++j) {
    const int64_t r = min(static_cast<int64_t>(8 * (wave + C::kWaves * j) + (lane >> 3)), p.m - 1 - m0);
    va[j] = static_cast<uint32_t>(r) * static_cast<uint32_t>(p.ldq) + rchunk * 16;
  }
#pragma unroll
  for (int j = 0; j < C::kPB; ++j) {
    const int r = min(8 * (wave + C::kWaves * j) + (lane >> 3), p.n - 1 - n0);
    vb[j] = static_cast<uint32_t>(r) * static_cast<uint32_t>(p.ldw) + rchunk * 16;
  }
  const char* const abase = reinterpret_cast<const char*>(p.q) + m0 * p.ldq;
  const char* const bbase = reinterpret_cast<const char*>(p.w) + static_cast<int64_t>(n0) * p.ldw;
  auto issue = [&](int kb, int slot) {
    // The last block of a K that is no multiple of 128: chunks past the row's end read its last one.
    const uint32_t back = ragged && kb == nkb - 1 ? 16u * max(0, rchunk - ((p.k & 127) / 16 - 1)) : 0u;
    const uint32_t dst = lds0 + slot * C::kStage + wave * 1024;
#pragma unroll
    for (int j = 0; j < C::kPA; ++j) load_lds_1k(abase + static_cast<int64_t>(kb) * 128, va[j] - back, dst + j * C::kWaves * 1024);
#pragma unroll
    for (int j = 0; j < C::kPB; ++j)
      load_lds_1k(bbase + static_cast<int64_t>(kb) * 128, vb[j] - back, dst + BM * 128 + j * C::kWaves * 1024);
  };

  v4i acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = v4i{0, 0, 0, 0};

  // Lane L reads row L % 16 at chunk 4 kk + L / 16 of a 16-row fragment.
  const int roff = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) * 16);
  const int aoff = wm * WM * 128 + roff, boff = BM * 128 + wn * WN * 128 + roff;

#pragma unroll
  for (int s = 0; s < ST - 1; ++s)
    if (s < nkb) issue(s, s);
  int slot = 0;
  for (int kb = 0; kb < nkb; ++kb) {
    // Younger than this stage's loads: those of the ST - 2 stages after it, where they exist.
    if (ST > 2 && kb + ST - 2 < nkb) wait_vm<(ST - 2) * (C::kPA + C::kPB)>();
    else wait_vm<0>();
    lds_done_barrier();  // all waves' loads of this stage have landed; all reads of the one before are done
    if (kb + ST - 1 < nkb) issue(kb + ST - 1, slot == 0 ? ST - 1 : slot - 1);
    const char* const st = lds + slot * C::kStage;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      v4i a[MI], b[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) a[i] = *reinterpret_cast<const v4i*>(st + ((aoff + i * 2048) ^ (kk * 64)));
#pragma unroll
      for (int j = 0; j < NI; ++j) b[j] = *reinterpret_cast<const v4i*>(st + ((boff + j * 2048) ^ (kk * 64)));
      if (ragged && kb == nkb - 1 && kk * 64 + (lane >> 4) * 16 >= (p.k & 127)) {
#pragma unroll
        for (int i = 0; i < MI; ++i) a[i] = v4i{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[j], a[i], acc[i][j], 0, 0, 0);
    }
    slot = slot == ST - 1 ? 0 : slot + 1;
  }
  lds_done_barrier();  // the ring becomes the staging of the output rows

  const Epilogue<T> epi(p);
  const int lrow = lane & 15, lcol = (lane >> 4) * 4;
  const int64_t mw = m0 + wm * WM;
  const int nw = n0 + wn * WN;
  float sw[NI][4], bias[NI][4];
#pragma unroll
  for (int j = 0; j < NI; ++j) epi.scales(nw + j * 16 + lcol, sw[j], bias[j]);
  T* const stage = reinterpret_cast<T*>(lds) + wave * 16 * C::kOutStride;
  T* const y = static_cast<T*>(p.y);
  const bool wide = (p.n & 7) == 0;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t row = mw + i * 16 + lrow;
    const float sq = p.sq[min(row, p.m - 1)];
#pragma unroll
    for (int j = 0; j < NI; ++j)
      *reinterpret_cast<vec4<T>*>(stage + lrow * C::kOutStride + j * 16 + lcol) =
          epi(acc[i][j], sq, sw[j], bias[j], row, nw + j * 16 + lcol);
    __builtin_amdgcn_wave_barrier();
    if (wide) {
      constexpr int LPR = WN / 8, RPI = 64 / LPR;  // lanes of a row, rows of one store
#pragma unroll
      for (int s = 0; s < 16 / RPI; ++s) {
        const int r = s * RPI + lane / LPR, c = (lane % LPR) * 8;
        const int64_t orow = mw + i * 16 + r;
        if (orow < p.m && nw + c < p.n)
          *reinterpret_cast<v4i*>(y + orow * p.n + nw + c) = *reinterpret_cast<const v4i*>(stage + r * C::kOutStride + c);
      }
    } else {
      for (int e = lane; e < 16 * WN; e += 64) {
        const int r = e / WN, c = e % WN;
        const int64_t orow = mw + i * 16 + r;
        if (orow < p.m && nw + c < p.n) y[orow * p.n + nw + c] = stage[r * C::kOutStride + c];
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ------------------------------------------------------------------ few rows
// A workgroup holds 16 MI rows and 32 columns; its four waves (and the ksplit workgroups of a
// tile) each take a run of the 64-deep blocks of K.  The sums of the waves meet in LDS.
constexpr int kStreamCols = 32;

template <typename T, int MI>
__global__ __launch_bounds__(256) void int8_stream_kernel(Int8GemmParams p) {
  constexpr int NI = kStreamCols / 16, U = 4;
  __shared__ v4i sums[3][MI * NI * 64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * kStreamCols;
  const int64_t m0 = static_cast<int64_t>(blockIdx.z) * (16 * MI);
  const int split = blockIdx.y;
  const int blocks = (p.k + 63) >> 6, parts = 4 * p.ksplit, part = 4 * split + wave;
  const int begin = static_cast<int>(static_cast<int64_t>(blocks) * part / parts);
  const int end = static_cast<int>(static_cast<int64_t>(blocks) * (part + 1) / parts);
  const int kl = (lane >> 4) * 16;  // this lane's k in a block
  const int8_t* ap[MI];
  const int8_t* bp[NI];
#pragma unroll
  for (int i = 0; i < MI; ++i) ap[i] = p.q + min(m0 + i * 16 + (lane & 15), p.m - 1) * p.ldq;
#pragma unroll
  for (int j = 0; j < NI; ++j) bp[j] = p.w + static_cast<int64_t>(min(n0 + j * 16 + (lane & 15), p.n - 1)) * p.ldw;
  v4i acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = v4i{0, 0, 0, 0};

  for (int kb = begin; kb < end; kb += U) {
    v4i a[U][MI], b[U][NI];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // Blocks past the wave's last one, and chunks past K, read the row's last chunk; their
      // activations are zeroed below.
      const int k = min((kb + u) * 64 + kl, p.k - 16);
#pragma unroll
      for (int j = 0; j < NI; ++j) b[u][j] = *reinterpret_cast<const v4i*>(bp[j] + k);
#pragma unroll
      for (int i = 0; i < MI; ++i) a[u][i] = *reinterpret_cast<const v4i*>(ap[i] + k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = kb + u < end && (kb + u) * 64 + kl < p.k;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const v4i ai = in ? a[u][i] : v4i{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[u][j], ai, acc[i][j], 0, 0, 0);
      }
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) sums[wave - 1][(i * NI + j) * 64 + lane] = acc[i][j];
  }
  __syncthreads();
  const Epilogue<T> epi(p);
  // Fragment f of the tile to wave f % 4; wave 0 holds its own sums in registers.
#pragma unroll
  for (int f = 0; f < MI * NI; ++f) {
    if (wave != 0) break;
    v4i s = acc[f / NI][f % NI];
#pragma unroll
    for (int w = 0; w < 3; ++w) s += sums[w][f * 64 + lane];
    const int64_t row = m0 + (f / NI) * 16 + (lane & 15);
    const int64_t col = n0 + (f % NI) * 16 + (lane >> 4) * 4;
    if (row >= p.m) continue;
    if (p.ksplit > 1) {
      int32_t* const o = p.partial + (static_cast<int64_t>(split) * p.m + row) * p.n + col;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < p.n) o[r] = s[r];
    } else {
      float sw[4], bias[4];
      epi.scales(col, sw, bias);
      const vec4<T> o = epi(s, p.sq[row], sw, bias, row, col);
      T* const y = static_cast<T*>(p.y) + row * p.n + col;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < p.n) y[r] = o[r];
    }
  }
}

// Sum of the K slices and the epilogue, four columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void int8_reduce_kernel(Int8GemmParams p) {
  const int quads = (p.n + 3) >> 2;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.m * quads) return;
  const int64_t row = i / quads, col = (i - row * quads) * 4;
  const int64_t plane = p.m * p.n;
  const int32_t* const s = p.partial + row * p.n + col;
  v4i acc{0, 0, 0, 0};
  for (int k = 0; k < p.ksplit; ++k) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col + r < p.n) acc[r] += s[k * plane + r];
  }
  const Epilogue<T> epi(p);
  float sw[4], bias[4];
  epi.scales(col, sw, bias);
  const vec4<T> o = epi(acc, p.sq[row], sw, bias, row, col);
  T* const y = static_cast<T*>(p.y) + row * p.n + col;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (col + r < p.n) y[r] = o[r];
}

enum : int { kTile128 = 0, kTile64 = 1, kStream16 = 2, kStream32 = 3, kStream64 = 4 };

template <typename T, int BM, int BN, int WM, int WN, int ST>
void launch_tile(Int8GemmParams& p, hipStream_t stream) {
  p.mtiles = static_cast<int32_t>((p.m + BM - 1) / BM);
  p.ntiles = (p.n + BN - 1) / BN;
  int8_tile_kernel<T, BM, BN, WM, WN, ST>
      <<<dim3(static_cast<unsigned>(p.mtiles * p.ntiles)), 64 * Int8Tile<BM, BN, WM, WN, ST>::kWaves, 0, stream>>>(p);
}

template <typename T, int MI>
void launch_stream(const Int8GemmParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.n + kStreamCols - 1) / kStreamCols), static_cast<unsigned>(p.ksplit),
                  static_cast<unsigned>((p.m + 16 * MI - 1) / (16 * MI)));
  int8_stream_kernel<T, MI><<<grid, 256, 0, stream>>>(p);
  if (p.ksplit > 1) {
    const int64_t items = p.m * ((p.n + 3) / 4);
    int8_reduce_kernel<T><<<dim3(static_cast<unsigned>((items + 255) / 256)), 256, 0, stream>>>(p);
  }
}

template <typename T>
void launch(Int8GemmParams& p, const Int8GemmPlan& plan, hipStream_t stream) {
  switch (plan.tile) {
    case kTile128: launch_tile<T, 128, 128, 64, 64, 2>(p, stream); break;
    case kTile64: launch_tile<T, 64, 64, 32, 32, 3>(p, stream); break;
    case kStream16: launch_stream<T, 1>(p, stream); break;
    case kStream32: launch_stream<T, 2>(p, stream); break;
    default: launch_stream<T, 4>(p, stream); break;
  }
}

}  // namespace

Int8GemmPlan int8_gemm_plan(int64_t m, int32_t n, int32_t k, int cus) {
  Int8GemmPlan plan{};
  plan.ksplit = 1;
  if (m <= 64) {
    plan.tile = m <= 16 ? kStream16 : m <= 32 ? kStream32 : kStream64;
    // K slices until every CU has two workgroups, each wave with at least four 64-deep blocks.
    const int64_t tiles = (n + kStreamCols - 1) / kStreamCols;
    while (plan.ksplit < 16 && tiles * plan.ksplit < 2 * cus && k / (plan.ksplit * 2) >= 4 * 4 * 64) plan.ksplit *= 2;
    return plan;
  }
  const int64_t big = ((m + 127) / 128) * ((n + 127) / 128);
  plan.tile = big >= cus ? kTile128 : kTile64;
  return plan;
}

hipError_t launch_int8_gemm(Int8GemmParams p, const Int8GemmPlan& plan, int elem, hipStream_t stream) {
  p.ksplit = plan.ksplit;
  if (elem == kFp16)
    launch<_Float16>(p, plan, stream);
  else
    launch<__bf16>(p, plan, stream);
  return hipGetLastError();
}

}  // namespace w4a4
