// Product of int8 codes with scales for each token (row of q) and channel (row of w):
//
//   y[m, n] = T( float(sum_k q[m, k] w[n, k]) * sq[m] * sw[n] + bias[n] + residual[m, n] )
//
// on the int8 MFMAs: the int32 sums are exact (K <= 65536), so neither tile, nor K split, nor
// order changes a result; the epilogue runs in fp32 and rounds once.  Both operands are row-major
// with K contiguous, as the quantizer writes them: no layout of the weights' own.
//
// The weights are MFMA operand A, so that a lane ends with four consecutive columns of one row.
// In a step of v_mfma_i32_16x16x64_i8 lane L holds k = 16 (L / 16) .. + 15 of row L % 16 of either operand.
//
// Three kernels:
//   int8_stream_kernel  up to 16 rows: the weights stream from memory straight into registers,
//                       the waves of a workgroup split K;
//   int8_tile_kernel    64 x 64 and 128 x 64 tiles through LDS, with K slices where tiles are few;
//   int8_big_kernel     256 x 256 tiles, for what fills the CUs with them.

#include "direct_load.h"
#include "int8_internal.h"

namespace w4a4 {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
template <typename T>
using vec4 = T __attribute__((ext_vector_type(4)));
// The same at the alignment of their elements: rows of an N that is no multiple of a vector (one
// access all the same: 1071 x 2048 x 15980 57 us, in elements 76).
typedef int v4i_w __attribute__((ext_vector_type(4), aligned(4)));
typedef int v4i_h __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
using vec4_h = T __attribute__((ext_vector_type(4), aligned(2)));

// y[row, col .. col + 3] of one accumulator quad, with the bias and (RES) the residual: fp32, one
// rounding.
template <typename T, bool RES = true>
struct Epilogue {
  const Int8GemmParams& p;
  __device__ explicit Epilogue(const Int8GemmParams& q) : p(q) {}
  __device__ __forceinline__ void scales(int64_t col, float (&sw)[4], float (&bias)[4]) const {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t c = min(col + r, static_cast<int64_t>(p.n) - 1);
      sw[r] = p.sw[c];
      bias[r] = p.bias != nullptr ? static_cast<float>(static_cast<const T*>(p.bias)[c]) : 0.0f;
    }
  }
  __device__ __forceinline__ vec4<T> residual(int64_t row, int64_t col) const {
    vec4<T> v{};
    if (RES && p.res != nullptr && row < p.m) {
      const T* const rp = static_cast<const T*>(p.res) + row * p.ldr + col;
      if (col + 4 <= p.n) {
        v = *reinterpret_cast<const vec4_h<T>*>(rp);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (col + r < p.n) v[r] = rp[r];
      }
    }
    return v;
  }
  __device__ __forceinline__ vec4<T> operator()(const v4i acc, float sq, const float (&sw)[4], const float (&bias)[4],
                                                const vec4<T> res) const {
    vec4<T> o;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float v = fmaf(static_cast<float>(acc[r]) * sq, sw[r], bias[r]);
      o[r] = static_cast<T>(RES ? v + static_cast<float>(res[r]) : v);
    }
    return o;
  }
};

// The sums of columns col .. col + 3 of a K slice, to its plane of partial sums.
__device__ __forceinline__ void store_partial(const Int8GemmParams& p, const v4i s, int split, int64_t row, int64_t col) {
  if (row >= p.m) return;
  int32_t* const o = p.partial + (split * p.m + row) * p.n + col;
  if (col + 4 <= p.n) {
    *reinterpret_cast<v4i_w*>(o) = s;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col + r < p.n) o[r] = s[r];
  }
}

// Eight staged columns of an output row, of which `left` (or fewer than none) are there.
template <typename T>
__device__ __forceinline__ void store_chunk(T* y, const T* staged, int left) {
  if (left >= 8) {
    *reinterpret_cast<v4i_h*>(y) = *reinterpret_cast<const v4i*>(staged);
  } else {
    for (int e = 0; e < left; ++e) y[e] = staged[e];
  }
}

// ------------------------------------------------------------------ LDS tiles
// BM x BN tiles of waves that each hold 64 x 64 of it and one KW-th of every 128-byte stage, on
// v_mfma_i32_32x32x32_i8: one wave a SIMD feeds it at its full rate (16 x 16 x 64: 28 clocks
// for 16), and the K split gives small tiles enough waves without more LDS reads.  A wave then
// owns 4 / KW of the four 32 x 32 blocks of its position, sums the other waves' parts of them
// through LDS and finishes them.
// Stage: BM rows of q, then BN rows of w, 128 bytes of K each, in a ring of ST.  A 1 KB direct
// load brings 8 rows; 16-byte chunk c of row r is kept at chunk c ^ (r % 8), so that eight rows
// read at one chunk meet eight different bank groups.
template <int BM, int BN, int KW, int ST>
struct Int8Tile {
  static constexpr int kPos = (BM / 64) * (BN / 64);
  static constexpr int kWaves = kPos * KW;
  static constexpr int kStage = (BM + BN) * 128;
  static constexpr int kPA = BM / 8 / kWaves, kPB = BN / 8 / kWaves;  // pieces of a wave
  static constexpr int kOwn = 4 / KW;                                 // blocks that a wave finishes
  static constexpr int kOutStride = 32 + 8;                           // staged output row, elements
  static constexpr int kBlock = KW > 1 ? (KW - 1) * 4096 : 4096;       // LDS of a block: its sums, then its output rows
  static constexpr int kScale = ST * kStage > kPos * 4 * kBlock ? ST * kStage : kPos * 4 * kBlock;  // fp32 sq, sw, bias
  static constexpr int kLds = kScale + (BM + 2 * BN) * 4;
  static_assert(BM + 2 * BN <= 64 * kWaves, "a scale or bias of a thread");
  static_assert(32 * kOutStride * 2 <= kBlock, "a block's output rows fit where its sums were");
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0, "pieces are dealt evenly");
};

// Two waves a SIMD in the bounds: the accumulators then stay in ordinary registers (given twice as
// many, the compiler moves them to the accumulation registers and back in every step).
// Measured (us, 2048 deep, 2560 columns): 128 rows 8.4, 776 rows 14.1 (6 of them for one step and the
// ends); a 64 x 64 step of a CU costs 0.25 us, a 128 x 64 step 0.36, where its MFMAs alone take 0.07
// and 0.13: a step lasts as long as its operands take to the CU, 16 or 24 KB at 64 to 67 GB/s, which is
// what this ring gets and no limit of the chip.  Of a wave's clocks at 776 rows 45% are waits for loads and
// barriers and 17% MFMAs; a deeper ring (four stages) does not help.
template <typename T, int BM, int BN, int KW, int ST>
__global__ __launch_bounds__(64 * (BM / 64) * (BN / 64) * KW, 2) void int8_tile_kernel(Int8GemmParams p) {
  using C = Int8Tile<BM, BN, KW, ST>;
  extern __shared__ __align__(1024) char lds[];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave % KW, pos = wave / KW;
  const int wm = pos / (BN / 64), wn = pos % (BN / 64);

  // XCD x = b % 8 owns a contiguous run of the tiles, which walk the m-tiles of a group of 8 under
  // each n-tile: the tiles that run together on an XCD share operands in its L2.
  int mt, nt, split;
  {
    const int tiles = p.mtiles * p.ntiles, total = tiles * p.ksplit;
    const int xcd = blockIdx.x & 7, q8 = total >> 3, r8 = total & 7;
    const int s = xcd * q8 + min(xcd, r8) + (static_cast<int>(blockIdx.x) >> 3);
    split = __builtin_amdgcn_readfirstlane(s / tiles);
    const int t = s - split * tiles;
    const int full = 8 * p.ntiles;
    const int g = t / full, rem = t - g * full;
    const int size = min(8, p.mtiles - 8 * g);
    nt = __builtin_amdgcn_readfirstlane(rem / size);  // uniform, and to be held in scalar registers
    mt = __builtin_amdgcn_readfirstlane(8 * g + (rem - nt * size));
  }
  const int64_t m0 = static_cast<int64_t>(mt) * BM;
  const int n0 = nt * BN;
  // The 128-byte blocks of this K slice; only the last slice ends inside one.
  const int blocks = (p.k + 127) >> 7;
  const int kb0 = static_cast<int>(static_cast<int64_t>(blocks) * split / p.ksplit);
  const int nkb = static_cast<int>(static_cast<int64_t>(blocks) * (split + 1) / p.ksplit) - kb0;
  const bool ragged = (p.k & 127) != 0 && split == p.ksplit - 1;

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
  const char* const abase = reinterpret_cast<const char*>(p.q) + m0 * p.ldq + static_cast<int64_t>(kb0) * 128;
  const char* const bbase = reinterpret_cast<const char*>(p.w) + static_cast<int64_t>(n0) * p.ldw + static_cast<int64_t>(kb0) * 128;
  constexpr int kPieces = C::kPA + C::kPB;
  auto issue = [&](int kb, int slot, int j) {  // piece j of this wave
    // The last block of a K that is no multiple of 128: chunks past the row's end read its last one.
    const uint32_t back = ragged && kb == nkb - 1 ? 16u * max(0, rchunk - ((p.k & 127) / 16 - 1)) : 0u;
    const uint32_t dst = lds0 + slot * C::kStage + wave * 1024;
    if (j < C::kPA) load_lds_1k(abase + static_cast<int64_t>(kb) * 128, va[j] - back, dst + j * C::kWaves * 1024);
    else load_lds_1k(bbase + static_cast<int64_t>(kb) * 128, vb[j - C::kPA] - back, dst + BM * 128 + (j - C::kPA) * C::kWaves * 1024);
  };

  v16i acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  // Lane L of a 32-deep MFMA holds k = 16 (L / 32) .. + 15 of row L % 32 of either operand: chunk
  // 2 kk + L / 32 of its row.
  const int roff = (lane & 31) * 128 + (((lane >> 5) ^ (lane & 7)) * 16);
  const int aoff = wm * 64 * 128 + roff, boff = BM * 128 + wn * 64 * 128 + roff;

  // The fragments of a stage are read one stage ahead of their MFMAs.  Reads and loads go out among
  // the MFMAs, the reads in the first half of a step and the loads in the second: in a bunch, each
  // holds a wave up until the one before is taken (128 x 128 tiles, a step of K = 8192 at 100 rows:
  // 0.27 us of MFMAs and 0.30 of reads and loads took 0.48).
  constexpr int kParts = 4 / KW, kMfmas = 4 * kParts;
  v4i a0[2 * kParts], b0[2 * kParts], a1[2 * kParts], b1[2 * kParts];
  auto read = [&](int slot, v4i (&a)[2 * kParts], v4i (&b)[2 * kParts], int f) {  // in the order of their use
    const char* const st = lds + slot * C::kStage;
    const int k4 = f >> 2, i = f & 1, kk = kg * kParts + k4;
    if (f & 2) a[2 * k4 + i] = *reinterpret_cast<const v4i*>(st + ((aoff + i * 4096) ^ (kk * 32)));
    else b[2 * k4 + i] = *reinterpret_cast<const v4i*>(st + ((boff + i * 4096) ^ (kk * 32)));
  };
  auto mfma = [&](const v4i (&a)[2 * kParts], const v4i (&b)[2 * kParts], int f) {
    const int k4 = f >> 2, i = (f >> 1) & 1, j = f & 1;
    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[2 * k4 + j], a[2 * k4 + i], acc[i][j], 0, 0, 0);
  };
  int slot = 0;  // of the stage that is multiplied
  auto step = [&](int kb, v4i (&a)[2 * kParts], v4i (&b)[2 * kParts], v4i (&an)[2 * kParts], v4i (&bn)[2 * kParts]) {
    const int next = slot == ST - 1 ? 0 : slot + 1;
    if (kb + 1 < nkb) {
      // Younger than the next stage's loads: those of the ST - 2 stages after it, where they exist.
      if (ST > 2 && kb + ST - 1 < nkb) wait_vm<(ST - 2) * kPieces>();
      else wait_vm<0>();
      lds_done_barrier();  // the next stage has landed for all waves, which hold this one in registers
    }
    if (ragged && kb == nkb - 1) {  // the activations past K count as zeros
#pragma unroll
      for (int k4 = 0; k4 < kParts; ++k4)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if ((kg * kParts + k4) * 32 + (lane >> 5) * 16 >= (p.k & 127)) a[2 * k4 + i] = v4i{0, 0, 0, 0};
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < kMfmas / 2; ++f) {
      mfma(a, b, f);
      read(next, an, bn, 2 * f);  // past the last stage: an old one's, not used
      read(next, an, bn, 2 * f + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    const bool more = kb + ST < nkb;
#pragma unroll
    for (int f = 0; f < kMfmas / 2; ++f) {
      mfma(a, b, kMfmas / 2 + f);
      if (more) {
#pragma unroll
        for (int j = f * kPieces / (kMfmas / 2); j < (f + 1) * kPieces / (kMfmas / 2); ++j) issue(kb + ST, slot, j);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    slot = next;
  };

  // A scale or bias of the tile for each thread, on its way before the operands (loaded in the
  // epilogue they cost 0.6 us there).
  float scale = 0.0f;
  if (p.ksplit == 1) {
    const int i = threadIdx.x;
    if (i < BM) scale = p.sq[min(m0 + i, p.m - 1)];
    else if (i < BM + BN) scale = p.sw[min(n0 + i - BM, p.n - 1)];
    else if (i < BM + 2 * BN && p.bias != nullptr)
      scale = static_cast<float>(static_cast<const T*>(p.bias)[min(n0 + i - BM - BN, p.n - 1)]);
  }
#pragma unroll
  for (int s = 0; s < ST; ++s)
    if (s < nkb) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j) issue(s, s, j);
    }
  if (nkb >= ST) wait_vm<(ST - 1) * kPieces>();
  else wait_vm<0>();
  lds_done_barrier();
#pragma unroll
  for (int f = 0; f < 4 * kParts; ++f) read(0, a0, b0, f);
#pragma unroll 1
  for (int kb = 0; kb < nkb; kb += 2) {
    step(kb, a0, b0, a1, b1);
    if (kb + 1 < nkb) step(kb + 1, a1, b1, a0, b0);
  }
  float* const sc = reinterpret_cast<float*>(lds + C::kScale);
  if (static_cast<int>(threadIdx.x) < BM + 2 * BN) sc[threadIdx.x] = scale;
  lds_done_barrier();  // the ring becomes the waves' sums and the staging of the output rows

  if constexpr (KW > 1) {
    // Block f = 2 i + j of a position belongs to K group f / kOwn; part q of it is that of group q
    // (q + 1 from the owner on).
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int owner = f / C::kOwn;
      if (kg == owner) continue;
      const int part = kg - (kg > owner);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const v16i v = acc[f >> 1][f & 1];
        reinterpret_cast<v4i*>(lds + (pos * 4 + f) * C::kBlock + part * 4096)[r * 64 + lane] =
            v4i{v[4 * r], v[4 * r + 1], v[4 * r + 2], v[4 * r + 3]};
      }
    }
    __syncthreads();
  }
  const Epilogue<T> epi(p);
  T* const y = static_cast<T*>(p.y);
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    if (f / C::kOwn != kg) continue;
    char* const mine = lds + (pos * 4 + f) * C::kBlock;
    T* const stage = reinterpret_cast<T*>(mine);
    const int64_t mb = m0 + wm * 64 + (f >> 1) * 32, row = mb + (lane & 31);
    const int nb = n0 + wn * 64 + (f & 1) * 32;
    const float sq = sc[wm * 64 + (f >> 1) * 32 + (lane & 31)];
    vec4<T> res[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) res[t] = p.ksplit == 1 ? epi.residual(row, nb + 8 * t + 4 * (lane >> 5)) : vec4<T>{};
    v4i sum[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {  // columns 8 t + 4 (L / 32) .. + 3 of row L % 32
      const v16i v = acc[f >> 1][f & 1];
      sum[t] = v4i{v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3]};
      if constexpr (KW > 1) {
#pragma unroll
        for (int q = 0; q < KW - 1; ++q) sum[t] += reinterpret_cast<const v4i*>(mine + q * 4096)[t * 64 + lane];
      }
    }
    if (p.ksplit > 1) {
#pragma unroll
      for (int t = 0; t < 4; ++t) store_partial(p, sum[t], split, row, nb + 8 * t + 4 * (lane >> 5));
      continue;
    }
    __builtin_amdgcn_wave_barrier();  // the sums are in registers: the output rows take their place
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int c = 8 * t + 4 * (lane >> 5);
      const float* const s = sc + BM + wn * 64 + (f & 1) * 32 + c;
      const float4 s4 = *reinterpret_cast<const float4*>(s), t4 = *reinterpret_cast<const float4*>(s + BN);
      const float sw[4] = {s4.x, s4.y, s4.z, s4.w}, bias[4] = {t4.x, t4.y, t4.z, t4.w};
      *reinterpret_cast<vec4<T>*>(stage + (lane & 31) * C::kOutStride + c) = epi(sum[t], sq, sw, bias, res[t]);
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int r = s * 16 + (lane >> 2), c = (lane & 3) * 8;
      if (mb + r < p.m) store_chunk(y + (mb + r) * p.n + nb + c, stage + r * C::kOutStride + c, p.n - nb - c);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ------------------------------------------------------------------ many rows
// 256 x 256 tiles, eight waves of 64 x 128 (two a SIMD), a ring of two 128-byte stages.  The loads
// of the next stage go out at the top of a step, before its MFMAs, and have all of them to land:
// spread among the MFMAs, or as 64-byte stages three steps ahead, they were no faster (8192^3,
// us: 431 / 469 / 462).
// The workgroups walk the tiles, one a CU; the loads run on into the next tile, so that its first
// stage lands during the epilogue, whose scales wait in LDS since the tile's first step.
// What bounds it: at 8192^3 the MFMAs are busy for 61% of the clocks, and the clock follows the power: 2.3 to
// 2.4 GHz with operands of ones (379, after hundreds of calls 358 us), 1.9 to 2.2 with random ones (448, 399);
// four waves of 128 x 128 on 32 x 32 x 32 MFMAs need a fifth fewer clocks and run them slower, in the same
// time.  MFMAs on random registers alone hold 3450 TOP/s of the 5000 that the matrix units issue.  With 16
// steps a tile (6208 x 2048 x 16384, 194 us) they are busy for 46%: the rest are a tile's ends.  A
// residual costs more than its bytes (270 us, 41 of them its bytes): it is read group by group in the epilogue.
// Tiles of 128 x 256 with two workgroups a CU, so that one's epilogue overlaps the other's product,
// lose more to their operand traffic (5% slower there).
struct Int8Big {
  static constexpr int kTile = 256, kWaves = 8, MI = 4, NI = 8;
  static constexpr int kStage = 2 * kTile * 128;
  static constexpr int kOutStride = 64 + 8;               // half of a wave's columns at a time
  static constexpr int kScale = 2 * kStage;               // fp32 sq, sw, bias of the tile
  static constexpr int kOut = kScale + 3 * kTile * 4;
  static constexpr int kLds = kOut + kWaves * 16 * kOutStride * 2;
};

template <typename T, bool RES>
__global__ __launch_bounds__(512) void int8_big_kernel(Int8GemmParams p) {
  using C = Int8Big;
  constexpr int MI = C::MI, NI = C::NI;
  extern __shared__ __align__(1024) char lds[];
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int nkb = (p.k + 127) >> 7;
  const bool ragged = (p.k & 127) != 0;

  // XCD b % 8 owns a contiguous run of the tiles, which its workgroups take in turn; the order
  // walks the m-tiles of a group of 8 under each n-tile, so that the 32 tiles that run together
  // on an XCD are 8 x 4 and share their operands in its L2.
  int t, t_end, t_stride;
  {
    const int total = p.ntiles * p.mtiles, grid = gridDim.x, xcd = blockIdx.x & 7;
    const int q = total >> 3, r = total & 7;
    const int begin = xcd * q + min(xcd, r);
    t = begin + (static_cast<int>(blockIdx.x) >> 3);
    t_end = begin + q + (xcd < r ? 1 : 0);
    t_stride = (grid >> 3) + (xcd < (grid & 7) ? 1 : 0);
  }
  if (t >= t_end) return;
  struct Tile { int64_t m0; int n0; };
  auto tile_at = [&](int i) {
    const int full = 8 * p.ntiles;
    const int g = i / full, rem = i - g * full;
    const int size = min(8, p.mtiles - 8 * g);
    const int nt = __builtin_amdgcn_readfirstlane(rem / size);
    const int mt = __builtin_amdgcn_readfirstlane(8 * g + (rem - nt * size));
    return Tile{static_cast<int64_t>(mt) * C::kTile, nt * C::kTile};
  };

  // Loader: four 1 KB pieces (8 rows) of either operand a wave and stage.  Rows past the matrix are
  // clamped to its last one, and chunks past K to the row's last one.
  const int rchunk = (lane & 7) ^ (lane >> 3);
  uint32_t va[4], vb[4];
  const char *abase, *bbase;
  auto load_tile = [&](const Tile& c) {
    abase = reinterpret_cast<const char*>(p.q) + c.m0 * p.ldq;
    bbase = reinterpret_cast<const char*>(p.w) + static_cast<int64_t>(c.n0) * p.ldw;
    const int mlast = static_cast<int>(min(p.m - 1 - c.m0, static_cast<int64_t>(C::kTile - 1))), nlast = min(p.n - 1 - c.n0, C::kTile - 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = 8 * (wave + 8 * j) + (lane >> 3);
      va[j] = static_cast<uint32_t>(min(r, mlast)) * static_cast<uint32_t>(p.ldq) + rchunk * 16;
      vb[j] = static_cast<uint32_t>(min(r, nlast)) * static_cast<uint32_t>(p.ldw) + rchunk * 16;
    }
  };
  auto issue = [&](int kb, int slot) {
    const uint32_t back = ragged && kb == nkb - 1 ? 16u * max(0, rchunk - ((p.k & 127) / 16 - 1)) : 0u;
    const uint32_t dst = lds0 + slot + wave * 1024;
#pragma unroll
    for (int j = 0; j < 4; ++j) load_lds_1k(abase + static_cast<int64_t>(kb) * 128, va[j] - back, dst + j * 8192);
#pragma unroll
    for (int j = 0; j < 4; ++j) load_lds_1k(bbase + static_cast<int64_t>(kb) * 128, vb[j] - back, dst + 32768 + j * 8192);
  };

  const int roff = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) * 16);
  const int aoff = wm * 64 * 128 + roff, boff = 32768 + wn * 128 * 128 + roff;
  const Epilogue<T, RES> epi(p);
  float* const sc = reinterpret_cast<float*>(lds + C::kScale);
  const bool lines = (p.n & 63) == 0;  // output rows are whole 128-byte lines

  Tile cur = tile_at(t);
  load_tile(cur);
  issue(0, 0);
  int slot = 0;
  for (;;) {
    const bool more = t + t_stride < t_end;
    // Threads 0..255: a row scale; 256..511: a column's scale and bias.
    float s0, s1 = 0.0f;
    if (tid < 256) {
      s0 = p.sq[min(cur.m0 + tid, p.m - 1)];
    } else {
      const int col = min(cur.n0 + tid - 256, p.n - 1);
      s0 = p.sw[col];
      if (p.bias != nullptr) s1 = static_cast<float>(static_cast<const T*>(p.bias)[col]);
    }
    v4i acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = v4i{0, 0, 0, 0};
    Tile nxt = cur;
    for (int kb = 0; kb < nkb; ++kb) {
      wait_vm<0>();
      lds_done_barrier();  // this stage has landed; every wave has read the one before (and the last tile's scales)
      if (kb + 1 < nkb) {
        issue(kb + 1, slot ^ C::kStage);
      } else if (more) {
        nxt = tile_at(t + t_stride);
        load_tile(nxt);
        issue(0, slot ^ C::kStage);
      }
      const char* const st = lds + slot;
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
      if (kb == 0) {
        sc[tid] = s0;
        if (tid >= 256) sc[256 + tid] = s1;
      }
      slot ^= C::kStage;
    }
    if (nkb == 1) lds_done_barrier();  // the scales

    // Epilogue: 16 rows x 64 columns at a time through the wave's own LDS rows to whole lines.
    const int l = opaque_copy(lane);
    const int lrow = l & 15, lcol = (l >> 4) * 4;
    const int64_t mw = cur.m0 + wm * 64;
    const int nw = cur.n0 + wn * 128;
    T* const stage = reinterpret_cast<T*>(lds + C::kOut) + wave * 16 * C::kOutStride;
    T* const y = static_cast<T*>(p.y);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float4 sw[4], bias[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float* const s = sc + 256 + wn * 128 + half * 64 + j * 16 + lcol;
        sw[j] = *reinterpret_cast<const float4*>(s);
        bias[j] = *reinterpret_cast<const float4*>(s + 256);
      }
      const int nh = nw + half * 64;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int64_t row = mw + i * 16 + lrow;
        const float sq = sc[wm * 64 + i * 16 + lrow];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float w4[4] = {sw[j].x, sw[j].y, sw[j].z, sw[j].w}, b4[4] = {bias[j].x, bias[j].y, bias[j].z, bias[j].w};
          *reinterpret_cast<vec4<T>*>(stage + lrow * C::kOutStride + j * 16 + lcol) =
              epi(acc[i][half * 4 + j], sq, w4, b4, epi.residual(row, nh + j * 16 + lcol));
        }
        __builtin_amdgcn_wave_barrier();
        // Whole lines go past the L2, which the operands need (us, past / through: 6208 x 2048 x 16384 194 / 203,
        // x 2560 34.3 / 34.9), parts of lines through it (1071 x 2048 x 15984 61 / 54).
        if (lines) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int r = s * 8 + (l >> 3), c = (l & 7) * 8;
            const int64_t orow = mw + i * 16 + r;
            if (orow < p.m && nh + c < p.n)
              __builtin_nontemporal_store(*reinterpret_cast<const v4i*>(stage + r * C::kOutStride + c),
                                          reinterpret_cast<v4i*>(y + orow * p.n + nh + c));
          }
        } else {
          for (int s = 0; s < 2; ++s) {
            const int r = s * 8 + (l >> 3), c = (l & 7) * 8;
            const int64_t orow = mw + i * 16 + r;
            if (orow < p.m) store_chunk(y + orow * p.n + nh + c, stage + r * C::kOutStride + c, p.n - nh - c);
          }
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
    if (!more) break;
    t += t_stride;
    cur = nxt;
  }
}

// ------------------------------------------------------------------ few rows
// A workgroup holds 16 rows and 32 columns; its four waves (and the ksplit workgroups of a tile)
// each take a run of the 64-deep blocks of K, eight blocks in flight.  Both operands go straight
// into registers; the sums of the waves meet in LDS.
constexpr int kStreamCols = 32;

template <typename T>
__global__ __launch_bounds__(256) void int8_stream_kernel(Int8GemmParams p) {
  constexpr int NI = kStreamCols / 16, U = 8;
  __shared__ v4i sums[3][NI * 64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * kStreamCols;
  const int64_t m0 = static_cast<int64_t>(blockIdx.z) * 16;
  const int split = blockIdx.y;
  const int blocks = (p.k + 63) >> 6, parts = 4 * p.ksplit, part = 4 * split + wave;
  const int begin = static_cast<int>(static_cast<int64_t>(blocks) * part / parts);
  const int end = static_cast<int>(static_cast<int64_t>(blocks) * (part + 1) / parts);
  const int kl = (lane >> 4) * 16;  // this lane's k in a block
  const int8_t* const ap = p.q + min(m0 + (lane & 15), p.m - 1) * p.ldq;
  const int8_t* bp[NI];
#pragma unroll
  for (int j = 0; j < NI; ++j) bp[j] = p.w + static_cast<int64_t>(min(n0 + j * 16 + (lane & 15), p.n - 1)) * p.ldw;
  // The wave that ends the tile has its scales, bias and residual on their way before the operands.
  const Epilogue<T> epi(p);
  const int64_t row = m0 + (lane & 15);
  const bool ends = wave == 0 && p.ksplit == 1;
  float sq = 0.0f, sw[NI][4] = {}, bias[NI][4] = {};
  vec4<T> res[NI] = {};
  if (ends) {
    sq = p.sq[min(row, p.m - 1)];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int64_t col = n0 + j * 16 + (lane >> 4) * 4;
      epi.scales(col, sw[j], bias[j]);
      res[j] = epi.residual(row, col);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  v4i acc[NI];
#pragma unroll
  for (int j = 0; j < NI; ++j) acc[j] = v4i{0, 0, 0, 0};

  for (int kb = begin; kb < end; kb += U) {
    v4i a[U], b[U][NI];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // Blocks past the wave's last one, and chunks past K, read the row's last chunk; their
      // activations are zeroed below.
      const int k = min((kb + u) * 64 + kl, p.k - 16);
#pragma unroll
      for (int j = 0; j < NI; ++j) b[u][j] = *reinterpret_cast<const v4i*>(bp[j] + k);
      a[u] = *reinterpret_cast<const v4i*>(ap + k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = kb + u < end && (kb + u) * 64 + kl < p.k;
      const v4i ai = in ? a[u] : v4i{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[u][j], ai, acc[j], 0, 0, 0);
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int j = 0; j < NI; ++j) sums[wave - 1][j * 64 + lane] = acc[j];
  }
  __syncthreads();
  if (wave != 0 || row >= p.m) return;
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    v4i s = acc[j];
#pragma unroll
    for (int w = 0; w < 3; ++w) s += sums[w][j * 64 + lane];
    const int64_t col = n0 + j * 16 + (lane >> 4) * 4;
    if (p.ksplit > 1) {
      store_partial(p, s, split, row, col);
    } else {
      const vec4<T> o = epi(s, sq, sw[j], bias[j], res[j]);
      T* const y = static_cast<T*>(p.y) + row * p.n + col;
      if (col + 4 <= p.n) {
        *reinterpret_cast<vec4_h<T>*>(y) = o;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (col + r < p.n) y[r] = o[r];
      }
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
  const Epilogue<T> epi(p);
  float sw[4], bias[4];
  epi.scales(col, sw, bias);
  const float sq = p.sq[row];
  const vec4<T> res = epi.residual(row, col);
  const int64_t plane = p.m * p.n;
  const int32_t* const s = p.partial + row * p.n + col;
  v4i acc{0, 0, 0, 0};
  if (col + 4 <= p.n) {
#pragma unroll 8
    for (int k = 0; k < p.ksplit; ++k) acc += *reinterpret_cast<const v4i_w*>(s + k * plane);
  } else {
    for (int k = 0; k < p.ksplit; ++k) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < p.n) acc[r] += s[k * plane + r];
    }
  }
  const vec4<T> o = epi(acc, sq, sw, bias, res);
  T* const y = static_cast<T*>(p.y) + row * p.n + col;
  if (col + 4 <= p.n) {
    *reinterpret_cast<vec4_h<T>*>(y) = o;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col + r < p.n) y[r] = o[r];
  }
}

enum : int { kTile128x64, kTile64, kStream, kBig };

template <typename T>
void launch_reduce(const Int8GemmParams& p, hipStream_t stream) {
  if (p.ksplit <= 1) return;
  const int64_t items = p.m * ((p.n + 3) / 4);
  int8_reduce_kernel<T><<<dim3(static_cast<unsigned>((items + 255) / 256)), 256, 0, stream>>>(p);
}

template <typename T, int BM, int BN, int KW, int ST>
void launch_tile(Int8GemmParams& p, hipStream_t stream) {
  using C = Int8Tile<BM, BN, KW, ST>;
  p.mtiles = static_cast<int32_t>((p.m + BM - 1) / BM);
  p.ntiles = (p.n + BN - 1) / BN;
  int8_tile_kernel<T, BM, BN, KW, ST>
      <<<dim3(static_cast<unsigned>(p.mtiles * p.ntiles * p.ksplit)), 64 * C::kWaves, C::kLds, stream>>>(p);
  launch_reduce<T>(p, stream);
}

template <typename T>
void launch_big(Int8GemmParams& p, hipStream_t stream) {
  p.mtiles = static_cast<int32_t>((p.m + Int8Big::kTile - 1) / Int8Big::kTile);
  p.ntiles = (p.n + Int8Big::kTile - 1) / Int8Big::kTile;
  const int tiles = p.mtiles * p.ntiles, cus = device_cu_count();
  const dim3 grid(static_cast<unsigned>(tiles < cus ? tiles : cus));
  if (p.res != nullptr)
    int8_big_kernel<T, true><<<grid, 512, Int8Big::kLds, stream>>>(p);
  else
    int8_big_kernel<T, false><<<grid, 512, Int8Big::kLds, stream>>>(p);
}

template <typename T>
void launch_stream(const Int8GemmParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.n + kStreamCols - 1) / kStreamCols), static_cast<unsigned>(p.ksplit),
                  static_cast<unsigned>((p.m + 15) / 16));
  int8_stream_kernel<T><<<grid, 256, 0, stream>>>(p);
  launch_reduce<T>(p, stream);
}

template <typename T>
void launch(Int8GemmParams& p, const Int8GemmPlan& plan, hipStream_t stream) {
  switch (plan.tile) {
    case kTile128x64: launch_tile<T, 128, 64, 2, 3>(p, stream); break;
    case kBig: launch_big<T>(p, stream); break;
    case kTile64: launch_tile<T, 64, 64, 4, 3>(p, stream); break;
    default: launch_stream<T>(p, stream); break;
  }
}

}  // namespace

Int8GemmPlan int8_gemm_plan(int64_t m, int32_t n, int32_t k, int cus) {
  Int8GemmPlan plan{};
  plan.ksplit = 1;
  if (m <= 16) {
    // K slices until every CU has a workgroup, each wave at least eight 64-deep blocks (one row, us
    // with 1 / 2 / 4 / 8 slices: 2048 deep and 2560 columns 5.9 / 6.4 / 7.1 / -, 16384 and 2048 columns
    // 20.2 / 13.9 / 10.7 / 11.6).  From 17 rows on the 64 x 64 tiles are faster (32 rows 15.3 / 12.8,
    // 64 rows 20.3 / 13.3 at 16384 deep; 64 rows x 16384 columns 20.7 / 10.7).
    plan.tile = kStream;
    const int64_t tiles = (n + kStreamCols - 1) / kStreamCols;
    while (plan.ksplit < 16 && tiles * plan.ksplit < cus && k / (plan.ksplit * 2) >= 4 * 8 * 64) plan.ksplit *= 2;
    return plan;
  }
  // The least of the times (us, beside a launch) that these measurements give, 128 bytes of K a step
  // and w workgroups on the CUs: 64 x 64 tiles 0.25 a step and workgroup of a CU and 1 for its end (2048
  // deep, 2560 columns: 128 rows 8.4 us, 1500 rows 21), 128 x 64 tiles 0.36 and 2 (11, 17), 256 x 256 tiles 1.4
  // a step and 6 for the end of a round of CUs (26, 28; 776 rows x 16384 columns 31.7 us, against 55 and
  // 49; 3355 rows, 256 deep, 2608 columns 12.5, against 16.6 and 16.4).  A K slice shortens the steps and costs
  // the sums' way through memory.
  const double steps = (k + 127) / 128;
  double best = 1e30;
  auto consider = [&](int tile, int64_t w, double step_us, double end_us, int ks) {
    if (w * ks >= 1 << 24) return;  // a launch holds fewer than 2^32 threads
    const double load = static_cast<double>(w) * ks / cus;
    const double us = ((steps / ks) * step_us + end_us) * (load < 1 ? 1 : load) +
                      (ks > 1 ? 3.0 + static_cast<double>(m) * n * (8.0 * ks + 2) / 5e6 : 0.0);
    if (us < best) {
      best = us;
      plan.tile = tile;
      plan.ksplit = ks;
    }
  };
  for (int ks = 1; ks <= 8; ks *= 2) {
    if (ks > 1 && steps / ks < 8) break;
    consider(kTile64, ((m + 63) / 64) * ((n + 63) / 64), 0.25, 1, ks);
    consider(kTile128x64, ((m + 127) / 128) * ((n + 63) / 64), 0.36, 2, ks);
  }
  const int64_t big = ((m + 255) / 256) * ((n + 255) / 256);
  if ((steps * 1.4 + 6) * static_cast<double>((big + cus - 1) / cus) < best) plan = {kBig, 1};
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
