// Query and key heads behind an RMSNorm of their own and the rotation by position, and the keys and
// values of new tokens into a 16-bit paged cache, in one pass.
//
//   f = x r g,  r = 1 / sqrt(mean_d(x^2) + eps),  g = 1 + w or w         (f = x without a norm)
//   pair j = (j, j + R/2), or (2j, 2j + 1) when interleaved:  angle = pos[axis(j)] freq[j]
//   (f1, f2) -> (f1 cos - f2 sin, f2 cos + f1 sin);  dimensions from R on stay f
//
// Everything is held in fp32 between the load and the one rounding at the end.  Angles are reduced in
// 64 bits: position * frequency / 2 pi, less its nearest integer, is exact to 2^-50 of the number of turns, so
// that far positions keep their angle.
//
// D / 16 lanes hold a head, 16 elements each: of a rotated pair both halves, so that nothing crosses
// lanes but the sum of squares.  A wave takes a token (or a part of its heads), each lane computes the sine and
// cosine of every 64th pair, and the heads share them through LDS.
// Bound by HBM where tokens are many: 4 x 1536 tokens of 32 + 8 heads of 128, 126 MB, 25.9 us, 4.9 TB/s, where the
// bytes alone take 23.6 in this form (fewer registers for a third more waves, or weights loaded a head: no faster); a single token by its loads' latency one behind the other, 4 us.

#include "quant_row.h"
#include "serving_internal.h"

namespace w4a4 {
namespace {

template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

// Addresses that are chosen among several tensors: the compiler takes them for global memory only when told.
template <typename T>
__device__ __forceinline__ vec8<T> load_global(uintptr_t a) {
  return *reinterpret_cast<const __attribute__((address_space(1))) vec8<T>*>(a);
}
template <typename T>
__device__ __forceinline__ void store_global(uintptr_t a, const vec8<T> v) {
  *reinterpret_cast<__attribute__((address_space(1))) vec8<T>*>(a) = v;
}

constexpr double kTurns = 0.15915494309189533577;  // 1 / (2 pi)

// The sum over a head's L lanes, which are all here or none.
template <int L>
__device__ __forceinline__ float head_sum(float v) {
  if constexpr (L > 1) v += lane_xor_f<0>(v);
  if constexpr (L > 2) v += lane_xor_f<1>(v);
  if constexpr (L > 4) v += lane_xor_f<2>(v);
  if constexpr (L > 8) v += lane_xor_f<3>(v);
  if constexpr (L > 16) v += __shfl_xor(v, 16, 64);
  return v;
}

// L lanes (a power of two, D / 16 or the next one) a head, 64 / L heads a round of the wave.  PAIRS: the two of a pair
// stand beside each other (interleaved).
template <typename T, int L, bool PAIRS>
__global__ __launch_bounds__(256) void head_rope_kernel(HeadRopeParams p) {
  constexpr int S = 64 / L;
  // The sines and cosines of the wave's token: each pair is computed by one lane.
  __shared__ __align__(16) float2 turns[4][8 * L];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned item = blockIdx.x * 4 + wave;  // tokens * parts < 2^26
  const unsigned token = item / p.parts, part = item - token * p.parts;
  if (token >= static_cast<unsigned>(p.b * p.t)) return;  // no barrier below: a wave has its part of LDS to itself
  const unsigned b = token / p.t, t = token - b * p.t;
  const int slot = lane / L, li = lane % L;
  const bool mine = li < p.d / 16;
  const bool turned = li < p.rot / 16;
  // The lane's two chunks of eight elements.
  const int c0 = PAIRS || !turned ? 16 * li : 8 * li;
  const int c1 = PAIRS || !turned ? 16 * li + 8 : 8 * li + p.rot / 2;
  const int hq = p.heads[0], hk = p.heads[1], all = hq + hk + p.heads[2];
  const int rounds = (all + S - 1) / S;

  auto side_of = [&](int head) { return head < hq ? 0 : head < hq + hk ? 1 : 2; };
  auto index_of = [&](int head, int side) { return head - (side == 0 ? 0 : side == 1 ? hq : hq + hk); };
  // The token's rows of the three tensors, and the strides of their heads, in bytes.
  const uintptr_t q0 = reinterpret_cast<uintptr_t>(p.x[0]) + 2 * (b * p.stride[0][0] + t * p.stride[0][1]);
  const uintptr_t k0 = reinterpret_cast<uintptr_t>(p.x[1]) + 2 * (b * p.stride[1][0] + t * p.stride[1][1]);
  const uintptr_t v0 = reinterpret_cast<uintptr_t>(p.x[2]) + 2 * (b * p.stride[2][0] + t * p.stride[2][1]);
  const int64_t qs = 2 * p.stride[0][2], ks = 2 * p.stride[1][2], vs = 2 * p.stride[2][2];
  const bool norm_q = p.w[0] != nullptr, norm_k = p.w[1] != nullptr, keys_out = p.k_out != nullptr;
  vec8<T> w[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i][0] = w[i][1] = vec8<T>{};
    if (p.w[i] != nullptr && mine) {
      w[i][0] = *reinterpret_cast<const vec8<T>*>(static_cast<const T*>(p.w[i]) + c0);
      w[i][1] = *reinterpret_cast<const vec8<T>*>(static_cast<const T*>(p.w[i]) + c1);
    }
  }

  const uintptr_t qo = reinterpret_cast<uintptr_t>(p.q_out) + static_cast<int64_t>(token) * hq * p.d * 2;
  const uintptr_t ko = reinterpret_cast<uintptr_t>(p.k_out) + static_cast<int64_t>(token) * hk * p.d * 2;
  const float inv_d = 1.0f / static_cast<float>(p.d), unit = p.unit_offset ? 1.0f : 0.0f;
  float co[8], si[8];
  int64_t row = -1;
  uintptr_t kc = 0, vc = 0;
  for (int base = part; base < rounds; base += p.parts) {
    const int head = base * S + slot;
    const int side = side_of(head), of = index_of(head, side);
    const int d0 = side == 2 ? 16 * li : c0, d1 = side == 2 ? 16 * li + 8 : c1;
    vec8<T> y0{}, y1{};
    if (mine && head < all) {
      const uintptr_t r = (side == 0 ? q0 : side == 1 ? k0 : v0) + of * (side == 0 ? qs : side == 1 ? ks : vs);
      y0 = load_global<T>(r + 2 * d0);
      y1 = load_global<T>(r + 2 * d1);
    }
    if (base == static_cast<int>(part)) {  // while the first head is under way
      // Where the token goes in the cache: nowhere behind the sequence's count, the table or the pool.
      if (p.c.lens != nullptr) {
        const int64_t len = max(p.c.lens[b], 0);
        const int count = min(max(p.counts != nullptr ? p.counts[b] : p.t, 0), p.t);
        const int64_t at = len + t, pg = at / kKvPage;
        if (static_cast<int>(t) < count && pg < p.c.table_pages) {
          const int page = p.c.table[b * p.c.table_stride + pg];
          if (page >= 0 && page < p.c.pages) row = static_cast<int64_t>(page) * p.c.kvh * kKvPage + at % kKvPage;
        }
      }
      kc = reinterpret_cast<uintptr_t>(p.c.k) + row * p.d * 2;
      vc = reinterpret_cast<uintptr_t>(p.c.v) + row * p.d * 2;
      if (p.rot > 0) {
        double pos[kRopeAxes];
#pragma unroll
        for (int a = 0; a < kRopeAxes; ++a) {
          pos[a] = 0.0;
          if (a < p.axes) {
            const int64_t i = a * p.pos_stride[0] + b * p.pos_stride[1] + t * p.pos_stride[2];
            pos[a] = p.pos64 ? static_cast<double>(static_cast<const int64_t*>(p.pos)[i])
                             : static_cast<double>(static_cast<const int32_t*>(p.pos)[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < (8 * L + 63) / 64; ++i) {
          const int j = 64 * i + lane;
          const uint64_t lo = p.axis[4 * i] | static_cast<uint64_t>(p.axis[4 * i + 1]) << 32;
          const uint64_t hi = p.axis[4 * i + 2] | static_cast<uint64_t>(p.axis[4 * i + 3]) << 32;
          const uint32_t a = static_cast<uint32_t>((lane & 32 ? hi : lo) >> (2 * (lane & 31))) & 3u;
          if (j < p.rot / 2) {
            const double at = a < 2u ? (a == 0u ? pos[0] : pos[1]) : (a == 2u ? pos[2] : pos[3]);
            const double turn = at * (static_cast<double>(p.freq[j]) * kTurns);
            float2 cs;
            sincospif(static_cast<float>(2.0 * (turn - __builtin_rint(turn))), &cs.y, &cs.x);
            turns[wave][j] = cs;
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (turned) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float4 v = *reinterpret_cast<const float4*>(&turns[wave][8 * li + e]);
            co[e] = v.x;
            si[e] = v.y;
            co[e + 1] = v.z;
            si[e + 1] = v.w;
          }
        }
      }
    }
    const bool norm = (side == 0 && norm_q) || (side == 1 && norm_k);
    if (side < 2 && (norm || turned)) {
      float f[16];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = static_cast<float>(y0[e]);
        f[8 + e] = static_cast<float>(y1[e]);
      }
      if (norm) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) ss = fmaf(f[e], f[e], ss);
        ss = head_sum<L>(ss);
        float mean = fmaf(ss, inv_d, p.eps);
        // bf16 heads whose squares leave fp32's range (the same for all lanes of a head): again at another scale.
        if (!(ss <= 1e37f) || mean < 1e-24f) {
          const float c = mean < 1e-24f ? 0x1p80f : 0x1p-80f;
          ss = 0.0f;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            f[e] *= c;
            ss = fmaf(f[e], f[e], ss);
          }
          mean = fmaf(head_sum<L>(ss), inv_d, p.eps * c * c);
        }
        const float r = __builtin_amdgcn_rsqf(mean);
        const vec8<T> g0 = side == 0 ? w[0][0] : w[1][0], g1 = side == 0 ? w[0][1] : w[1][1];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f[e] = f[e] * r * (unit + static_cast<float>(g0[e]));
          f[8 + e] = f[8 + e] * r * (unit + static_cast<float>(g1[e]));
        }
      }
      if (turned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = PAIRS ? 2 * e : e, j2 = PAIRS ? 2 * e + 1 : 8 + e;
          const float u = f[i], v = f[j2];
          f[i] = u * co[e] - v * si[e];
          f[j2] = v * co[e] + u * si[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y0[e] = static_cast<T>(f[e]);
        y1[e] = static_cast<T>(f[8 + e]);
      }
    }
    if (!mine || head >= all) continue;
    uintptr_t out;
    if (side == 0 || (side == 1 && keys_out)) {
      out = side == 0 ? qo + of * p.d * 2 : ko + of * p.d * 2;
    } else {
      if (row < 0) continue;
      out = (side == 1 ? kc : vc) + static_cast<int64_t>(of) * (kKvPage * p.d * 2);
    }
    store_global<T>(out + 2 * d0, y0);
    store_global<T>(out + 2 * d1, y1);
  }
}

template <typename T, int L>
void launch_pairs(const HeadRopeParams& p, hipStream_t stream) {
  const unsigned items = static_cast<unsigned>(p.b) * p.t * p.parts;
  const dim3 grid((items + 3) / 4);
  if (p.interleaved) head_rope_kernel<T, L, true><<<grid, 256, 0, stream>>>(p);
  else head_rope_kernel<T, L, false><<<grid, 256, 0, stream>>>(p);
}

template <typename T>
void launch_lanes(const HeadRopeParams& p, int lanes, hipStream_t stream) {
  switch (lanes) {
    case 1: launch_pairs<T, 1>(p, stream); break;
    case 2: launch_pairs<T, 2>(p, stream); break;
    case 4: launch_pairs<T, 4>(p, stream); break;
    case 8: launch_pairs<T, 8>(p, stream); break;
    case 16: launch_pairs<T, 16>(p, stream); break;
    default: launch_pairs<T, 32>(p, stream); break;
  }
}

}  // namespace

static int head_lanes(int32_t d) {
  int lanes = 1;
  while (lanes < d / 16) lanes *= 2;
  return lanes;
}

// A wave for each round of heads where tokens are few, else up to three rounds a wave (4 x 1536 tokens of 32 + 8 heads
// of 128, five rounds, in 1 / 2 parts: 28.1 / 26.6 us; 8 x 776 of 8 + 1 + 1 heads of 256, three rounds: 17.3 / 20.1).
int32_t head_rope_parts(const HeadRopeParams& p, int cus) {
  const int64_t heads_a_round = 64 / head_lanes(p.d), tokens = static_cast<int64_t>(p.b) * p.t;
  const int64_t rounds = (static_cast<int64_t>(p.heads[0]) + p.heads[1] + p.heads[2] + heads_a_round - 1) / heads_a_round;
  const int64_t want = (8LL * cus + tokens - 1) / tokens, few = want < rounds ? want : rounds, least = (rounds + 2) / 3;
  return static_cast<int32_t>(few > least ? few : least);
}

hipError_t launch_head_rope(const HeadRopeParams& p, int elem, hipStream_t stream) {
  if (p.b <= 0 || p.t <= 0) return hipSuccess;
  if (elem == kFp16)
    launch_lanes<_Float16>(p, head_lanes(p.d), stream);
  else
    launch_lanes<__bf16>(p, head_lanes(p.d), stream);
  return hipGetLastError();
}

}  // namespace w4a4
