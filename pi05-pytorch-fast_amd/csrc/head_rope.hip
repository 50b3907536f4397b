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
// lanes but the sum of squares.  A wave takes a token (or a part of its heads) and keeps its sines
// and cosines over the heads.

#include "serving_internal.h"

namespace w4a4 {
namespace {

template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

constexpr double kTurns = 0.15915494309189533577;  // 1 / (2 pi)

// L lanes (a power of two, D / 16 or the next one) a head.
template <typename T, int L>
__global__ __launch_bounds__(256) void head_rope_kernel(HeadRopeParams p) {
  constexpr int S = 64 / L, kAhead = 4;
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t token = item / p.parts;
  const int part = static_cast<int>(item - token * p.parts);
  if (token >= static_cast<int64_t>(p.b) * p.t) return;
  const int b = static_cast<int>(token / p.t), t = static_cast<int>(token - static_cast<int64_t>(b) * p.t);
  const int slot = lane / L, li = lane % L;
  const bool mine = li < p.d / 16;
  const bool turned = li < p.rot / 16;
  // The lane's two chunks of eight elements.
  const int c0 = p.interleaved || !turned ? 16 * li : 8 * li;
  const int c1 = p.interleaved || !turned ? 16 * li + 8 : 8 * li + p.rot / 2;

  // Where the token goes in the cache: nowhere behind the sequence's count, the table or the pool.
  int64_t row = -1;
  if (p.c.lens != nullptr) {
    const int64_t len = max(p.c.lens[b], 0);
    const int count = min(max(p.counts != nullptr ? p.counts[b] : p.t, 0), p.t);
    const int64_t at = len + t, pg = at / kKvPage;
    if (t < count && pg < p.c.table_pages) {
      const int page = p.c.table[b * p.c.table_stride + pg];
      if (page >= 0 && page < p.c.pages) row = static_cast<int64_t>(page) * p.c.kvh * kKvPage + at % kKvPage;
    }
  }

  float co[8], si[8];
  if (turned) {
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
    const uint32_t axis = p.axis[li >> 1] >> (16 * (li & 1));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t a = (axis >> (2 * e)) & 3u;
      const double at = a < 2u ? (a == 0u ? pos[0] : pos[1]) : (a == 2u ? pos[2] : pos[3]);
      const double turns = at * (static_cast<double>(p.freq[8 * li + e]) * kTurns);
      sincospif(static_cast<float>(2.0 * (turns - __builtin_rint(turns))), &si[e], &co[e]);
    }
  }

  const int hq = p.heads[0], hk = p.heads[1], all = hq + hk + p.heads[2];
  const int rounds = (all + S - 1) / S;
  for (int base = part; base < rounds; base += kAhead * p.parts) {
    vec8<T> x[kAhead][2];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int head = (base + j * p.parts) * S + slot;
      x[j][0] = x[j][1] = vec8<T>{};
      if (mine && head < all) {
        const int side = head < hq ? 0 : head < hq + hk ? 1 : 2;
        const int of = head - (side == 0 ? 0 : side == 1 ? hq : hq + hk);
        const T* const src = static_cast<const T*>(side == 0 ? p.x[0] : side == 1 ? p.x[1] : p.x[2]);
        const int64_t sb = side == 0 ? p.stride[0][0] : side == 1 ? p.stride[1][0] : p.stride[2][0];
        const int64_t st = side == 0 ? p.stride[0][1] : side == 1 ? p.stride[1][1] : p.stride[2][1];
        const int64_t sh = side == 0 ? p.stride[0][2] : side == 1 ? p.stride[1][2] : p.stride[2][2];
        const T* const r = src + b * sb + t * st + of * sh;
        const int d0 = side == 2 ? 16 * li : c0, d1 = side == 2 ? 16 * li + 8 : c1;
        x[j][0] = *reinterpret_cast<const vec8<T>*>(r + d0);
        x[j][1] = *reinterpret_cast<const vec8<T>*>(r + d1);
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (base + j * p.parts >= rounds) break;  // uniform
      const int head = (base + j * p.parts) * S + slot;
      const int side = head < hq ? 0 : head < hq + hk ? 1 : 2;
      const int of = head - (side == 0 ? 0 : side == 1 ? hq : hq + hk);
      vec8<T> y0 = x[j][0], y1 = x[j][1];
      const T* const w = static_cast<const T*>(side == 0 ? p.w[0] : p.w[1]);
      if (side != 2 && (w != nullptr || turned)) {
        float f[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f[e] = static_cast<float>(x[j][0][e]);
          f[8 + e] = static_cast<float>(x[j][1][e]);
        }
        if (w != nullptr) {
          float ss = 0.0f;
#pragma unroll
          for (int e = 0; e < 16; ++e) ss = fmaf(f[e], f[e], ss);
#pragma unroll
          for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
          float r = 1.0f / __builtin_sqrtf(ss / static_cast<float>(p.d) + p.eps);
          vec8<T> w0{}, w1{};
          if (mine) {
            w0 = *reinterpret_cast<const vec8<T>*>(w + c0);
            w1 = *reinterpret_cast<const vec8<T>*>(w + c1);
          }
          // bf16 heads whose squares leave fp32's range (the same for all lanes of a head): in 64 bits.
          if (!(ss <= 1e37f && ss >= 1e-25f)) {
            double s = 0.0;
#pragma unroll
            for (int e = 0; e < 16; ++e) s += static_cast<double>(f[e]) * f[e];
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
            const double rd = 1.0 / sqrt(s / p.d + p.eps);
#pragma unroll
            for (int e = 0; e < 16; ++e) f[e] = static_cast<float>(f[e] * rd);
            r = 1.0f;
          }
          const float unit = p.unit_offset ? 1.0f : 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[e] = f[e] * r * (unit + static_cast<float>(w0[e]));
            f[8 + e] = f[8 + e] * r * (unit + static_cast<float>(w1[e]));
          }
        }
        if (turned) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float& u = p.interleaved ? f[2 * e] : f[e];
            float& v = p.interleaved ? f[2 * e + 1] : f[8 + e];
            const float a = u, c = v;
            u = a * co[e] - c * si[e];
            v = c * co[e] + a * si[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y0[e] = static_cast<T>(f[e]);
          y1[e] = static_cast<T>(f[8 + e]);
        }
      }
      if (!mine || head >= all) continue;
      T* out;
      if (side == 0) {
        out = static_cast<T*>(p.q_out) + (token * hq + of) * p.d;
      } else if (side == 1 && p.k_out != nullptr) {
        out = static_cast<T*>(p.k_out) + (token * hk + of) * p.d;
      } else {
        if (row < 0) continue;
        out = static_cast<T*>(side == 1 ? p.c.k : p.c.v) + (row + static_cast<int64_t>(of) * kKvPage) * p.d;
      }
      const int d0 = side == 2 ? 16 * li : c0, d1 = side == 2 ? 16 * li + 8 : c1;
      *reinterpret_cast<vec8<T>*>(out + d0) = y0;
      *reinterpret_cast<vec8<T>*>(out + d1) = y1;
    }
  }
}

template <typename T>
void launch_lanes(const HeadRopeParams& p, int lanes, hipStream_t stream) {
  const int64_t items = static_cast<int64_t>(p.b) * p.t * p.parts;
  const dim3 grid(static_cast<unsigned>((items + 3) / 4));
  switch (lanes) {
    case 1: head_rope_kernel<T, 1><<<grid, 256, 0, stream>>>(p); break;
    case 2: head_rope_kernel<T, 2><<<grid, 256, 0, stream>>>(p); break;
    case 4: head_rope_kernel<T, 4><<<grid, 256, 0, stream>>>(p); break;
    case 8: head_rope_kernel<T, 8><<<grid, 256, 0, stream>>>(p); break;
    case 16: head_rope_kernel<T, 16><<<grid, 256, 0, stream>>>(p); break;
    default: head_rope_kernel<T, 32><<<grid, 256, 0, stream>>>(p); break;
  }
}

}  // namespace

hipError_t launch_head_rope(HeadRopeParams p, int elem, hipStream_t stream) {
  if (p.b <= 0 || p.t <= 0) return hipSuccess;
  int lanes = 1;
  while (lanes < p.d / 16) lanes *= 2;
  // Few tokens: a wave for each round of heads.
  const int rounds = (p.heads[0] + p.heads[1] + p.heads[2] + 64 / lanes - 1) / (64 / lanes);
  const int64_t tokens = static_cast<int64_t>(p.b) * p.t;
  const int64_t want = (8LL * device_cu_count() + tokens - 1) / tokens;
  p.parts = static_cast<int>(want < rounds ? want : rounds);
  if (elem == kFp16)
    launch_lanes<_Float16>(p, lanes, stream);
  else
    launch_lanes<__bf16>(p, lanes, stream);
  return hipGetLastError();
}

}  // namespace w4a4
