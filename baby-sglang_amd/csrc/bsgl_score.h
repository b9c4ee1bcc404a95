// The score shapes of the scored attention kernels (ScoreMods), in units of log2: what the online
// softmax in base 2 works on.
#pragma once

#include "bsgl_device.h"
#include "bsgl_launch.h"

#include <type_traits>

namespace bsgl {

// {first visible position, number of visible positions} of a row, inside [0, seq): `to_default` is the end
// where mods.to is not given.  An interval that is empty or upside down has no positions.
__device__ __forceinline__ int2 visible_range(const ScoreMods& m, int64_t row, int seq, int to_default) {
  int lo = m.from != nullptr ? m.from[row] : 0;
  int hi = m.to != nullptr ? m.to[row] : to_default;
  lo = max(0, min(lo, seq));
  hi = max(lo, min(hi, seq));
  return make_int2(lo, hi - lo);
}

// cap * tanh(s / cap) - slope * distance of one head, s = scale * (q . k), times log2(e).
//   tanh(x) = 1 - 2 / (e^{2x} + 1): one exp2 and one reciprocal, and no overflow: e^{2x} = inf gives exactly 1
// fast(): about 1.5e-7 of the cap in absolute error (1 - 2r cancels near zero), 7e-6 for a cap of 50: a
// hundredth of what the rounding of bf16 / f16 inputs puts on a score.  precise(), for f32 rows, where 7e-6 would be the
// largest error of all: relative to the result, 3e-7.  Below x = 0.55 x + x^3 P(x^2), P a polynomial of degree 4
// interpolated at the Chebyshev nodes of [0, 0.55^2] (2^-24 of the result off), above it 1 - 2 e / (1 + e) with e = e^{-2x} <= 1/3.
// (The device library's tanh is as good and three times as long: 24 of them for every four tokens of a decode row.)
struct ScoreShape {
  float lin;     // scale * log2(e)
  float arg;     // 2 * scale * log2(e) / cap, 0: no cap
  float top;     // cap * log2(e)
  float slope;   // slope * log2(e)
  __device__ __forceinline__ ScoreShape() {}
  __device__ __forceinline__ ScoreShape(const ScoreMods& m, float scale, int head) {
    lin = scale * kLog2e;
    arg = m.cap > 0.f ? 2.f * scale * kLog2e / m.cap : 0.f;
    top = m.cap * kLog2e;
    slope = m.slopes != nullptr ? m.slopes[head] * kLog2e : 0.f;
  }
  __device__ __forceinline__ float fast(float qk, float dist) const {
    float s = qk * lin;
    if (top > 0.f) s = fmaf(-2.f * top, __builtin_amdgcn_rcpf(fast_exp2(qk * arg) + 1.f), top);
    return fmaf(-slope, dist, s);
  }
  __device__ __forceinline__ float precise(float qk, float dist) const {
    float s = qk * lin;
    if (top > 0.f) {
      const float y = fabsf(qk * arg), e = fast_exp2(-y);  // y = 2 x log2 e
      const float x = y * (0.5f / kLog2e), z = x * x;
      const float p = fmaf(fmaf(fmaf(fmaf(-0.0066157547f, z, 0.021312745f), z, -0.053910065f), z, 0.13333118f), z, -0.33333331f);
      const float th = y < 1.1f * kLog2e ? fmaf(x * z, p, x) : fmaf(-2.f * e, __builtin_amdgcn_rcpf(1.f + e), 1.f);
      s = top * __builtin_copysignf(th, qk * arg);
    }
    return fmaf(-slope, dist, s);
  }
};

// a 16-byte piece of a row holds an infinity or a NaN
template <typename Tag> __device__ __forceinline__ bool not_finite(const uint4& x) {
  constexpr uint32_t e = std::is_same<Tag, f32_tag>::value ? 0x7f800000u : std::is_same<Tag, bf16_tag>::value ? 0x7f80u : 0x7c00u;
  bool bad = false;
  for (uint32_t w : {x.x, x.y, x.z, x.w}) {
    bad |= (w & e) == e;
    if constexpr (!std::is_same<Tag, f32_tag>::value) bad |= (w >> 16 & e) == e;
  }
  return bad;
}

// Extend kernels: whether this lane's row has met the values of a token that it does not see -- P . V multiplies them by an exact zero -- and
// one of them is no number.  That can only be in a step of 32 places that some row of the wave does not see whole; places are counted from the last
// token back, those past `kv_len` repeat it, the row sees [lo, hi) of them and every live row sees [full_from, full_to).  `v`: byte 0 of the kv head's
// part of slot 0.  (Run only where a row came out NaN: the tokens are read once, 16 bytes a lane.)
template <typename Tag, int ROW>
__device__ __forceinline__ bool met_unseen(const char* v, int64_t slab_row_bytes, const int32_t* table_row, uint32_t max_slot, int kv_len, int wave_len,
                                           int full_from, int full_to, int lo, int hi) {
  constexpr int LPT = ROW / 16, TPL = 64 / LPT;  // lanes per token, tokens per load
  const int lane = threadIdx.x & 63;
  bool met = false;
  for (int t0 = 0; t0 < min(kv_len, wave_len); t0 += 32) {
    if (t0 >= full_from && t0 + 32 <= full_to) continue;
    uint32_t odd = 0;  // the step's tokens with such a value
#pragma unroll 4
    for (int q = 0; q < 32; q += TPL) {
      uint32_t slot = (uint32_t)table_row[max(kv_len - 1 - (t0 + q + lane / LPT), 0)];
      slot = slot > max_slot ? max_slot : slot;
      const unsigned long long b = __ballot(not_finite<Tag>(*(const uint4*)(v + slot * slab_row_bytes + 16 * (lane % LPT))));
#pragma unroll
      for (int k = 0; k < TPL; ++k) odd |= (b >> (k * LPT) & ((1ull << LPT) - 1)) != 0 ? 1u << (q + k) : 0u;
    }
    auto below = [&](int t) { return t <= t0 ? 0u : t >= t0 + 32 ? ~0u : (1u << (t - t0)) - 1; };
    met |= (odd & ~(below(hi) & ~below(lo))) != 0;
  }
  return met;
}

}  // namespace bsgl
