// The score shapes of the scored attention kernels (ScoreMods), in units of log2: what the online
// softmax in base 2 works on.
#pragma once

#include "bsgl_device.h"
#include "bsgl_launch.h"

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
// hundredth of what the rounding of bf16 / f16 inputs puts on a score.  precise(): the library's tanh,
// for f32 rows, where 7e-6 would be the largest error of all.
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
    if (top > 0.f) s = top * tanhf(s / top);
    return fmaf(-slope, dist, s);
  }
};

}  // namespace bsgl
