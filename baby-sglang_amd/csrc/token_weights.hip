// Accumulated attention weight of cached tokens: what a decode step's softmax gave every visible token,
// summed over the q heads, added to a table that runs parallel to the page table.
//
//   weights[req_i, from_i + t] += sum_h exp2(score[i, h, t] - lse[i, h] * log2 e)
//
// The decode kernel leaves its scores behind (4 bytes per head and token, an eighth to a twentieth of the K/V rows it
// reads); a second pass is needed because a weight is known only once its whole row has been summed up.  Bound
// by those bytes, mostly from the caches they were just written to.  A thread owns four consecutive tokens and
// sums the heads in order, so the result does not depend on the launch.
//
// Two requests of a batch may name the same row: the first of them adds up all of its namesakes, in batch
// order, and the others leave, so that no two workgroups touch the same entry.
#include "bsgl_device.h"
#include "bsgl_launch.h"
#include "bsgl_score.h"

namespace bsgl {

namespace {

constexpr int kTokens = 256;  // tokens per workgroup of 64 lanes: four per lane

__global__ __launch_bounds__(64) void token_weights_kernel(WeightsArgs a) {
  const int lane = threadIdx.x;
  const int row = blockIdx.y;
  auto req_of = [&](int i) {
    const int64_t r = a.req_idx[i];
    return r < 0 ? (int64_t)0 : (r >= a.table_rows ? a.table_rows - 1 : r);
  };
  auto len_of = [&](int i) {
    const int64_t s = a.seq_lens[i];
    return (int)(s < 0 ? 0 : (s > a.table_cols ? a.table_cols : s));
  };
  const int64_t req = req_of(row);
  // the request's namesakes: one before it owns the row; `later`: there is one behind it
  bool before = false, later = false;
  for (int i0 = 0; i0 < a.rows; i0 += 64) {
    const int i = i0 + lane;
    const bool same = i < a.rows && i != row && req_of(min(i, a.rows - 1)) == req;
    before |= __any(same && i < row);
    later |= __any(same && i > row);
  }
  if (before) return;
  const int seq = len_of(row);
  const int2 seen = visible_range(a.mods, row, seq, seq);
  const float* src = a.mods.scores + (int64_t)row * a.n_q_heads * a.mods.score_stride;
  const float* lse = a.lse + (int64_t)row * a.n_q_heads;
  if (!later) {
    // (grid-stride: the grid is made for the longest request the host knows of)
    for (int64_t t0 = (int64_t)blockIdx.x * kTokens; t0 < seen.y; t0 += (int64_t)gridDim.x * kTokens) {
      const int t = (int)t0 + 4 * lane;
      if (t >= seen.y) continue;
      float w[4] = {0.f, 0.f, 0.f, 0.f};
      for (int h = 0; h < a.n_q_heads; ++h) {
        // (a score row has room for whole groups of 16: the last group's tail is never used)
        const float4 s = *(const float4*)(src + h * a.mods.score_stride + t);
        const float l = lse[h] * kLog2e;
        w[0] += fast_exp2(s.x - l);
        w[1] += fast_exp2(s.y - l);
        w[2] += fast_exp2(s.z - l);
        w[3] += fast_exp2(s.w - l);
      }
      const int64_t at = req * a.row_stride + seen.x + t;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (t + k < seen.y) a.out[at + k] = a.old[at + k] + w[k];
      }
    }
    return;
  }
  // (rare) several requests on one row: column by column, every one of them that sees it
  for (int64_t c = (int64_t)blockIdx.x * 64 + lane; c < a.table_cols; c += (int64_t)gridDim.x * 64) {
    float w = 0.f;
    bool any = false;
    for (int i = row; i < a.rows; ++i) {
      if (req_of(i) != req) continue;
      const int s = len_of(i);
      const int2 r = visible_range(a.mods, i, s, s);
      const int64_t t = c - r.x;
      if (t < 0 || t >= r.y) continue;
      any = true;
      const float* si = a.mods.scores + (int64_t)i * a.n_q_heads * a.mods.score_stride;
      for (int h = 0; h < a.n_q_heads; ++h) w += fast_exp2(si[h * a.mods.score_stride + t] - a.lse[(int64_t)i * a.n_q_heads + h] * kLog2e);
    }
    const int64_t at = req * a.row_stride + c;
    if (any) a.out[at] = a.old[at] + w;
  }
}

}  // namespace

hipError_t launch_token_weights(const WeightsArgs& a, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  const int64_t longest = a.len_hint > 0 && a.len_hint < a.table_cols ? a.len_hint : a.table_cols;
  const int64_t blocks = (longest + kTokens - 1) / kTokens;
  const dim3 grid((unsigned)(blocks < 1024 ? blocks : 1024), (unsigned)a.rows);
  hipLaunchKernelGGL(token_weights_kernel, grid, dim3(64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace bsgl
