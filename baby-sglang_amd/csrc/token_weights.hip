// Accumulated attention weight of cached tokens: what a decode step's softmax gave every visible token,
// summed over the q heads, added to a table that runs parallel to the page table.
//
//   weights[req_i, from_i + t] += sum_h exp2(score[i, h, t] - lse[i, h] * log2 e)
//
// The decode kernel leaves its scores behind (4 bytes per head and token, an eighth to a twentieth of the K/V rows it
// reads); a second pass is needed because a weight is known only once its whole row has been summed up.  Bound
// by those bytes, mostly from the caches they were just written to.  A workgroup owns 256 consecutive tokens: its
// four waves take the heads in turn, four tokens per lane, and their sums are added in LDS in wave order, so
// the result does not depend on the launch.
//
// Two requests of a batch may name the same row: the first of them adds up all of its namesakes, in batch
// order, and the others leave, so that no two workgroups touch the same entry.
#include "bsgl_device.h"
#include "bsgl_launch.h"
#include "bsgl_score.h"

namespace bsgl {

namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;

constexpr int kTokens = 256;  // tokens per workgroup: four per lane of a wave
constexpr int kWaves = 4;     // that share the heads

// a head's log-sum-exp as what its scores are taken against.  A head whose visible scores are all -inf (an infinity in K) has one of
// -inf and gives its tokens nothing: -inf - -inf would be NaN, which a weight never loses again.  (A NaN among the scores passes.)
__device__ __forceinline__ float against(float lse) { return lse == kNegInf ? -kNegInf : lse * kLog2e; }

__global__ __launch_bounds__(64 * kWaves) void token_weights_kernel(WeightsArgs a) {
  __shared__ f32x4 s_sum[kWaves][64];
  __shared__ int s_same[kWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
  int mine = 0;  // bit 0: one before, bit 1: one behind
  for (int i = tid; i < a.rows; i += 64 * kWaves) {
    if (i != row && req_of(i) == req) mine |= i < row ? 1 : 2;
  }
  mine = (__any(mine & 1) ? 1 : 0) | (__any(mine & 2) ? 2 : 0);
  const int seq = len_of(row);
  const int2 seen = visible_range(a.mods, row, seq, seq);
  const float* src = a.mods.scores + (int64_t)row * a.n_q_heads * a.mods.score_stride;
  const float* lse = a.lse + (int64_t)row * a.n_q_heads;
  // the wave's head sums of the first 256 tokens leave before it is known whose row this is
  auto head_sums = [&](int64_t t0) {
    f32x4 w = {0.f, 0.f, 0.f, 0.f};
    const int t = (int)t0 + 4 * lane;
    if (t < seen.y) {
      // (a score row has room for whole groups of 16: the last group's tail is never used)
#pragma unroll 4
      for (int h = wave; h < a.n_q_heads; h += kWaves) {
        const f32x4 s = *(const f32x4*)(src + h * a.mods.score_stride + t);
        const float l = against(lse[h]);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] += fast_exp2(s[k] - l);
      }
    }
    return w;
  };
  const int64_t t_first = (int64_t)blockIdx.x * kTokens;
  if (lane == 0) s_same[wave] = mine;
  f32x4 w = head_sums(t_first);
  __syncthreads();
  mine = s_same[0] | s_same[1] | s_same[2] | s_same[3];
  if (mine & 1) return;
  if (mine == 0) {
    // (grid-stride: the grid is made for the longest request the host knows of)
    for (int64_t t0 = t_first; t0 < seen.y; t0 += (int64_t)gridDim.x * kTokens) {
      if (t0 != t_first) {
        w = head_sums(t0);
        __syncthreads();  // (the sums before these have been read)
      }
      s_sum[wave][lane] = w;
      __syncthreads();
      const int64_t t = t0 + tid;
      if (t < seen.y) {
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) sum += ((const float*)s_sum[v])[tid];
        const int64_t at = req * a.row_stride + seen.x + t;
        a.out[at] = a.old[at] + sum;
      }
    }
    return;
  }
  // (rare) several requests on one row: column by column, every one of them that sees it
  for (int64_t c = (int64_t)blockIdx.x * kTokens + tid; c < a.table_cols; c += (int64_t)gridDim.x * kTokens) {
    float sum = 0.f;
    bool any = false;
    for (int i = row; i < a.rows; ++i) {
      if (req_of(i) != req) continue;
      const int s = len_of(i);
      const int2 r = visible_range(a.mods, i, s, s);
      const int64_t t = c - r.x;
      if (t < 0 || t >= r.y) continue;
      any = true;
      const float* si = a.mods.scores + (int64_t)i * a.n_q_heads * a.mods.score_stride;
      for (int h = 0; h < a.n_q_heads; ++h) sum += fast_exp2(si[h * a.mods.score_stride + t] - against(a.lse[(int64_t)i * a.n_q_heads + h]));
    }
    const int64_t at = req * a.row_stride + c;
    if (any) a.out[at] = a.old[at] + sum;
  }
}

}  // namespace

hipError_t launch_token_weights(const WeightsArgs& a, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  const int64_t longest = a.len_hint > 0 && a.len_hint < a.table_cols ? a.len_hint : a.table_cols;
  const int64_t blocks = (longest + kTokens - 1) / kTokens;
  const dim3 grid((unsigned)(blocks < 1024 ? blocks : 1024), (unsigned)a.rows);
  hipLaunchKernelGGL(token_weights_kernel, grid, dim3(64 * kWaves), 0, stream, a);
  return hipGetLastError();
}

}  // namespace bsgl
