// KV scatter and prefill row expansion for gfx950.
//
// kv_scatter_kernel: k_slab[loc[t]] = k_new[t]; v_slab[loc[t]] = v_new[t]
// (reference: memory_pool.py:152-171).  Pure byte movement, 16 B per lane, so one
// instance serves every dtype; source rows may be strided views.
//
// prefill_expand: turns the per-request (prefix_lens, extended_lens) of an
// extend batch into one (page-table row, visible length) pair per q row, so
// that row r of request i sees positions 0 .. prefix_lens[i] + r -- the
// causal-with-prefix mask of attn_backend.py:74-92 expressed as a length.
#include "bsgl_device.h"
#include "bsgl_launch.h"

namespace bsgl {

namespace {

__global__ __launch_bounds__(256) void kv_scatter_kernel(ScatterArgs a) {
  const int pieces = a.row_bytes >> 4;
  const int64_t gid = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t total = (int64_t)a.n_tok * pieces;
  if (gid >= total) return;
  const int t = (int)(gid / pieces);
  const int p = (int)(gid % pieces);
  const int64_t slot = a.loc[t];
  if (slot < 0 || slot >= a.n_slots) return;
  const int64_t dst = slot * a.slab_row_stride * a.elem_bytes + (int64_t)p * 16;
  const uint4 kv = *(const uint4*)((const char*)a.k_new + (int64_t)t * a.k_row_stride * a.elem_bytes + (int64_t)p * 16);
  const uint4 vv = *(const uint4*)((const char*)a.v_new + (int64_t)t * a.v_row_stride * a.elem_bytes + (int64_t)p * 16);
  *(uint4*)((char*)a.k_slab + dst) = kv;
  *(uint4*)((char*)a.v_slab + dst) = vv;
}

// exclusive running sums of extended_lens and of the block groups of each request,
// ceil(ceil(extended_lens / blk_rows) / grp_blocks)  (negative lengths count as 0, lengths above
// the number of q rows as that number)
// (`starts`: the groups' sums once more, in LDS, or NULL)
__device__ __forceinline__ void running_sums(const ExpandArgs& a, int* starts = nullptr) {
  __shared__ int64_t s_ext[256], s_blk[256];
  const int tid = threadIdx.x;
  const int per = (a.batch + 255) / 256;
  const int lo = min(tid * per, a.batch), hi = min(lo + per, a.batch);
  // (lengths are bounded by the number of q rows, an int: 32-bit unsigned divisions, a fraction of the
  // instructions of 64-bit ones)
  const uint32_t br = a.blk_rows > 0 ? (uint32_t)a.blk_rows : 16u;
  const uint32_t gb = a.grp_blocks > 0 ? (uint32_t)a.grp_blocks : 1u;
  auto groups_of = [&](int64_t e) { return (int64_t)((((uint32_t)e + br - 1) / br + gb - 1) / gb); };
  int64_t sum = 0, blocks = 0;
  for (int i = lo; i < hi; ++i) {
    const int64_t e = min(max((int64_t)0, a.extended_lens[i]), (int64_t)a.total_q_tokens);  // (bounded: the sums cannot overflow)
    sum += e;
    blocks += groups_of(e);
  }
  // exclusive scan over the 256 threads' partial sums: inside a wave by shuffles, across the four waves
  // through LDS (one thread walking all 256 entries took 4 of this launch's 8 microseconds)
  const int lane = tid & 63, wave = tid >> 6;
  int64_t inc_e = sum, inc_b = blocks;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t oe = __shfl_up(inc_e, d), ob = __shfl_up(inc_b, d);
    if (lane >= d) { inc_e += oe; inc_b += ob; }
  }
  if (lane == 63) { s_ext[wave] = inc_e; s_blk[wave] = inc_b; }
  __syncthreads();
  int64_t run = inc_e - sum, brun = inc_b - blocks;
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    if (w < wave) { run += s_ext[w]; brun += s_blk[w]; }
  }
  if (tid == 255) {
    a.cu_ext[a.batch] = run + sum;
    if (a.cu_blk != nullptr) {
      a.cu_blk[a.batch] = brun + blocks;
      a.cu_blk[a.batch + 1] = a.order != nullptr;
    }
    if (starts != nullptr) starts[a.batch] = (int)min(brun + blocks, (int64_t)0x7fffffff);
  }
  for (int i = lo; i < hi; ++i) {
    const int64_t e = min(max((int64_t)0, a.extended_lens[i]), (int64_t)a.total_q_tokens);  // (bounded: the sums cannot overflow)
    a.cu_ext[i] = run;
    if (a.cu_blk != nullptr) a.cu_blk[i] = brun;
    if (starts != nullptr) starts[i] = (int)brun;
    run += e;
    brun += groups_of(e);
  }
}

__global__ __launch_bounds__(256) void prefill_cu_kernel(ExpandArgs a) { running_sums(a); }

// The same and the order in which the scored extend kernel launches its groups: the longest streams first, so that the launch does not end
// on a few of them (what a group streams is taken from its first row's beginning and its last row's end, exact for
// causal, prefix, window and document masks).  A counting sort by 256 lengths; the order inside one is any.
__global__ __launch_bounds__(256) void prefill_order_kernel(ExpandArgs a) {
  __shared__ int s_start[kMaxOrder + 1];
  __shared__ int s_bucket[256];
  __shared__ int s_part[4], s_max[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  running_sums(a, s_start);
  s_bucket[tid] = 0;
  __threadfence_block();
  __syncthreads();
  const int n = s_start[a.batch];
  if (n > a.n_order) {
    for (int g = tid; g < a.n_order; g += 256) a.order[g] = g;
    return;
  }
  constexpr int PER = kMaxOrder / 256;
  const int64_t rows = (int64_t)max(a.grp_blocks, 1) * max(a.blk_rows, 1);
  int key[PER], longest = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int g = tid + 256 * k;
    key[k] = -1;
    if (g >= n) continue;
    int lo = 0, hi = a.batch;  // the last request that starts at g or before
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_start[mid] <= g) lo = mid; else hi = mid;
    }
    const int64_t ext = min(max((int64_t)0, a.extended_lens[lo]), (int64_t)a.total_q_tokens);
    const int64_t seq = min(max((int64_t)0, a.seq_lens[lo]), a.table_cols);
    const int64_t prefix = min(max((int64_t)0, a.prefix_lens[lo]), seq);
    const int64_t r0 = (g - s_start[lo]) * rows, r1 = min(r0 + rows, ext) - 1;
    const int64_t at = a.cu_ext[lo], last_row = (int64_t)a.total_q_tokens - 1;
    int64_t end = min(seq, prefix + r1 + 1), begin = 0;
    if (a.to != nullptr) end = min(seq, (int64_t)a.to[min(at + r1, last_row)]);
    if (a.from != nullptr) begin = max((int64_t)0, (int64_t)a.from[min(at + r0, last_row)]);
    key[k] = (int)max((int64_t)0, min(end - begin, (int64_t)0x7fffffff));  // (never negative: every group has a place)
    longest = max(longest, key[k]);
  }
  longest = __builtin_amdgcn_readlane(wave_inclusive_scan<ScanMax>(longest), 63);
  if (lane == 0) s_max[wave] = longest;
  __syncthreads();
  longest = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
  const float f = 255.f / (float)max(longest, 1);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (key[k] < 0) continue;
    key[k] = 255 - min(255, (int)((float)key[k] * f));
    atomicAdd(&s_bucket[key[k]], 1);
  }
  __syncthreads();
  const int incl = wave_inclusive_scan<ScanAdd>(s_bucket[tid]);
  if (lane == 63) s_part[wave] = incl;
  __syncthreads();
  int before = incl - s_bucket[tid];
  for (int w = 0; w < wave; ++w) before += s_part[w];
  s_bucket[tid] = before;  // (its own entry only)
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PER; ++k)
    if (key[k] >= 0) a.order[atomicAdd(&s_bucket[key[k]], 1)] = tid + 256 * k;
}

// what the decode kernels have to know about extend token t
__device__ __forceinline__ void expand_row(const ExpandArgs& a, int t) {
  // last request i with cu_ext[i] <= t
  int lo = 0, hi = a.batch;  // invariant: cu_ext[lo] <= t (cu_ext[0] == 0), answer in [lo, hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_ext[mid] <= t) lo = mid; else hi = mid;
  }
  // requests with extended_lens == 0 share a start with their successor; the
  // search above lands on the LAST request starting at or before t, which is
  // the one that owns the row.
  int64_t len = 0, req = 0;
  if (a.rows4 != nullptr) {
    int4 r4 = make_int4(0, 0, 0, 0);
    if (a.batch > 0 && t < a.cu_ext[a.batch]) {
      auto i32 = [](int64_t x) { return (int)max((int64_t)0, min(x, (int64_t)0x7fffffff)); };
      const int64_t full = max((int64_t)0, a.seq_lens[lo]);
      const int64_t prefix = max((int64_t)0, min(a.prefix_lens[lo], full));
      r4 = make_int4(i32(a.req_pool_indices[lo]), i32(full), i32(prefix + (t - a.cu_ext[lo])), 1);
    }
    a.rows4[t] = r4;
    return;
  }
  if (a.batch > 0 && t < a.cu_ext[a.batch]) {
    const int64_t r = t - a.cu_ext[lo];
    req = a.req_pool_indices[lo];
    len = a.prefix_lens[lo] + r + 1;
    const int64_t full = a.seq_lens[lo];
    len = len > full ? full : len;
    len = len < 0 ? 0 : len;
  }
  a.row_req[t] = req;
  a.row_len[t] = len;
}

__global__ __launch_bounds__(256) void prefill_rows_kernel(ExpandArgs a) {
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= a.total_q_tokens) return;
  expand_row(a, t);
}

// A few extend tokens that run as rows of the decode kernel: sums, rows and zeroed tickets in one workgroup.
__global__ __launch_bounds__(256) void prefill_few_kernel(ExpandArgs a) {
  for (int i = threadIdx.x; i < a.n_clear; i += 256) a.clear[i] = 0;
  running_sums(a);
  __threadfence_block();
  __syncthreads();
  for (int t = threadIdx.x; t < a.total_q_tokens; t += 256) expand_row(a, t);
}

}  // namespace

hipError_t launch_kv_scatter(const ScatterArgs& a, hipStream_t stream) {
  if (a.n_tok == 0) return hipSuccess;
  const int64_t total = (int64_t)a.n_tok * (a.row_bytes >> 4);
  hipLaunchKernelGGL(kv_scatter_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_prefill_expand(const ExpandArgs& a, hipStream_t stream) {
  if (a.clear != nullptr) {
    hipLaunchKernelGGL(prefill_few_kernel, dim3(1), dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  if (a.order != nullptr && (a.batch > kMaxOrder || a.n_order > kMaxOrder)) return hipErrorInvalidValue;
  if (a.order != nullptr) hipLaunchKernelGGL(prefill_order_kernel, dim3(1), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(prefill_cu_kernel, dim3(1), dim3(256), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.total_q_tokens == 0 || (a.row_req == nullptr && a.rows4 == nullptr)) return e;
  hipLaunchKernelGGL(prefill_rows_kernel, dim3((a.total_q_tokens + 255) / 256), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace bsgl
