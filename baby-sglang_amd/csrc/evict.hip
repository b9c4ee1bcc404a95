// Eviction from the paged cache by accumulated attention weight: of every request the first `sinks` and the
// last `recent` tokens and, of those between, the ones with the largest weight are kept, `budget` in all
// (ties: the earlier token).  Page-table and weight rows are compacted in order; the slots of the others are
// listed.
//
// One workgroup per request.  The m-th largest of the middle is found by radix selection on the weights as
// ordered integers: three histograms in LDS (11, 11 and 10 bits), each followed by one scan that finds the
// digit.  Then one pass in order: wave w owns the w-th contiguous stretch of a chunk, so that positions come from wave-local
// scans and one exchange of the waves' totals per chunk.  A chunk is in registers -- slots and weights -- before anything of
// it is written, and what is written never lies behind what has been read: the rows may be compacted in place.
// Bound by latency: 12 barriers and four trips to memory; the bytes (8 per token) are read at a CU's own rate.
#include "bsgl_device.h"
#include "bsgl_launch.h"

namespace bsgl {

namespace {

// weights as unsigned integers in the same order: NaN above everything (whatever its sign), -0 equal to 0
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = as_u32(w + 0.f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

constexpr int kBins = 2048;

// NT threads, V values of each thread and chunk (V a multiple of 4): lane l of wave w holds the tokens
// w * 64 V + 256 j + 4 l .. + 3 of the chunk, j = 0 .. V / 4 - 1
template <int NT, int V>
__global__ __launch_bounds__(NT) void evict_kernel(EvictArgs a) {
  constexpr int WAVES = NT / 64;
  constexpr int CHUNK = NT * V;
  constexpr int NJ = V / 4;
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint32_t s_part[WAVES];
  __shared__ uint32_t s_pick[3];  // digit found, elements above it, elements in it
  __shared__ int2 s_wave[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x;
  const int64_t r64 = a.req_idx[row];
  const int64_t req = r64 < 0 ? 0 : (r64 >= a.table_rows ? a.table_rows - 1 : r64);
  const int64_t s64 = a.seq_lens[row];
  const int n = (int)(s64 < 0 ? 0 : (s64 > a.table_cols ? a.table_cols : s64));
  // a row named twice is compacted for its first request only
  bool mine = true;
  for (int i = tid; i < row; i += NT) {
    const int64_t o = a.req_idx[i];
    mine &= (o < 0 ? 0 : (o >= a.table_rows ? a.table_rows - 1 : o)) != req;
  }
  mine = __syncthreads_and(mine);
  const int n_keep = min(n, a.budget);
  if (tid == 0) a.new_lens[row] = n_keep;
  int32_t* gone = a.evicted == nullptr ? nullptr : a.evicted + (int64_t)row * a.evicted_row_stride;
  const int n_gone = mine ? n - n_keep : 0;
  if (gone != nullptr)
    for (int i = min(n_gone, a.evicted_cols) + tid; i < a.evicted_cols; i += NT) gone[i] = -1;
  if (!mine) return;
  const int32_t* t_in = a.table + req * a.table_row_stride;
  const float* w_in = a.weights + req * a.weights_row_stride;
  int32_t* t_out = a.out_table + req * a.table_row_stride;
  float* w_out = a.out_weights + req * a.weights_row_stride;
  if (n <= a.budget) {
    if (t_out != t_in)
      for (int i = tid; i < n; i += NT) t_out[i] = t_in[i];
    if (w_out != w_in)
      for (int i = tid; i < n; i += NT) w_out[i] = w_in[i];
    return;
  }
  const int lo = a.sinks, hi = n - a.recent;           // the middle
  const int m = a.budget - a.sinks - a.recent;         // how many of it stay: 0 <= m < hi - lo
  const bool rows16 = (((uintptr_t)t_in | (uintptr_t)w_in) & 15) == 0;  // whole groups of four may be read at once

  uint32_t key[V];
  auto load_keys = [&](int base) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int at = base + wave * (64 * V) + 256 * j + 4 * lane;
      float w[4] = {0.f, 0.f, 0.f, 0.f};
      if (rows16 && at + 3 < n) {
        const float4 x = *(const float4*)(w_in + at);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (at + k < n) w[k] = w_in[at + k];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) key[4 * j + k] = as_u32(w[k]);
    }
  };
  const bool one_chunk = n <= CHUNK;
  if (one_chunk) load_keys(0);

  // ---- the m-th largest key of the middle, and how many of its equals stay --------------------------
  uint32_t thresh = 0xffffffffu, prefix = 0;
  int need_eq = 0;
  if (m > 0) {
    int left = m;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const int bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < kBins; i += NT) s_hist[i] = 0;
      __syncthreads();
      for (int base = 0; base < n; base += CHUNK) {
        if (!one_chunk) load_keys(base);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int at = base + wave * (64 * V) + 256 * (i / 4) + 4 * lane + (i & 3);
          const uint32_t kx = weight_key(as_f32(key[i]));
          const bool in = at >= lo && at < hi && (pass == 0 || (kx >> (shift + bits)) == prefix);
          const uint32_t d = (kx >> shift) & ((1u << bits) - 1);
          const unsigned long long act = __ballot(in);
          if (act == 0) continue;
          // (a wave whose values share the digit -- weights that were never added to, say -- counts them at once: 64 adds to
          // one address take 64 turns)
          const uint32_t first = __builtin_amdgcn_readlane(d, __ffsll((long long)act) - 1);
          if (__all(!in || d == first)) {
            if (lane == 0) atomicAdd(&s_hist[first], (uint32_t)__popcll(act));
          } else if (in) {
            atomicAdd(&s_hist[d], 1u);
          }
        }
      }
      __syncthreads();
      // from the top: the digit in which the running count passes `left`.  Thread t owns kBins / NT bins, the
      // highest bins with thread 0
      constexpr int BPT = kBins / NT;
      uint32_t c[BPT], sum = 0;
#pragma unroll
      for (int b = 0; b < BPT; ++b) {
        c[b] = s_hist[kBins - 1 - (tid * BPT + b)];
        sum += c[b];
      }
      const uint32_t incl = (uint32_t)wave_inclusive_scan<ScanAdd>((int)sum);
      if (lane == 63) s_part[wave] = incl;
      __syncthreads();
      uint32_t run = incl - sum;
      for (int w = 0; w < wave; ++w) run += s_part[w];
#pragma unroll
      for (int b = 0; b < BPT; ++b) {
        if (run < (uint32_t)left && run + c[b] >= (uint32_t)left) {  // one thread, one bin
          s_pick[0] = (uint32_t)(kBins - 1 - (tid * BPT + b));
          s_pick[1] = run;
        }
        run += c[b];
      }
      __syncthreads();
      prefix = (prefix << bits) | s_pick[0];
      left -= (int)s_pick[1];
    }
    thresh = prefix;
    need_eq = left;
  }

  // ---- compaction, chunk by chunk ------------------------------------------------------------------
  int kept_base = 0, eq_base = 0;  // of the chunks before this one
#pragma unroll 1
  for (int base = 0; base < n; base += CHUNK) {
    if (!one_chunk) load_keys(base);
    int32_t slot[V];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int at = base + wave * (64 * V) + 256 * j + 4 * lane;
      if (rows16 && at + 3 < n) {
        const int4 x = *(const int4*)(t_in + at);
        slot[4 * j] = x.x; slot[4 * j + 1] = x.y; slot[4 * j + 2] = x.z; slot[4 * j + 3] = x.w;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) slot[4 * j + k] = at + k < n ? t_in[at + k] : 0;
      }
    }
    // what each value is: 2 = stays, 1 = equal to the threshold (stays if early enough), 0 = goes
    auto kind = [&](int i, int at) {
      if (at >= n) return 0;
      if (at < lo || at >= hi) return 2;
      if (m == 0) return 0;
      const uint32_t kx = weight_key(as_f32(key[i]));
      return kx > thresh ? 2 : kx == thresh ? 1 : 0;
    };
    int n2 = 0, n1 = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int k = kind(i, base + wave * (64 * V) + 256 * (i / 4) + 4 * lane + (i & 3));
      n2 += k == 2;
      n1 += k == 1;
    }
    n2 = __builtin_amdgcn_readlane(wave_inclusive_scan<ScanAdd>(n2), 63);
    n1 = __builtin_amdgcn_readlane(wave_inclusive_scan<ScanAdd>(n1), 63);
    __syncthreads();  // (s_wave of the chunk before has been read; in place: everybody's values are in registers below)
    if (lane == 0) s_wave[wave] = make_int2(n2, n1);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // this wave's slots and weights have arrived
    __syncthreads();
    int kept = kept_base, eq = eq_base, chunk2 = 0, chunk1 = 0;
    for (int w = 0; w < WAVES; ++w) {
      const int2 x = s_wave[w];
      if (w < wave) {
        kept += x.x + max(0, min(eq + x.y, need_eq) - min(eq, need_eq));
        eq += x.y;
      }
      chunk2 += x.x;
      chunk1 += x.y;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int at0 = base + wave * (64 * V) + 256 * j + 4 * lane;
      int kd[4], e4 = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        kd[k] = kind(4 * j + k, at0 + k);
        e4 += kd[k] == 1;
      }
      const int e_incl = wave_inclusive_scan<ScanAdd>(e4);
      int e_at = eq + e_incl - e4, k4 = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (kd[k] == 1) kd[k] = e_at++ < need_eq ? 2 : 0;
        k4 += kd[k] == 2;
      }
      const int k_incl = wave_inclusive_scan<ScanAdd>(k4);
      int k_at = kept + k_incl - k4;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int at = at0 + k;
        if (at >= n) continue;
        if (kd[k] == 2) {
          t_out[k_at] = slot[4 * j + k];
          w_out[k_at] = as_f32(key[4 * j + k]);
          ++k_at;
        } else {
          const int g = at - k_at;  // tokens before this one that go
          if (gone != nullptr && g < a.evicted_cols) gone[g] = slot[4 * j + k];
        }
      }
      kept += __builtin_amdgcn_readlane(k_incl, 63);
      eq += __builtin_amdgcn_readlane(e_incl, 63);
    }
    kept_base += chunk2 + max(0, min(eq_base + chunk1, need_eq) - min(eq_base, need_eq));
    eq_base += chunk1;
  }
}

}  // namespace

hipError_t launch_evict(const EvictArgs& a, hipStream_t stream) {
  if (a.batch == 0) return hipSuccess;
  const dim3 grid((unsigned)a.batch);
  if (a.longest <= 1024) hipLaunchKernelGGL((evict_kernel<256, 4>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((evict_kernel<1024, 16>), grid, dim3(1024), 0, stream, a);
  return hipGetLastError();
}

}  // namespace bsgl
