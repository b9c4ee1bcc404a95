// Eviction from the paged cache by accumulated attention weight: of every request the first `sinks` and the
// last `recent` tokens and, of those between, the ones with the largest weight are kept, `budget` in all
// (ties: the earlier token).  Page-table and weight rows are compacted in order; the slots of the others are
// listed.
//
// The m-th largest of the middle is found by radix selection on the weights as ordered integers: up to three
// histograms in LDS (11, 11 and 10 bits), each followed by one scan that finds the digit, ended early when the digit's
// bin holds exactly what is still wanted.  Then the tokens are dealt out in order: a wave owns a contiguous stretch, so
// positions come from wave-local scans and one exchange of the waves' totals.
//
//   evict_kernel    one workgroup per request, up to 16384 tokens in registers, longer rows chunk by chunk.  A chunk is in
//                   registers -- slots and weights -- before anything of it is written, and what is written never lies
//                   behind what has been read: the rows may be compacted in place.  Bound by latency: four trips to memory and
//                   a dozen barriers; the bytes (8 per token) hardly count.
//   split_* kernels for longer rows (kSplitFrom): a row is dealt over workgroups of 2048 tokens.  Each pass of the selection
//                   is a launch; the last workgroup of a row to arrive scans the row's histogram.  In place, the launch that
//                   clears the histograms also copies the row into the workspace, which everything behind it reads (a workgroup
//                   would otherwise write where another has not read yet).  Bound by its six launches.
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
__device__ __forceinline__ constexpr int pass_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ constexpr int pass_bits(int pass) { return pass == 2 ? 10 : 11; }

// A request's row and what is to be done with it.
struct Row {
  int n, n_keep;
  int lo, hi;  // the middle
  int m;       // how many of it stay: 0 <= m < hi - lo when n > budget
  const int32_t* t_in;
  const float* w_in;
  int32_t* t_out;
  float* w_out;
  int32_t* gone;
  bool rows16;  // whole groups of four may be read at once
  bool mine;    // no request before this one names the same row
};

// (NT threads, all of them)
template <int NT> __device__ __forceinline__ Row take_row(const EvictArgs& a, int row) {
  Row r;
  auto clamp_req = [&](int64_t x) { return x < 0 ? 0 : (x >= a.table_rows ? a.table_rows - 1 : x); };
  const int64_t req = clamp_req(a.req_idx[row]);
  const int64_t s64 = a.seq_lens[row];
  r.n = (int)(s64 < 0 ? 0 : (s64 > a.table_cols ? a.table_cols : s64));
  r.n_keep = min(r.n, a.budget);
  r.lo = a.sinks;
  r.hi = r.n - a.recent;
  r.m = a.budget - a.sinks - a.recent;
  r.t_in = a.table + req * a.table_row_stride;
  r.w_in = a.weights + req * a.weights_row_stride;
  r.t_out = a.out_table + req * a.table_row_stride;
  r.w_out = a.out_weights + req * a.weights_row_stride;
  r.gone = a.evicted == nullptr ? nullptr : a.evicted + (int64_t)row * a.evicted_row_stride;
  r.rows16 = (((uintptr_t)r.t_in | (uintptr_t)r.w_in) & 15) == 0;
  // a row named twice is compacted for its first request only
  bool mine = true;
  for (int i = threadIdx.x; i < row; i += NT) mine &= clamp_req(a.req_idx[i]) != req;
  r.mine = row == 0 || __syncthreads_and(mine);
  return r;
}

// Thread t of wave w holds the tokens base + w * 64 V + 256 j + 4 lane .. + 3, j = 0 .. V / 4 - 1.
template <int NT, int V> __device__ __forceinline__ int token_at(int base, int i) {
  return base + (int)(threadIdx.x >> 6) * (64 * V) + 256 * (i / 4) + 4 * (int)(threadIdx.x & 63) + (i & 3);
}
template <int NT, int V, typename T> __device__ __forceinline__ void load_row(const T* src, bool vec, int base, int n, T (&out)[V]) {
  typedef __attribute__((ext_vector_type(4))) T T4;
#pragma unroll
  for (int j = 0; j < V / 4; ++j) {
    const int at = token_at<NT, V>(base, 4 * j);
    if (vec && at + 3 < n) {
      const T4 x = *(const T4*)(src + at);
#pragma unroll
      for (int k = 0; k < 4; ++k) out[4 * j + k] = x[k];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) out[4 * j + k] = at + k < n ? src[at + k] : T(0);
    }
  }
}

// this chunk's part of a pass's histogram (LDS, zeroed by the caller)
template <int NT, int V> __device__ __forceinline__ void count_digits(uint32_t* hist, const float (&w)[V], const Row& r, int base, int pass, uint32_t prefix) {
  const int shift = pass_shift(pass), bits = pass_bits(pass);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int at = token_at<NT, V>(base, i);
    const uint32_t k = weight_key(w[i]);
    const bool in = at >= r.lo && at < r.hi && (pass == 0 || (k >> (shift + bits)) == prefix);
    const uint32_t d = (k >> shift) & ((1u << bits) - 1);
    const unsigned long long act = __ballot(in);
    if (act == 0) continue;
    // (a wave whose values share the digit -- weights that were never added to, say -- counts them at once: 64 adds to
    // one address take 64 turns)
    const uint32_t first = __builtin_amdgcn_readlane(d, __ffsll((long long)act) - 1);
    if (__all(!in || d == first)) {
      if ((threadIdx.x & 63) == 0) atomicAdd(&hist[first], (uint32_t)__popcll(act));
    } else if (in) {
      atomicAdd(&hist[d], 1u);
    }
  }
}

// The digit, counted from the top, in which the running count reaches `left`: {digit, count above it, its own count}.
// Thread t owns kBins / NT bins, the highest ones with thread 0; `bin(b)` reads one.
template <int NT, typename Bin> __device__ __forceinline__ void pick_digit(Bin bin, int left, uint32_t (&s_part)[NT / 64], uint32_t (&s_pick)[3]) {
  constexpr int BPT = kBins / NT;
  const int tid = threadIdx.x, wave = tid >> 6;
  uint32_t c[BPT], sum = 0;
#pragma unroll
  for (int b = 0; b < BPT; ++b) {
    c[b] = bin(kBins - 1 - (tid * BPT + b));
    sum += c[b];
  }
  const uint32_t incl = (uint32_t)wave_inclusive_scan<ScanAdd>((int)sum);
  if ((tid & 63) == 63) s_part[wave] = incl;
  __syncthreads();
  uint32_t run = incl - sum;
#pragma unroll
  for (int w = 0; w < NT / 64 - 1; ++w) run += w < wave ? s_part[w] : 0u;
#pragma unroll
  for (int b = 0; b < BPT; ++b) {
    if (run < (uint32_t)left && run + c[b] >= (uint32_t)left) {  // one thread, one bin
      s_pick[0] = (uint32_t)(kBins - 1 - (tid * BPT + b));
      s_pick[1] = run;
      s_pick[2] = c[b];
    }
    run += c[b];
  }
  __syncthreads();
}

// Where the selection stands: keys above `prefix` in their top `known` bits stay, `left` of the ones equal in them are
// still wanted.  done: exactly that many are there (or all bits are known, and the earliest `left` of them stay).
struct Pick {
  uint32_t prefix;
  int left;
  int known;
  bool all;  // every key with this prefix stays
};

// What a value is: 2 = stays, 1 = equal to the threshold (stays if early enough), 0 = goes
__device__ __forceinline__ int kind_of(float w, int at, const Row& r, const Pick& p) {
  if (at >= r.n) return 0;
  if (at < r.lo || at >= r.hi) return 2;
  if (r.m == 0) return 0;
  const uint32_t k = weight_key(w) >> (32 - p.known);
  return k > p.prefix ? 2 : k == p.prefix ? (p.all ? 2 : 1) : 0;
}

template <int NT, int V> __device__ __forceinline__ int2 count_kinds(const float (&w)[V], const Row& r, const Pick& p, int base) {
  int n2 = 0, n1 = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int k = kind_of(w[i], token_at<NT, V>(base, i), r, p);
    n2 += k == 2;
    n1 += k == 1;
  }
  return make_int2(__builtin_amdgcn_readlane(wave_inclusive_scan<ScanAdd>(n2), 63), __builtin_amdgcn_readlane(wave_inclusive_scan<ScanAdd>(n1), 63));
}

// how many of `count` equals stay when `before` equals stand ahead of them
__device__ __forceinline__ int equals_kept(int before, int count, int left) { return max(0, min(before + count, left) - min(before, left)); }

// deals out this wave's tokens: kept ones to t_out / w_out from `kept` on, the others' slots to r.gone
template <int NT, int V>
__device__ __forceinline__ void deal_out(const float (&w)[V], const int32_t (&slot)[V], const Row& r, const Pick& p, int base, int kept, int eq, int32_t* t_out,
                                         float* w_out, int gone_cols) {
#pragma unroll
  for (int j = 0; j < V / 4; ++j) {
    const int at0 = token_at<NT, V>(base, 4 * j);
    int kd[4], e4 = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      kd[k] = kind_of(w[4 * j + k], at0 + k, r, p);
      e4 += kd[k] == 1;
    }
    int e_at = eq, e_all = 0;
    if (__any(e4 != 0)) {
      const int e_incl = wave_inclusive_scan<ScanAdd>(e4);
      e_at += e_incl - e4;
      e_all = __builtin_amdgcn_readlane(e_incl, 63);
    }
    int k4 = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (kd[k] == 1) kd[k] = e_at++ < p.left ? 2 : 0;
      k4 += kd[k] == 2;
    }
    const int k_incl = wave_inclusive_scan<ScanAdd>(k4);
    int k_at = kept + k_incl - k4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int at = at0 + k;
      if (at >= r.n) continue;
      if (kd[k] == 2) {
        t_out[k_at] = slot[4 * j + k];
        w_out[k_at] = w[4 * j + k];
        ++k_at;
      } else {
        const int g = at - k_at;  // tokens before this one that go
        if (r.gone != nullptr && g < gone_cols) r.gone[g] = slot[4 * j + k];
      }
    }
    kept += __builtin_amdgcn_readlane(k_incl, 63);
    eq += e_all;
  }
}

// ---- one workgroup per request ------------------------------------------------------------------------
template <int NT, int V>
__global__ __launch_bounds__(NT) void evict_kernel(EvictArgs a) {
  constexpr int WAVES = NT / 64;
  constexpr int CHUNK = NT * V;
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint32_t s_part[WAVES];
  __shared__ uint32_t s_pick[3];
  __shared__ int2 s_wave[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x;
  for (int i = tid; i < kBins; i += NT) s_hist[i] = 0;
  const Row r = take_row<NT>(a, row);
  const int n = r.n;
  float w[V];
  const bool one_chunk = n <= CHUNK;
  if (one_chunk && n > a.budget) load_row<NT, V>(r.w_in, r.rows16, 0, n, w);
  if (tid == 0) a.new_lens[row] = r.n_keep;
  const int n_gone = r.mine ? n - r.n_keep : 0;
  if (r.gone != nullptr)
    for (int i = min(n_gone, a.evicted_cols) + tid; i < a.evicted_cols; i += NT) r.gone[i] = -1;
  if (!r.mine) return;
  if (n <= a.budget) {
    if (r.t_out != r.t_in)
      for (int i = tid; i < n; i += NT) r.t_out[i] = r.t_in[i];
    if (r.w_out != r.w_in)
      for (int i = tid; i < n; i += NT) r.w_out[i] = r.w_in[i];
    return;
  }
  int32_t slot[V];
  if (one_chunk) load_row<NT, V>(r.t_in, r.rows16, 0, n, slot);  // (travels while the threshold is looked for)
  Pick p = {0, r.m, 0, false};
  if (r.m > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      if (pass > 0)
        for (int i = tid; i < kBins; i += NT) s_hist[i] = 0;
      __syncthreads();
      for (int base = 0; base < n; base += CHUNK) {
        if (!one_chunk) load_row<NT, V>(r.w_in, r.rows16, base, n, w);
        count_digits<NT, V>(s_hist, w, r, base, pass, p.prefix);
      }
      __syncthreads();
      pick_digit<NT>([&](int b) { return s_hist[b]; }, p.left, s_part, s_pick);
      p.prefix = (p.prefix << pass_bits(pass)) | s_pick[0];
      p.left -= (int)s_pick[1];
      p.known += pass_bits(pass);
      p.all = (int)s_pick[2] == p.left;
      if (p.all) break;
    }
  }

  // ---- deal out, chunk by chunk
  int kept_base = 0, eq_base = 0;  // of the chunks before this one
#pragma unroll 1
  for (int base = 0; base < n; base += CHUNK) {
    if (!one_chunk) {
      load_row<NT, V>(r.w_in, r.rows16, base, n, w);
      load_row<NT, V>(r.t_in, r.rows16, base, n, slot);
    }
    const int2 mine = count_kinds<NT, V>(w, r, p, base);
    __syncthreads();  // (s_wave of the chunk before has been read)
    if (lane == 0) s_wave[wave] = mine;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // this wave's slots and weights have arrived: nothing is written before everybody's have
    __syncthreads();
    int kept = kept_base, eq = eq_base, chunk2 = 0, chunk1 = 0;
    for (int v = 0; v < WAVES; ++v) {
      const int2 x = s_wave[v];
      if (v < wave) {
        kept += x.x + equals_kept(eq, x.y, p.left);
        eq += x.y;
      }
      chunk2 += x.x;
      chunk1 += x.y;
    }
    deal_out<NT, V>(w, slot, r, p, base, kept, eq, r.t_out, r.w_out, a.evicted_cols);
    kept_base += chunk2 + equals_kept(eq_base, chunk1, p.left);
    eq_base += chunk1;
  }
}

// ---- a row over several workgroups ----------------------------------------------------------------------
constexpr int kNT = 256, kV = 8;
constexpr int kSlice = kNT * kV;
constexpr int kSplitFrom = 16384;  // rows up to this many tokens stay with one workgroup

// of a request, in the workspace
struct SplitState {
  uint32_t hist[3][kBins];
  uint32_t arrived[3];
  Pick pick[3];  // after each pass
};
// behind the batch's states: per request [slices] counts, then the row's slots and weights

__device__ __forceinline__ SplitState* state_of(const EvictArgs& a, int row) { return (SplitState*)a.workspace + row; }
__device__ __forceinline__ int2* counts_of(const EvictArgs& a, int row) {
  return (int2*)((char*)a.workspace + a.counts_at) + (int64_t)row * a.slices;
}
__device__ __forceinline__ int32_t* staged_of(const EvictArgs& a, int row) {
  return (int32_t*)((char*)a.workspace + a.staged_at) + (int64_t)row * 2 * a.staged_row;
}

__global__ __launch_bounds__(kNT) void split_start_kernel(EvictArgs a) {
  const int row = blockIdx.y;
  uint32_t* dst = (uint32_t*)state_of(a, row);
  for (int i = blockIdx.x * kNT + threadIdx.x; i < (int)(sizeof(SplitState) / 4); i += gridDim.x * kNT) dst[i] = 0;
  if (!a.staged) return;
  const Row r = take_row<kNT>(a, row);
  const int base = blockIdx.x * kSlice;
  if (!r.mine || r.n <= a.budget || base >= r.n) return;
  int32_t* t = staged_of(a, row);
  float* w = (float*)(t + a.staged_row);
  const int end = min(r.n, base + kSlice);
  for (int i = base + (int)threadIdx.x; i < end; i += kNT) {
    t[i] = r.t_in[i];
    w[i] = r.w_in[i];
  }
}

// a row of the kernels behind that one, if it is to be cut: read from its copy where there is one
__device__ __forceinline__ Row take_staged_row(const EvictArgs& a, int row) {
  Row r = take_row<kNT>(a, row);
  if (a.staged && r.n > a.budget) {
    r.t_in = staged_of(a, row);
    r.w_in = (const float*)(r.t_in + a.staged_row);
    r.rows16 = true;
  }
  return r;
}

// the selection as it stood before `pass`
__device__ __forceinline__ Pick pick_before(const SplitState* st, const Row& r, int pass) {
  if (pass == 0) return {0, r.m, 0, false};
  return st->pick[pass - 1];
}

__global__ __launch_bounds__(kNT) void split_pass_kernel(EvictArgs a, int pass) {
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint32_t s_part[kNT / 64];
  __shared__ uint32_t s_pick[3];
  __shared__ uint32_t s_ticket;
  const int tid = threadIdx.x;
  const int row = blockIdx.y;
  const int base = blockIdx.x * kSlice;
  for (int i = tid; i < kBins; i += kNT) s_hist[i] = 0;
  const Row r = take_staged_row(a, row);
  SplitState* st = state_of(a, row);
  const Pick before = pick_before(st, r, pass);
  // (nothing to select, or the selection has ended: the same for every workgroup of the row)
  if (!r.mine || r.n <= a.budget || r.m == 0 || base >= r.n) return;
  if (before.all) {
    if (blockIdx.x == 0 && tid == 0) st->pick[pass] = before;
    return;
  }
  float w[kV];
  load_row<kNT, kV>(r.w_in, r.rows16, base, r.n, w);
  __syncthreads();
  count_digits<kNT, kV>(s_hist, w, r, base, pass, before.prefix);
  __syncthreads();
  for (int i = tid; i < kBins; i += kNT) {
    const uint32_t c = s_hist[i];
    if (c != 0) __hip_atomic_fetch_add(&st->hist[pass][i], c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // The last workgroup of the row looks at the whole.  The adds, the ticket and the loads below are agent-scope atomics, all made
  // where the XCDs' caches meet, so all it takes is that this workgroup's adds have been made before its ticket is drawn
  // (a release fence would write back the whole L2: 64 rows x 131072 tokens 451 us with it)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const uint32_t n_wg = (uint32_t)((r.n + kSlice - 1) / kSlice);
  if (tid == 0) s_ticket = __hip_atomic_fetch_add(&st->arrived[pass], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_ticket != n_wg - 1) return;
  pick_digit<kNT>([&](int b) { return __hip_atomic_load(&st->hist[pass][b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }, before.left, s_part, s_pick);
  if (tid == 0) {
    Pick p;
    p.prefix = (before.prefix << pass_bits(pass)) | s_pick[0];
    p.left = before.left - (int)s_pick[1];
    p.known = before.known + pass_bits(pass);
    p.all = (int)s_pick[2] == p.left;
    st->pick[pass] = p;
  }
}

__global__ __launch_bounds__(kNT) void split_count_kernel(EvictArgs a) {
  __shared__ int2 s_wave[kNT / 64];
  const int row = blockIdx.y;
  const int base = blockIdx.x * kSlice;
  const Row r = take_staged_row(a, row);
  if (!r.mine || r.n <= a.budget || base >= r.n) return;
  const Pick p = r.m > 0 ? state_of(a, row)->pick[2] : Pick{0, 0, 0, false};
  float w[kV];
  load_row<kNT, kV>(r.w_in, r.rows16, base, r.n, w);
  const int2 mine = count_kinds<kNT, kV>(w, r, p, base);
  if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    int2 sum = make_int2(0, 0);
    for (int v = 0; v < kNT / 64; ++v) {
      sum.x += s_wave[v].x;
      sum.y += s_wave[v].y;
    }
    counts_of(a, row)[blockIdx.x] = sum;
  }
}

__global__ __launch_bounds__(kNT) void split_deal_kernel(EvictArgs a) {
  __shared__ int2 s_wave[kNT / 64];
  __shared__ int2 s_before[kNT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.y;
  const int base = blockIdx.x * kSlice;
  const Row r = take_staged_row(a, row);
  const int n = r.n;
  const int n_gone = r.mine ? n - r.n_keep : 0;
  if (blockIdx.x == 0 && tid == 0) a.new_lens[row] = r.n_keep;
  if (r.gone != nullptr)
    for (int64_t i = min(n_gone, a.evicted_cols) + (int64_t)blockIdx.x * kNT + tid; i < a.evicted_cols; i += (int64_t)gridDim.x * kNT) r.gone[i] = -1;
  if (!r.mine || base >= n) return;
  if (n <= a.budget) {
    const int end = min(n, base + kSlice);
    if (r.t_out != r.t_in)
      for (int i = base + tid; i < end; i += kNT) r.t_out[i] = r.t_in[i];
    if (r.w_out != r.w_in)
      for (int i = base + tid; i < end; i += kNT) r.w_out[i] = r.w_in[i];
    return;
  }
  const Pick p = r.m > 0 ? state_of(a, row)->pick[2] : Pick{0, 0, 0, false};
  float w[kV];
  int32_t slot[kV];
  load_row<kNT, kV>(r.w_in, r.rows16, base, n, w);
  load_row<kNT, kV>(r.t_in, r.rows16, base, n, slot);
  // what the slices before this one keep
  const int2* counts = counts_of(a, row);
  int2 sum = make_int2(0, 0);
  for (int i = tid; i < (int)blockIdx.x; i += kNT) {
    const int2 c = counts[i];
    sum.x += c.x;
    sum.y += c.y;
  }
  const int b2 = __builtin_amdgcn_readlane(wave_inclusive_scan<ScanAdd>(sum.x), 63), b1 = __builtin_amdgcn_readlane(wave_inclusive_scan<ScanAdd>(sum.y), 63);
  const int2 mine = count_kinds<kNT, kV>(w, r, p, base);
  if (lane == 0) {
    s_before[wave] = make_int2(b2, b1);
    s_wave[wave] = mine;
  }
  __syncthreads();
  int kept = 0, eq = 0;
  for (int v = 0; v < kNT / 64; ++v) {
    kept += s_before[v].x;
    eq += s_before[v].y;
  }
  kept += min(eq, p.left);
  for (int v = 0; v < wave; ++v) {
    kept += s_wave[v].x + equals_kept(eq, s_wave[v].y, p.left);
    eq += s_wave[v].y;
  }
  deal_out<kNT, kV>(w, slot, r, p, base, kept, eq, r.t_out, r.w_out, a.evicted_cols);
}

}  // namespace

// Rows longer than kSplitFrom are split; the workspace is for them.
size_t evict_workspace(int64_t batch, int64_t longest, int64_t* counts_at, int64_t* staged_at, int64_t* staged_row) {
  if (longest <= kSplitFrom || batch <= 0) return 0;
  const int64_t slices = (longest + kSlice - 1) / kSlice;
  const int64_t row = (longest + 63) / 64 * 64;
  const int64_t counts = (batch * (int64_t)sizeof(SplitState) + 255) / 256 * 256;
  const int64_t staged = counts + (batch * slices * 8 + 255) / 256 * 256;
  if (counts_at != nullptr) *counts_at = counts;
  if (staged_at != nullptr) *staged_at = staged;
  if (staged_row != nullptr) *staged_row = row;
  return (size_t)(staged + batch * row * 8);
}

hipError_t launch_evict(const EvictArgs& a_in, hipStream_t stream) {
  EvictArgs a = a_in;
  if (a.batch == 0) return hipSuccess;
  if (a.longest > kSplitFrom) {
    // one workgroup takes 1.2 us per 1000 tokens there, the split form's six launches some 20 us whatever the length
    a.slices = (int32_t)((a.table_cols + kSlice - 1) / kSlice);  // (a hint that is too small must not cost a token)
    evict_workspace(a.batch, a.table_cols, &a.counts_at, &a.staged_at, &a.staged_row);
    a.staged = a.out_table == a.table || a.out_weights == a.weights;
    const dim3 grid((unsigned)a.slices, (unsigned)a.batch);
    hipLaunchKernelGGL(split_start_kernel, grid, dim3(kNT), 0, stream, a);
    for (int pass = 0; pass < 3; ++pass) hipLaunchKernelGGL(split_pass_kernel, grid, dim3(kNT), 0, stream, a, pass);
    hipLaunchKernelGGL(split_count_kernel, grid, dim3(kNT), 0, stream, a);
    hipLaunchKernelGGL(split_deal_kernel, grid, dim3(kNT), 0, stream, a);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)a.batch);
  auto go = [&](auto kernel, int nt) { hipLaunchKernelGGL(kernel, grid, dim3(nt), 0, stream, a); };
  if (a.longest <= 1024) go(evict_kernel<256, 4>, 256);
  else if (a.longest <= 2048) go(evict_kernel<512, 4>, 512);
  else if (a.longest <= 4096) go(evict_kernel<1024, 4>, 1024);
  else if (a.longest <= 8192) go(evict_kernel<1024, 8>, 1024);
  else go(evict_kernel<1024, 16>, 1024);
  return hipGetLastError();
}

}  // namespace bsgl
