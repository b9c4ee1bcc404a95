// Scored decode attention in 32 bits for gfx950 (the scores: ScoreMods; the plain f32 rows and what this kernel does not
// take stay with paged_decode_valu.hip): head_dim 64 or 128, up to 16 q heads per kv head.
//
// One workgroup per (request, kv head, piece of its visible tokens), four waves that take the piece's tiles of 16 tokens in
// turn.  The products are v_mfma_f32_16x16x4_f32, f32 by f32, with every operand loaded from memory as the product wants it,
// so nothing passes through LDS and no lane adds up another's sums (those sums, two dozen per lane and step in the generic
// kernel, and a tanh of each on every lane of the row, are what made a capped f32 decode run at half its bandwidth):
//   S^T = K Q^T   lane (c, u) = (lane & 15, lane >> 4) reads 16 bytes of token c per load, values 16 j + 4 u ..; Q in the
//                 same order.  It then owns the scores of head c and tokens 4 u .. 4 u + 3.
//   O  += P V     product i takes token 4 u + i of each u: P from the register it is in, V as D / 16 neighbouring values
//                 of the token per lane (which columns of the product they are is this kernel's choice).
// The next tile's K is asked for as soon as the scores are made of this one's, its V behind the last product: both are
// always on their way, in the registers of one tile (two tiles' worth spilled); bound by memory (see launch_decode_scored_f32 for what it
// reached).  The waves' results meet in LDS, pieces in the workspace: the last workgroup of a (request, kv head) to finish
// -- a ticket -- merges them, or a launch of its own where the tickets do not fit.
#include "bsgl_device.h"
#include "bsgl_launch.h"
#include "bsgl_mfma.h"
#include "bsgl_score.h"

namespace bsgl {

namespace {

using namespace mfma;

typedef __attribute__((ext_vector_type(4))) float f32x4v;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4v;

constexpr int kWaves = 4;
constexpr int kTokens = 16;  // per tile

template <int D>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(3)))
void decode_scored_f32_kernel(DecodeArgs a) {
  constexpr int KN = D / 16;  // loads of K per lane and tile
  constexpr int VN = D / 64;  // loads of V per lane and token
  constexpr int PAD = D + 4;
  constexpr int C4 = D / 4;
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][16][PAD];
  __shared__ float s_m[kWaves][16], s_l[kWaves][16];
  __shared__ float s_w[16][64];  // merge: weight of a head's part
  __shared__ uint32_t s_ticket;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, u = lane >> 4;
  const int row = blockIdx.x, kvh = blockIdx.y, split = blockIdx.z;
  const int G = a.n_q_heads / a.n_kv_heads;

  // ---- the row's visible tokens and this workgroup's piece of them
  int64_t req = a.req_idx[row];
  req = req < 0 ? 0 : (req >= a.kv.table_rows ? a.kv.table_rows - 1 : req);
  const int64_t seq64 = a.seq_lens[row];
  const int len = (int)(seq64 < 0 ? 0 : (seq64 > a.kv.table_cols ? a.kv.table_cols : seq64));
  const int2 seen = visible_range(a.mods, row, len, len);
  const int seq = seen.y;
  const bool fused = a.counters != nullptr;
  // (fused: no piece is shorter than a tile per wave, or than four where the pieces would be more than two per CU -- 64 x 2048
  // tokens, 12 / 2 heads: 16 pieces 67 us, 8 63, both before the loads were cached; 16 x 2048: 17 pieces 21.6, 8 19.9; 9 requests of 700 or so: 13 pieces
  // stay; not fused: the merge expects all n_splits)
  const int shortest = (int64_t)a.rows * a.n_kv_heads * a.n_splits > 512 ? 4 * kTokens * kWaves : kTokens * kWaves;
  const int n_parts = fused ? max(1, min(a.n_splits, (seq + shortest - 1) / shortest)) : a.n_splits;
  if (split >= n_parts) return;
  const int chunk = ((seq + n_parts - 1) / n_parts + kTokens - 1) / kTokens * kTokens;
  const int start = min(split * (int64_t)chunk, (int64_t)seq), end = min(start + (int64_t)chunk, (int64_t)seq);
  const int n_tiles = (end - start + kTokens - 1) / kTokens;
  const int32_t* table_row = a.kv.table + req * a.kv.table_row_stride + seen.x;
  const uint32_t max_slot = (uint32_t)(a.kv.n_slots - 1);
  const int head = kvh * G + min(c, G - 1);

  f32x4v qf[KN];
  {
    const float* q_ptr = (const float*)a.q + (int64_t)row * a.q_row_stride + (int64_t)head * D + 4 * u;
#pragma unroll
    for (int j = 0; j < KN; ++j) qf[j] = *(const f32x4v*)(q_ptr + 16 * j);
  }
  const ScoreShape shape(a.mods, a.scale, head);
  float* const score_dst = a.mods.scores == nullptr ? nullptr : a.mods.scores + ((int64_t)row * a.n_q_heads + head) * a.mods.score_stride + start + 4 * u;
  const float far = (float)(len - 1 - seen.x - start);  // distance of the piece's first token

  // (cached loads: a line comes in two pieces; non-temporal, 64 x 2048 tokens of 12 / 2 heads took 67 us instead of 53)
  f32x4v xk[KN], xv[4][VN];
  // the slot of the tile's token c (places past the end repeat the last one)
  auto entry = [&](int tile) {
    const uint32_t e = (uint32_t)table_row[min(start + tile * kTokens + c, end - 1)];
    return (int)(e > max_slot ? max_slot : e);
  };
  auto load_k = [&](int slot) {
    const float* k_ptr = (const float*)a.kv.k_slab + (int64_t)slot * a.kv.slab_row_stride + (int64_t)kvh * D + 4 * u;
#pragma unroll
    for (int j = 0; j < KN; ++j) xk[j] = *(const f32x4v*)(k_ptr + 16 * j);
  };
  auto load_v = [&](int slot) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* v_ptr = (const float*)a.kv.v_slab + (int64_t)__shfl(slot, 4 * u + i) * a.kv.slab_row_stride + (int64_t)kvh * D + c * (D / 16);
#pragma unroll
      for (int n = 0; n < VN; ++n) xv[i][n] = *(const f32x4v*)(v_ptr + 4 * n);
    }
  };

  float m_run = kNegInf, m_sub = 0.f, l_run = 0.f;
  f32x4v o_acc[D / 16];
#pragma unroll
  for (int n = 0; n < D / 16; ++n) o_acc[n] = f32x4v{0.f, 0.f, 0.f, 0.f};

  // ---- the wave's tiles: wave, wave + 4, ..
  int slot = wave < n_tiles ? entry(wave) : 0;
  if (wave < n_tiles) {
    load_k(slot);
    load_v(slot);
    slot = entry(wave + kWaves);
  }
  for (int tile = wave; tile < n_tiles; tile += kWaves) {
    const bool more = tile + kWaves < n_tiles;
    const int left = end - start - tile * kTokens - 4 * u;  // this lane's tokens that exist: the first `left` of four
    f32x4v s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KN; ++j)
#pragma unroll
      for (int m = 0; m < 4; ++m) s = __builtin_amdgcn_mfma_f32_16x16x4f32(xk[j][m], qf[j][m], s, 0, 0, 0);
    if (more) load_k(slot);
    float t_max = kNegInf;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float y = shape.precise(s[r], fabsf(far - (float)(tile * kTokens + 4 * u + r)));
      s[r] = r < left ? y : kNegInf;
      t_max = fmaxf(t_max, s[r]);
    }
    // (a row of the buffer has room for whole tiles)
    if (score_dst != nullptr && c < G) *(f32x4v*)(score_dst + tile * kTokens) = s;
    t_max = fmaxf(t_max, __shfl_xor(t_max, 16));
    t_max = fmaxf(t_max, __shfl_xor(t_max, 32));
    if (__any(t_max > m_run)) {
      const float m_new = fmaxf(m_run, t_max);
      const float alpha = m_new == kNegInf ? 1.f : fast_exp2(m_run - m_new);
      m_run = m_new;
      m_sub = m_new == kNegInf ? 0.f : m_new;
      l_run *= alpha;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float ar = __shfl(alpha, 4 * u + r);  // (O: head 4 u + r in register r)
#pragma unroll
        for (int n = 0; n < D / 16; ++n) o_acc[n][r] *= ar;
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[r] = fast_exp2(s[r] - m_sub);
      l_run += s[r];
    }
    if (!more && n_tiles * kTokens > end - start) {
      // (the repeated token's values meet a probability of 0: they must be numbers)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < VN; ++n)
          if (i >= left) xv[i][n] = f32x4v{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < D / 16; ++n) o_acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(s[i], xv[i][n / 4][n % 4], o_acc[n], 0, 0, 0);
    if (more) load_v(slot);
    slot = entry(tile + 2 * kWaves);
  }

  // ---- the four waves' results: lane (c, u) holds values c (D / 16) .. of heads 4 u .. 4 u + 3
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int n = 0; n < D / 16; n += 4)
      *(f32x4v*)&s_o[wave][4 * u + r][c * (D / 16) + n] = f32x4v{o_acc[n][r], o_acc[n + 1][r], o_acc[n + 2][r], o_acc[n + 3][r]};
  l_run += __shfl_xor(l_run, 16);
  l_run += __shfl_xor(l_run, 32);
  if (u == 0) {
    s_m[wave][c] = m_run;
    s_l[wave][c] = l_run;
  }
  __syncthreads();
  const int64_t n_rh = (int64_t)a.rows * a.n_q_heads;
  const int64_t rh0 = (int64_t)row * a.n_q_heads + (int64_t)kvh * G;
  const bool direct = n_parts == 1;
  float* const part_o = direct ? nullptr : a.ws_o + ((int64_t)split * n_rh + rh0) * D;
  auto part_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)part_o, 0, direct ? 0 : G * D * 4, 0x00020000);
  for (int idx = tid; idx < G * C4; idx += 64 * kWaves) {
    const int h = idx / C4, c4 = idx % C4;
    float m = kNegInf, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s_m[w][h]);
    f32x4v o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = s_m[w][h] == kNegInf ? (s_l[w][h] == 0.f ? 0.f : 1.f) : fast_exp2(s_m[w][h] - m);  // (nothing seen; NaN passes)
      l += s_l[w][h] * f;
      const f32x4v x = *(const f32x4v*)&s_o[w][h][4 * c4];
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = fmaf(x[k], f, o[k]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const float lse = l == 0.f ? kNegInf : ((m == kNegInf ? 0.f : m) + __builtin_amdgcn_logf(l)) * kLn2;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] *= inv;
    if (direct) {
      *(f32x4v*)((float*)a.out + (int64_t)row * a.out_row_stride + (int64_t)(kvh * G + h) * D + 4 * c4) = o;
      if (a.lse != nullptr && c4 == 0) a.lse[rh0 + h] = lse;
    } else {
      // (aux 16 = sc1: written through, so that the merging workgroup's sc1 loads see the bytes)
      if (fused) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4v, o), part_rsrc, (h * D + 4 * c4) * 4, 0, 16);
      else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4v, o), part_rsrc, (h * D + 4 * c4) * 4, 0, 0);
      if (c4 == 0) {
        float* pl = a.ws_lse + (int64_t)split * n_rh + rh0 + h;
        if (fused) __hip_atomic_store(pl, lse, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        else *pl = lse;
      }
    }
  }
  if (direct || !fused) return;

  // ---- ticket: the last workgroup of this (row, kv head) merges the pieces
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's bytes have left
  __syncthreads();                                  // and everybody's
  uint32_t* counter = a.counters + (int64_t)row * a.n_kv_heads + kvh;
  if (tid == 0) s_ticket = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_ticket != (uint32_t)n_parts - 1) return;
  // lane p of a wave: part p of a head
  for (int h = wave; h < G; h += kWaves) {
    const float l = lane < n_parts ? __hip_atomic_load(a.ws_lse + (int64_t)lane * n_rh + rh0 + h, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : kNegInf;
    const float mx = group_max<64>(l);
    const float w = l == kNegInf ? 0.f : fast_exp2((l - mx) * kLog2e);  // (NaN passes)
    const float sum = group_sum<64>(w);
    s_w[h][lane] = sum == 0.f ? 0.f : w / sum;
    if (a.lse != nullptr && lane == 0) a.lse[rh0 + h] = sum == 0.f ? kNegInf : mx + __builtin_amdgcn_logf(sum) * kLn2;
  }
  __syncthreads();
  // (the parts' distance fits 31 bits: the caller checked)
  auto all_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(a.ws_o + rh0 * D), 0, (int)((((int64_t)(n_parts - 1) * n_rh + G) * D) * 4), 0x00020000);
  const int part_stride = (int)(n_rh * D * 4);
  for (int idx = tid; idx < G * C4; idx += 64 * kWaves) {
    const int h = idx / C4, c4 = idx % C4;
    f32x4v o = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < n_parts; p0 += 8) {
      f32x4v x[8];
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int p = min(p0 + j, n_parts - 1);
        x[j] = __builtin_bit_cast(f32x4v, __builtin_amdgcn_raw_buffer_load_b128(all_rsrc, p * part_stride + (h * D + 4 * c4) * 4, 0, 16));
        w[j] = p0 + j < n_parts ? s_w[h][p] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = fmaf(w[j], x[j][k], o[k]);
      }
    }
    *(f32x4v*)((float*)a.out + (int64_t)row * a.out_row_stride + (int64_t)(kvh * G + h) * D + 4 * c4) = o;
  }
  if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // (the next launch's tickets)
}

}  // namespace

bool decode_scored_f32_supported(const DecodeArgs& a) {
  return a.scored && a.mods.rows == nullptr && a.dtype == kF32 && (a.head_dim == 64 || a.head_dim == 128) && a.n_kv_heads > 0 && a.n_kv_heads <= 65535 &&
         a.n_q_heads % a.n_kv_heads == 0 && a.n_q_heads / a.n_kv_heads <= 16 && a.kv.table_cols <= 0x7fff0000 &&
         ((uintptr_t)a.kv.k_slab | (uintptr_t)a.kv.v_slab | (uintptr_t)a.q | (uintptr_t)a.out) % 16 == 0 && a.kv.slab_row_stride % 4 == 0 &&
         a.q_row_stride % 4 == 0 && a.out_row_stride % 4 == 0;
}

// Per call, with a cap: 64 requests of 2048 tokens, 12 / 2 heads of 128: 53 us (268 MB; 5.1 TB/s, what a large copy reaches), the
// generic kernel and its merge 96; 14 / 2 heads of 64: 29 and 56; 9 requests of 700 tokens 11 and 18.
hipError_t launch_decode_scored_f32(const DecodeArgs& a, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  const dim3 grid((unsigned)a.rows, (unsigned)a.n_kv_heads, (unsigned)a.n_splits);
  if (a.head_dim == 128) hipLaunchKernelGGL((decode_scored_f32_kernel<128>), grid, dim3(64 * kWaves), 0, stream, a);
  else hipLaunchKernelGGL((decode_scored_f32_kernel<64>), grid, dim3(64 * kWaves), 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.n_splits == 1 || a.counters != nullptr) return e;
  MergeArgs mg;
  mg.out = a.out;
  mg.out_row_stride = a.out_row_stride;
  mg.lse_out = a.lse;
  mg.parts_o = a.ws_o;
  mg.parts_lse = a.ws_lse;
  mg.n_parts = a.n_splits;
  mg.rows = a.rows;
  mg.n_heads = a.n_q_heads;
  mg.head_dim = a.head_dim;
  mg.dtype = a.out_dtype;
  return launch_merge(mg, stream);
}

}  // namespace bsgl
