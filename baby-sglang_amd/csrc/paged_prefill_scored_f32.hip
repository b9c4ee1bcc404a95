// Scored extend attention in 32 bits for gfx950 (see paged_prefill_scored.hip for the scores, the work list and the
// order of the tokens): f32 rows, head_dim 64 or 128, up to 16 q heads per kv head.
//
// v_mfma_f32_32x32x2_f32 multiplies f32 by f32 with nothing rounded on the way in, at a sixteenth of the bf16 rate (157
// TFLOP/s), so the products set the time and the rest is kept simple: a step is 32 tokens, its K and V (32 KB at
// head_dim 128) come by LDS-DMA into one of two buffers while the other is worked on, and two workgroups fit a CU: the
// exponentials of one run beside the products of the other.  Nothing changes places between the two products:
//   S^T = K Q^T   a lane owns one column (a query row of one head) and 16 of the step's tokens, as it gets them from the products
//   O  += P V     the product over two tokens per instruction takes P from the register it is in -- register r holds the
//                 tokens acc_row(r, 0) of the lower lanes and acc_row(r, 1) of the upper ones -- and V's rows in that order
// LDS: a row's 16-byte pieces are dealt by an XOR with the token's number (bit 2 of it also flips bit 3), so that both the
// K reads (16 bytes of one token per lane) and the V reads (4 bytes, tokens t and t + 4 of the two halves) use all banks.
// The largest score is not tracked exactly: the reference moves when a score exceeds it by 2^6.
//
// What it measured: see launch_prefill_scored_f32.
#include "bsgl_device.h"
#include "bsgl_launch.h"
#include "bsgl_mfma.h"
#include "bsgl_score.h"

namespace bsgl {

namespace {

using namespace mfma;

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4v;

constexpr int kWaves = 4;
constexpr int kStep = 32;  // tokens

// row of the 32x32 accumulator that register r of a lane in half `hi` holds
__device__ __forceinline__ constexpr int acc_row(int r, int hi) { return (r & 3) + 8 * (r >> 2) + 4 * hi; }
// where token t's 16-byte piece p stands in its row: p ^ deal(t)
__device__ __forceinline__ constexpr int deal(int t) { return t ^ (((t >> 2) & 1) << 3); }

// One query row of one head by itself, from the tokens [lo, hi) it sees, 8 of them on their way at a time.  Slow, and only ever run for
// rows that met_unseen names: a product multiplies the values of a token that the row must not see by an exact zero, and
// 0 * NaN is NaN.
template <int D>
__device__ __forceinline__ void rescue_row(const PrefillArgs& a, int64_t q_row, int head, int kvh, int64_t req, int pos, int lo, int hi, int split) {
  constexpr int N = D / 64;
  const int lane = threadIdx.x & 63;
  const ScoreShape shape(a.mods, a.scale, head);
  const float* q_ptr = (const float*)a.q + q_row * a.q_row_stride + (int64_t)head * D + N * lane;
  float q[N], o[N], m = kNegInf, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = q_ptr[i];
    o[i] = 0.f;
  }
  const int32_t* table_row = a.kv.table + req * a.kv.table_row_stride;
  const uint32_t max_slot = (uint32_t)(a.kv.n_slots - 1);
  constexpr int B = 8;
  for (int j0 = lo; j0 < hi; j0 += B) {
    float k[B][N], v[B][N], s[B], mn = m;
#pragma unroll
    for (int i = 0; i < B; ++i) {
      uint32_t slot = (uint32_t)table_row[min(j0 + i, hi - 1)];
      slot = slot > max_slot ? max_slot : slot;
      const int64_t at = (int64_t)slot * a.kv.slab_row_stride + (int64_t)kvh * D + N * lane;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        k[i][n] = ((const float*)a.kv.k_slab)[at + n];
        v[i][n] = ((const float*)a.kv.v_slab)[at + n];
      }
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      float dot = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n) dot = fmaf(q[n], k[i][n], dot);
      s[i] = shape.precise(group_sum<64>(dot), (float)abs(pos - (j0 + i)));
      if (j0 + i >= hi) {
        s[i] = kNegInf;
#pragma unroll
        for (int n = 0; n < N; ++n) v[i][n] = 0.f;
      }
      mn = s[i] > mn ? s[i] : mn;
    }
    const float alpha = mn == kNegInf ? 1.f : fast_exp2(m - mn);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int n = 0; n < N; ++n) o[n] *= alpha;
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const float p = s[i] == kNegInf ? 0.f : fast_exp2(s[i] - mn);
      l += p;
#pragma unroll
      for (int n = 0; n < N; ++n) o[n] += p * v[i][n];
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float* dst = (float*)a.out + q_row * a.out_row_stride + (int64_t)head * D + N * lane;
  if (a.splits > 1) {
    const int64_t part = ((int64_t)split * a.total_q_tokens + q_row) * a.n_q_heads + head;
    dst = a.parts_o + part * D + N * lane;
    if (lane == 0) a.parts_lse[part] = l == 0.f ? kNegInf : (m + __builtin_amdgcn_logf(l)) * kLn2;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) dst[i] = o[i] * inv;
}

// PW: positions among a wave's 32 columns; 32: 64 positions x 2 q heads per workgroup, 16: 16 positions x 8 q heads.
template <int D, int PW>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2)))
void prefill_scored_f32_kernel(PrefillArgs a) {
  constexpr int CH = 32 / PW;                      // q heads among a wave's columns
  constexpr int HPW = PW == 32 ? 2 : kWaves * CH;  // q heads per workgroup
  constexpr int ROWS = PW == 32 ? 64 : PW;         // positions per workgroup
  constexpr int ROW = D * 4;
  constexpr int HALF = kStep * ROW;      // K, or V, of a step
  constexpr int PIECES = ROW / 16;       // of a row
  constexpr int TPD = 64 / PIECES;       // tokens per DMA instruction
  constexpr int TPW = kStep / kWaves;    // tokens a wave brings per step
  constexpr int NDMA = TPW / TPD;        // instructions for their K, and as many for V
  constexpr int DB = D / 32;
  __shared__ __attribute__((aligned(1024))) char smem[2 * 2 * HALF];
  __shared__ int2 s_rng[kWaves];
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lp = lane & 31, hi = lane >> 5;
  const int pos = lp % PW, hsub = lp / PW;
  const int G = a.n_q_heads / a.n_kv_heads;

  // ---- which (request, block of positions, kv head, q heads): the launch order of paged_prefill_scored.hip
  const int n_z = (G + HPW - 1) / HPW;
  const int per_group = a.grp_blocks * n_z;
  const unsigned slot = blockIdx.x >> 3;
  const int64_t g = (int64_t)(slot / (unsigned)per_group) * 8 + ((blockIdx.x + 8 - (blockIdx.y & 7)) & 7);
  if (g >= a.cu_blk[a.batch] * a.n_kv_heads) return;
  const int within = (int)(slot % (unsigned)per_group);
  const int kvh = (int)(g % a.n_kv_heads);
  int64_t pg = g / a.n_kv_heads;
  // (longest streams first, if the launch that made the list sorted it; whatever stands there, it is a group of this launch)
  if (pg < a.n_order && a.cu_blk[a.batch + 1] != 0) pg = max((int64_t)0, min((int64_t)a.order[pg], a.cu_blk[a.batch] - 1));
  const int rt0 = (within % n_z) * HPW;
  const int n_rt = min(HPW, G - rt0);
  int i_req = 0;
  for (int base = 1; base <= a.batch; base += 64) {
    const int j = base + lane;
    const bool le = j <= a.batch && a.cu_blk[j] <= pg;
    i_req += __popcll(__ballot(le));
  }
  i_req = min(i_req, a.batch - 1);
  const int64_t q_first = a.cu_ext[i_req];
  const int64_t ext_raw = max((int64_t)0, min(a.extended_lens[i_req], (int64_t)a.total_q_tokens - q_first));
  const int n_blocks = (int)((ext_raw + ROWS - 1) / ROWS);
  const int bg0 = (int)(pg - a.cu_blk[i_req]) * a.grp_blocks;
  const int nb = min(a.grp_blocks, n_blocks - bg0);
  const int bi = within / n_z;  // block of the group, counted from the request's end
  if (bi >= nb) return;
  const int hw = PW == 32 ? wave >> 1 : wave * CH;  // first of this wave's q heads among the workgroup's
  const int q0_blk = (bg0 + nb - 1 - bi) * ROWS;
  const int rows_blk = (int)min((int64_t)ROWS, ext_raw - q0_blk);
  const int pos_off = PW == 32 ? 32 * (wave & 1) : 0;
  const int q0 = q0_blk + pos_off;
  const int n_heads = max(0, min(CH, n_rt - hw));
  const int n_rows = n_heads > 0 ? max(0, min(PW, rows_blk - pos_off)) : 0;
  const bool col_ok = pos < n_rows && hsub < n_heads;
  const int64_t q_row0 = q_first + q0;
  int64_t req = a.req_idx[i_req];
  req = req < 0 ? 0 : (req >= a.kv.table_rows ? a.kv.table_rows - 1 : req);
  const int64_t seq64 = a.seq_lens[i_req];
  const int seq = (int)(seq64 < 0 ? 0 : (seq64 > a.kv.table_cols ? a.kv.table_cols : seq64));
  const int64_t pre64 = a.prefix_lens[i_req];
  const int prefix = (int)(pre64 < 0 ? 0 : (pre64 > seq ? seq : pre64));

  // ---- what this lane's row sees, and what the wave and the workgroup have to stream
  const int own = prefix + q0 + pos;
  int2 seen = make_int2(0, 0);  // {first, number}
  if (col_ok) seen = visible_range(a.mods, q_row0 + pos, seq, min(seq, own + 1));
  const bool live = seen.y > 0;
  int2 rng;
  {
    int f0 = live ? seen.x : 0x7fffffff, f1 = live ? seen.x + seen.y : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      f0 = min(f0, __shfl_xor(f0, d));
      f1 = max(f1, __shfl_xor(f1, d));
    }
    rng = make_int2(__builtin_amdgcn_readfirstlane(f0), __builtin_amdgcn_readfirstlane(f1));
  }
  if (lane == 0) s_rng[wave] = rng;
  __syncthreads();
  int first = 0x7fffffff, last = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    first = min(first, __builtin_amdgcn_readfirstlane(s_rng[w].x));
    last = max(last, __builtin_amdgcn_readfirstlane(s_rng[w].y));
  }
  if (last == 0) first = 0;  // nobody sees anything
  if (a.splits > 1) {
    // this workgroup's piece of the stream: whole steps, counted from the last token back
    const int all = last - first;
    const int chunk = ((all + a.splits - 1) / a.splits + kStep - 1) / kStep * kStep;
    const int s0 = min((int)blockIdx.y * chunk, all), s1 = min(s0 + chunk, all);
    first = last - s1;
    last -= s0;
  }
  // Everything below counts tokens from the last one back: place t is position last - 1 - t
  const int kv_len = last - first;
  const int n_steps = (kv_len + kStep - 1) / kStep;
  const int my_lo = last - (seen.x + seen.y);
  const int my_hi = live ? my_lo + seen.y : -0x7fffffff;
  const int my_pos = last - 1 - own;
  const int wave_lo = last - rng.y, wave_hi = rng.y > 0 ? last - rng.x : 0;  // places any row of the wave sees
  const int32_t* table_row = a.kv.table + req * a.kv.table_row_stride + first;
  const uint32_t max_slot = (uint32_t)(a.kv.n_slots - 1);
  const int head0 = kvh * G + rt0 + hw;
  const int head = head0 + hsub;

  // ---- Q: lane (column lp, half hi) holds values 8 j + 4 hi + m of its row, the order the K reads give
  f32x4v qf[D / 8];
  {
    const float* q_ptr = (const float*)a.q + (q_row0 + pos) * a.q_row_stride + (int64_t)head * D + 4 * hi;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      qf[j] = f32x4v{0.f, 0.f, 0.f, 0.f};
      if (col_ok) qf[j] = *(const f32x4v*)(q_ptr + 8 * j);
    }
  }
  const ScoreShape shape(a.mods, a.scale, min(head, a.n_q_heads - 1));

  // ---- LDS-DMA: instruction i of a wave brings TPD tokens, one 16-byte piece per lane
  const int lane_tok = lane / PIECES, piece = lane % PIECES;
  uint32_t entry[NDMA];
  auto read_entries = [&](int step) {
#pragma unroll
    for (int i = 0; i < NDMA; ++i) {
      const int t = step * kStep + wave * TPW + i * TPD + lane_tok;
      entry[i] = (uint32_t)table_row[max(kv_len - 1 - t, 0)];  // (places past the end repeat the last one)
    }
  };
  auto issue = [&](int step) {
#pragma unroll
    for (int i = 0; i < NDMA; ++i) {
      const int t = wave * TPW + i * TPD;
      const int64_t row = (int64_t)(entry[i] > max_slot ? max_slot : entry[i]) * a.kv.slab_row_stride + (int64_t)kvh * D;
      const int64_t at = row * 4 + ((piece ^ (deal(t + lane_tok) & (PIECES - 1))) << 4);
      const uint32_t dst = __builtin_amdgcn_readfirstlane(lds + (uint32_t)(step & 1) * (2 * HALF) + (uint32_t)t * ROW);
      dma_1k<false>((const char*)a.kv.k_slab + at, dst);
      dma_1k<false>((const char*)a.kv.v_slab + at, dst + HALF);
    }
  };

  const int k_at = lp * ROW + ((hi ^ (deal(lp) & (PIECES - 1))) << 4);  // ^ (j << 5): piece 2 j + hi of token lp
  int v_at[4][2];  // token r + 4 hi of a group of eight, value lp of an even / odd block of 32 (as `deal` leaves it, bit 3 of the token clear)
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int odd = 0; odd < 2; ++odd)
      v_at[r][odd] = HALF + (r + 4 * hi) * ROW + 128 * (odd ^ hi) + ((((lp >> 2) ^ (r + 4 * hi)) & 7) << 4) + 4 * (lp & 3);

  float m_run = kNegInf, m_sub = 0.f, l_run = 0.f;
  f32x16 o_acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o_acc[db][r] = 0.f;

  if (n_steps > 0) {
    read_entries(0);
    issue(0);
    if (n_steps > 1) read_entries(1);
  }
  for (int step = 0; step < n_steps; ++step) {
    // the step has arrived, everybody's share of it, and everybody is done with the one before
    __builtin_amdgcn_s_waitcnt(0x0F70);
    dma_wait<0>();
    __syncthreads();
    if (step + 1 < n_steps) {
      issue(step + 1);
      if (step + 2 < n_steps) read_entries(step + 2);
    }
    const int t_step = step * kStep;
    if (t_step >= wave_hi || t_step + kStep <= wave_lo) continue;  // nothing this wave's rows see
    const char* st = smem + (step & 1) * (2 * HALF);

    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      const f32x4v k = *(const f32x4v*)(st + (k_at ^ (j << 5)));
#pragma unroll
      for (int m = 0; m < 4; ++m) s = __builtin_amdgcn_mfma_f32_32x32x2f32(k[m], qf[j][m], s, 0, 0, 0);
    }
    float t_max = kNegInf;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int t = t_step + acc_row(r, 0) + 4 * hi;
      const float x = shape.precise(s[r], fabsf((float)(t - my_pos)));
      s[r] = (t >= my_lo && t < my_hi) ? x : kNegInf;
      t_max = fmaxf(t_max, s[r]);
    }
    if (__any(t_max > m_run + 6.f)) {
      const float m_new = fmaxf(m_run, fmaxf(t_max, __shfl_xor(t_max, 32)));
      const float alpha = m_new == kNegInf ? 1.f : fast_exp2(m_run - m_new);
      m_run = m_new;
      m_sub = m_new == kNegInf ? 0.f : m_new;
      l_run *= alpha;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float ar = __shfl(alpha, acc_row(r, 0) + 4 * hi);
#pragma unroll
        for (int db = 0; db < DB; ++db) o_acc[db][r] *= ar;
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = fast_exp2(s[r] - m_sub);
      l_run += s[r];
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        // (bit 3 of the token flips the block's parity, bit 4 its half: the rest of `deal`)
        const int block = db ^ (((r >> 2) & 1) | (DB > 2 ? (r >> 3) << 1 : 0));
        const float v = *(const float*)(st + v_at[r & 3][block & 1] + 8 * (r >> 2) * ROW + 256 * (block >> 1));
        o_acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(s[r], v, o_acc[db], 0, 0, 0);
      }
    }
  }

  // ---- normalise and write: 32 lanes hold 32 neighbouring values of a row
  const float l_all = l_run + __shfl_xor(l_run, 32);
  const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
  const uint32_t live_rows = (uint32_t)__ballot(live);
  if (a.splits > 1 && hi == 0 && col_ok) {
    const float lse = live && l_all != 0.f ? (m_sub + __builtin_amdgcn_logf(l_all)) * kLn2 : kNegInf;
    a.parts_lse[((int64_t)blockIdx.y * a.total_q_tokens + q_row0 + pos) * a.n_q_heads + head] = lse;
  }
  uint32_t bad = 0;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = acc_row(r, 0) + 4 * hi;
    const float ir = __shfl(inv, row);
    const bool ok = row % PW < n_rows && row / PW < n_heads;
    const bool on = (live_rows >> row) & 1;
    const int64_t q_row = q_row0 + row % PW;
    const int h = head0 + row / PW;
    float* dst = (float*)a.out + q_row * a.out_row_stride + (int64_t)h * D;
    if (a.splits > 1) dst = a.parts_o + (((int64_t)blockIdx.y * a.total_q_tokens + q_row) * a.n_q_heads + h) * D;
    bool nan = false;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const float x = on ? o_acc[db][r] * ir : 0.f;
      nan |= x != x;
      if (ok) dst[32 * db + lp] = x;
    }
    const unsigned long long b = __ballot(nan && ok);
    if (b & 0xffffffffull) bad |= 1u << acc_row(r, 0);
    if (b >> 32) bad |= 1u << acc_row(r, 1);
  }
  // rows that came out NaN and have met a value that they do not see (not those with a NaN among the scores they do see): again, by themselves
  bad &= ~(uint32_t)__ballot(l_all != l_all);
  if (bad != 0) {
    int g0 = live ? my_lo : 0, g1 = live ? my_hi : 0x7fffffff;  // what every row of the wave sees
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      g0 = max(g0, __shfl_xor(g0, d));
      g1 = min(g1, __shfl_xor(g1, d));
    }
    bad &= (uint32_t)__ballot(met_unseen<f32_tag, ROW>((const char*)a.kv.v_slab + (int64_t)kvh * ROW, a.kv.slab_row_stride * 4, table_row, max_slot, kv_len,
                                                       wave_hi, __builtin_amdgcn_readfirstlane(g0), __builtin_amdgcn_readfirstlane(g1), my_lo, my_hi));
  }
  if (bad != 0) __builtin_amdgcn_s_waitcnt(0x0F70);  // (behind the stores above, which went to the same rows)
  while (bad != 0) {
    const int r = __ffs((int)bad) - 1;
    bad &= bad - 1;
    const int lo = __builtin_amdgcn_readlane(seen.x, r), n = __builtin_amdgcn_readlane(seen.y, r);
    rescue_row<D>(a, q_row0 + r % PW, head0 + r / PW, kvh, req, prefix + q0 + r % PW, max(lo, first), min(lo + n, last), (int)blockIdx.y);
  }
}

}  // namespace

bool prefill_scored_f32_supported(const PrefillArgs& a, const char** why) {
  if (a.fold_group > 0 || (a.head_dim != 128 && a.head_dim != 64)) {
    *why = "matrix-core extend in f32 needs head_dim 64 or 128";
    return false;
  }
  if (a.n_kv_heads <= 0 || a.n_q_heads % a.n_kv_heads != 0 || a.n_q_heads / a.n_kv_heads > 16) {
    *why = "matrix-core extend in f32 needs 1..16 query heads per kv head";
    return false;
  }
  if (((uintptr_t)a.kv.k_slab | (uintptr_t)a.kv.v_slab | (uintptr_t)a.q) % 16 != 0 || a.kv.slab_row_stride % 4 != 0 || a.q_row_stride % 4 != 0) {
    *why = "matrix-core extend in f32 needs 16-byte aligned rows";
    return false;
  }
  return true;
}

// Against the tokens as rows of the generic kernel, with a cap (12 / 2 heads of 128): 1 token over 300 29.8 us / 40, 64 over
// 300 33 / 46, 4 x 200 over 300 66 / 247, 8 x 512 over 1536 551 / 4081 (82 TFLOP/s; 384 workgroups for 512 places, the one
// with two to a CU sets the time); 28 / 4 heads, 4 x 300 over 800: 298 / 1575.  Two accumulators for the scores instead
// of one chain of products: no difference.
hipError_t launch_prefill_scored_f32(const PrefillArgs& a, dim3 grid, hipStream_t stream) {
  const dim3 block(64 * kWaves);
  if (a.head_dim == 128) {
    if (a.blk_rows == 64) hipLaunchKernelGGL((prefill_scored_f32_kernel<128, 32>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((prefill_scored_f32_kernel<128, 16>), grid, block, 0, stream, a);
  } else {
    if (a.blk_rows == 64) hipLaunchKernelGGL((prefill_scored_f32_kernel<64, 32>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((prefill_scored_f32_kernel<64, 16>), grid, block, 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace bsgl
