// Scored extend attention for gfx950: cap * tanh(s / cap), minus slope[head] * |i - j|, over an interval
// [from, to) of positions per query row (ScoreMods); bf16 / f16, head_dim 128 or two kv heads of 64 folded.
//
// The frame is paged_prefill_mfma32.hip's: the same work list (launched longest stream first, see prefill_order_kernel), four waves on 64 positions x 2
// q heads (or 16 x 8 for short extends), one K/V stream per workgroup through a four-stage ring, per 32-token
// step 8 products for the scores of the NEXT step beside the exponentials of this one and 8 for P . V.  What is
// new sits between the products:
//
//   * a finished score is kept as u with t = A u + C, t the score in units of log2 and C one number per lane
//     and step, so that the exponent's multiply-add takes in the rest:
//       plain        u = scale log2 e q.k             A = 1               C = 0
//       cap          u = 1 / (2^{2 s / cap} + 1)      A = -2 cap log2 e   C = cap log2 e
//       bias         u = q.k - (slope / A) row        A = scale log2 e    C = slope (step's first - i)
//       cap and bias u = 1 / (..) - (slope / A) row   A = -2 cap log2 e   C = both
//     (tanh(x) = 1 - 2 / (e^{2x} + 1); `row` is the token's place in the step, a literal of the multiply-add: as
//     slope x row in registers the bias cost 200 us of a 780 us launch, sixteen registers too many).  A cap costs 24 issue
//     cycles a score -- multiply, exp2, add, reciprocal -- beside the 20 of the plain softmax: this kernel is bound by
//     vector issue where the plain one is bound by both pipes.
//   * probabilities are rounded once, to bf16 (2^-8 of each) or f16 (2^-11), on their way into the second product; sums and
//     statistics are f32.  bf16 results are 1.35 times as far from 64 bits as their own rounding puts them; the decode kernel's two
//     halves would double the products of P V and add 24 vector instructions to a step that is bound by their issue.
//   * the tokens are streamed from the last one back (the page-table entries are staged in that order, nothing else
//     changes): a bias makes the nearest tokens the largest, so going forward a steep slope raises the running maximum in
//     every step, and every step then rescales the output (48 x 512 over 1536, 28 / 4 heads: 983 us forward, 768 back; without a
//     bias there is no difference).
//   * the workgroup streams the tokens from the first that any of its rows sees to the last: a document mask
//     skips what lies before the document, a prefix mask reaches past the diagonal.  Steps that every row of
//     a wave sees whole take no mask.
//   * where a launch has far fewer workgroups than the machine takes (one long request, say), every block's stream is cut into pieces
//     (PrefillArgs::splits) whose normalised fp32 results a second launch merges.
//   * rows that see nothing are left out of the ranges and written as zeros.
//   * 0 * NaN: a token that one row must not see can share a step with a row that sees it, and P . V multiplies its
//     values by an exact zero.  Where such a token holds NaN or an infinity the product is NaN; rows that come out NaN and
//     have met such a token are therefore computed again, one by one, from the tokens they see (met_unseen, rescue_row; costs a
//     test per output value when there are none).  A NaN among the tokens that a row does see starts none of that: 300 tokens over
//     4000, 12 / 2 heads, 57 us, with a NaN in the prefix 61 (13 ms where all rows that came out NaN were computed again), with
//     one among the new tokens 5.5 ms, for the rows ahead of it in its step.
//
// NaN is honoured here (the plain kernel's build assumes none).  The maxima are taken of u, never of a raw product:
// u is a result of float arithmetic, which the compiler knows to be canonical, so three-way maxima stay one
// instruction each.
#include "bsgl_device.h"
#include "bsgl_launch.h"
#include "bsgl_mfma.h"
#include "bsgl_score.h"

#include <type_traits>

namespace bsgl {

namespace {

using namespace mfma;

typedef __attribute__((ext_vector_type(16))) float f32x16;

template <typename Tag> struct Mma32;
template <> struct Mma32<bf16_tag> {
  __device__ static __forceinline__ f32x16 mm(const uint4& a, const uint4& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
};
template <> struct Mma32<f16_tag> {
  __device__ static __forceinline__ f32x16 mm(const uint4& a, const uint4& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
};

// row of the 32x32 accumulator that register r of a lane in half `hi` holds
__device__ __forceinline__ constexpr int acc_row(int r, int hi) { return (r & 3) + 8 * (r >> 2) + 4 * hi; }

__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
__device__ __forceinline__ float min3(float a, float b, float c) { return fminf(fminf(a, b), c); }

// One query row of one head by itself, from the tokens [lo, hi) it sees: the wave's lanes hold two values of the
// head each, 16 tokens are on their way at a time.  Slow, and only ever run for rows that met_unseen names.
template <typename Tag>
__device__ __forceinline__ void rescue_row(const PrefillArgs& a, int64_t q_row, int head, int kvh, int64_t req, int pos, int lo, int hi, int split) {
  using E = Elem<Tag>;
  const int lane = threadIdx.x & 63;
  const bool on = a.fold_group == 0 || lane < 32;
  const int dim = a.fold_group == 0 ? 128 : 64;
  // (folded: kv head head / fold_group of the pair, 64 values each)
  const int64_t kv_off = (a.fold_group == 0 ? (int64_t)kvh * 128 : (int64_t)(head / a.fold_group) * 64) + 2 * lane;
  const ScoreShape shape(a.mods, a.scale, head);
  auto two = [&](const void* base, int64_t elem, float (&f)[2]) {
    const uint32_t w = on ? *(const uint32_t*)((const char*)base + elem * 2) : 0;
    float g[8];
    E::unpack(make_uint4(w, 0, 0, 0), g);
    f[0] = g[0];
    f[1] = g[1];
  };
  float q[2], o[2] = {0.f, 0.f}, m = kNegInf, l = 0.f;
  two(a.q, q_row * a.q_row_stride + (int64_t)head * dim + 2 * lane, q);
  const int32_t* table_row = a.kv.table + req * a.kv.table_row_stride;
  const uint32_t max_slot = (uint32_t)(a.kv.n_slots - 1);
  constexpr int B = 16;
  for (int j0 = lo; j0 < hi; j0 += B) {
    float k[B][2], v[B][2], s[B], mn = m;
#pragma unroll
    for (int i = 0; i < B; ++i) {
      uint32_t slot = (uint32_t)table_row[min(j0 + i, hi - 1)];
      slot = slot > max_slot ? max_slot : slot;
      two(a.kv.k_slab, (int64_t)slot * a.kv.slab_row_stride + kv_off, k[i]);
      two(a.kv.v_slab, (int64_t)slot * a.kv.slab_row_stride + kv_off, v[i]);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      s[i] = shape.fast(group_sum<64>(fmaf(q[0], k[i][0], q[1] * k[i][1])), (float)abs(pos - (j0 + i)));
      if (j0 + i >= hi) s[i] = kNegInf, v[i][0] = v[i][1] = 0.f;
      mn = s[i] > mn ? s[i] : mn;
    }
    const float alpha = mn == kNegInf ? 1.f : fast_exp2(m - mn);
    m = mn;
    l *= alpha;
    o[0] *= alpha;
    o[1] *= alpha;
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const float p = s[i] == kNegInf ? 0.f : fast_exp2(s[i] - mn);
      l += p;
      o[0] += p * v[i][0];
      o[1] += p * v[i][1];
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (a.splits > 1) {
    const int64_t part = ((int64_t)split * a.total_q_tokens + q_row) * a.n_q_heads + head;
    if (on) *(float2*)(a.parts_o + part * dim + 2 * lane) = make_float2(o[0] * inv, o[1] * inv);
    if (lane == 0) a.parts_lse[part] = l == 0.f ? kNegInf : (m + __builtin_amdgcn_logf(l)) * kLn2;
    return;
  }
  if (on) *(uint32_t*)((char*)a.out + (q_row * a.out_row_stride + (int64_t)head * dim + 2 * lane) * 2) = E::pack2(o[0] * inv, o[1] * inv);
}

// PW = positions among a wave's 32 columns.  32: the layout above (64 positions x 2 q heads per
// workgroup).  16: for batches of short extends a wave's columns are 2 q heads x 16 positions and
// the workgroup covers 16 positions x 8 q heads, so a kv head's K/V is streamed by ONE workgroup
// for up to 8 q heads instead of once per pair of heads.
// CAP, BIAS: which of the two the call has (see the head of this file).
template <typename Tag, int PW, bool CAP, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void prefill_scored_kernel(PrefillArgs a) {
  using E = Elem<Tag>;
  constexpr int D = 128;
  constexpr int REC = 512;  // K row | V row of one kv head
  constexpr int WAVES = 4;
  constexpr int CH = 32 / PW;                    // q heads among a wave's columns
  constexpr int HPW = PW == 32 ? 2 : WAVES * CH;  // q heads per workgroup
  constexpr int ROWS = PW == 32 ? 64 : PW;  // positions per workgroup
  constexpr int NSTAGE = 4;
  constexpr int TILE_BYTES = kTile * REC;
  constexpr int STEP = 2 * kTile;                  // tokens per step: two tiles
  constexpr int STEP_BYTES = 2 * TILE_BYTES;
  constexpr int DMA_PER_STEP = STEP_BYTES / 1024;  // 16 instructions, two tokens each
  constexpr int DPW = DMA_PER_STEP / WAVES;        // instructions per wave and step
  constexpr int RING = NSTAGE * STEP_BYTES;
  constexpr int kOPad = D + 4;
  constexpr int STAGE_OUT = 32 * kOPad * 4;        // output staging of one wave
  constexpr int BUF = RING > WAVES * STAGE_OUT ? RING : WAVES * STAGE_OUT;
  constexpr int SLOTS = kSlotBlock;
  constexpr int NTHR = 64 * WAVES;
  constexpr int EPT = SLOTS / NTHR;  // page-table entries of a block per thread
  static_assert(SLOTS == EPT * NTHR && SLOTS / STEP == 16, "whole entries per thread and block; steps per block as shifted below");

  __shared__ __attribute__((aligned(1024))) char smem[BUF + 2 * SLOTS * 4];
  __shared__ int2 s_rng[WAVES];
  __shared__ uint32_t s_bad[WAVES];     // columns of a wave that came out NaN
  __shared__ uint8_t s_live[WAVES][32];  // columns that see something
  int32_t* s_slots = (int32_t*)(smem + BUF);
  const uint32_t lds_ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lp = lane & 31;  // column of S^T, row of O
  const int pos = lp % PW;   // its position inside the wave's PW ...
  const int hsub = lp / PW;  // ... and its q head among the wave's CH
  const int hi = lane >> 5;
  const int G = a.n_q_heads / a.n_kv_heads;
  const int fold = a.fold_group;  // folded heads: see paged_prefill_mfma.hip

  // ---- which (request, block of 64 positions, kv head, pair of q heads) is this? ------------
  // (the launch order of paged_prefill_mfma.hip: index = 8 * slot + xcd)
  const int n_z = (G + HPW - 1) / HPW;
  const int per_group = a.grp_blocks * n_z;
  const unsigned slot = blockIdx.x >> 3;
  // (the pieces of a block's stream share nothing: each on the next XCD)
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
  // rows this request may own: never past the last row of q / out, whatever extended_lens says
  // (inconsistent metadata gives wrong numbers, not an access outside the tensors)
  const int64_t q_first = a.cu_ext[i_req];
  const int64_t ext_raw = max((int64_t)0, min(a.extended_lens[i_req], (int64_t)a.total_q_tokens - q_first));
  const int n_blocks = (int)((ext_raw + ROWS - 1) / ROWS);
  const int bg0 = (int)(pg - a.cu_blk[i_req]) * a.grp_blocks;
  const int nb = min(a.grp_blocks, n_blocks - bg0);
  const int bi = within / n_z;  // block of the group, counted from the request's end (last blocks first)
  if (bi >= nb) return;
  // The last pair of an odd GQA group holds one q head.  Its workgroups then take TWO blocks of
  // that head each (waves 2, 3 the block before the one of waves 0, 1; the stream is the longer
  // one's) instead of leaving half their waves without work, and every second one of them retires.
  const bool two_blocks = PW == 32 && n_rt == 1;
  if (two_blocks && (bi & 1)) return;
  const int hw = PW == 32 ? wave >> 1 : wave * CH;  // first of this wave's q heads among the workgroup's (or its block)
  const int my_bi = bi + (two_blocks ? hw : 0);
  const bool head_ok = two_blocks ? my_bi < nb : hw < n_rt;  // no such head / block: the wave only helps to load
  const int q0_blk = (bg0 + nb - 1 - (head_ok ? my_bi : bi)) * ROWS;
  const int rows_blk = (int)min((int64_t)ROWS, ext_raw - q0_blk);
  const int pos_off = PW == 32 ? 32 * (wave & 1) : 0;
  const int q0 = q0_blk + pos_off;
  const int n_heads = PW == 32 ? (head_ok ? 1 : 0) : max(0, min(CH, n_rt - hw));  // q heads this wave really has
  const int n_rows = n_heads > 0 ? max(0, min(PW, rows_blk - pos_off)) : 0;       // positions it really has
  const bool col_ok = pos < n_rows && hsub < n_heads;
  const int64_t q_row0 = q_first + q0;
  int64_t req = a.req_idx[i_req];
  req = req < 0 ? 0 : (req >= a.kv.table_rows ? a.kv.table_rows - 1 : req);
  const int64_t seq64 = a.seq_lens[i_req];
  const int seq = (int)(seq64 < 0 ? 0 : (seq64 > a.kv.table_cols ? a.kv.table_cols : seq64));
  const int64_t pre64 = a.prefix_lens[i_req];
  const int prefix = (int)(pre64 < 0 ? 0 : (pre64 > seq ? seq : pre64));
  // ---- what this lane's row sees, and what the wave and the workgroup have to stream ---------------
  const int own = prefix + q0 + pos;  // its position in the request
  int2 seen = make_int2(0, 0);        // {first, number} of the positions it sees
  if (col_ok) seen = visible_range(a.mods, q_row0 + pos, seq, min(seq, own + 1));
  // (rows that see nothing are left out: their scores may be anything, they are written as zeros)
  const bool live = seen.y > 0;
  int2 rng;                 // the wave's rows: first position any of them sees, one past the last
  int full_from, full_to;   // ... and the positions all of them see
  {
    int f0 = live ? seen.x : 0x7fffffff, f1 = live ? seen.x + seen.y : 0, g0 = live ? seen.x : 0, g1 = live ? seen.x + seen.y : 0x7fffffff;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      f0 = min(f0, __shfl_xor(f0, d));
      f1 = max(f1, __shfl_xor(f1, d));
      g0 = max(g0, __shfl_xor(g0, d));
      g1 = min(g1, __shfl_xor(g1, d));
    }
    rng = make_int2(__builtin_amdgcn_readfirstlane(f0), __builtin_amdgcn_readfirstlane(f1));
    full_from = __builtin_amdgcn_readfirstlane(g0);
    full_to = __builtin_amdgcn_readfirstlane(g1);
  }
  if (lane == 0) s_rng[wave] = rng;
  __syncthreads();
  int first = 0x7fffffff, last = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    first = min(first, __builtin_amdgcn_readfirstlane(s_rng[w].x));
    last = max(last, __builtin_amdgcn_readfirstlane(s_rng[w].y));
  }
  if (last == 0) first = 0;  // nobody sees anything
  if (a.splits > 1) {
    // this workgroup's piece of the stream: whole steps, counted from the last token back
    const int all = last - first;
    const int chunk = ((all + a.splits - 1) / a.splits + STEP - 1) / STEP * STEP;
    const int s0 = min((int)blockIdx.y * chunk, all), s1 = min(s0 + chunk, all);
    first = last - s1;
    last -= s0;
  }
  // Everything below counts tokens in the order they are streamed, from the last one back (see the head of this
  // file): place t is position last - 1 - t.
  const int kv_len = last - first;
  const int wave_len = rng.y > 0 ? last - rng.x : 0;
  {
    const int f = full_from;
    full_from = last - min(full_to, last);
    full_to = last - max(f, first);
  }
  const int my_lo = last - (seen.x + seen.y);
  const int my_hi = live ? my_lo + seen.y : 0x7fffffff;
  const int my_pos = last - 1 - own;
  const int wave_pos = last - 1 - (prefix + q0);  // places before this one stand ahead of some row of the wave
  const int32_t* table_row = a.kv.table + req * a.kv.table_row_stride + first;
  const uint32_t max_slot = (uint32_t)(a.kv.n_slots - 1);
  const uint32_t row_units = (uint32_t)(a.kv.slab_row_stride * 2 / 16);
  const int head0 = kvh * G + rt0 + (two_blocks ? 0 : hw);  // (folded: kvh = 0 and G counts the heads of both halves)
  const int head = head0 + hsub;                            // the q head of this lane's column

  // ---- Q^T fragments: lane (position lp, half hi) holds Q[q_row0 + lp][head][16 kb + 8 hi ..] ----
  uint4 qf[8];
  {
    const char* qrow = (const char*)a.q + (q_row0 + pos) * a.q_row_stride * 2;
#pragma unroll
    for (int kb = 0; kb < 8; ++kb) {
      qf[kb] = make_uint4(0, 0, 0, 0);
      if (col_ok) {
        if (fold == 0) {
          qf[kb] = *(const uint4*)(qrow + ((int64_t)head * D + 16 * kb + 8 * hi) * 2);
        } else if ((16 * kb + 8 * hi) / 64 == head / fold) {
          qf[kb] = *(const uint4*)(qrow + ((int64_t)head * 64 + (16 * kb + 8 * hi) % 64) * 2);
        }
      }
    }
  }
  const float scale_log2e = a.scale * kLog2e;
  const float arg = CAP ? 2.f * scale_log2e / a.mods.cap : 0.f;
  const float top2 = CAP ? a.mods.cap * kLog2e : 0.f;
  const float slope = BIAS ? a.mods.slopes[min(head, a.n_q_heads - 1)] * kLog2e : 0.f;
  const float A = CAP ? -2.f * top2 : BIAS ? scale_log2e : 1.f;
  const float slope_u = BIAS ? slope / A : 0.f;
  // raw score of register r -> u (see the head of this file)
  auto shape = [&](float raw, int r) {
    float u = raw;
    if constexpr (CAP) u = __builtin_amdgcn_rcpf(fast_exp2(raw * arg) + 1.f);
    if constexpr (BIAS) u = fmaf(-slope_u, (float)acc_row(r, 0), u);
    if constexpr (!CAP && !BIAS) u *= scale_log2e;
    return u;
  };
  constexpr bool FLIP = CAP;  // A is negative: the largest score has the smallest u
  constexpr float kHidden = FLIP ? -kNegInf : kNegInf;
  // the part of a score that the step and the lane decide
  auto step_c = [&](int step) {
    return BIAS ? fmaf(-slope, (float)(step * STEP + 4 * hi - my_pos), top2) : CAP ? top2 : 0.f;
  };
  auto ext3 = [](float x, float y, float z) { return FLIP ? min3(x, y, z) : max3(x, y, z); };

  // ---- DMA source pieces: two tokens per instruction, [K 256 B | V 256 B] per token -----
  const int piece = lane & 31;
  const bool piece_is_v = piece >= 16;
  const int lane_tok = lane >> 5;
  const uint64_t lane_src = (uint64_t)(piece_is_v ? a.kv.v_slab : a.kv.k_slab) + (uint64_t)kvh * (D * 2) +
                            (uint64_t)((((piece & 15)) ^ (lane_tok << 2)) << 4);

  // K as the A operand: lane (token lp of the step, half hi) reads K[token][16 kb + 8 hi ..]
  const int k_rec = rec_of_token(lp & 15);
  int k_off[8];
#pragma unroll
  for (int kb = 0; kb < 8; ++kb)
    k_off[kb] = (lp >> 4) * TILE_BYTES + k_rec * REC + (((2 * kb + hi) ^ xr_of_rec(k_rec)) << 4);
  // V as the B operand through transposing reads: a 16-lane group fetches 4 tokens x 16 values
  // (lane i of it: token i >> 2, values 4 (i & 3) ..) and lane i receives value column i of the
  // four tokens.  The group's tokens: 8 jh + 4 hi + 0..3 of the tile, its columns
  // 32 db + 16 (group & 1) ..
  int v_off[2][4];
  {
    const int i16 = lane & 15, dh = (lane >> 4) & 1;
#pragma unroll
    for (int jh = 0; jh < 2; ++jh) {
      const int rec = rec_of_token(8 * jh + 4 * hi + (i16 >> 2));
#pragma unroll
      for (int db = 0; db < 4; ++db)
        v_off[jh][db] = rec * REC + 256 + (((4 * db + 2 * dh + ((i16 & 3) >> 1)) ^ xr_of_rec(rec)) << 4) + ((i16 & 1) << 3);
    }
  }

  // m_run: largest score of the lane's position when it was last looked for, units of log2; m_sub: what its scores are taken
  // against.  The maximum of a step is looked for only until every row of the wave has seen a token, and where tokens are
  // masked.  Otherwise the step's probabilities are made first and their sum, which is wanted anyway, tells: if a lane's 16 pass
  // 2^kTop, the reference moves and they are made again, before a product has met a value.  A move is dear (every lane's 64
  // sums), so the largest score stands at 2^kLift, well below that.  bf16 has f32's exponents and stands in the middle of them:
  // 2^-10 to 2^10, 20 of the 2^+-126 that the products with the values have.  f16 ends at 2^16, and what is below 2^-25 is lost from the
  // product (not from the sum): from the largest score, at 2^6, that is 2^-31, 2^-14 in all for 131072 tokens.
  // (A cap bounds the scores, and a fixed reference of 0 needs no looking at all; but 2^(cap log2 e) times a value is not in range
  // whatever the value is.)
  constexpr bool HALF = std::is_same<Tag, f16_tag>::value;
  constexpr float kLift = HALF ? 6.f : -10.f, kTop = HALF ? 15.f : 10.f;
  constexpr float kMostSum = HALF ? 0x1p15f : 0x1p10f;
  constexpr float kSlack = kTop - kLift - 4.f;  // (16 scores this far above m_run come to 2^kTop)
  float m_run = kNegInf, m_sub = 0.f;           // (while nothing has been seen)
  bool all_seen = false;                        // (wave-uniform)
  float l_run = 0.f;  // sum of this lane's probabilities (its 16 tokens of every step)
  f32x16 o_acc[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o_acc[db][r] = 0.f;

  // The page-table entries of the sequence are staged SLOTS at a time into the two halves of
  // s_slots; block b + 1 is fetched while block b is being worked on, so the K/V stream never
  // drains between blocks.  Each thread fetches two entries of a block.
  const int n_steps = (kv_len + STEP - 1) / STEP;
  auto entry_ptr = [&](int e) {  // the entry of place e; places past the end repeat the last one
    return table_row + max(kv_len - 1 - max(e, 0), 0);
  };
  auto entry_off = [&](uint32_t s) { return (int32_t)((s > max_slot ? max_slot : s) * row_units); };
  {
    uint32_t e[EPT];
#pragma unroll
    for (int k = 0; k < EPT; ++k) e[k] = (uint32_t)*entry_ptr(tid + k * NTHR);
#pragma unroll
    for (int k = 0; k < EPT; ++k) s_slots[tid + k * NTHR] = entry_off(e[k]);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // retire every compiler-visible load before the step loop
  __syncthreads();
  // (the entries of block b + 1 come in by LDS-DMA, raw, and are turned into row offsets in place by
  // the threads whose wave brought them: no register ever holds data that is still on its way --
  // an asm load INTO a register counts as complete where its statement ends, and under register
  // pressure the compiler may copy that register before the data lands)
  const uint32_t lds_slots = lds_ring + BUF;

  // a step is loaded by all waves together: wave w issues instructions w*DPW .. w*DPW+DPW-1;
  // instruction i brings tokens 2i, 2i+1 of the step (tile i / 8)
  // (the row offsets of a step are read from s_slots one request early, so that the request
  // itself does not start with an LDS round trip)
  // a step's requests of this wave: request r (0 .. NREQ-1) is
  // group g and is instruction wave * DPW + r of that step
  constexpr int NREQ = DPW;
  static_assert(NREQ == 4, "four requests per wave and step");
  uint32_t off[NREQ];
  auto read_offsets = [&](int group) {
#pragma unroll
    for (int r = 0; r < NREQ; ++r) {
      const int step = group;
      off[r] = (uint32_t)s_slots[((step * STEP) & (2 * SLOTS - 1)) + 2 * (wave * DPW + r) + lane_tok];
    }
  };
  // The four source addresses are made ahead of the wait and the barrier of the step that issues them
  // (make_src), and the requests then go out as ONE statement, M0 set per request and restored once
  // (four statements with their address arithmetic in between: 78 cycles per request, this form 54).
  uint64_t src4[NREQ];
  auto make_src = [&]() {
#pragma unroll
    for (int r = 0; r < NREQ; ++r) {
      const int i = wave * DPW + r;  // wave-uniform: instruction i brings tokens 2i, 2i+1 of its step (tile i / 8)
      const uint32_t xr = (uint32_t)xr_of_rec(rec_of_token(2 * (i & 7)));
      src4[r] = (((uint64_t)off[r] << 4) + lane_src) ^ (uint64_t)(xr << 4);
    }
  };
  auto issue_group = [&](int group) {
    uint32_t dst[NREQ];
#pragma unroll
    for (int r = 0; r < NREQ; ++r) {
      const int i = wave * DPW + r;
      const uint32_t stage = lds_ring + (uint32_t)((group) % NSTAGE) * STEP_BYTES;
      dst[r] = __builtin_amdgcn_readfirstlane(stage + (uint32_t)(i >> 3) * TILE_BYTES + (uint32_t)rec_of_token(2 * (i & 7)) * REC);
    }
    uint32_t keep;
      asm volatile(
          "s_mov_b32 %0, m0\n\t"
          "s_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\t"
          "s_mov_b32 m0, %6\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\t"
          "s_mov_b32 m0, %7\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, off\n\t"
          "s_mov_b32 m0, %8\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, off\n\t"
          "s_mov_b32 m0, %0"
          : "=&s"(keep)
          : "v"(src4[0]), "v"(src4[1]), "v"(src4[2]), "v"(src4[3]), "s"(dst[0]), "s"(dst[1]), "s"(dst[2]), "s"(dst[3])
          : "memory");
  };

  const int n_groups = n_steps;  // (a step is the unit of requests, waits and barriers)
  f32x16 sc_a, sc_b;
  if (n_groups > 0) {
    read_offsets(0);
    make_src();
    issue_group(0);
  }
  if (n_groups > 1) { read_offsets(1); make_src(); issue_group(1); }
  if (n_groups > 2) { read_offsets(2); make_src(); issue_group(2); }
  if (n_groups > 3) read_offsets(3);

  // sc_a, sc_b: the u of the step about to be consumed, and the raw scores, then u, of the one after it: the
  // two trade places from step to step.  ext16: the extreme u of a lane
  auto ext16 = [&](const f32x16& v) {
    float m = ext3(v[0], v[1], v[2]);
#pragma unroll
    for (int r = 3; r < 15; r += 2) m = ext3(m, v[r], v[r + 1]);
    return ext3(m, v[15], v[15]);
  };
  auto load_k = [&](uint4 (&kf)[8], const char* st) {
#pragma unroll
    for (int kb = 0; kb < 8; ++kb) kf[kb] = *(const uint4*)(st + k_off[kb]);
  };
  auto scores = [&](const uint4 (&kf)[8]) {
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int kb = 0; kb < 8; ++kb) s = Mma32<Tag>::mm(kf[kb], qf[kb], s);
    return s;
  };
  {
    if (n_groups > 2) dma_wait<2 * NREQ>(); else if (n_groups > 1) dma_wait<NREQ>(); else dma_wait<0>();
    __syncthreads();
    if (0 < wave_len) {
      uint4 kf[8];
      load_k(kf, smem);
      sc_a = scores(kf);
#pragma unroll
      for (int r = 0; r < 16; ++r) sc_a[r] = shape(sc_a[r], r);
    }
  }

  {
    // the head of a step: wait for this wave's share of the next group, the workgroup barrier, the
    // requests of the group three ahead
    auto top = [&](int step) {
      // the entries of block b + 1 are asked for at the head of step 16 b + 2 (behind that group's K/V
      // requests), have arrived by the wait one group after the next and are turned into row offsets
      // there; their half of s_slots was last read for step 16 b - 1 and is first read for step
      // 16 b + 16, whose requests go out three groups ahead of it
      const int in_blk = step & (SLOTS / STEP - 1);
      const int group = step;
      const bool more_entries = ((step >> 4) + 1) * SLOTS < kv_len;  // wave-uniform
      const bool has_next = group + 1 < n_groups;           // wave-uniform
      const bool issue_ok = has_next && group + 3 < n_groups;  // wave-uniform
      if (issue_ok) make_src();  // the addresses of this group's requests, ahead of the wait
      if (has_next) {
        // this wave's share of the next group has landed (one younger group may stay in flight, and
        // one group after the entries were asked for, those behind it) ...
        if (group + 2 >= n_groups) dma_wait<0>();
        else if (in_blk == 3 && more_entries) dma_wait<NREQ + EPT>();
        else dma_wait<NREQ>();
        if (in_blk == 4 && more_entries) {
          // (this wave's own pieces, landed by the wait above; the barrier below publishes them)
          int32_t* half = s_slots + (((step >> 4) + 1) & 1) * SLOTS;
          uint32_t e[EPT];
#pragma unroll
          for (int k = 0; k < EPT; ++k) e[k] = (uint32_t)half[tid + k * NTHR];
#pragma unroll
          for (int k = 0; k < EPT; ++k) half[tid + k * NTHR] = entry_off(e[k]);
        }
        // ... and so has everybody's; all waves are also done reading the group before this one
        __syncthreads();
        // the row offsets of the group after the one requested now are asked for first (any entries if
        // there is no such group: they are then never used) and travel while the requests go out
        read_offsets(group + 4);
        if (issue_ok) issue_group(group + 3);  // into the stages the group before this one used
        if (in_blk == 2 && more_entries) {
          const int e = ((step >> 4) + 1) * SLOTS + tid;
          const uint32_t half = lds_slots + (uint32_t)((((step >> 4) + 1) & 1) * SLOTS * 4) + (uint32_t)wave * 256u;
#pragma unroll
          for (int k = 0; k < EPT; ++k)
            dma_256((const void*)entry_ptr(e + k * NTHR), __builtin_amdgcn_readfirstlane(half + (uint32_t)(k * NTHR * 4)));
        }
      }
    };
    auto do_step = [&](int step, auto stage_c, f32x16& sc, f32x16& sn) {
      constexpr int STAGE = decltype(stage_c)::value;
      constexpr int NEXT = (STAGE + 1) % NSTAGE;
      top(step);
      const char* st = smem + STAGE * STEP_BYTES;
      if (step * STEP >= wave_len) return;  // nothing this wave's rows may see (wave-uniform)

      // The body runs at raised priority (four waves: the SIMD's other wave belongs to another workgroup and
      // is wherever it is): where both waves have an instruction ready, the one inside its products goes first
      // and the one at the head of its step (wait, barrier, requests) fills in.  + 0.6 to + 1.8 % by shape.
      __builtin_amdgcn_s_setprio(2);
      // K fragments of step + 1 (whatever the stage holds if there is no such step: the scores
      // made of them are then never used); they travel while the maximum is looked at
      uint4 kf[8];
      load_k(kf, smem + NEXT * STEP_BYTES);

      const bool hides = step * STEP < full_from || step * STEP + STEP > full_to;  // wave-uniform
      const bool looks_ahead = BIAS && step * STEP < wave_pos;
      const float c_step = step_c(step);
      // moves the reference of every row to its largest score so far (`lmax`: the lane's)
      auto move_reference = [&](float lmax) __attribute__((always_inline)) {
        float x = lmax, y = lmax;
        swap32(x, y);  // the partner lane holds the position's other 16 tokens
        const float m_new = max3(m_run, x, y);
        // a position with nothing visible yet keeps m = -inf: its factor is 1, not exp2(nan)
        const float alpha = m_new == kNegInf ? 1.f : fast_exp2(m_run - m_new);
        m_run = m_new;
        m_sub = m_new == kNegInf ? 0.f : m_new - kLift;  // masked scores: exp2(-inf) = 0
        l_run *= alpha;
        // O has its positions in the registers: register r of this lane belongs to position
        // acc_row(r, hi), whose factor lives on lane acc_row(r, hi)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float ar = __shfl(alpha, acc_row(r, 0) + 4 * hi);
#pragma unroll
          for (int db = 0; db < 4; ++db) o_acc[db][r] *= ar;
        }
      };
      if (__builtin_expect(hides || looks_ahead || !all_seen, 0)) {  // (rare: the ends of the rows' intervals, and prefixes read both ways)
        int t0m = step * STEP + 4 * hi;
        asm volatile("" : "+v"(t0m));
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int t = t0m + acc_row(r, 0);
          // (the bias above is slope * (j - i), which is what is wanted up to the row's own position)
          if constexpr (BIAS) sc[r] = fmaf(-2.f * slope_u, (float)max(my_pos - t, 0), sc[r]);
          sc[r] = (t >= my_lo && t < my_hi) ? sc[r] : kHidden;
        }
        const float lmax = fmaf(ext16(sc), A, c_step);
        if (__any(lmax > m_run + kSlack)) move_reference(lmax);
        all_seen = !__any(live && m_run == kNegInf);
      }
      float c0 = c_step - m_sub;

      // ---- from here to the end of the step: one basic block, issued in the order written ----
      // (a scheduling barrier after every product: the compiler's own order puts the vector
      // work in clumps and waits for every LDS read right behind its issue).  A product holds
      // the vector issue for 8 of its 32 cycles; the gap takes one or two exponentials (8
      // cycles each) and a few 4-cycle instructions.
      auto v_frag = [&](int i) {  // V fragment of PV product i: tile i >> 2, value columns 32 (i & 3) ..
        const s16x4_t va = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4_t*)(st + (i >> 2) * TILE_BYTES + v_off[0][i & 3]));
        const s16x4_t vb = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4_t*)(st + (i >> 2) * TILE_BYTES + v_off[1][i & 3]));
        const uint2 va2 = __builtin_bit_cast(uint2, va), vb2 = __builtin_bit_cast(uint2, vb);
        return make_uint4(va2.x, va2.y, vb2.x, vb2.y);
      };
#pragma unroll
      for (int r = 0; r < 16; ++r) sn[r] = 0.f;
      float e[16], p[16];
      float sum = 0.f;  // of the lane's probabilities of this step
      uint32_t pw[8];  // probabilities, two to a word: words 4 kk .. 4 kk + 3 = the A operand of tile kk
      uint4 vf[4];  // V fragments travel three products ahead of their use
      e[0] = fmaf(sc[0], A, c0);
      e[1] = fmaf(sc[1], A, c0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kb = 0; kb < 8; ++kb) {
        sn = Mma32<Tag>::mm(kf[kb], qf[kb], sn);
        p[2 * kb] = fast_exp2(e[2 * kb]);
        p[2 * kb + 1] = fast_exp2(e[2 * kb + 1]);
        if (kb < 7) {
          e[2 * kb + 2] = fmaf(sc[2 * kb + 2], A, c0);
          e[2 * kb + 3] = fmaf(sc[2 * kb + 3], A, c0);
        }
        if (kb >= 4) pw[kb - 4] = E::pack2(p[2 * (kb - 4)], p[2 * (kb - 4) + 1]);
        if (kb >= 5) vf[kb - 5] = v_frag(kb - 5);
        if (kb >= 1) sum = (sum + p[2 * kb - 2]) + p[2 * kb - 1];
        __builtin_amdgcn_sched_barrier(0);
      }
      sum = (sum + p[14]) + p[15];
      if (__builtin_expect(__any(sum > kMostSum), 0)) {
        move_reference(fmaf(ext16(sc), A, c_step));
        c0 = c_step - m_sub;
        sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[r] = fast_exp2(fmaf(sc[r], A, c0));
          sum += p[r];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) pw[r] = E::pack2(p[2 * r], p[2 * r + 1]);
      }
      l_run += sum;
      // k-values of a lane in PV product i: registers 8 kk .. 8 kk + 7 of the score accumulator,
      // i.e. tokens {0-3, 8-11} + 4 hi of tile kk = i >> 2
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int kk = i >> 2;
        o_acc[i & 3] = Mma32<Tag>::mm(make_uint4(pw[4 * kk], pw[4 * kk + 1], pw[4 * kk + 2], pw[4 * kk + 3]), vf[i % 4], o_acc[i & 3]);
        if (i + 3 < 8) vf[(i + 3) % 4] = v_frag(i + 3);
        if (i < 4) pw[4 + i] = E::pack2(p[8 + 2 * i], p[8 + 2 * i + 1]);
        // (the next step's scores are complete by now: three of them per gap)
        if (i >= 2) {
#pragma unroll
          for (int r = 3 * (i - 2); r < (i == 7 ? 16 : 3 * (i - 1)); ++r) sn[r] = shape(sn[r], r);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
    };
    static_assert(NSTAGE == 4, "the step loop below is unrolled over the ring");
    for (int step = 0; step < n_steps; step += NSTAGE) {
      do_step(step, std::integral_constant<int, 0>{}, sc_a, sc_b);
      if (step + 1 < n_steps) do_step(step + 1, std::integral_constant<int, 1>{}, sc_b, sc_a);
      if (step + 2 < n_steps) do_step(step + 2, std::integral_constant<int, 2>{}, sc_a, sc_b);
      if (step + 3 < n_steps) do_step(step + 3, std::integral_constant<int, 3>{}, sc_b, sc_a);
    }
  }

  // ---- normalise and write: rows through LDS so that a lane stores 16 contiguous bytes ----
  __syncthreads();  // the ring is free: each wave stages its rows in its own region
  float* o_lds = (float*)(smem + wave * STAGE_OUT);
  uint32_t sums_nan;  // columns with a NaN among the scores they see: nothing to be done
  {
    float x = l_run, y = l_run;
    swap32(x, y);
    const float l_pos = x + y;  // both halves of the position's tokens
    // (a NaN sum stays NaN; a row that sees nothing is zeroed by the write below)
    const float inv = l_pos == 0.f ? 0.f : 1.f / l_pos;
    sums_nan = (uint32_t)__ballot(l_pos != l_pos);
    if (lane == 0) s_bad[wave] = 0;
    if (hi == 0) s_live[wave][lp] = live;
    if (a.splits > 1 && hi == 0 && col_ok) {
      const float lse = live && l_pos != 0.f ? (m_sub + __builtin_amdgcn_logf(l_pos)) * kLn2 : kNegInf;
      a.parts_lse[((int64_t)blockIdx.y * a.total_q_tokens + q_row0 + pos) * a.n_q_heads + head] = lse;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float ir = __shfl(inv, acc_row(r, 0) + 4 * hi);
#pragma unroll
      for (int db = 0; db < 4; ++db) o_lds[(acc_row(r, 0) + 4 * hi) * kOPad + 32 * db + lp] = o_acc[db][r] * ir;
    }
    for (int idx = lane; idx < 32 * (D / 8); idx += 64) {
      const int r = idx / (D / 8), c8 = idx % (D / 8);  // r: column of S^T = (q head r / PW, position r % PW)
      if (r % PW >= n_rows || r / PW >= n_heads) continue;
      const int64_t orow = q_row0 + r % PW;
      const int oh = head0 + r / PW;
      const float* src = o_lds + r * kOPad + c8 * 8;
      const bool ok = s_live[wave][r] != 0;
      float f[8];
      bool nan = false;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f[k] = ok ? src[k] : 0.f;
        nan |= f[k] != f[k];
      }
      if (nan && (fold == 0 || (c8 * 8) / 64 == oh / fold)) atomicOr(&s_bad[wave], 1u << r);
      if (a.splits > 1) {
        const int dim = fold == 0 ? D : 64;
        if (fold != 0 && (c8 * 8) / 64 != oh / fold) continue;
        float* dst = a.parts_o + (((int64_t)blockIdx.y * a.total_q_tokens + orow) * a.n_q_heads + oh) * dim + (c8 * 8) % dim;
        *(float4*)dst = make_float4(f[0], f[1], f[2], f[3]);
        *(float4*)(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
        continue;
      }
      const uint4 packed = E::pack(f);
      if (fold == 0) {
        *(uint4*)((char*)a.out + (orow * a.out_row_stride + (int64_t)oh * D + c8 * 8) * 2) = packed;
      } else if ((c8 * 8) / 64 == oh / fold) {
        *(uint4*)((char*)a.out + (orow * a.out_row_stride + (int64_t)oh * 64 + (c8 * 8) % 64) * 2) = packed;
      }
    }
  }
  // rows that came out NaN and have met a value that they do not see: again, by themselves
  uint32_t bad = __builtin_amdgcn_readfirstlane(s_bad[wave]) & ~sums_nan;
  if (bad != 0)
    bad &= (uint32_t)__ballot(met_unseen<Tag, 256>((const char*)a.kv.v_slab + (int64_t)kvh * (D * 2), a.kv.slab_row_stride * 2, table_row, max_slot, kv_len,
                                                   wave_len, full_from, full_to, my_lo, my_hi));
  if (bad != 0) __builtin_amdgcn_s_waitcnt(0x0F70);  // (behind the stores above, which went to the same rows)
  while (bad != 0) {
    const int r = __ffs((int)bad) - 1;
    bad &= bad - 1;
    const int lo = __builtin_amdgcn_readlane(seen.x, r), n = __builtin_amdgcn_readlane(seen.y, r);
    rescue_row<Tag>(a, q_row0 + r % PW, head0 + r / PW, kvh, req, prefix + q0 + r % PW, max(lo, first), min(lo + n, last), (int)blockIdx.y);
  }
}

template <typename Tag, int PW>
void launch_shape(const PrefillArgs& a, dim3 grid, hipStream_t stream) {
  const bool cap = a.mods.cap > 0.f, bias = a.mods.slopes != nullptr;
  if (cap && bias) hipLaunchKernelGGL((prefill_scored_kernel<Tag, PW, true, true>), grid, dim3(256), 0, stream, a);
  else if (cap) hipLaunchKernelGGL((prefill_scored_kernel<Tag, PW, true, false>), grid, dim3(256), 0, stream, a);
  else if (bias) hipLaunchKernelGGL((prefill_scored_kernel<Tag, PW, false, true>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((prefill_scored_kernel<Tag, PW, false, false>), grid, dim3(256), 0, stream, a);
}

}  // namespace

// the extend kernels' conditions, with up to 16 q heads per kv head (a workgroup takes them two or eight at a time)
bool prefill_scored_supported(const PrefillArgs& a, const char** why) {
  if (a.dtype == kF32) return prefill_scored_f32_supported(a, why);
  // (without a cap the largest score is taken to be the largest product, and a bias is carried in units of the scale)
  if (!(a.mods.cap > 0.f) && !(a.scale > 1e-30f)) {
    *why = "the matrix-core kernel needs a positive scale";
    return false;
  }
  PrefillArgs b = a;
  if (a.n_kv_heads > 0 && a.n_q_heads % a.n_kv_heads == 0 && a.n_q_heads / a.n_kv_heads <= 16) b.n_q_heads = a.n_kv_heads;
  return prefill_mfma_supported(b, why);
}

// the grid of launch_prefill_mfma32: 2 (64-position blocks) or 8 (16-position blocks) q heads per workgroup
hipError_t launch_prefill_scored(const PrefillArgs& a, hipStream_t stream) {
  const int group = a.n_q_heads / a.n_kv_heads;
  const int hpw = a.blk_rows == 64 ? 2 : 8;
  const int n_z = (group + hpw - 1) / hpw;
  const int64_t local_groups = ((int64_t)a.max_groups * a.n_kv_heads + 7) / 8;
  const int64_t n_wg = 8 * local_groups * a.grp_blocks * n_z;
  if (n_wg > 0x7fffffffll) return hipErrorInvalidValue;
  const dim3 grid((unsigned)n_wg, (unsigned)(a.splits > 1 ? a.splits : 1), 1);
  if (a.dtype == kF32) (void)launch_prefill_scored_f32(a, grid, stream);
  else if (a.dtype == kBF16) a.blk_rows == 64 ? launch_shape<bf16_tag, 32>(a, grid, stream) : launch_shape<bf16_tag, 16>(a, grid, stream);
  else a.blk_rows == 64 ? launch_shape<f16_tag, 32>(a, grid, stream) : launch_shape<f16_tag, 16>(a, grid, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits <= 1) return e;
  MergeArgs mg;
  mg.out = a.out;
  mg.out_row_stride = a.out_row_stride;
  mg.lse_out = nullptr;
  mg.parts_o = a.parts_o;
  mg.parts_lse = a.parts_lse;
  mg.n_parts = a.splits;
  mg.rows = a.total_q_tokens;
  mg.n_heads = a.n_q_heads;
  mg.head_dim = a.fold_group > 0 ? 64 : a.head_dim;
  mg.dtype = a.dtype;
  mg.row_end = a.cu_ext + a.batch;
  return launch_merge(mg, stream);
}

}  // namespace bsgl
