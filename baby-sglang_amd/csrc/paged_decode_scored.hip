// Scored decode attention for gfx950 (the scores: ScoreMods): bf16, f16 and f32 rows, head_dim 64 or 128, up to 16 q heads per
// kv head, requests or (ScoreMods::rows) extend tokens as rows.
//
// One workgroup per (row, kv head, piece of its visible tokens), four waves that take the piece's tiles of 16 tokens in
// turn.  Every operand is loaded from memory as its product wants it, so nothing passes through LDS, a wave needs the
// registers of one tile only, and three or four waves per SIMD keep the memory busy whatever the lengths are:
//   S^T = K Q^T   lane (c, u) = (lane & 15, lane >> 4) reads 16 bytes of token c per load, bytes 64 j + 16 u ..; Q in the
//                 same order.  It then owns the scores of head c and tokens 4 u .. 4 u + 3.
//   O  += P V     the k-values of a lane are its own four tokens: P from the registers it is in, V as D / 16 neighbouring values
//                 of each token per lane -- which columns of the product they are is this kernel's choice.  f32
//                 (v_mfma_f32_16x16x4_f32, f32 by f32) takes one token per product; 16 bits take all four, the tokens'
//                 values brought together by byte permutes, and bf16 takes them twice, with P as a high and a low half (P to 16
//                 bits, as the plain decode has it; f16 rounds it once, 2^-11).
// The next tile's K is asked for as soon as the scores are made of this one's, its V behind the last product: both are
// always on their way; bound by memory (see launch_decode_scored for what it reached).  The waves' results meet in LDS, pieces
// in the workspace: the last workgroup of a (row, kv head) to finish -- a ticket -- merges them, or a launch of its own where
// the tickets do not fit.
#include "bsgl_device.h"
#include "bsgl_launch.h"
#include "bsgl_mfma.h"
#include "bsgl_score.h"

#include <type_traits>

namespace bsgl {

namespace {

using namespace mfma;

typedef __attribute__((ext_vector_type(4))) float f32x4v;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4v;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2v;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4v;

constexpr int kWaves = 4;
constexpr int kTokens = 16;  // per tile

// S^T += K Q^T over the 16 bytes a lane has of a token and of a head
template <typename Tag> __device__ __forceinline__ f32x4v score_product(u32x4v k, u32x4v q, f32x4v s) {
  if constexpr (std::is_same<Tag, f32_tag>::value) {
    const f32x4v kf = __builtin_bit_cast(f32x4v, k), qf = __builtin_bit_cast(f32x4v, q);
#pragma unroll
    for (int m = 0; m < 4; ++m) s = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[m], qf[m], s, 0, 0, 0);
    return s;
  } else if constexpr (std::is_same<Tag, bf16_tag>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k), __builtin_bit_cast(bf16x8_t, q), s, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, k), __builtin_bit_cast(f16x8_t, q), s, 0, 0, 0);
  }
}

// waves per SIMD the registers of an instance allow
// The largest score of a tile stands at 2^kLift: f16, whose probabilities enter the second product as they are, ends at 2^16, and what is
// below 2^-25 is lost from the product but not from the sum -- 2^-40 from the largest score, nothing for rows of any length; with it
// at 1, a tail of 60000 tokens of 2^-26 each loses 2^-10 of the row.
template <typename Tag> constexpr float kLift = std::is_same<Tag, f16_tag>::value ? 15.f : 0.f;

template <typename Tag, int D> constexpr int occupancy() { return std::is_same<Tag, f32_tag>::value && D == 128 ? 3 : 4; }

// ROWS: extend tokens as rows (ScoreMods::rows), else requests
template <typename Tag, int D, bool ROWS>
__global__ __launch_bounds__(64 * kWaves, (occupancy<Tag, D>()))
void decode_scored_kernel(DecodeArgs a) {
  using E = Elem<Tag>;
  constexpr bool F32 = E::BYTES == 4;
  constexpr int ROW = D * E::BYTES;    // bytes of a head
  constexpr int KN = ROW / 64;         // loads of K per lane and tile
  constexpr int VB = ROW / 16;         // bytes of V per lane and token: 8, 16 or 32
  constexpr int VW = VB / 4;           // words
  constexpr int NB = D / 16;           // blocks of 16 output columns = values of V per lane and token
  constexpr int PAD = D + 4;
  constexpr int C4 = D / 4;
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][16][PAD];
  __shared__ float s_m[kWaves][16], s_l[kWaves][16];
  __shared__ float s_w[16][64];  // merge: weight of a head's part
  __shared__ uint32_t s_ticket;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, u = lane >> 4;
  const int G = a.n_q_heads / a.n_kv_heads;
  const bool fused = a.counters != nullptr;

  // ---- which row, and what it sees: row i's page-table row, own position and visible tokens
  struct RowView {
    int req, own, first, seq;
    bool owned;
  };
  auto view = [&](int i) {
    int64_t req, len64;
    int own = 0;
    RowView v;
    v.owned = true;
    if constexpr (ROWS) {
      const int4 r4 = a.mods.rows[i];
      req = r4.x;
      len64 = r4.y;
      own = r4.z;
      v.owned = r4.w != 0;
    } else {
      req = a.req_idx[i];
      len64 = a.seq_lens[i];
    }
    v.req = (int)(req < 0 ? 0 : (req >= a.kv.table_rows ? a.kv.table_rows - 1 : req));
    const int len = (int)(len64 < 0 ? 0 : (len64 > a.kv.table_cols ? a.kv.table_cols : len64));
    v.own = ROWS ? own : len - 1;
    const int2 seen = visible_range(a.mods, i, len, min(len, v.own + 1));
    v.first = seen.x;
    v.seq = v.owned ? seen.y : 0;
    return v;
  };
  int row, kvh, split, n_parts;
  RowView me;
  if (a.balance_target > 0) {
    // Pieces of one length for the whole batch, dealt out in row order: with some target of pieces per kv head, a batch of
    // any lengths takes target + rows workgroups of them at most.  Every wave finds its own by itself (1 us).
    // (extend tokens of a request read the same K/V: their workgroups for one piece of it are a multiple of kv heads x pieces apart
    // in the launch, on one XCD and its L2 where that is a multiple of eight -- 8 x 8 over 1000, 28 / 4 heads: 23 us, with rows
    // side by side 32; requests share nothing, and kv head by kv head streams a little better)
    int nth;
    if constexpr (!ROWS) {
      const unsigned per = (unsigned)(a.balance_target + a.rows);
      kvh = blockIdx.x / per;
      nth = blockIdx.x % per;
    } else {
      kvh = blockIdx.x % (unsigned)a.n_kv_heads;
      nth = blockIdx.x / (unsigned)a.n_kv_heads;
    }
    RowView v0 = {0, 0, 0, 0, false};
    int total = 0, longest = 0;
    for (int r0 = 0; r0 < a.rows; r0 += 64) {
      RowView v = {0, 0, 0, 0, false};
      if (r0 + lane < a.rows) v = view(r0 + lane);
      if (r0 == 0) v0 = v;
      total += __builtin_amdgcn_readlane(wave_inclusive_scan<ScanAdd>(v.seq), 63);
      longest = max(longest, __builtin_amdgcn_readlane(wave_inclusive_scan<ScanMax>(v.seq), 63));
    }
    int piece = max((total + a.balance_target - 1) / a.balance_target, (longest + a.n_splits - 1) / a.n_splits);
    piece = (max(piece, a.piece_len) + kTokens - 1) / kTokens * kTokens;
    int before = 0;
    row = -1;
    split = n_parts = 0;
    for (int r0 = 0; r0 < a.rows; r0 += 64) {
      RowView v = {0, 0, 0, 0, false};
      if (r0 == 0) v = v0;
      else if (r0 + lane < a.rows) v = view(r0 + lane);
      const int parts = !v.owned ? 0 : v.seq <= a.whole_len ? 1 : (v.seq + piece - 1) / piece;
      const int incl = wave_inclusive_scan<ScanAdd>(parts);
      const int all = __builtin_amdgcn_readlane(incl, 63);
      if (nth < before + all) {
        const int at = __popcll(__ballot(before + incl <= nth));
        row = r0 + at;
        n_parts = __builtin_amdgcn_readlane(parts, at);
        split = nth - before - (__builtin_amdgcn_readlane(incl, at) - n_parts);
        me.req = __builtin_amdgcn_readlane(v.req, at);
        me.own = __builtin_amdgcn_readlane(v.own, at);
        me.first = __builtin_amdgcn_readlane(v.first, at);
        me.seq = __builtin_amdgcn_readlane(v.seq, at);
        break;
      }
      before += all;
    }
    if (row < 0) return;
  } else {
    // (requests side by side on the XCDs: 16 x 2048 f32 tokens 20 us, 25 the other way round; extend tokens: as above)
    if constexpr (!ROWS) {
      row = blockIdx.x % (unsigned)a.rows;
      kvh = blockIdx.x / (unsigned)a.rows % (unsigned)a.n_kv_heads;
      split = blockIdx.x / ((unsigned)a.rows * (unsigned)a.n_kv_heads);
    } else {
      kvh = blockIdx.x % (unsigned)a.n_kv_heads;
      split = blockIdx.x / (unsigned)a.n_kv_heads % (unsigned)a.n_splits;
      row = blockIdx.x / ((unsigned)a.n_kv_heads * (unsigned)a.n_splits);
    }
    me = view(row);
    if (!me.owned) return;  // (every workgroup of the row: no ticket is drawn)
    // (fused: no piece is shorter than piece_len; else the merge expects all n_splits)
    n_parts = !fused ? a.n_splits : me.seq <= a.whole_len ? 1 : min(a.n_splits, (me.seq + a.piece_len - 1) / a.piece_len);
    if (split >= n_parts) return;
  }
  const int64_t req = me.req;
  const int seq = me.seq;
  const int chunk = ((seq + n_parts - 1) / n_parts + kTokens - 1) / kTokens * kTokens;
  const int start = (int)min(split * (int64_t)chunk, (int64_t)seq), end = (int)min(start + (int64_t)chunk, (int64_t)seq);
  const int n_tiles = (end - start + kTokens - 1) / kTokens;
  const int32_t* table_row = a.kv.table + req * a.kv.table_row_stride + me.first;
  const uint32_t max_slot = (uint32_t)(a.kv.n_slots - 1);
  const int head = kvh * G + min(c, G - 1);

  // ---- this row's new token: written here, and read from where it comes from
  int new_slot = -1;
  const char *k_new = nullptr, *v_new = nullptr;
  if (a.new_loc != nullptr) {
    const int loc = a.new_loc[row];
    if (loc >= 0 && (uint32_t)loc <= max_slot) {
      new_slot = loc;
      k_new = (const char*)a.k_new + ((int64_t)row * a.k_new_stride + (int64_t)kvh * D) * E::BYTES;
      v_new = (const char*)a.v_new + ((int64_t)row * a.v_new_stride + (int64_t)kvh * D) * E::BYTES;
      if (split == 0 && tid < 2 * (ROW / 16)) {
        const int piece = tid % (ROW / 16);
        const bool is_v = tid >= ROW / 16;
        const int64_t at = ((int64_t)loc * a.kv.slab_row_stride + (int64_t)kvh * D) * E::BYTES + 16 * piece;
        *(u32x4v*)((char*)(is_v ? a.kv.v_slab : a.kv.k_slab) + at) = *(const u32x4v*)((is_v ? v_new : k_new) + 16 * piece);
      }
    }
  }

  u32x4v qf[KN];
  {
    const char* q_ptr = (const char*)a.q + ((int64_t)row * a.q_row_stride + (int64_t)head * D) * E::BYTES + 16 * u;
#pragma unroll
    for (int j = 0; j < KN; ++j) qf[j] = *(const u32x4v*)(q_ptr + 64 * j);
  }
  const ScoreShape shape(a.mods, a.scale, head);
  float* const score_dst = a.mods.scores == nullptr ? nullptr : a.mods.scores + ((int64_t)row * a.n_q_heads + head) * a.mods.score_stride + start + 4 * u;
  const float far = (float)(me.own - me.first - start);  // distance of the piece's first token

  u32x4v xk[KN];
  uint32_t xv[4][VW];
  const int64_t slab_row = a.kv.slab_row_stride * E::BYTES;
  const char* const k_lane = (const char*)a.kv.k_slab + (int64_t)kvh * ROW + 16 * u;
  const char* const v_lane = (const char*)a.kv.v_slab + (int64_t)kvh * ROW + VB * c;
  // the slot of the tile's token c (places past the end repeat the last one)
  auto entry = [&](int tile) {
    const uint32_t e = (uint32_t)table_row[min(start + tile * kTokens + c, end - 1)];
    return (int)(e > max_slot ? max_slot : e);
  };
  // (K/V of a request are read once: non-temporal, 64 x 2048 bf16 tokens of 12 / 2 heads 30.5 us from memory, 33 through the caches.  f32
  // is not: its lines come in more pieces, 62 us against 59.5; nor is what the rows of an extend share)
  auto fetch = [&](auto* p) {
    if constexpr (!F32 && !ROWS) return __builtin_nontemporal_load(p);
    else return *p;
  };
  auto load_k = [&](int slot) {
    const char* p = slot == new_slot ? k_new + 16 * u : k_lane + slot * slab_row;
#pragma unroll
    for (int j = 0; j < KN; ++j) xk[j] = fetch((const u32x4v*)(p + 64 * j));
  };
  auto load_v = [&](int slot) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int of = __shfl(slot, 4 * u + i);
      const char* p = of == new_slot ? v_new + VB * c : v_lane + of * slab_row;
      if constexpr (VB == 8) {
        const u32x2v x = fetch((const u32x2v*)p);
        xv[i][0] = x[0];
        xv[i][1] = x[1];
      } else {
#pragma unroll
        for (int n = 0; n < VB / 16; ++n) {
          const u32x4v x = fetch((const u32x4v*)(p + 16 * n));
#pragma unroll
          for (int k = 0; k < 4; ++k) xv[i][4 * n + k] = x[k];
        }
      }
    }
  };

  float m_run = kNegInf, m_sub = 0.f, l_run = 0.f;
  f32x4v o_acc[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) o_acc[n] = f32x4v{0.f, 0.f, 0.f, 0.f};

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
    if constexpr (F32) {
      // (two chains: a sum of D terms in one rounds as often as in any, but at its full size; 16 x 300 - 900 tokens, 12 / 2 heads,
      // 9.4e-7 off their 64-bit result so, 6.4e-7 in two, 4.5e-7 in four, which spill; 15.6, 15.8 and 16.0 us)
      f32x4v s2 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KN; j += 2) {
        s = score_product<Tag>(xk[j], qf[j], s);
        s2 = score_product<Tag>(xk[j + 1], qf[j + 1], s2);
      }
      s += s2;
    } else {
#pragma unroll
      for (int j = 0; j < KN; ++j) s = score_product<Tag>(xk[j], qf[j], s);
    }
    if (more) load_k(slot);
    float t_max = kNegInf;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float dist = fabsf(far - (float)(tile * kTokens + 4 * u + r));
      const float y = F32 ? shape.precise(s[r], dist) : shape.fast(s[r], dist);
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
      m_sub = m_new == kNegInf ? 0.f : m_new - kLift<Tag>;
      l_run *= alpha;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float ar = __shfl(alpha, 4 * u + r);  // (O: head 4 u + r in register r)
#pragma unroll
        for (int n = 0; n < NB; ++n) o_acc[n][r] *= ar;
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
        for (int w = 0; w < VW; ++w) xv[i][w] = i >= left ? 0u : xv[i][w];
    }
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NB; ++n) o_acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(s[i], as_f32(xv[i][n]), o_acc[n], 0, 0, 0);
    } else {
      // value n of the four tokens: half n & 1 of word n / 2 of each
      const uint32_t p01 = E::pack2(s[0], s[1]), p23 = E::pack2(s[2], s[3]);
      uint32_t q01 = 0, q23 = 0;  // bf16: what the rounding to p left over
      if constexpr (std::is_same<Tag, bf16_tag>::value) {
        q01 = E::pack2(s[0] - as_f32(p01 << 16), s[1] - as_f32(p01 & 0xffff0000u));
        q23 = E::pack2(s[2] - as_f32(p23 << 16), s[3] - as_f32(p23 & 0xffff0000u));
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const uint32_t sel = n & 1 ? 0x07060302u : 0x05040100u;
        const uint32_t v01 = __builtin_amdgcn_perm(xv[1][n / 2], xv[0][n / 2], sel), v23 = __builtin_amdgcn_perm(xv[3][n / 2], xv[2][n / 2], sel);
        if constexpr (std::is_same<Tag, bf16_tag>::value)
          o_acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, u32x4v{p01, p23, q01, q23}),
                                                             __builtin_bit_cast(bf16x8_t, u32x4v{v01, v23, v01, v23}), o_acc[n], 0, 0, 0);
        else
          o_acc[n] = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4v, u32x2v{p01, p23}), __builtin_bit_cast(f16x4v, u32x2v{v01, v23}), o_acc[n], 0, 0, 0);
      }
    }
    if (more) load_v(slot);
    slot = entry(tile + 2 * kWaves);
  }

  // ---- the four waves' results: lane (c, u) holds values c (D / 16) .. of heads 4 u .. 4 u + 3
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int n = 0; n < NB; n += 4)
      *(f32x4v*)&s_o[wave][4 * u + r][c * NB + n] = f32x4v{o_acc[n][r], o_acc[n + 1][r], o_acc[n + 2][r], o_acc[n + 3][r]};
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
  // four finished values of a head to `out`, in its type
  auto store_out = [&](int h, int c4, f32x4v o) {
    const int64_t at = (int64_t)row * a.out_row_stride + (int64_t)(kvh * G + h) * D + 4 * c4;
    if constexpr (!F32) {
      if (a.out_dtype != kF32) {
        *(u32x2v*)((uint16_t*)a.out + at) = u32x2v{E::pack2(o[0], o[1]), E::pack2(o[2], o[3])};
        return;
      }
    }
    *(f32x4v*)((float*)a.out + at) = o;
  };
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
    const float lse = l == 0.f ? kNegInf : ((m == kNegInf ? 0.f : m - kLift<Tag>) + __builtin_amdgcn_logf(l)) * kLn2;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] *= inv;
    if (direct) {
      store_out(h, c4, o);
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
        if (p0 + j >= n_parts) x[j] = f32x4v{0.f, 0.f, 0.f, 0.f};  // (0 times an infinity is none)
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = fmaf(w[j], x[j][k], o[k]);
      }
    }
    store_out(h, c4, o);
  }
  if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // (the next launch's tickets)
}

}  // namespace

bool decode_scored_supported(const DecodeArgs& a) {
  const int64_t eb = dtype_bytes(a.dtype);
  return a.scored && (a.head_dim == 64 || a.head_dim == 128) && a.n_kv_heads > 0 && a.n_kv_heads <= 65535 && a.n_q_heads % a.n_kv_heads == 0 &&
         a.n_q_heads / a.n_kv_heads <= 16 && a.kv.table_cols <= 0x7fff0000 &&
         ((uintptr_t)a.kv.k_slab | (uintptr_t)a.kv.v_slab | (uintptr_t)a.q | (uintptr_t)a.out) % 16 == 0 &&
         (a.kv.slab_row_stride * eb | a.q_row_stride * eb | a.out_row_stride * dtype_bytes(a.out_dtype)) % 16 == 0;
}

template <typename Tag>
static void launch_scored_tag(const DecodeArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)(a.balance_target > 0 ? (a.balance_target + a.rows) * a.n_kv_heads : a.rows * a.n_kv_heads * a.n_splits));
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, stream, a); };
  if (a.mods.rows != nullptr) a.head_dim == 128 ? go(decode_scored_kernel<Tag, 128, true>) : go(decode_scored_kernel<Tag, 64, true>);
  else a.head_dim == 128 ? go(decode_scored_kernel<Tag, 128, false>) : go(decode_scored_kernel<Tag, 64, false>);
}

// Per call, with a cap, K/V from memory: 64 requests of 2048 tokens, 12 / 2 heads of 128: bf16 29.8 us (135 MB; the plain decode 28.6), f32
// 60.5 (270 MB; the generic kernel 98); 128 of 2048 - 4096, 28 / 4 heads, 161 (the copy rate; the plain decode 157); 96 documents of 1 - 3363
// tokens, 28 / 4 heads, f16, 39 (143 MB); one request of 4000 tokens 10.6 (the plain decode 12.8).
hipError_t launch_decode_scored(const DecodeArgs& a_in, hipStream_t stream) {
  if (a_in.rows == 0) return hipSuccess;
  DecodeArgs a = a_in;
  a.balance_target = 0;
  a.whole_len = 0;
  a.piece_len = kTokens;
  if ((int64_t)a.rows * a.n_kv_heads * a.n_splits > 0x7fffffffll) return hipErrorInvalidValue;
  if (a.counters != nullptr && !a.uniform) {
    const int64_t units = (int64_t)a.rows * a.n_kv_heads;
    // Short rows are not cut: one piece has no merge to wait for.  131 tokens 6.2 us, in two pieces 8.1, 200 7.2 / 8.3, 300 8.1 / 8.3;
    // five turns of 3 - 41 tokens over 333 11.8 / 13.8; 500 10.9 / 8.4, f32 16 / 10, whose tiles take longer.
    // Few workgroups for a page table's width: pieces of 256 tokens (128 where that makes 256 workgroups at most: one request of 4000 tokens
    // 10.1 us, 10.6 in pieces of 256; 64 where that makes 64: one of 500 7.5 us, 8.4 in pieces of 128, 8 of 1000 10.6 / 9.5), cut without
    // looking at the other rows (1 us less than finding a piece).  Else the rows' lengths decide: pieces of one length, some 512 workgroups -- two
    // per CU (64 x 2048 tokens of 12 / 2 heads of 128: 30.5 us from memory, 32 in 1024, 37.5 in 768; heads of 64, with weights, 1024 27 us,
    // 512 30.5) --, 768 from 257 (row, kv head) pairs on (96 documents of 28 / 4 heads: 40 us, 48 in 512, 45.5 in 1024) and
    // from 512 pairs on no cut at all but of rows twice the mean (128 x 2048 - 4096, 28 / 4 heads: 161 us; 221 with pieces of the
    // mean, which cut every second row; 171 in four times as many).
    // (no request is longer than the page table is wide; a hint that is too small makes its pieces longer)
    const int64_t longest = a.len_hint > 0 && a.len_hint < a.kv.table_cols ? a.len_hint : a.kv.table_cols;
    a.whole_len = a.dtype == kF32 ? 128 : 384;
    a.piece_len = units * ((longest + 63) / 64) <= 64 ? 64 : units * ((longest + 127) / 128) <= 256 ? 128 : 256;
    const int64_t most = longest <= a.whole_len ? 1 : (longest + a.piece_len - 1) / a.piece_len;
    if (units * most <= 512) {
      if (a.n_splits > most) a.n_splits = (int32_t)most;
    } else if (a.rows <= 1024 && a.kv.table_cols <= (1 << 20)) {
      const int64_t pieces = units > 256 ? (units < 512 ? 768 : units / 2) : a.head_dim == 64 && a.dtype != kF32 ? 1024 : 512;
      a.balance_target = (int32_t)((pieces + a.n_kv_heads - 1) / a.n_kv_heads);
    } else if (a.base_splits > 0) {
      a.n_splits = a.base_splits;
    }
  }
  switch (a.dtype) {
    case kBF16: launch_scored_tag<bf16_tag>(a, stream); break;
    case kF16: launch_scored_tag<f16_tag>(a, stream); break;
    case kF32: launch_scored_tag<f32_tag>(a, stream); break;
    default: return hipErrorInvalidValue;
  }
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
  mg.owned = a.mods.rows;
  return launch_merge(mg, stream);
}

}  // namespace bsgl
