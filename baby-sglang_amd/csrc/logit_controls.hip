// Penalties, biases and token masks on a step's logits, one launch:
//   x = logits[b, t]
//   t among the request's tokens so far:   x = x > 0 ? x / repetition[b] : x * repetition[b]
//   t among those it has produced, n times: x -= frequency[b] * n + presence[b]
//   x += the biases of t
//   x = -inf where the request's token mask has no bit t
//
// Bound by the logits' bytes.  A workgroup owns kChunk consecutive tokens of one request.  It asks for its logits
// and mask words first, then walks the request's token list (which comes from L2: every workgroup of the request reads
// it) and counts the ones inside its chunk in LDS -- integer adds, so the order in which lanes arrive changes nothing --
// and finishes the logits from registers.  So neither a dense count table [requests, vocabulary] nor a second
// pass over the logits exists.  To keep the finish short, which nearly every wave runs for some marked token, the biases
// of a token are summed up before; a marked token carries the number of one of its entries.  (Where a token stands in
// several, each of them walks the request's biases in their order for the sum.  Without the test for that the walk was
// most of a launch: 300 biases, 64 x 151936 f32, 42 us against 20.  A penalty divides: multiplied by 1 / repetition, which is
// rounded once more and infinite for the smallest ones, 1 x 151936 bf16 took 4.9 us for 5.4 and 64 x 151936 f32 20.2 for 20.6.)
#include "bsgl_device.h"
#include "bsgl_launch.h"

namespace bsgl {

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;  // tokens per workgroup
// the mark of a token: how often it was produced, the number of a bias entry, and two flags
constexpr int kCountBits = 18;
constexpr uint32_t kCount = (1u << kCountBits) - 1;
constexpr uint32_t kEntry = kLogitMaxBias - 1;
constexpr uint32_t kBiased = 1u << 30;
constexpr uint32_t kPrompt = 1u << 31;  // seen in the prompt part
static_assert(kCount == kLogitMaxHistory && kCountBits + 12 == 30 && kLogitMaxBias == 1 << 12, "the fields fit");

template <typename Tag> struct Logit;
template <> struct Logit<bf16_tag> {
  typedef uint16_t type;
  __device__ static __forceinline__ float to_f32(uint16_t v) { return as_f32((uint32_t)v << 16); }
};
template <> struct Logit<f16_tag> {
  typedef uint16_t type;
  __device__ static __forceinline__ float to_f32(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
};
template <> struct Logit<f32_tag> {
  typedef uint32_t type;
  __device__ static __forceinline__ float to_f32(uint32_t v) { return as_f32(v); }
};

template <typename Tag, bool VECTORS>
__global__ __launch_bounds__(kThreads) void logit_controls_kernel(LogitArgs a) {
  using E = Elem<Tag>;
  using T = typename Logit<Tag>::type;
  constexpr int VEC = VECTORS ? E::VEC : 1;
  constexpr int PER = VECTORS ? kChunk / kThreads / VEC : 1;  // pieces per lane
  extern __shared__ uint32_t smem[];
  uint32_t* s_mark = smem;                     // [kChunk]
  int32_t* s_ids = (int32_t*)(smem + kChunk);  // [n_bias]
  float* s_vals = (float*)(s_ids + a.n_bias);  // [n_bias] the biases
  float* s_sums = s_vals + a.n_bias;           // [n_bias] the sum of all biases of an entry's token
  __shared__ int s_twice;                      // a token stands in several entries
  const int tid = threadIdx.x;
  const int row = blockIdx.y;
  const int v0 = blockIdx.x * kChunk;
  const int n = min(kChunk, a.vocab - v0);
  const T* src = (const T*)a.logits + (int64_t)row * a.logits_row_stride + v0;
  T* dst = (T*)a.out + (int64_t)row * a.out_row_stride + v0;
  const bool marks = a.history != nullptr || a.bias_ids != nullptr;

  // ---- everything whose address is known, in one trip ---------------------------------------------------
  float rep = 1.f, pres = 0.f, freq = 0.f;
  int64_t h = row, l64 = 0, p64 = 0, mr = row;
  if (a.history != nullptr) {
    if (a.history_rows != nullptr) h = a.history_rows[row];
    l64 = a.history_lens[row];
    if (a.prompt_lens != nullptr) p64 = a.prompt_lens[row];
    if (a.repetition != nullptr) rep = a.repetition[row];
    if (a.presence != nullptr) pres = a.presence[row];
    if (a.frequency != nullptr) freq = a.frequency[row];
  }
  if (a.token_mask != nullptr && a.mask_rows != nullptr) mr = a.mask_rows[row];
  uint4 raw[PER];
  if constexpr (VECTORS) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = (p * kThreads + tid) * VEC;
      if (at < n) raw[p] = *(const uint4*)(src + at);  // (the vocabulary is whole vectors here)
    }
  }
  const uint32_t* mask = nullptr;
  if (a.token_mask != nullptr && mr >= 0 && mr < a.mask_n_rows) mask = (const uint32_t*)a.token_mask + mr * a.mask_row_stride;
  uint32_t word[PER];
#pragma unroll
  for (int p = 0; p < PER; ++p) word[p] = 0xffffffffu;
  if (VECTORS && mask != nullptr) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = (p * kThreads + tid) * VEC;
      if (at < n) word[p] = mask[(v0 + at) >> 5] >> (at & 31);  // (VEC tokens of one word)
    }
  }

  // ---- marks ---------------------------------------------------------------------------------------------
  if (marks) {
#pragma unroll
    for (int i = 0; i < kChunk / kThreads / 4; ++i) ((uint4*)s_mark)[i * kThreads + tid] = make_uint4(0, 0, 0, 0);
    if (tid == 0) s_twice = 0;
    for (int i = tid; i < a.n_bias; i += kThreads) {
      s_ids[i] = a.bias_ids[(int64_t)row * a.bias_row_stride + i];
      s_vals[i] = a.bias_values[(int64_t)row * a.bias_row_stride + i];
    }
    __syncthreads();
    if (a.history != nullptr) {
      const int32_t* ids = a.history + (h < 0 ? 0 : (h >= a.history_n_rows ? a.history_n_rows - 1 : h)) * a.history_row_stride;
      const int len = (int)(l64 < 0 ? 0 : (l64 > a.history_cols ? a.history_cols : l64));
      const int prompt = (int)(p64 < 0 ? 0 : (p64 > len ? len : p64));
      auto count = [&](int32_t id, int at) {
        const uint32_t t = (uint32_t)id - (uint32_t)v0;
        if (t >= (uint32_t)n) return;  // (a negative id wraps past every chunk)
        if (at < prompt) atomicOr(&s_mark[t], kPrompt);
        else atomicAdd(&s_mark[t], 1u);
      };
      if (((uintptr_t)ids & 15) == 0) {
        const int whole = len & ~3;
        for (int i = tid * 4; i < whole; i += kThreads * 16) {
          // (four trips' loads together)
          int4 x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = i + k * kThreads * 4 < whole ? *(const int4*)(ids + i + k * kThreads * 4) : make_int4(-1, -1, -1, -1);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int at = i + k * kThreads * 4;
            count(x[k].x, at);
            count(x[k].y, at + 1);
            count(x[k].z, at + 2);
            count(x[k].w, at + 3);
          }
        }
        if (tid < len - whole) count(ids[whole + tid], whole + tid);
      } else {
        for (int i = tid; i < len; i += kThreads) count(ids[i], i);
      }
    }
    for (int i = tid; i < a.n_bias; i += kThreads) {
      const uint32_t t = (uint32_t)s_ids[i] - (uint32_t)v0;
      if (t >= (uint32_t)n) continue;
      s_sums[i] = s_vals[i];
      if ((atomicOr(&s_mark[t], kBiased) & kBiased) == 0) atomicAdd(&s_mark[t], (uint32_t)i << kCountBits);
      else s_twice = 1;
    }
    __syncthreads();
    if (a.n_bias > 0 && s_twice != 0) {
      for (int i = tid; i < a.n_bias; i += kThreads) {
        const int32_t id = s_ids[i];
        if ((uint32_t)id - (uint32_t)v0 >= (uint32_t)n) continue;
        // (every entry of a token comes to the same sum, in the same order: it does not matter whose number the token got)
        float sum = 0.f;
#pragma unroll 8
        for (int b = 0; b < a.n_bias; ++b) {
          const float v = s_vals[b];
          sum += s_ids[b] == id ? v : 0.f;
        }
        s_sums[i] = sum;
      }
      __syncthreads();
    }
  }

  // ---- finish --------------------------------------------------------------------------------------------
  auto finish = [&](float x, uint32_t c) {
    const uint32_t made = c & kCount;
    if (c & (kPrompt | kCount)) x = x > 0.f ? x / rep : x * rep;
    if (made != 0) x = (x - freq * (float)made) - pres;  // (only then: an infinite penalty times 0 is NaN)
    if (c & kBiased) x += s_sums[(c >> kCountBits) & kEntry];
    return x;
  };
  if constexpr (VECTORS) {
    constexpr uint32_t kAll = (1u << VEC) - 1;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = (p * kThreads + tid) * VEC;
      if (at >= n) continue;
      uint32_t c[VEC], any = 0;
#pragma unroll
      for (int k = 0; k < VEC; ++k) c[k] = 0;
      if (marks) {
#pragma unroll
        for (int k = 0; k < VEC; k += 4) {
          const uint4 m = *(const uint4*)(s_mark + at + k);
          c[k] = m.x;
          c[k + 1] = m.y;
          c[k + 2] = m.z;
          c[k + 3] = m.w;
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) any |= c[k];
      }
      if (any != 0 || (word[p] & kAll) != kAll) {
        float f[VEC];
        E::unpack(raw[p], f);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          if (c[k] != 0) f[k] = finish(f[k], c[k]);
          f[k] = (word[p] >> k) & 1u ? f[k] : kNegInf;
        }
        raw[p] = E::pack(f);
      }
      *(uint4*)(dst + at) = raw[p];
    }
  } else {
    for (int at = tid; at < n; at += kThreads) {
      const bool allowed = mask == nullptr || (mask[(v0 + at) >> 5] >> (at & 31)) & 1u;
      const uint32_t c = marks ? s_mark[at] : 0u;
      T v = src[at];
      if (c != 0 || !allowed) {
        const float x = allowed ? finish(Logit<Tag>::to_f32(v), c) : kNegInf;
        if constexpr (E::BYTES == 4) v = as_u32(x);
        else v = (T)E::pack2(x, 0.f);
      }
      dst[at] = v;
    }
  }
}

template <typename Tag>
hipError_t launch_tag(const LogitArgs& a, hipStream_t stream) {
  using E = Elem<Tag>;
  const dim3 grid((unsigned)((a.vocab + kChunk - 1) / kChunk), (unsigned)a.batch);
  size_t lds = 0;
  if (a.history != nullptr || a.bias_ids != nullptr) lds = kChunk * 4 + (size_t)a.n_bias * 12;
  // 16-byte pieces where every row of both tensors starts on 16 bytes and ends on a whole piece
  const bool vectors = ((uintptr_t)a.logits | (uintptr_t)a.out) % 16 == 0 && a.logits_row_stride * E::BYTES % 16 == 0 &&
                       a.out_row_stride * E::BYTES % 16 == 0 && a.vocab % E::VEC == 0;
  if (vectors) hipLaunchKernelGGL((logit_controls_kernel<Tag, true>), grid, dim3(kThreads), lds, stream, a);
  else hipLaunchKernelGGL((logit_controls_kernel<Tag, false>), grid, dim3(kThreads), lds, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_logit_controls(const LogitArgs& a, hipStream_t stream) {
  if (a.batch == 0 || a.vocab == 0) return hipSuccess;
  switch (a.dtype) {
    case kBF16: return launch_tag<bf16_tag>(a, stream);
    case kF16: return launch_tag<f16_tag>(a, stream);
    case kF32: return launch_tag<f32_tag>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace bsgl
