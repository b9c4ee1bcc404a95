// Penalties, biases and token masks on a step's logits, one launch:
//   x = logits[b, t]
//   t among the request's tokens so far:   x = x > 0 ? x / repetition[b] : x * repetition[b]
//   t among those it has produced, n times: x -= frequency[b] * n + presence[b]
//   x += the biases of t
//   x = -inf where the request's token mask has no bit t
//
// Bound by the logits' bytes.  A workgroup owns kChunk consecutive tokens of one request: it asks for its logits
// first, then walks the request's token list (which comes from L2: every workgroup of the request reads it) and counts the
// ones inside its chunk in LDS -- integer adds, so the order in which lanes arrive changes nothing -- and
// then finishes the logits from registers.  So neither a dense count table [requests, vocabulary] nor a second
// pass over the logits exists.
#include "bsgl_device.h"
#include "bsgl_launch.h"

namespace bsgl {

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;            // tokens per workgroup
constexpr uint32_t kPrompt = 1u << 31;  // seen in the prompt part; the bits below count the produced ones

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
  constexpr int PER = kChunk / kThreads / VEC;  // pieces per lane
  extern __shared__ uint32_t smem[];
  uint32_t* s_count = smem;                                   // [kChunk], with a history
  float* s_bias = (float*)(smem + (a.history ? kChunk : 0));  // [kChunk], with biases
  int32_t* s_ids = (int32_t*)(s_bias + kChunk);               // [kThreads]
  float* s_vals = (float*)(s_ids + kThreads);                 // [kThreads]
  const int tid = threadIdx.x;
  const int row = blockIdx.y;
  const int v0 = blockIdx.x * kChunk;
  const int n = min(kChunk, a.vocab - v0);
  const T* src = (const T*)a.logits + (int64_t)row * a.logits_row_stride + v0;
  T* dst = (T*)a.out + (int64_t)row * a.out_row_stride + v0;

  uint4 raw[VECTORS ? PER : 1];
  if constexpr (VECTORS) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = (p * kThreads + tid) * VEC;
      if (at < n) raw[p] = *(const uint4*)(src + at);  // (the vocabulary is whole vectors here)
    }
  }

  float rep = 1.f, pres = 0.f, freq = 0.f;
  if (a.history != nullptr) {
    for (int i = tid; i < kChunk; i += kThreads) s_count[i] = 0;
    const int64_t h64 = a.history_rows != nullptr ? a.history_rows[row] : row;
    const int64_t h = h64 < 0 ? 0 : (h64 >= a.history_n_rows ? a.history_n_rows - 1 : h64);
    const int64_t l64 = a.history_lens[row];
    const int len = (int)(l64 < 0 ? 0 : (l64 > a.history_cols ? a.history_cols : l64));
    const int64_t p64 = a.prompt_lens != nullptr ? a.prompt_lens[row] : 0;
    const int prompt = (int)(p64 < 0 ? 0 : (p64 > len ? len : p64));
    if (a.repetition != nullptr) rep = a.repetition[row];
    if (a.presence != nullptr) pres = a.presence[row];
    if (a.frequency != nullptr) freq = a.frequency[row];
    const int32_t* ids = a.history + h * a.history_row_stride;
    __syncthreads();
    auto count = [&](int32_t id, int at) {
      const uint32_t t = (uint32_t)(id - v0);
      if (id < 0 || t >= (uint32_t)n) return;
      if (at < prompt) atomicOr(&s_count[t], kPrompt);
      else atomicAdd(&s_count[t], 1u);
    };
    if (((uintptr_t)ids & 15) == 0) {
      for (int i = tid * 4; i < len; i += kThreads * 4) {
        if (i + 3 < len) {
          const int4 x = *(const int4*)(ids + i);
          count(x.x, i);
          count(x.y, i + 1);
          count(x.z, i + 2);
          count(x.w, i + 3);
        } else {
          for (int k = i; k < len; ++k) count(ids[k], k);
        }
      }
    } else {
      for (int i = tid; i < len; i += kThreads) count(ids[i], i);
    }
  }
  if (a.bias_ids != nullptr) {
    for (int i = tid; i < kChunk; i += kThreads) s_bias[i] = 0.f;
    // kThreads entries at a time; an id that stands there several times is summed by its first entry, in order, so the
    // result does not depend on which lane comes first
    for (int k0 = 0; k0 < a.n_bias; k0 += kThreads) {
      __syncthreads();
      const bool have = k0 + tid < a.n_bias;
      const int32_t id = have ? a.bias_ids[(int64_t)row * a.bias_row_stride + k0 + tid] : -1;
      s_ids[tid] = id;
      s_vals[tid] = have ? a.bias_values[(int64_t)row * a.bias_row_stride + k0 + tid] : 0.f;
      __syncthreads();
      if (id >= v0 && id < v0 + n) {
        bool owner = true;
        float sum = 0.f;
        const int m = min(kThreads, a.n_bias - k0);
        for (int j = 0; j < m; ++j) {
          if (s_ids[j] != id) continue;
          owner &= j >= tid;
          sum += s_vals[j];
        }
        if (owner) s_bias[id - v0] += sum;
      }
    }
  }
  const uint32_t* mask = nullptr;
  if (a.token_mask != nullptr) {
    const int64_t mr = a.mask_rows != nullptr ? a.mask_rows[row] : row;
    if (mr >= 0 && mr < a.mask_n_rows) mask = (const uint32_t*)a.token_mask + mr * a.mask_row_stride;
  }
  if (a.history != nullptr || a.bias_ids != nullptr) __syncthreads();

  auto finish = [&](float x, int at, uint32_t word) {
    if (a.history != nullptr) {
      const uint32_t c = s_count[at];
      if (c != 0) {
        x = x > 0.f ? x / rep : x * rep;
        const uint32_t made = c & ~kPrompt;
        x -= freq * (float)made;
        if (made != 0) x -= pres;
      }
    }
    if (a.bias_ids != nullptr) x += s_bias[at];
    return (word >> ((v0 + at) & 31)) & 1u ? x : kNegInf;
  };
  if constexpr (VECTORS) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = (p * kThreads + tid) * VEC;
      if (at >= n) continue;
      const uint32_t word = mask != nullptr ? mask[(v0 + at) >> 5] : 0xffffffffu;  // (VEC tokens of one word)
      float f[VEC];
      E::unpack(raw[p], f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = finish(f[k], at + k, word);
      *(uint4*)(dst + at) = E::pack(f);
    }
  } else {
    for (int at = tid; at < n; at += kThreads) {
      const uint32_t word = mask != nullptr ? mask[(v0 + at) >> 5] : 0xffffffffu;
      const float x = finish(Logit<Tag>::to_f32(src[at]), at, word);
      if constexpr (E::BYTES == 4) dst[at] = as_u32(x);
      else dst[at] = (T)E::pack2(x, 0.f);
    }
  }
}

template <typename Tag>
hipError_t launch_tag(const LogitArgs& a, hipStream_t stream) {
  using E = Elem<Tag>;
  const dim3 grid((unsigned)((a.vocab + kChunk - 1) / kChunk), (unsigned)a.batch);
  size_t lds = 0;
  if (a.history != nullptr) lds += kChunk * 4;
  if (a.bias_ids != nullptr) lds += kChunk * 4 + kThreads * 8;
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
