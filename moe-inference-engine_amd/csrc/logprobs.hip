// Log probabilities of given tokens, the entropy and the top alternatives of
// rows of logits (mie_token_logprobs).
//
// Mathematics: with m the row's maximum, s = sum exp(x - m) and
// e = sum exp(x - m) (x - m): log p_t = x_t - m - log s, and the entropy
// log s - e / s.
#include <math.h>

#include <algorithm>

#include "mie_common.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kMaxTop = 64;

struct LogprobsArgs {
  const char* logits;
  int64_t stride;  // elements
  int32_t rows, vocab, top;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_tokens;
};

// The order of the alternatives as one number: the value's rank among the
// floats (NaN above all, -0 as 0), then the lower index.
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  const uint32_t u = __float_as_uint(x + 0.f);
  uint32_t rank = u & 0x80000000u ? ~u : u | 0x80000000u;
  rank = x != x ? 0xfffffffeu : rank;
  return static_cast<uint64_t>(rank) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}

template <typename F>
__device__ __forceinline__ float block_reduce(float x, float* s, F f) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = f(x, __shfl_xor(x, off));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
  __syncthreads();
  x = s[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) x = f(x, s[w]);
  return x;
}

__device__ __forceinline__ uint64_t block_max(uint64_t x, uint64_t* s) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const uint64_t y = __shfl_xor(static_cast<unsigned long long>(x), off);
    x = y > x ? y : x;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
  __syncthreads();
  x = s[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) x = s[w] > x ? s[w] : x;
  return x;
}

// grid = rows.
template <typename T>
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(LogprobsArgs a) {
  __shared__ float s_f[kThreads / 64];
  __shared__ uint64_t s_k[kThreads / 64];
  const int64_t r = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.logits) + r * a.stride;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) m = fmaxf(m, mie::Mem<T>::get(x + i));
  m = block_reduce(m, s_f, [](float p, float q) { return fmaxf(p, q); });
  float s = 0.f, e = 0.f;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
    const float d = mie::Mem<T>::get(x + i) - m, w = expf(d);
    s += w;
    e += w == 0.f ? 0.f : w * d;
  }
  s = block_reduce(s, s_f, [](float p, float q) { return p + q; });
  e = block_reduce(e, s_f, [](float p, float q) { return p + q; });
  const float z = logf(s);
  if (threadIdx.x == 0) {
    if (a.logprobs) {
      const int64_t t = a.tokens[r];
      a.logprobs[r] = t >= 0 && t < a.vocab ? mie::Mem<T>::get(x + t) - m - z : NAN;
    }
    if (a.entropy) a.entropy[r] = z - e / s;
  }
  uint64_t last = ~0ull;  // above every key
  for (int j = 0; j < a.top; ++j) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const uint64_t key = key_of(mie::Mem<T>::get(x + i), i);
      best = key < last && key > best ? key : best;
    }
    last = block_max(best, s_k);
    if (threadIdx.x == 0) {
      const int i = static_cast<int>(0xffffffffu - static_cast<uint32_t>(last));
      a.top_tokens[r * a.top + j] = i;
      a.top_logprobs[r * a.top + j] = mie::Mem<T>::get(x + i) - m - z;
    }
  }
}

}  // namespace

extern "C" int64_t mie_token_logprobs_workspace(int32_t rows, int32_t vocab, int32_t top) {
  (void)rows;
  (void)vocab;
  (void)top;
  return 0;
}

extern "C" int32_t mie_token_logprobs(const void* logits, int64_t stride, int32_t rows, int32_t vocab,
                                      const int64_t* tokens, int32_t top, float* logprobs, float* entropy,
                                      float* top_logprobs, int64_t* top_tokens, void* workspace,
                                      int64_t workspace_bytes, int32_t dtype, void* stream) {
  if (dtype != MIE_DTYPE_F32 && dtype != MIE_DTYPE_BF16)
    return mie::fail(MIE_ERR_UNSUPPORTED, "mie_token_logprobs: dtype %d; float32 or bfloat16 only", dtype);
  if (rows < 0 || rows > 1 << 20 || vocab < 1 || vocab > 1 << 30 || stride < vocab)
    return mie::fail(MIE_ERR_INVALID, "mie_token_logprobs: rows=%d (at most 2^20) vocab=%d stride=%lld", rows, vocab,
                     static_cast<long long>(stride));
  if (top < 0 || top > kMaxTop || top > vocab)
    return mie::fail(MIE_ERR_INVALID, "mie_token_logprobs: top %d outside [0, min(vocab, %d)]", top, kMaxTop);
  if (rows == 0) return MIE_OK;
  if (!logits || (logprobs && !tokens) || (top > 0 && (!top_logprobs || !top_tokens)))
    return mie::fail(MIE_ERR_INVALID, "mie_token_logprobs: null pointer");
  const int64_t need = mie_token_logprobs_workspace(rows, vocab, top);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return mie::fail(MIE_ERR_WORKSPACE, "mie_token_logprobs: workspace of %lld bytes, %lld needed",
                     static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  const LogprobsArgs a{static_cast<const char*>(logits), stride, rows, vocab, top, tokens, logprobs, entropy,
                       top_logprobs, top_tokens};
  mie::clear_error();
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MIE_DTYPE_F32)
    token_logprobs_kernel<float><<<rows, kThreads, 0, st>>>(a);
  else
    token_logprobs_kernel<uint16_t><<<rows, kThreads, 0, st>>>(a);
  return mie::check_launch("mie_token_logprobs");
}
