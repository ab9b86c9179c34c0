// Log probabilities of given tokens, the entropy and the top alternatives of
// rows of logits (mie_token_logprobs).
//
// Mathematics: with m a reference near the row's maximum, s = sum exp(x - m)
// and e = sum exp(x - m) (x - m): log p_t = x_t - m - log s, and the entropy
// log s - e / s.  Sums over parts of a row are shifted to one reference
// when they are joined.
//
// One pass over the logits (bound by reading them).  A workgroup takes a row,
// or one of several slices of it where the rows alone do not fill the GPU (a
// second launch joins them).  Each thread keeps its own reference, raised only
// when a value exceeds it by 10, and four sums of each kind.
//
// Alternatives.  A row's `top` best keys (value, then the lower index) are
// found in the same pass.  A wave keeps a bound that at least `top` of its
// values so far reach: what the top-th largest of its lanes' maxima is (each
// lane has one for each of the vectors it loads at a time), found bit by bit
// with ballots and left at 16 bits, from the first chunk (64 lanes x 16
// values) and again after the 2nd, 4th, 8th, ...  The few values above it
// go to a list in LDS; a list that fills up is cut to its `top` best, which
// raises the bound too.  A wave's values come in the order of their indices,
// so one equal to a bound that earlier values set is never among the best.  In
// the end the lists of the four waves are ranked by counting.
//
// On MI355X, float32: 1000 rows of 50257 40 us with the top 5 (5.0 TB/s, the rate
// of a copy), 57 with 20, 115 with 64; 64 rows 13 us; one row 11 us, two
// launches.
//
// A row with a NaN or +inf has no finite result: only the order of its
// alternatives is left, which is found by one pass for each.
#include <float.h>
#include <math.h>

#include <algorithm>

#include "mie_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 64;
constexpr int kCap = 1024;     // keys of a wave's list
constexpr int kRanked = 128;   // the most of them that are ranked
constexpr float kRaise = 10.f;
constexpr float kLog2e = 1.4426950408889634f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct LogprobsArgs {
  const char* logits;
  int64_t stride;  // elements
  int32_t rows, vocab, top, slices;
  const int64_t* tokens;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_tokens;
  // Slices > 1, for each (row, slice): its best keys and (m, s, e, unused).
  uint64_t* ws_keys;
  f32x4* ws_sums;
};

// The order of the alternatives as one number: the value's rank among the
// floats (NaN above all, -0 as 0), then the lower index.
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  const uint32_t u = __float_as_uint(x + 0.f);
  uint32_t rank = u & 0x80000000u ? ~u : u | 0x80000000u;
  rank = x != x ? 0xfffffffeu : rank;
  return static_cast<uint64_t>(rank) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ int index_of(uint64_t key) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t rank = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(rank & 0x80000000u ? rank & 0x7fffffffu : ~rank);
}

__device__ __forceinline__ uint64_t wave_max(uint64_t x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const uint64_t y = __shfl_xor(static_cast<unsigned long long>(x), off);
    x = y > x ? y : x;
  }
  return x;
}

// s = sum exp(x - m), e = sum exp(x - m) (x - m).
struct Sums {
  float m, s, e;
};
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  auto shift = [&](Sums& x) {
    const float d = x.m - m, f = mie::fast_exp2(d * kLog2e);
    // What is out of reach is dropped: sums of float32's lowest values would
    // overflow on the way to 0.
    x.e = f == 0.f ? 0.f : (x.e + x.s * d) * f;
    x.s = f == 0.f ? 0.f : x.s * f;
  };
  shift(a);
  shift(b);
  return Sums{m, a.s + b.s, a.e + b.e};
}
__device__ __forceinline__ Sums block_join(Sums x) {
  __shared__ Sums s_part[kWaves];
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = join(x, Sums{__shfl_xor(x.m, off), __shfl_xor(x.s, off), __shfl_xor(x.e, off)});
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = x;
  __syncthreads();
  x = s_part[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) x = join(x, s_part[w]);
  return x;
}

// A wave's list of keys: `count` of them, and the bound.
struct List {
  uint64_t* keys;  // LDS
  int count;
  float bound;
};

// A value that at least k of the lanes' values reach (k <= 64): the k-th
// largest, down to 16 bits of its rank.
template <int N>
__device__ __forceinline__ float reached_by(const float (&x)[N], int k) {
  uint32_t rank[N], bound = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t u = __float_as_uint(x[j]);
    rank[j] = u & 0x80000000u ? ~u : u | 0x80000000u;
  }
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t higher = bound | 1u << bit;
    int reach = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) reach += __popcll(__ballot(rank[j] >= higher));
    if (reach >= k) bound = higher;
  }
  // Below the smallest rank of a number every value reaches -inf.
  return bound < 0x00800000u ? -INFINITY : __uint_as_float(bound & 0x80000000u ? bound & 0x7fffffffu : ~bound);
}

// Cuts `count` keys to the `top` best, best first; the last one's value, or
// -inf where there are fewer.  Apart from the kernels, whose registers it
// would take: everything goes in and out by value.
__device__ __attribute__((noinline)) float best_of(__attribute__((address_space(3))) uint64_t* keys, int count,
                                                   int top) {
  const int lane = threadIdx.x & 63;
  uint64_t mine[kCap / 64];
#pragma unroll
  for (int j = 0; j < kCap / 64; ++j) mine[j] = j * 64 + lane < count ? keys[j * 64 + lane] : 0;
  uint64_t last = ~0ull;
  for (int k = 0; k < min(count, top); ++k) {
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < kCap / 64; ++j) best = mine[j] < last && mine[j] > best ? mine[j] : best;
    last = wave_max(best);
    if (lane == 0) keys[k] = last;
  }
  return count < top ? -INFINITY : value_of(last);
}
__device__ __forceinline__ void cut(List& list, int top) {
  const float bound = best_of((__attribute__((address_space(3))) uint64_t*)list.keys, list.count, top);
  list.count = __builtin_amdgcn_readfirstlane(min(list.count, top));
  list.bound = fmaxf(list.bound, bound);
}

// Adds the lanes' keys for which `want` holds; there is room.
__device__ __forceinline__ void push(List& list, float x, int index, bool want) {
  const uint64_t who = __ballot(want);
  if (who == 0) return;
  const int lane = threadIdx.x & 63;
  if (want) list.keys[list.count + __popcll(who & ((1ull << lane) - 1))] = key_of(x, index);
  list.count += __popcll(who);
}

template <typename T> struct Chunk;
template <> struct Chunk<float> {
  static constexpr int VEC = 4, U = 4;
  u32x4 v[U];
  __device__ __forceinline__ float get(int u, int j) const { return __uint_as_float(v[u][j]); }
  static constexpr uint32_t kLowest = 0xff800000u;  // -inf
};
template <> struct Chunk<uint16_t> {
  static constexpr int VEC = 8, U = 2;
  u32x4 v[U];
  __device__ __forceinline__ float get(int u, int j) const {
    return j % 2 ? mie::bf16_hi(v[u][j / 2]) : mie::bf16_lo(v[u][j / 2]);
  }
  static constexpr uint32_t kLowest = 0xff80ff80u;
};

// What is left to do once a row's sums and keys are known: `n` keys in LDS, in
// any order and all different.
__device__ __forceinline__ void finish(const LogprobsArgs& a, int64_t row, Sums sums, float target,
                                       const uint64_t* keys, int n) {
  const float z = logf(sums.s);
  if (threadIdx.x == 0) {
    if (a.logprobs) a.logprobs[row] = target - sums.m - z;
    if (a.entropy) a.entropy[row] = z - sums.e / sums.s;
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t key = keys[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += keys[j] > key;
    if (above < a.top) {
      a.top_tokens[row * a.top + above] = index_of(key);
      a.top_logprobs[row * a.top + above] = value_of(key) - sums.m - z;
    }
  }
}

// A row without finite results: NaN, and the alternatives one after the other.
template <typename T>
__device__ __attribute__((noinline)) void finish_not_finite(LogprobsArgs a, int64_t row) {
  __shared__ uint64_t s_best[kWaves];
  const T* x = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  if (threadIdx.x == 0) {
    if (a.logprobs) a.logprobs[row] = NAN;
    if (a.entropy) a.entropy[row] = NAN;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const uint64_t key = key_of(mie::Mem<T>::get(x + i), i);
      best = key < last && key > best ? key : best;
    }
    best = wave_max(best);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_best[threadIdx.x >> 6] = best;
    __syncthreads();
    last = s_best[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) last = s_best[w] > last ? s_best[w] : last;
    if (threadIdx.x == 0) {
      a.top_tokens[row * a.top + k] = index_of(last);
      a.top_logprobs[row * a.top + k] = NAN;
    }
  }
}

// The row's value at its token, NaN for a token outside the vocabulary.
template <typename T>
__device__ __forceinline__ float target_of(const LogprobsArgs& a, int64_t row) {
  if (!a.logprobs) return NAN;
  const int64_t t = a.tokens[row];
  return t < 0 || t >= a.vocab ? NAN
                               : mie::Mem<T>::get(reinterpret_cast<const T*>(a.logits) + row * a.stride + t);
}

// grid = rows x slices, a row's slices side by side.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads, 4) void token_logprobs_kernel(LogprobsArgs a) {
  using C = Chunk<T>;
  constexpr int VEC = C::VEC, U = C::U;
  __shared__ uint64_t s_keys[TOP ? kWaves * kCap : 1];
  __shared__ int s_count[kWaves];
  const int64_t row = static_cast<int>(blockIdx.x) / a.slices;
  const int slice = static_cast<int>(blockIdx.x) % a.slices;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T* x = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  const float target = target_of<T>(a, row);

  // 16-byte vectors from the first aligned value on; slice s takes the s-th
  // share of them, the first also the values before and behind.
  const int head = min(a.vocab, static_cast<int>((0 - reinterpret_cast<uintptr_t>(x)) % 16 / sizeof(T)));
  const int vectors = (a.vocab - head) / VEC, tail = a.vocab - head - vectors * VEC;
  const int share = (vectors + a.slices - 1) / a.slices;
  const int first = min(slice * share, vectors), last = min(first + share, vectors);
  const u32x4* xv = reinterpret_cast<const u32x4*>(x + head);

  List list{s_keys + wave * kCap, 0, -INFINITY};
  float m = -FLT_MAX, s[4] = {0.f, 0.f, 0.f, 0.f}, e[4] = {0.f, 0.f, 0.f, 0.f};
  auto raise = [&](float top) {
    if (__any(top > m + kRaise)) {
      const float to = fmaxf(top, m), d = m - to, f = mie::fast_exp2(d * kLog2e);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e[j] = f == 0.f ? 0.f : (e[j] + s[j] * d) * f;  // as in join
        s[j] = f == 0.f ? 0.f : s[j] * f;
      }
      m = to;
    }
  };
  auto add = [&](float v, int j) {
    const float d = v - m, w = mie::fast_exp2(d * kLog2e);
    s[j] += w;
    e[j] = fmaf(w, fmaxf(d, -FLT_MAX), e[j]);  // 0 for -inf
  };
  // One value of each of the first n threads, in the wave's order of indices.
  auto edge = [&](int from, int n) {
    const bool have = static_cast<int>(threadIdx.x) < n;
    const float v = have ? mie::Mem<T>::get(x + from + threadIdx.x) : -INFINITY;
    raise(v);
    add(v, 0);
    if constexpr (TOP) {
      if (list.count + 64 > kCap) cut(list, a.top);
      push(list, v, from + threadIdx.x, have && (v > list.bound || list.count < a.top));
    }
  };
  if (slice == 0 && wave == 0 && head > 0) edge(0, head);

  auto load = [&](C& chunk, int c) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = c + u * kThreads + threadIdx.x;
      chunk.v[u] = __builtin_nontemporal_load(xv + min(i, last - 1));
    }
  };
  C chunk, next;
  float lane_most[U];
#pragma unroll
  for (int u = 0; u < U; ++u) lane_most[u] = -INFINITY;
  if (first < last) load(chunk, first);
  for (int c = first, n = 1; c < last; c += U * kThreads, ++n, chunk = next) {
    load(next, c + U * kThreads);
    // What was loaded past the end counts as -inf; looked at here, where the
    // loads of the next chunk are under way.
    if (c + U * kThreads > last) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * kThreads + static_cast<int>(threadIdx.x) >= last)
          chunk.v[u] = u32x4{C::kLowest, C::kLowest, C::kLowest, C::kLowest};
    }
    float top[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      top[u] = chunk.get(u, 0);
#pragma unroll
      for (int j = 1; j < VEC; ++j) top[u] = fmaxf(top[u], chunk.get(u, j));
    }
    float most = top[0];
#pragma unroll
    for (int u = 1; u < U; ++u) most = fmaxf(most, top[u]);
    raise(most);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) add(chunk.get(u, j), j % 4);
    if constexpr (TOP) {
      // Values equal to the bound are taken where this chunk raised it.
      bool start = c == first;
#pragma unroll
      for (int u = 0; u < U; ++u) lane_most[u] = fmaxf(lane_most[u], top[u]);
      if ((n & (n - 1)) == 0) {
        // One maximum a lane is a cheap and close bound for few alternatives
        // (1000 x 50257: top 5 37.8 us, 39.1 with four each), not for as many
        // as there are lanes (top 64: 170 us, 115).
        float bound;
        if (a.top <= 32) {
          float one[1] = {lane_most[0]};
#pragma unroll
          for (int u = 1; u < U; ++u) one[0] = fmaxf(one[0], lane_most[u]);
          bound = reached_by(one, a.top);
        } else {
          bound = reached_by(lane_most, a.top);
        }
        start |= bound > list.bound;
        list.bound = fmaxf(list.bound, bound);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!__any(start ? top[u] >= list.bound : top[u] > list.bound)) continue;
        if (list.count + 64 * VEC > kCap) cut(list, a.top);
        const int i = c + u * kThreads + threadIdx.x;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float v = chunk.get(u, j);
          push(list, v, head + i * VEC + j, i < last && (start ? v >= list.bound : v > list.bound));
        }
      }
    }
  }
  if (slice == 0 && wave == 0 && tail > 0) edge(head + vectors * VEC, tail);

  Sums sums{m, s[0], e[0]};
#pragma unroll
  for (int j = 1; j < 4; ++j) {
    sums.s += s[j];
    sums.e += e[j];
  }
  sums = block_join(sums);
  int n = 0;
  if constexpr (TOP) {
    if (list.count > kRanked) cut(list, a.top);
    if (lane == 0) s_count[wave] = list.count;
    __syncthreads();
    // The lists, one behind the other at the front.
    uint64_t mine[kRanked / 64];
    int at = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      at += w < wave ? s_count[w] : 0;
      n += s_count[w];
    }
#pragma unroll
    for (int j = 0; j < kRanked / 64; ++j)
      if (j * 64 + lane < list.count) mine[j] = list.keys[j * 64 + lane];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kRanked / 64; ++j)
      if (j * 64 + lane < list.count) s_keys[at + j * 64 + lane] = mine[j];
    __syncthreads();
  }
  if (a.slices == 1) {
    if (sums.s != sums.s)
      finish_not_finite<T>(a, row);
    else
      finish(a, row, sums, target, s_keys, n);
    return;
  }
  const int64_t piece = row * a.slices + slice;
  if (threadIdx.x == 0) a.ws_sums[piece] = f32x4{sums.m, sums.s, sums.e, 0.f};
  if constexpr (TOP) {
    for (int i = threadIdx.x; i < a.top; i += kThreads)
      if (i >= n) a.ws_keys[piece * a.top + i] = 0;  // a slice with fewer values
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t key = s_keys[i];
      int above = 0;
      for (int j = 0; j < n; ++j) above += s_keys[j] > key;
      if (above < a.top) a.ws_keys[piece * a.top + above] = key;
    }
  }
}

// grid = rows: joins a row's slices.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_slices_kernel(LogprobsArgs a) {
  __shared__ uint64_t s_keys[kWaves * kCap];
  const int64_t row = blockIdx.x;
  const float target = target_of<T>(a, row);
  const int total = a.slices * a.top;
  Sums sums{-FLT_MAX, 0.f, 0.f};
  for (int i = threadIdx.x; i < a.slices; i += kThreads) {
    const f32x4 p = a.ws_sums[row * a.slices + i];
    sums = join(sums, Sums{p.x, p.y, p.z});
  }
  for (int i = threadIdx.x; i < total; i += kThreads) s_keys[i] = a.ws_keys[row * total + i];
  sums = block_join(sums);  // a barrier: the keys are there
  if (sums.s != sums.s) {
    finish_not_finite<T>(a, row);
    return;
  }
  // Keys of 0, the places a short slice left, are below the others, of which
  // there are `top` at least.
  finish(a, row, sums, target, s_keys, total);
}

// Slices of a row: as many as make 512 workgroups with the rows, of 4096 values at least.
int slices_for(int rows, int vocab, int top) {
  const int want = std::max(1, 512 / std::max(rows, 1)), most = std::max(1, vocab / 4096);
  return std::min({want, most, 64, std::max(1, 512 / std::max(top, 1))});
}

template <typename T>
void launch(const LogprobsArgs& a, hipStream_t st) {
  const int grid = a.rows * a.slices;
  if (a.top > 0)
    token_logprobs_kernel<T, true><<<grid, kThreads, 0, st>>>(a);
  else
    token_logprobs_kernel<T, false><<<grid, kThreads, 0, st>>>(a);
  if (a.slices > 1) join_slices_kernel<T><<<a.rows, kThreads, 0, st>>>(a);
}

}  // namespace

extern "C" int64_t mie_token_logprobs_workspace(int32_t rows, int32_t vocab, int32_t top) {
  if (rows < 1 || vocab < 1 || top < 0 || top > kMaxTop) return 0;
  const int slices = slices_for(rows, vocab, top);
  return slices == 1 ? 0 : static_cast<int64_t>(rows) * slices * (static_cast<int64_t>(sizeof(f32x4)) + 8 * top);
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
  if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15))
    return mie::fail(MIE_ERR_INVALID, "mie_token_logprobs: the workspace must be 16-byte aligned");
  LogprobsArgs a{static_cast<const char*>(logits), stride, rows, vocab, top, slices_for(rows, vocab, top), tokens,
                 logprobs, entropy, top_logprobs, top_tokens, nullptr, static_cast<f32x4*>(workspace)};
  a.ws_keys = reinterpret_cast<uint64_t*>(a.ws_sums + static_cast<int64_t>(rows) * a.slices);
  mie::clear_error();
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MIE_DTYPE_F32)
    launch<float>(a, st);
  else
    launch<uint16_t>(a, st);
  return mie::check_launch("mie_token_logprobs");
}
