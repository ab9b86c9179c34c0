// Rotary positions for a step's packed tokens and their K and V into the pool
// (mie_rope_append).
//
// Mathematics: each pair of a head's values is turned by the angle a =
// position * frequency.  The angle in turns, a / 2 pi, is formed and reduced
// to [-1/2, 1/2] in float64 (a far position leaves float32 no digits behind
// the point); what is left is a float32 with an error of 2^-26 turns at most,
// and its sine and cosine serve every head of the token.
//
// Bound by memory: q, k and v are read once and written once.  A workgroup
// takes a token: its threads first form the token's cosines and sines in LDS,
// then each moves units of VEC pairs (two 16-byte vectors), all heads of q, k
// and v in one flat range.  On MI355X 8192 bfloat16 tokens of 32 + 8 + 8 heads
// x 128 (201 MB) take 39.7 us, the rate of a device copy (5.0 TB/s); 64 float32
// tokens of 8 heads x 96 3.6 us in a graph, a launch.
#include <algorithm>

#include "mie_common.h"

namespace {

constexpr int kThreads = 256;

struct RopeArgs {
  const char* q;
  const char* k;
  const char* v;
  char* q_out;
  char* k_pool;
  char* v_pool;
  int64_t q_st, q_sh, kv_st, kv_sh, out_st, out_sh, sblk, shead;  // elements
  int64_t num_slots;
  const int64_t* slots;
  const int32_t* positions;
  const double* freq;
  int32_t tokens, heads, kv_heads, head_dim, pairs;  // pairs: rotary_dim / 2
  float factor;
  int32_t units;                // units of VEC pairs in a token
  mie::FastDiv head_units, bs;  // those in a head
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};
template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  return mie::Mem<T>::get(&x);
}
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  T y;
  mie::Mem<T>::put(&y, x);
  return y;
}

// grid = tokens; LDS: (cos, sin) of the token's pairs (dynamic).
template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rope_append_kernel(RopeArgs a) {
  using V = Vec<T, VEC>;
  extern __shared__ float2 s_turn[];
  const int token = blockIdx.x;
  for (int i = threadIdx.x; i < a.pairs; i += kThreads) {
    double turns = static_cast<double>(a.positions[token]) * (a.freq[i] * 0.15915494309189533577);  // 1 / 2 pi
    turns -= rint(turns);
    float sn, cs;
    sincospif(2.f * static_cast<float>(turns), &sn, &cs);
    s_turn[i] = make_float2(cs * a.factor, sn * a.factor);
  }
  __syncthreads();

  const int rotating = a.pairs / VEC;  // units of a head that turn; the rest are copied
  for (int u = threadIdx.x; u < a.units; u += kThreads) {
    const int row = a.head_units.div(u), j = u - row * a.head_units.d;
    const bool turns = j < rotating && row < a.heads + a.kv_heads;
    // The unit's two vectors.
    int d1 = 2 * j * VEC, d2 = d1 + VEC;
    if (!INTERLEAVED && j < rotating) {
      d1 = j * VEC;
      d2 = d1 + a.pairs;
    }
    const T* src;
    T* dst;
    if (row < a.heads) {
      src = reinterpret_cast<const T*>(a.q) + token * a.q_st + row * a.q_sh;
      dst = reinterpret_cast<T*>(a.q_out) + token * a.out_st + row * a.out_sh;
    } else {
      const bool value = row >= a.heads + a.kv_heads;
      const int h = row - a.heads - (value ? a.kv_heads : 0);
      const int64_t slot = a.slots[token];
      if (slot < 0 || slot >= a.num_slots) continue;
      const int64_t blk = static_cast<int64_t>(static_cast<uint64_t>(slot) / a.bs.d);
      src = reinterpret_cast<const T*>(value ? a.v : a.k) + token * a.kv_st + h * a.kv_sh;
      dst = reinterpret_cast<T*>(value ? a.v_pool : a.k_pool) + blk * a.sblk + h * a.shead +
            (slot - blk * a.bs.d) * a.head_dim;
    }
    V x = *reinterpret_cast<const V*>(src + d1), y = *reinterpret_cast<const V*>(src + d2);
    if (turns) {
      const float2* turn = s_turn + j * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float2 cs = turn[e];
        if constexpr (INTERLEAVED) {
          // Pair e of the unit: elements 2 e, 2 e + 1 of its 2 VEC consecutive ones.
          T* first = 2 * e < VEC ? &x.v[2 * e % VEC] : &y.v[2 * e % VEC];
          T* second = 2 * e + 1 < VEC ? &x.v[(2 * e + 1) % VEC] : &y.v[(2 * e + 1) % VEC];
          const float f = to_f32(*first), s = to_f32(*second);
          *first = from_f32<T>(f * cs.x - s * cs.y);
          *second = from_f32<T>(s * cs.x + f * cs.y);
        } else {
          const float f = to_f32(x.v[e]), s = to_f32(y.v[e]);
          x.v[e] = from_f32<T>(f * cs.x - s * cs.y);
          y.v[e] = from_f32<T>(s * cs.x + f * cs.y);
        }
      }
    }
    *reinterpret_cast<V*>(dst + d1) = x;
    *reinterpret_cast<V*>(dst + d2) = y;
  }
}

template <typename T>
void launch_rope(RopeArgs a, bool wide, bool interleaved, hipStream_t st) {
  constexpr int W = 16 / sizeof(T);
  const int vec = wide ? W : 1;
  const int rows = a.heads + 2 * a.kv_heads;
  a.head_units = mie::FastDiv::make(a.head_dim / (2 * vec));
  a.units = rows * (a.head_dim / (2 * vec));
  const int groups = a.tokens;
  const size_t lds = sizeof(float2) * a.pairs;
  if (wide && interleaved)
    rope_append_kernel<T, W, true><<<groups, kThreads, lds, st>>>(a);
  else if (wide)
    rope_append_kernel<T, W, false><<<groups, kThreads, lds, st>>>(a);
  else if (interleaved)
    rope_append_kernel<T, 1, true><<<groups, kThreads, lds, st>>>(a);
  else
    rope_append_kernel<T, 1, false><<<groups, kThreads, lds, st>>>(a);
}

}  // namespace

extern "C" int32_t mie_rope_append(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
                                   const void* v, int64_t kv_stride_t, int64_t kv_stride_h, void* k_pool,
                                   void* v_pool, int64_t pool_stride_block, int64_t pool_stride_head,
                                   int32_t num_blocks, const int64_t* slots, const int32_t* positions,
                                   const double* frequencies, int32_t rotary_dim, int32_t interleaved, float factor,
                                   int32_t tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                   int32_t block_size, void* q_out, int64_t out_stride_t, int64_t out_stride_h,
                                   int32_t dtype, void* stream) {
  if (dtype != MIE_DTYPE_F32 && dtype != MIE_DTYPE_BF16)
    return mie::fail(MIE_ERR_UNSUPPORTED, "mie_rope_append: dtype %d; float32 or bfloat16 only", dtype);
  const int elt = mie::elt_size(dtype);
  if (tokens < 0 || tokens > 1 << 23 || num_heads < 1 || num_kv_heads < 1 || num_blocks < 1 || block_size < 1)
    return mie::fail(MIE_ERR_INVALID, "mie_rope_append: bad shape tokens=%d heads=%d/%d num_blocks=%d block_size=%d",
                     tokens, num_heads, num_kv_heads, num_blocks, block_size);
  if (num_heads > 4096 || num_kv_heads > 4096)
    return mie::fail(MIE_ERR_INVALID, "mie_rope_append: heads=%d/%d above 4096", num_heads, num_kv_heads);
  if (head_dim < 2 || head_dim > 1024 || head_dim % 2 || rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim)
    return mie::fail(MIE_ERR_INVALID, "mie_rope_append: rotary_dim %d of head_dim %d (even, at most 1024)", rotary_dim,
                     head_dim);
  if (tokens == 0) return MIE_OK;
  if (!q || !k || !v || !k_pool || !v_pool || !slots || !positions || !frequencies || !q_out)
    return mie::fail(MIE_ERR_INVALID, "mie_rope_append: null pointer");
  if (pool_stride_head < static_cast<int64_t>(block_size) * head_dim ||
      pool_stride_block < static_cast<int64_t>(num_kv_heads) * pool_stride_head)
    return mie::fail(MIE_ERR_INVALID, "mie_rope_append: pool strides overlap");
  RopeArgs a;
  a.q = static_cast<const char*>(q);
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  a.q_out = static_cast<char*>(q_out);
  a.k_pool = static_cast<char*>(k_pool);
  a.v_pool = static_cast<char*>(v_pool);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.kv_st = kv_stride_t;
  a.kv_sh = kv_stride_h;
  a.out_st = out_stride_t;
  a.out_sh = out_stride_h;
  a.sblk = pool_stride_block;
  a.shead = pool_stride_head;
  a.num_slots = static_cast<int64_t>(num_blocks) * block_size;
  a.slots = slots;
  a.positions = positions;
  a.freq = frequencies;
  a.tokens = tokens;
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.pairs = rotary_dim / 2;
  a.factor = factor;
  a.bs = mie::FastDiv::make(static_cast<uint32_t>(block_size));
  // 16-byte vectors where every row, half and tail starts on one; single
  // elements otherwise.
  const int w = 16 / elt;
  const bool wide = rotary_dim % (2 * w) == 0 && head_dim % (2 * w) == 0 &&
                    (q_stride_t | q_stride_h | kv_stride_t | kv_stride_h | out_stride_t | out_stride_h |
                     pool_stride_block | pool_stride_head) % w == 0 &&
                    ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                      reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_pool) |
                      reinterpret_cast<uintptr_t>(v_pool)) & 15) == 0;
  mie::clear_error();
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MIE_DTYPE_F32)
    launch_rope<float>(a, wide, interleaved != 0, st);
  else
    launch_rope<uint16_t>(a, wide, interleaved != 0, st);
  return mie::check_launch("mie_rope_append");
}
