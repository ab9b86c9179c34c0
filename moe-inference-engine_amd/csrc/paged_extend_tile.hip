// mie_paged_extend for many rows: tiles of 128 rows whose keys and values go
// through LDS.
//
// One workgroup per (128 rows, K/V head, partition of the keys), 32 rows per
// wave.  K and V come in tiles of KT keys straight from the pool into two LDS
// buffers (16 bytes per lane, no registers between): tile t + 1 is in flight
// while tile t is multiplied, one barrier per tile.  A wave forms S^T = K Q^T
// on the 32 x 32 matrix instructions, so a lane holds scores of one row only
// (its other half of the keys is in the lane 32 further on): maxima and sums
// are in-lane but for one exchange, and the probabilities are, without moving,
// the second operand of O^T = V^T P^T.  bfloat16 V is transposed by the LDS
// read.
//
// The running maximum is raised only where a row's scores outgrow it by 2^8:
// sums and outputs are then at most 2^8 times larger than with the true one,
// which costs nothing in floating point, and the rescaling of O is rare.
// bfloat16 probabilities are rounded once to bfloat16 on the way into the
// second product: a relative error of 2^-9 at most per term, of the size of
// the output's own rounding and averaged over the keys; their sum is taken
// before the rounding.
//
// Bound by the matrix cores together with the softmax's vector instructions and
// the issue of the loads: on MI355X two chunks of 4096 bfloat16 tokens, 32 heads
// over 8 x 128, 550 to 575 us or 935 to 980 TFLOP/s (an 8192^3 library product:
// 1230); 12 x 64 83 us, 620 TFLOP/s (half the products per exponential), with
// capped scores 131.  Without the next tile's loads 410 of 548 us, without the softmax 477,
// products and LDS reads alone 326.
//
// Rows of K and V in LDS are as they lie in the pool, except that the 16-byte
// pieces of a row are exchanged (XOR with bits of the key) so that a read's
// lanes fall on different banks; the exchange is made in the addresses the
// lanes load from.
#include <algorithm>

#include "paged_extend.h"

namespace {

using mie::Mem;
using mie::extend::Args;
using mie::extend::f32x4;
using mie::extend::kLog2e;
using mie::extend::kTileRows;
using mie::extend::Place;
using mie::extend::u32x4;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
using mie::gemm::bf16x8;

typedef __attribute__((address_space(3))) char lds_char;

// The XOR of a key's 16-byte pieces, CH pieces per row.  K is read 16 keys at
// a time at one piece: rows that start on the same bank differ in the XOR.
template <int CH>
__device__ __forceinline__ int key_swizzle(int key) {
  if constexpr (CH % 16 == 0) return key & 15;
  if constexpr (CH % 8 == 0) return key >> 1 & 7;
  return key >> 2 & 3;
}
// V is read four keys at a time at four pieces (bfloat16), or two keys four
// apart at eight (float32).
template <typename T, int CH>
__device__ __forceinline__ int value_swizzle(int key) {
  if constexpr (sizeof(T) == 4) return CH % 16 == 0 ? (key >> 2 & 1) << 3 : 0;
  if constexpr (CH % 16 == 0) return (key & 3) << 2;
  return CH == 8 ? (key >> 1 & 1) << 2 : 0;
}

// A value the compiler must take as new here: what is computed from it in a
// rare path stays there, neither kept in registers across the loop nor done on
// every path.
template <typename X>
__device__ __forceinline__ X fresh(X x) {
  asm volatile("" : "+v"(x));
  return x;
}

// max / sum over the two lanes of a row (l, l + 32).
template <bool MAX>
__device__ __forceinline__ float across_halves(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float u = __uint_as_float(a[0]), v = __uint_as_float(a[1]);
  return MAX ? fmaxf(u, v) : u + v;
}

template <typename T> struct Products;
template <> struct Products<uint16_t> {
  static constexpr int KT = 64;     // keys per tile
  static constexpr int kDims = 16;  // dims one 16-byte piece per lane covers
  static __device__ __forceinline__ f32x16 scores(u32x4 k, u32x4 q, f32x16 s) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, q), s, 0,
                                                   0, 0);
  }
};
template <> struct Products<float> {
  static constexpr int KT = 32;
  static constexpr int kDims = 8;
  static __device__ __forceinline__ f32x16 scores(u32x4 k, u32x4 q, f32x16 s) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k[e]), __uint_as_float(q[e]), s, 0, 0, 0);
    return s;
  }
};

// Key of register i of a 32-key block in lane half h, and dim likewise.
__device__ __forceinline__ int in_block(int i, int h) { return 8 * (i / 4) + 4 * h + i % 4; }

template <typename T, int D>
struct Tile {
  static constexpr int KT = Products<T>::KT;
  static constexpr int kRowBytes = D * static_cast<int>(sizeof(T));
  static constexpr int CH = kRowBytes / 16;
  static constexpr int kBytes = KT * kRowBytes;
  static constexpr int kLoads = kBytes / 4096;  // 16-byte loads per lane for K, and as many for V
  static constexpr int kKeys = KT / 4;          // keys a wave loads
  static constexpr int NQ = D / Products<T>::kDims, NB = KT / 32, ND = D / 32;
  static_assert(kBytes % 4096 == 0 && 16 % kKeys == 0, "a tile divides among the waves");
};

// Where a lane reads in a tile.  XORs touch the bits below a row only, so an
// address is a lane's constant plus the row's.
template <typename T, int D>
struct Reads {
  using L = Tile<T, D>;
  int k_row, k_xor, v_row, v_xor;
  __device__ __forceinline__ Reads() {
    const int lane = threadIdx.x & 63, q = lane & 31, h = lane >> 5;
    k_row = q * L::kRowBytes;
    k_xor = (h ^ key_swizzle<L::CH>(q)) * 16;
    if constexpr (sizeof(T) == 4) {
      // Keys 8 (i / 4) + 4 h + i % 4, dim q of a block of 32.
      v_row = 4 * h * L::kRowBytes + q * 4;
      v_xor = value_swizzle<T, L::CH>(4 * h) * 16;
    } else {
      // The transposing read: 16 lanes take four keys x 16 dims.
      const int key = 4 * h + ((lane & 15) >> 2);
      v_row = key * L::kRowBytes + (lane >> 4 & 1) * 32 + (lane & 3) * 8;
      v_xor = value_swizzle<T, L::CH>(key) * 16;
    }
  }
  // Piece 2 c + h of key 32 b + q.
  __device__ __forceinline__ int key(int b, int c) const { return k_row + ((c * 32) ^ k_xor) + b * 32 * L::kRowBytes; }
  // Dim block n (32 dims) of the lane's keys from `first` on.
  __device__ __forceinline__ int value(int first, int n) const {
    return v_row + ((n * 32 * static_cast<int>(sizeof(T))) ^ v_xor) + first * L::kRowBytes;
  }
};

// What a wave holds of its 32 rows.
template <typename T, int D>
struct State {
  using L = Tile<T, D>;
  u32x4 q[L::NQ];
  f32x16 o[L::ND];
  float m, l;  // m: what the sums are relative to; l: this lane's half of the keys
  int position, row_head;
  float slope;
  mie::extend::Range keys;         // this row sees
  mie::extend::Range some, shared;  // some / every row of the wave sees
};

template <typename T, int D>
__device__ __forceinline__ void rescale(State<T, D>& w, float top) {
  // top: the row's largest exponent in this tile, -inf if it sees none.
  if (__any(top > w.m + 8.f)) {
    const float raised = fmaxf(top, w.m);
    const float alpha = raised == -INFINITY ? 1.f : mie::fast_exp2(w.m - raised);
    w.m = raised;
    w.l *= alpha;
#pragma unroll
    for (int n = 0; n < Tile<T, D>::ND; ++n) w.o[n] *= alpha;
  }
}

// O^T += V^T P^T.
template <typename T, int D>
__device__ __forceinline__ void multiply_values(State<T, D>& w, const Reads<T, D>& at, const char* tile,
                                                const f32x16 (&p)[Tile<T, D>::NB]) {
  using L = Tile<T, D>;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int b = 0; b < L::NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int n = 0; n < L::ND; ++n)
          w.o[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(
              *reinterpret_cast<const float*>(tile + at.value(b * 32 + in_block(i, 0), n)), p[b][i], w.o[n], 0, 0, 0);
  } else {
#pragma unroll
    for (int b = 0; b < L::NB; ++b)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        u32x4 pk;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pk[e] = __builtin_bit_cast(
              uint32_t, __builtin_convertvector(f32x2{p[b][half * 8 + 2 * e], p[b][half * 8 + 2 * e + 1]}, bf16x2));
#pragma unroll
        for (int n = 0; n < L::ND; ++n) {
          s16x4 v[2];
#pragma unroll
          for (int r = 0; r < 2; ++r)
            v[r] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(tile + at.value(b * 32 + half * 16 + r * 8, n)));
          const u32x4 a = __builtin_bit_cast(u32x4, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
          w.o[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                           __builtin_bit_cast(bf16x8, pk), w.o[n], 0, 0, 0);
        }
      }
  }
}

// Replaces this wave's share of a tile's values that are not finite by 0;
// whether there were any.
template <typename T, int D>
__device__ __forceinline__ bool drop_not_finite(char* tile, int wave) {
  const int lane = threadIdx.x & 63;
  bool any = false;
#pragma unroll 1
  for (int c = (wave * 64 + lane) * 16; c < Tile<T, D>::kBytes; c += 4096) {
    u32x4 x = *reinterpret_cast<const u32x4*>(tile + c), y = x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4) {
        y[e] = mie::extend::not_finite(__uint_as_float(x[e])) ? 0u : x[e];
      } else {
        const uint32_t low = (x[e] & 0x7f80u) == 0x7f80u ? 0u : x[e] & 0xffffu;
        const uint32_t high = (x[e] & 0x7f800000u) == 0x7f800000u ? 0u : x[e] & 0xffff0000u;
        y[e] = low | high;
      }
      any |= x[e] != y[e];
    }
    *reinterpret_cast<u32x4*>(tile + c) = y;
  }
  return __any(any);
}

// What the loop left out, for the wave's rows: the values drop_not_finite
// replaced, to the rows that see them (a weight above 0 times such a value is
// the value itself), and NaN for the rows that see a key without a block.
template <typename T, int D>
__device__ __attribute__((noinline)) void mend_rows(Args a, Place p, const char* v_head, int first, int end, int position, bool odd, f32x4* out, float& sum) {
  using L = Tile<T, D>;
  const int h = (threadIdx.x & 63) >> 5;
  const mie::extend::Range keys = mie::extend::keys_of(a, p, position);
  const mie::extend::Range shared = mie::extend::shared_keys(a, p, p.p_first, p.p_last);
  for (int k0 = first; k0 < end; k0 += L::KT) {
    const bool whole = mie::extend::holds(shared, k0, k0 + L::KT);
    for (int key = k0; key < min(k0 + L::KT, end); ++key) {
      bool bad;
      const int64_t off = mie::extend::row_offset(a, key, mie::extend::entry_of(a, p.b, key), L::kRowBytes, bad);
      const bool seen = mie::extend::holds(keys, key);
      if (bad && seen) sum = NAN;
      if (bad || whole || !odd) continue;
      const T* v = reinterpret_cast<const T*>(v_head + off);
      for (int n = 0; n < L::ND * 4; ++n)
        for (int e = 0; e < 4; ++e) {
          const float x = Mem<T>::get(v + n / 4 * 32 + in_block(n % 4 * 4 + e, h));
          out[n][e] += seen && mie::extend::not_finite(x) ? x : 0.f;
        }
    }
  }
}

template <typename T, int D>
__device__ __forceinline__ void attend(const Args& a, State<T, D>& w, const Reads<T, D>& at,
                                       const char* k_tile, const char* v_tile, int k0) {
  using L = Tile<T, D>;
  f32x16 s[L::NB];
#pragma unroll
  for (int b = 0; b < L::NB; ++b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
    for (int c = 0; c < L::NQ; ++c) {
      s[b] = Products<T>::scores(*reinterpret_cast<const u32x4*>(k_tile + at.key(b, c)), w.q[c], s[b]);
    }
  }
  float top = -INFINITY, scale = a.scale;  // a positive scale goes into the exponential's operand
  const int key0 = fresh(k0 + 4 * ((threadIdx.x & 63) >> 5));
  if (a.cap > 0.f || a.slopes || !(a.scale > 0.f)) {
    const float dot_scale = fresh(a.scale);
    scale = 1.f;
    if (a.cap > 0.f) {
      const float cap = fresh(a.cap);
#pragma unroll
      for (int b = 0; b < L::NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[b][i] = mie::extend::capped<T>(s[b][i], cap, dot_scale, a.cap_ratio);
    } else {
#pragma unroll
      for (int b = 0; b < L::NB; ++b) s[b] *= dot_scale;
    }
    if (a.slopes) {
      const float away = fresh(static_cast<float>(w.position - key0));
#pragma unroll
      for (int b = 0; b < L::NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[b][i] = fmaf(-w.slope, fabsf(away - static_cast<float>(b * 32 + in_block(i, 0))), s[b][i]);
    }
  }
  if (!mie::extend::holds(w.shared, k0, k0 + L::KT)) {
    const mie::extend::Range seen{fresh(w.keys.low - key0), w.keys.high - key0};
#pragma unroll
    for (int b = 0; b < L::NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[b][i] = mie::extend::holds(seen, b * 32 + in_block(i, 0)) ? s[b][i] : -INFINITY;
  }
#pragma unroll
  for (int b = 0; b < L::NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
  rescale(w, across_halves<true>(top) * scale);
  const float ref = w.m == -INFINITY ? 0.f : w.m;
  float sum = 0.f;
#pragma unroll
  for (int b = 0; b < L::NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[b][i] = mie::fast_exp2(fmaf(s[b][i], scale, -ref));
      sum += s[b][i];
    }
  w.l += sum;
  multiply_values<T, D>(w, at, v_tile, s);
}

// grid = tiles x parts x kv_heads, the K/V head fastest, a sequence's last
// tiles (the longest) first.  WHOLE: blocks hold a multiple of 16 keys.
template <typename T, int D, bool WHOLE>
__global__ __launch_bounds__(256, D * sizeof(T) <= 384 ? 2 : 1) void extend_tile_kernel(Args a) {
  using L = Tile<T, D>;
  __shared__ __align__(16) char s_k0[L::kBytes];
  __shared__ __align__(16) char s_v0[L::kBytes];
  __shared__ __align__(16) char s_k1[L::kBytes];
  __shared__ __align__(16) char s_v1[L::kBytes];
  __shared__ int s_bad, s_odd;  // a key without a block; a dropped value
  const int lane = threadIdx.x & 63, q = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const mie::extend::Item item = mie::extend::item_of(a);
  const int kvh = item.kvh, part = item.part, tile = a.tiles - 1 - item.tile;
  const Place p = mie::extend::find_place<kTileRows>(a, tile);
  if (p.b < 0) return;
  const mie::extend::Split split = mie::extend::split_of(a, p);
  const int parts = split.parts;
  if (part >= parts) return;
  const int first = p.low + part * split.keys;
  const int end = parts == 1 ? p.high : min(p.high, first + split.keys);
  if (threadIdx.x == 0) s_bad = s_odd = 0;

  State<T, D> w;
  const Reads<T, D> at;
  const int row0 = p.row0 + wave * 32;
  const int row = min(row0 + q, p.rows - 1);
  const int token = a.group.div(row);
  const int base = p.len - p.count;
  w.row_head = kvh * a.group.d + row - token * a.group.d;
  w.position = base + token;
  w.slope = a.slopes ? a.slopes[w.row_head] * kLog2e : 0.f;
  const int p_first = base + static_cast<int>(a.group.div(min(row0, p.rows - 1)));
  const int p_last = base + static_cast<int>(a.group.div(min(row0 + 32, p.rows) - 1));
  w.keys = mie::extend::keys_of(a, p, w.position);
  w.shared = mie::extend::shared_keys(a, p, p_first, p_last);
  w.some = mie::extend::Range{mie::extend::keys_of(a, p, p_first).low,
                              row0 < p.rows ? mie::extend::keys_of(a, p, p_last).high : 0};
  const mie::extend::Range shared = mie::extend::shared_keys(a, p, p.p_first, p.p_last);  // by every row of the tile
  const char* qp = a.q + (p.start + token) * a.q_st + w.row_head * a.q_sh + h * 16;
#pragma unroll
  for (int c = 0; c < L::NQ; ++c) w.q[c] = *reinterpret_cast<const u32x4*>(qp + c * 32);
  w.m = -INFINITY;
  w.l = 0.f;
#pragma unroll
  for (int n = 0; n < L::ND; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) w.o[n][i] = 0.f;

  // Loading.  A wave brings kKeys consecutive keys of a tile, the lane's n-th
  // 16-byte piece to byte ((wave kLoads + n) 64 + lane) 16 of the LDS buffer.
  const char* k_head = a.k_pool + kvh * a.shead;
  const char* v_head = a.v_pool + kvh * a.shead;
  const int32_t* table = a.tables + p.b * a.table_stride;
  int in_wave[L::kLoads], k_piece[L::kLoads], v_piece[L::kLoads];  // the piece's key and its bytes in that key's row
#pragma unroll
  for (int n = 0; n < L::kLoads; ++n) {
    const int at = n * 64 + lane;
    in_wave[n] = at / L::CH;
    k_piece[n] = ((at - in_wave[n] * L::CH) ^ key_swizzle<L::CH>(wave * L::kKeys + in_wave[n])) * 16;
    v_piece[n] = ((at - in_wave[n] * L::CH) ^ value_swizzle<T, L::CH>(wave * L::kKeys + in_wave[n])) * 16;
  }
  auto to_lds = [&](const char* from, char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
  };
  // Table entries are loaded a tile ahead and looked at when they are used:
  // waiting for one is waiting for every load before it.  Where blocks hold
  // whole multiples of kKeys the wave's keys are one block's, and its address
  // is the wave's; keys past the end are places behind the last one's in its
  // block.  Otherwise every lane finds its own, the last key again past the end.
  int32_t id[WHOLE ? 1 : L::kLoads];
  auto group_of = [&](int k0) { return min(k0 + wave * L::kKeys, (end - 1) & -L::kKeys); };
  auto key_of = [&](int k0, int n) { return min(k0 + wave * L::kKeys + in_wave[n], end - 1); };
  auto look_up = [&](int k0) {
    if constexpr (WHOLE) {
      id[0] = table[min(static_cast<int>(a.bs.div(group_of(k0))), a.table_width - 1)];
    } else {
#pragma unroll
      for (int n = 0; n < L::kLoads; ++n)
        id[n] = table[min(static_cast<int>(a.bs.div(key_of(k0, n))), a.table_width - 1)];
    }
  };
  auto row_of = [&](int key, int32_t block, bool& bad) {
    const int blk = a.bs.div(key);
    bad = static_cast<uint32_t>(block) >= static_cast<uint32_t>(a.num_blocks) || blk >= a.table_width;
    return (bad ? 0 : block) * a.sblk + static_cast<int64_t>(key - blk * static_cast<int>(a.bs.d)) * L::kRowBytes;
  };
  int64_t next_off = 0;  // WHOLE: the next tile's row of this wave
  auto aim = [&](int k0) {
    if constexpr (WHOLE) {
      bool bad;
      next_off = row_of(group_of(k0), __builtin_amdgcn_readfirstlane(id[0]), bad);
      if (bad) s_bad = 1;
    }
  };
  auto bring = [&](int k0, int n, char* k_tile, char* v_tile) {
    const int to = (wave * L::kLoads + n) * 1024;
    if constexpr (WHOLE) {
      to_lds(k_head + next_off + static_cast<uint32_t>(in_wave[n] * L::kRowBytes + k_piece[n]), k_tile + to);
      to_lds(v_head + next_off + static_cast<uint32_t>(in_wave[n] * L::kRowBytes + v_piece[n]), v_tile + to);
    } else {
      bool bad;
      const int64_t off = row_of(key_of(k0, n), id[n], bad);
      to_lds(k_head + off + k_piece[n], k_tile + to);
      to_lds(v_head + off + v_piece[n], v_tile + to);
      if (__any(bad)) s_bad = 1;
    }
  };
  // Everything this wave has loaded is in LDS, and every wave's is after the barrier.
  auto arrive = [&]() {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  };

  __syncthreads();  // the flags are clear
  int k0 = first;
  if (k0 < end) {
    look_up(k0);
    aim(k0);
#pragma unroll
    for (int n = 0; n < L::kLoads; ++n) bring(k0, n, s_k0, s_v0);
    look_up(k0 + L::KT);
  }
  auto step = [&](char* k_here, char* v_here, char* k_next, char* v_next) {
    arrive();
    if (!mie::extend::holds(shared, k0, k0 + L::KT)) {
      if (drop_not_finite<T, D>(v_here, wave)) s_odd = 1;
      __syncthreads();
    }
    // (Past the last tile its last keys come again, and nobody reads them.)
    if (k0 + L::KT < end) {
      aim(k0 + L::KT);
#pragma unroll
      for (int n = 0; n < L::kLoads; ++n) bring(k0 + L::KT, n, k_next, v_next);
      look_up(k0 + 2 * L::KT);
    }
    if (k0 < w.some.high && k0 + L::KT > w.some.low) attend<T, D>(a, w, at, k_here, v_here, k0);
    k0 += L::KT;
  };
  while (k0 < end) {
    step(s_k0, s_v0, s_k1, s_v1);
    if (k0 >= end) break;
    step(s_k1, s_v1, s_k0, s_v0);
  }

  float sum = across_halves<false>(w.l);
  f32x4 o[L::ND * 4];
#pragma unroll
  for (int n = 0; n < L::ND * 4; ++n)
    o[n] = f32x4{w.o[n / 4][n % 4 * 4], w.o[n / 4][n % 4 * 4 + 1], w.o[n / 4][n % 4 * 4 + 2], w.o[n / 4][n % 4 * 4 + 3]};
  arrive();
  if (s_bad | s_odd) {
    f32x4 mended[L::ND * 4];
    float mended_sum = sum;
#pragma unroll
    for (int n = 0; n < L::ND * 4; ++n) mended[n] = o[n];
    mend_rows<T, D>(a, p, v_head, first, end, w.position, s_odd != 0, mended, mended_sum);
#pragma unroll
    for (int n = 0; n < L::ND * 4; ++n) o[n] = mended[n];
    sum = mended_sum;
  }
  if (row0 + q >= p.rows) return;
  if (parts == 1) {
    const float f = p.bad ? NAN : sum == 0.f ? 0.f : 1.f / sum;
    T* out = reinterpret_cast<T*>(a.out + (p.start + token) * a.out_st + w.row_head * a.out_sh);
#pragma unroll
    for (int n = 0; n < L::ND * 4; ++n) Mem<T>::put4(out + n / 4 * 32 + in_block(n % 4 * 4, h), o[n] * f);
    return;
  }
  const int64_t ws_row =
      ((static_cast<int64_t>(tile) * a.kv_heads + kvh) * a.parts + part) * kTileRows + wave * 32 + q;
#pragma unroll
  for (int n = 0; n < L::ND * 4; ++n)
    *reinterpret_cast<f32x4*>(a.ws_acc + ws_row * D + n / 4 * 32 + in_block(n % 4 * 4, h)) = o[n];
  if (h == 0) {
    a.ws_ml[ws_row * 2] = w.m;
    a.ws_ml[ws_row * 2 + 1] = sum;
  }
}

template <typename T, int D>
void launch_tile(const Args& a, uint32_t groups, hipStream_t st) {
  if (a.whole_blocks)
    extend_tile_kernel<T, D, true><<<groups, 256, 0, st>>>(a);
  else
    extend_tile_kernel<T, D, false><<<groups, 256, 0, st>>>(a);
}

template <typename T>
void launch_dim(const Args& a, int head_dim, uint32_t groups, hipStream_t st) {
  switch (head_dim) {
    case 32: launch_tile<T, 32>(a, groups, st); break;
    case 64: launch_tile<T, 64>(a, groups, st); break;
    case 96: launch_tile<T, 96>(a, groups, st); break;
    case 128: launch_tile<T, 128>(a, groups, st); break;
    default: launch_tile<T, 256>(a, groups, st); break;
  }
}

}  // namespace

namespace mie {
namespace extend {

void launch_tiles(const Args& a, int dtype, int head_dim, hipStream_t stream) {
  const uint32_t groups = static_cast<uint32_t>(static_cast<int64_t>(a.tiles) * a.parts * a.kv_heads);
  if (dtype == MIE_DTYPE_F32)
    launch_dim<float>(a, head_dim, groups, stream);
  else
    launch_dim<uint16_t>(a, head_dim, groups, stream);
}

}  // namespace extend
}  // namespace mie
