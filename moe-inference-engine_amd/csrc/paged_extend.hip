// Attention of a step's packed tokens over the paged pool (mie_paged_extend).
//
// Mathematics: one pass over a row's keys with the running maximum m, sum l
// and output o of a softmax in base 2; a block of keys with maximum m' scales
// l and o by 2^(m - m') first.  Pieces of the same row (waves, partitions) are
// joined the same way.
//
// One workgroup per (16 rows, K/V head, partition of the keys).  Its four
// waves take every fourth block of 32 keys and merge their states in LDS once;
// there is no barrier in the loop.  Scores are computed transposed, S^T =
// K Q^T, so a lane holds four consecutive keys of one row - the second operand
// of O^T = V^T P^T: the probabilities never leave their registers.  V is read
// in rows: lane i's vector holds dims 4 i .. 4 i + 3, operand rows i of four
// 16-row blocks (block j: dims 4 i + j).  With bfloat16 V the probabilities go
// in as the sum of two bfloat16 values, 16 bits of significand.
//
// What a token does not see has no part in its row even where it is not
// finite: a masked probability is 0, and a block in which some row masks a key
// is multiplied key by key, skipping zeros, if its V holds a NaN or infinity
// (0 times those would be NaN).  bfloat16 does so for every block with such a
// V: an infinity times the second of a probability's two values may be NaN.
//
// Bound by reading K and V where a sequence has one tile: 64 tokens over 512
// to 8192 cached ones, 32 heads over 8 x 128 bfloat16, capped, 207 us (1145 MB
// at 5.5 TB/s); one over 100000 75 us; 4 tokens at 2048, 12 x 64, 8.7 us, two
// launches of dependent rounds.
#include <limits.h>

#include <algorithm>

#include "paged_extend.h"

namespace {

using mie::Mem;
using mie::extend::across_groups;
using mie::extend::Args;
using mie::extend::f32x4;
using mie::extend::kFewRows;
using mie::extend::kLog2e;
using mie::extend::kTileRows;
using mie::extend::Place;
using mie::extend::u32x4;
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

constexpr int kRows = mie::extend::kFewRows;

// A load of data that is read once, in whole cache lines per instruction, goes
// around the caches: V's (K's operands are half lines).
template <bool ONCE, typename V>
__device__ __forceinline__ V fetch(const V* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(p);
  return *p;
}

// V's operands of one 64- or 32-dim group for 32 keys, and their products.
// Lane (i, g): keys 16 t + 4 g + r (t < 2, r < 4), dims VEC i .. VEC i + VEC - 1.
template <typename T, int VEC> struct Values;
template <int VEC> struct Values<float, VEC> {
  typedef float vec __attribute__((ext_vector_type(VEC)));
  vec v[2][4];
  template <bool ONCE>
  __device__ __forceinline__ void load(int t, int r, const char* p) {
    v[t][r] = fetch<ONCE>(reinterpret_cast<const vec*>(p));
  }
  __device__ __forceinline__ bool not_finite() const {
    bool any = false;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VEC; ++j) any |= mie::extend::not_finite(v[t][r][j]);
    return any;
  }
  __device__ __forceinline__ void multiply(const float (&p)[2][4], f32x4* o) const {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[t][r][j], p[t][r], o[j], 0, 0, 0);
  }
};
template <int VEC> struct Values<uint16_t, VEC> {
  uint32_t v[2][4][VEC / 2];
  template <bool ONCE>
  __device__ __forceinline__ void load(int t, int r, const char* p) {
    if constexpr (VEC == 4) {
      const u32x2 x = fetch<ONCE>(reinterpret_cast<const u32x2*>(p));
      v[t][r][0] = x.x;
      v[t][r][1] = x.y;
    } else {
      v[t][r][0] = fetch<ONCE>(reinterpret_cast<const uint32_t*>(p));
    }
  }
  __device__ __forceinline__ bool not_finite() const {
    mie::extend::u16x2 most = {0, 0};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int w = 0; w < VEC / 2; ++w) mie::extend::take_magnitudes(most, v[t][r][w]);
    return mie::extend::not_finite(most);
  }
  // Contraction slot 4 t + r of lane group g is key 16 t + 4 g + r in both operands.
  __device__ __forceinline__ void multiply(const float (&p)[2][4], f32x4* o) const {
    u32x4 hi, lo;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float x = p[w / 2][2 * (w % 2)], y = p[w / 2][2 * (w % 2) + 1];
      hi[w] = mie::pack_bf16x2(x, y);
      lo[w] = mie::pack_bf16x2(x - mie::bf16_lo(hi[w]), y - mie::bf16_hi(hi[w]));
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      u32x4 a;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t x = v[w / 2][2 * (w % 2)][j / 2], y = v[w / 2][2 * (w % 2) + 1][j / 2];
        a[w] = __builtin_amdgcn_perm(y, x, j % 2 ? 0x07060302u : 0x05040100u);  // the two keys' dim j
      }
      o[j] = mie::gemm::mfma_fragment<uint16_t>(a, hi, o[j]);
      o[j] = mie::gemm::mfma_fragment<uint16_t>(a, lo, o[j]);
    }
  }
};

// Dim of register r of 16-dim block n in lane group g (the layout above).
template <int D>
__device__ __forceinline__ int dim_of(int n, int r, int g) {
  constexpr int G4 = D / 64;
  return n < G4 * 4 ? n / 4 * 64 + g * 16 + r * 4 + n % 4 : G4 * 64 + (n - G4 * 4) / 2 * 32 + g * 8 + r * 2 + n % 2;
}

// grid = tiles x parts x kv_heads, the K/V head fastest.  ONCE: a sequence has
// one tile, so nobody else reads its keys.
template <typename T, int D, bool ONCE>
__global__ __launch_bounds__(256, D * sizeof(T) <= 384 ? 2 : 1) void extend_rows_kernel(Args a) {
  constexpr int NCH = D * static_cast<int>(sizeof(T)) / 64;  // 64-byte pieces of a row
  constexpr int G4 = D / 64, G2 = D % 64 / 32;               // 64- and 32-dim groups
  constexpr int NO = G4 * 4 + G2 * 2;                        // 16-dim blocks
  constexpr int kRowBytes = D * static_cast<int>(sizeof(T));
  __shared__ float s_max[4][kRows], s_sum[4][kRows];
  __shared__ __align__(16) float s_out[4][kRows][D + 4];
  __shared__ __align__(16) int64_t s_off[4][2][32];  // each wave's row offsets, this block's and the next one's
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const mie::extend::Item item = mie::extend::item_of(a);
  const int kvh = item.kvh, part = item.part, tile = item.tile;
  const Place p = mie::extend::find_place<kRows>(a, tile);
  if (p.b < 0) return;
  const mie::extend::Split split = mie::extend::split_of(a, p);
  const int parts = split.parts;
  if (part >= parts) return;
  const int first = p.low + part * split.keys;
  const int end = parts == 1 ? p.high : min(p.high, first + split.keys);

  // This lane's row (the last one again past the end), its head and position.
  const int row = min(p.row0 + i, p.rows - 1);
  const int token = a.group.div(row);
  const int head = kvh * a.group.d + row - token * a.group.d;
  const int position = p.len - p.count + token;
  const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.f;
  const mie::extend::Range keys = mie::extend::keys_of(a, p, position);
  const mie::extend::Range shared = mie::extend::shared_keys(a, p, p.p_first, p.p_last);
  const char* qp = a.q + (p.start + token) * a.q_st + head * a.q_sh + g * 16;
  u32x4 q[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) q[c] = *reinterpret_cast<const u32x4*>(qp + c * 64);

  f32x4 o[NO];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int n = 0; n < NO; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};

  const char* k_head = a.k_pool + kvh * a.shead;
  const char* v_head = a.v_pool + kvh * a.shead;
  // Lanes l and l + 32 look up key l of a block (its last key again past the end).
  auto key_at = [&](int k0) { return min(k0 + (lane & 31), end - 1); };
  auto place_rows = [&](int k0, int32_t id, int buffer) {
    bool bad;
    s_off[wave][buffer][lane & 31] = mie::extend::row_offset(a, key_at(k0), id, kRowBytes, bad);
    __builtin_amdgcn_wave_barrier();
    return static_cast<uint32_t>(__ballot(bad));
  };
  u32x4 kf[2][NCH];
  auto load_keys = [&](int buffer) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* rows = k_head + s_off[wave][buffer][t * 16 + i] + g * 16;
#pragma unroll
      for (int c = 0; c < NCH; ++c) kf[t][c] = *reinterpret_cast<const u32x4*>(rows + c * 64);
    }
  };

  int k0 = first + wave * 32, buffer = 0;
  uint32_t bad_keys = 0;
  int32_t id = -1;  // the next block's entry
  if (k0 < end) {
    id = mie::extend::entry_of(a, p.b, key_at(k0));
    bad_keys = place_rows(k0, id, 0);
    load_keys(0);
    if (k0 + 128 < end) id = mie::extend::entry_of(a, p.b, key_at(k0 + 128));
  }
  for (; k0 < end; k0 += 128, buffer ^= 1) {
    Values<T, 4> v4[G4 > 0 ? G4 : 1];
    Values<T, 2> v2[G2 > 0 ? G2 : 1];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const char* v = v_head + s_off[wave][buffer][t * 16 + g * 4 + r];
#pragma unroll
        for (int n = 0; n < G4; ++n) v4[n].template load<ONCE>(t, r, v + (n * 64 + i * 4) * sizeof(T));
#pragma unroll
        for (int n = 0; n < G2; ++n) v2[n].template load<ONCE>(t, r, v + (G4 * 64 + n * 32 + i * 2) * sizeof(T));
      }
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NCH; ++c) s[u] = mie::gemm::mfma_fragment<T>(kf[u][c], q[c], s[u]);
    }
    const uint32_t bad = bad_keys;
    if (k0 + 128 < end) {
      bad_keys = place_rows(k0 + 128, id, buffer ^ 1);
      load_keys(buffer ^ 1);
      if (k0 + 256 < end) id = mie::extend::entry_of(a, p.b, key_at(k0 + 256));
    }
    float w[2][4];
    float top = m;
    const bool whole = mie::extend::holds(shared, k0, k0 + 32);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int in_block = u * 16 + g * 4 + r, key = k0 + in_block;
        float x = mie::extend::exponent<T>(a, s[u][r], slope, static_cast<float>(position - key));
        if (bad) x = bad >> in_block & 1 ? NAN : x;
        if (!whole) x = mie::extend::holds(keys, key) ? x : -INFINITY;
        w[u][r] = x;
        top = fmaxf(top, x);
      }
    top = across_groups<true>(top);
    const float ref = top == -INFINITY ? 0.f : top;
    if (__any(top > m)) {  // a later maximum: the sums so far shrink
      const float alpha = mie::fast_exp2(m - ref);
      l *= alpha;
#pragma unroll
      for (int n = 0; n < NO; ++n) o[n] *= alpha;
    }
    m = top;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        w[u][r] = mie::fast_exp2(w[u][r] - ref);
        l += w[u][r];
      }
    bool odd = false;
    if (!whole || sizeof(T) == 2) {
#pragma unroll
      for (int n = 0; n < G4; ++n) odd |= v4[n].not_finite();
#pragma unroll
      for (int n = 0; n < G2; ++n) odd |= v2[n].not_finite();
    }
    if (__any(odd)) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          for (int from = 0; from < 4; ++from) {
            const float weight = __shfl(w[t][r], i + 16 * from);
            const T* v = reinterpret_cast<const T*>(v_head + s_off[wave][buffer][t * 16 + from * 4 + r]);
#pragma unroll
            for (int n = 0; n < NO; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float x = Mem<T>::get(v + dim_of<D>(n, e, g));
                o[n][e] = weight == 0.f ? o[n][e] : o[n][e] + weight * x;
              }
          }
      continue;
    }
#pragma unroll
    for (int n = 0; n < G4; ++n) v4[n].multiply(w, &o[n * 4]);
#pragma unroll
    for (int n = 0; n < G2; ++n) v2[n].multiply(w, &o[G4 * 4 + n * 2]);
  }

  // Merge the waves: the largest maximum, then the rescaled sums and outputs.
  l = across_groups<false>(l);
  if (g == 0) {
    s_max[wave][i] = m;
    s_sum[wave][i] = l;
  }
  __syncthreads();
  const float top = fmaxf(fmaxf(s_max[0][i], s_max[1][i]), fmaxf(s_max[2][i], s_max[3][i]));
  const float f = m == -INFINITY ? 1.f : mie::fast_exp2(m - top);
  // Lane (i, g) holds, of a 64-dim group, dims 16 g + 4 r + j in o[j][r]; of a
  // 32-dim group, dims 8 g + 2 r + j.
#pragma unroll
  for (int n = 0; n < G4; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const f32x4* u = &o[n * 4];
      *reinterpret_cast<f32x4*>(&s_out[wave][i][n * 64 + g * 16 + r * 4]) =
          f32x4{u[0][r] * f, u[1][r] * f, u[2][r] * f, u[3][r] * f};
    }
#pragma unroll
  for (int n = 0; n < G2; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const f32x4* u = &o[G4 * 4 + n * 2];
      float* dst = &s_out[wave][i][G4 * 64 + n * 32 + g * 8 + r * 2];
      dst[0] = u[0][r] * f;
      dst[1] = u[1][r] * f;
    }
  __syncthreads();
  const int64_t piece = (static_cast<int64_t>(tile) * a.kv_heads + kvh) * a.parts + part;
  for (int e = threadIdx.x; e < kRows * (D / 4); e += 256) {
    const int in_tile = e / (D / 4), c = e % (D / 4) * 4;
    const int r = p.row0 + in_tile;
    if (r >= p.rows) break;
    float top = s_max[0][in_tile];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, s_max[w][in_tile]);
    float sum = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = s_max[w][in_tile];
      sum += mw == -INFINITY ? s_sum[w][in_tile] : s_sum[w][in_tile] * mie::fast_exp2(mw - top);
      v += *reinterpret_cast<const f32x4*>(&s_out[w][in_tile][c]);
    }
    if (parts == 1) {
      if (p.bad) sum = NAN;
      v = sum == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : v / sum;
      const int t = a.group.div(r);
      Mem<T>::put4(reinterpret_cast<T*>(a.out + (p.start + t) * a.out_st +
                                        (kvh * a.group.d + r - t * a.group.d) * a.out_sh) + c, v);
    } else {
      *reinterpret_cast<f32x4*>(a.ws_acc + (piece * kRows + in_tile) * D + c) = v;
      if (c == 0) {
        a.ws_ml[(piece * kRows + in_tile) * 2] = top;
        a.ws_ml[(piece * kRows + in_tile) * 2 + 1] = sum;
      }
    }
  }
}

// Partitions that are summed side by side, a power of two: many where there
// are many partitions (then few rows), so that a column's chain is short.
template <int D>
constexpr int join_lanes(int parts) {
  int lanes = 1;
  while (lanes * 2 <= parts && lanes * 2 <= 1024 / D) lanes *= 2;
  return lanes;
}

// Joins the partitions of a tile's rows in one pass over them, with a running
// maximum like the kernels'.  A row takes D / 4 columns of four dims by `lanes`
// partitions at a time, a workgroup as many rows as that leaves.
// grid = (tiles x kv_heads, ceil(rows of a tile / per group)).
template <typename T, int D, int ROWS>
__global__ __launch_bounds__(256) void extend_join_kernel(Args a, int lanes) {
  constexpr int kCols = D / 4, kAtOnce = 256 / kCols;  // 24 columns leave 16 threads over
  __shared__ __align__(16) f32x4 s_v[kAtOnce][kCols];
  __shared__ float s_top[kAtOnce], s_sum[kAtOnce];
  const int kvh = blockIdx.x % a.kv_heads, tile = blockIdx.x / a.kv_heads;
  const Place p = mie::extend::find_place<ROWS>(a, tile);
  if (p.b < 0) return;
  const int parts = mie::extend::split_of(a, p).parts;
  if (parts == 1) return;
  const int col = threadIdx.x % kCols, at = threadIdx.x / kCols;
  const int lane = at & (lanes - 1), in_tile = blockIdx.y * (kAtOnce / lanes) + at / lanes;
  const int r = p.row0 + in_tile;
  const bool have = at / lanes < kAtOnce / lanes && in_tile < ROWS && r < p.rows;
  const int64_t piece = (static_cast<int64_t>(tile) * a.kv_heads + kvh) * a.parts;
  float top = -INFINITY, sum = 0.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  // A part without seen keys has no weight: sum and values 0 (or NaN, kept).
  auto take = [&](float m, float s, f32x4 x) {
    const float to = fmaxf(top, m);
    const float f = m == -INFINITY ? 1.f : mie::fast_exp2(m - to);
    const float g = top == -INFINITY ? 1.f : mie::fast_exp2(top - to);
    sum = sum * g + s * f;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] * g + x[e] * f;
    top = to;
  };
  if (have) {
    const float* ml = a.ws_ml + (piece * ROWS + in_tile) * 2;
    const float* acc = a.ws_acc + (piece * ROWS + in_tile) * D + col * 4;
#pragma unroll 4
    for (int j = lane; j < parts; j += lanes)
      take(ml[static_cast<int64_t>(j) * ROWS * 2], ml[static_cast<int64_t>(j) * ROWS * 2 + 1],
           *reinterpret_cast<const f32x4*>(acc + static_cast<int64_t>(j) * ROWS * D));
    s_v[at][col] = v;
    if (col == 0) {
      s_top[at] = top;
      s_sum[at] = sum;
    }
  }
  __syncthreads();
  if (!have || lane != 0) return;
  for (int j = 1; j < lanes; ++j) take(s_top[at + j], s_sum[at + j], s_v[at + j][col]);
  v = sum == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : v / sum;
  const int t = a.group.div(r);
  Mem<T>::put4(reinterpret_cast<T*>(a.out + (p.start + t) * a.out_st +
                                    (kvh * a.group.d + r - t * a.group.d) * a.out_sh) + col * 4, v);
}

// ---- host ------------------------------------------------------------------

// Workgroups that the keys are split for, and the keys of the smallest
// partition: of 16 rows; where a sequence has one such tile, so that its keys
// are read once and reading them is the work (its partitions also even out
// ragged lengths); of 128 rows in float32 and in bfloat16 (whose products take
// an eighth of the time, so that partitions and their join weigh more).
// Measured on MI355X, us, once: 64 sequences of 512 to 8192 tokens (32 heads
// over 8 x 128, bfloat16) 210 with 2048 workgroups, 212 with 4096, 228 with
// 8192, (12 x 64) 175, 156, 152; 1 x 2048 (12 x 64) 10.2 with partitions of
// 256, 8.8 with 128, 13.5 with 512; 1 x 100000 76 with 256 and 87 with 128
// (many more to join).  128 rows, bfloat16: 512 + 1500 (12 x 64) 23.3 with 1024
// workgroups of 256 keys, 20.5 with 512 of 384; 1000 + 0 21.5, 18.5; two of 512
// + 3500 (32 over 8 x 128) 114, 98; four of 50 to 300 + up to 8000 63, 57.
// float32: 512 + 1500 (12 x 64) 53 with 256 keys, 51 with 128; six of up to 700
// + 1300 (8 x 96) 80 with 1024 workgroups, 102 with 2048.  Up to 256 keys stay in one piece: the join
// costs more (1 and 8 tokens at 200, 12 x 64: 6.3 and 6.4 against 8.4 and 8.7;
// at 400 9.5 against 8.7).
constexpr int kGroups = 1024, kMinPart = 256;
constexpr int kGroupsOnce = 4096, kMinPartOnce = 128;
constexpr int kGroupsTileF32 = 1024, kMinPartTileF32 = 128;
constexpr int kGroupsTile = 512, kMinPartTile = 384;
constexpr int kOnePiece = 256;

struct Plan {
  int rows;  // of a tile
  int64_t tiles;
  int parts, part_keys;
  int64_t bytes;
};

// Tiles of 128 rows read K and V an eighth as often as those of 16, but take
// a wave per 32 rows and stage through LDS: they pay from some work on, and
// where a sequence has more rows than the small ones hold.  The work is
// tokens x heads x keys x head_dim, the keys those of a middle token.
// Measured on MI355X, us with 16 / 128 rows (new tokens per sequence + those
// before), the work in millions behind it:
//   bfloat16, 12 heads x 64: 1 x 16 + 2000 (25) 12.9 / 14.0; 1 x 256 + 0 (25)
//   8.6 / 10.9; 8 x 16 + 1000 (99) 14.6 / 14.3; 1 x 64 + 4000 (198) 21.9 /
//   18.7; 1 x 1000 + 0 (384) 25.2 / 19.6; 8 x 256 + 1000 (1774) 60.7 / 35.6.
//   32 heads over 8 x 128: 1 x 16 + 2000 (132) 17.0 / 18.1; 1 x 256 + 0 (134)
//   13.1 / 14.2; 8 x 16 + 1000 (528) 33.8 / 23.8; 1 x 256 + 4000 (4328) 119 / 56.
//   float32, 12 x 64: 1 x 1000 + 0 (384) 39.9 / 50.3; 8 x 64 + 1000 (406) 42 /
//   47; 1 x 256 + 4000 (812) 75 / 60; 8 x 256 + 1000 (1774) 121 / 102.  32 over
//   8 x 128: 1 x 256 + 0 (134) 25 / 43; 8 x 16 + 1000 (528) 66 / 51; 1 x 1000
//   + 0 (2048) 193 / 137; 64 x 4 + 2000 (2099, 16 rows) 214 / 566.
bool many_rows(int64_t tokens, int max_new, int64_t keys, int group, int kv_heads, int head_dim, int dtype) {
  const double work = static_cast<double>(tokens) * group * kv_heads * (keys - std::min<int64_t>(max_new, keys) / 2) *
                      head_dim;
  if (dtype == MIE_DTYPE_F32) return static_cast<int64_t>(max_new) * group >= 64 && work >= 500e6;
  return static_cast<int64_t>(max_new) * group > kFewRows && work >= 160e6;
}

// Row tiles: as many as the batch can have (the lengths are on the device).
// The keys are split until the tiles make the workgroups wanted.
Plan make_plan(int tokens, int batch, int max_new, int max_len, int window, int group, int kv_heads, int head_dim,
               int dtype) {
  Plan p;
  const int64_t keys = window > 0 ? std::min(max_len, window) : max_len;
  const int rows = p.rows =
      many_rows(tokens, max_new, keys, group, kv_heads, head_dim, dtype) ? kTileRows : kFewRows;
  const int64_t most = (static_cast<int64_t>(max_new) * group + rows - 1) / rows;
  p.tiles = static_cast<int64_t>(max_new) * group <= rows
                ? batch
                : std::min<int64_t>(batch * most, static_cast<int64_t>(tokens) * group / rows + batch);
  // Keys a tile can see: all, or a window back from each of its tokens.
  const int64_t span = (rows + group - 1) / group + 1;
  const int64_t range = window > 0 ? std::min<int64_t>(max_len, static_cast<int64_t>(window) + span + 32) : max_len;
  const bool once = static_cast<int64_t>(max_new) * group <= kFewRows;
  int groups = once ? kGroupsOnce : kGroups, min_part = once ? kMinPartOnce : kMinPart;
  if (rows == kTileRows) {
    groups = dtype == MIE_DTYPE_F32 ? kGroupsTileF32 : kGroupsTile;
    min_part = dtype == MIE_DTYPE_F32 ? kMinPartTileF32 : kMinPartTile;
  }
  const int64_t want = std::max<int64_t>(1, groups / (p.tiles * kv_heads));
  const int64_t parts = range <= kOnePiece ? 1 : std::min<int64_t>(want, (range + min_part - 1) / min_part);
  if (parts <= 1) {
    p.parts = 1;
    p.part_keys = INT_MAX;
    p.bytes = 0;
    return p;
  }
  p.part_keys = static_cast<int>(((range + parts - 1) / parts + 127) & ~127);
  // The first key may lie up to 31 before the first one seen.
  p.parts = static_cast<int>((range + 31 + p.part_keys - 1) / p.part_keys);
  p.bytes = p.tiles * kv_heads * p.parts * rows * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
  return p;
}

int32_t check_shape(int32_t tokens, int32_t batch, int32_t max_new, int32_t max_len, int32_t window,
                    int32_t num_heads, int32_t kv_heads, int32_t head_dim, int32_t dtype) {
  const char* what = "mie_paged_extend";
  if (dtype != MIE_DTYPE_F32 && dtype != MIE_DTYPE_BF16)
    return mie::fail(MIE_ERR_UNSUPPORTED, "%s: dtype %d; float32 or bfloat16 only", what, dtype);
  if (head_dim != 32 && head_dim != 64 && head_dim != 96 && head_dim != 128 && head_dim != 256)
    return mie::fail(MIE_ERR_UNSUPPORTED, "%s: head_dim %d; 32, 64, 96, 128 or 256", what, head_dim);
  if (tokens < 0 || tokens > 1 << 22 || batch < 1 || batch > 1 << 16 || max_new < 0 || max_len < 0 || max_len > 1 << 30 ||
      window < 0)
    return mie::fail(MIE_ERR_INVALID, "%s: bad shape tokens=%d batch=%d max_new=%d max_context_len=%d window=%d", what,
                     tokens, batch, max_new, max_len, window);
  if (kv_heads < 1 || num_heads < kv_heads || num_heads % kv_heads || num_heads / kv_heads > 128 || kv_heads > 1024)
    return mie::fail(MIE_ERR_INVALID, "%s: num_heads=%d num_kv_heads=%d (at most 128 to one, 1024 of them)", what,
                     num_heads, kv_heads);
  return MIE_OK;
}

template <typename T, int D>
void launch(const Args& a, const Plan& plan, hipStream_t st) {
  const uint32_t rows = static_cast<uint32_t>(plan.tiles * a.kv_heads);
  if (plan.rows == kTileRows)
    mie::extend::launch_tiles(a, sizeof(T) == 4 ? MIE_DTYPE_F32 : MIE_DTYPE_BF16, D, st);
  else if (static_cast<int64_t>(a.max_new) * a.group.d <= kFewRows)
    extend_rows_kernel<T, D, true><<<rows * plan.parts, 256, 0, st>>>(a);
  else
    extend_rows_kernel<T, D, false><<<rows * plan.parts, 256, 0, st>>>(a);
  if (plan.parts == 1) return;
  const int lanes = join_lanes<D>(plan.parts), per_group = 256 / (D / 4) / lanes;
  const int64_t most = std::min<int64_t>(plan.rows, static_cast<int64_t>(a.max_new) * a.group.d);
  const dim3 grid(rows, static_cast<uint32_t>((most + per_group - 1) / per_group));
  if (plan.rows == kFewRows)
    extend_join_kernel<T, D, kFewRows><<<grid, 256, 0, st>>>(a, lanes);
  else
    extend_join_kernel<T, D, kTileRows><<<grid, 256, 0, st>>>(a, lanes);
}

template <typename T>
void launch_dim(const Args& a, const Plan& plan, int head_dim, hipStream_t st) {
  switch (head_dim) {
    case 32: launch<T, 32>(a, plan, st); break;
    case 64: launch<T, 64>(a, plan, st); break;
    case 96: launch<T, 96>(a, plan, st); break;
    case 128: launch<T, 128>(a, plan, st); break;
    default: launch<T, 256>(a, plan, st); break;
  }
}

}  // namespace

extern "C" int64_t mie_paged_extend_workspace(int32_t tokens, int32_t batch, int32_t max_new, int32_t max_context_len,
                                              int32_t window, int32_t num_heads, int32_t num_kv_heads,
                                              int32_t head_dim, int32_t dtype) {
  if (int32_t rc = check_shape(tokens, batch, max_new, max_context_len, window, num_heads, num_kv_heads, head_dim, dtype))
    return -rc;
  if (tokens == 0 || max_new == 0) return 0;
  return make_plan(tokens, batch, std::min(max_new, tokens), max_context_len, window, num_heads / num_kv_heads,
                   num_kv_heads, head_dim, dtype)
      .bytes;
}

extern "C" int32_t mie_paged_extend(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_pool,
                                    const void* v_pool, int64_t pool_stride_block, int64_t pool_stride_head,
                                    int32_t num_blocks, const int32_t* block_tables, int64_t table_stride,
                                    int32_t table_width, const int32_t* starts, const int32_t* context_lens,
                                    int32_t tokens, int32_t batch, int32_t max_new, int32_t max_context_len,
                                    int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                    float scale, float softcap, const float* slopes, int32_t window,
                                    const int32_t* prefix_lens, void* out, int64_t out_stride_t, int64_t out_stride_h,
                                    void* workspace, int64_t workspace_bytes, int32_t dtype, void* stream) {
  const char* what = "mie_paged_extend";
  if (int32_t rc = check_shape(tokens, batch, max_new, max_context_len, window, num_heads, num_kv_heads, head_dim, dtype))
    return rc;
  if (block_size < 1 || num_blocks < 1 || table_width < 1 || table_stride < table_width)
    return mie::fail(MIE_ERR_INVALID, "%s: block_size=%d num_blocks=%d table rows of %d, %lld apart", what, block_size,
                     num_blocks, table_width, static_cast<long long>(table_stride));
  // A larger cap would show what tanh leaves of small scores in float32.
  if (!(softcap >= 0.f) || !(softcap <= mie::extend::kMaxSoftcap) || !(fabsf(scale * kLog2e) < INFINITY) ||
      (softcap > 0.f && !(fabsf(2.f * kLog2e * scale / softcap) < INFINITY)))
    return mie::fail(MIE_ERR_INVALID, "%s: scale %g, softcap %g", what, scale, softcap);
  if (tokens == 0 || max_new == 0) return MIE_OK;
  if (!q || !k_pool || !v_pool || !starts || !context_lens || !out || !block_tables)
    return mie::fail(MIE_ERR_INVALID, "%s: null pointer", what);
  if (pool_stride_head < static_cast<int64_t>(block_size) * head_dim ||
      pool_stride_block < static_cast<int64_t>(num_kv_heads) * pool_stride_head)
    return mie::fail(MIE_ERR_INVALID, "%s: pool strides overlap", what);
  if (out_stride_h < head_dim || out_stride_t < head_dim)
    return mie::fail(MIE_ERR_INVALID, "%s: rows of out overlap", what);
  const int elt = mie::elt_size(dtype), w = 16 / elt;
  if ((q_stride_t | q_stride_h | out_stride_t | out_stride_h | pool_stride_block | pool_stride_head) % w ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool) |
        reinterpret_cast<uintptr_t>(out)) & 15))
    return mie::fail(MIE_ERR_INVALID, "%s: rows of q, out and the pools must be 16-byte aligned", what);
  max_new = std::min(max_new, tokens);
  const int group = num_heads / num_kv_heads;
  const Plan plan = make_plan(tokens, batch, max_new, max_context_len, window, group, num_kv_heads, head_dim, dtype);
  if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return mie::fail(MIE_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed (16-byte aligned)", what,
                     static_cast<long long>(workspace_bytes), static_cast<long long>(plan.bytes));
  if (plan.tiles * plan.parts * num_kv_heads > 1 << 23)
    return mie::fail(MIE_ERR_INVALID, "%s: %lld row tiles of %d heads are too many for a launch", what,
                     static_cast<long long>(plan.tiles), num_kv_heads);
  Args a;
  a.q = static_cast<const char*>(q);
  a.k_pool = static_cast<const char*>(k_pool);
  a.v_pool = static_cast<const char*>(v_pool);
  a.out = static_cast<char*>(out);
  a.q_st = q_stride_t * elt;
  a.q_sh = q_stride_h * elt;
  a.out_st = out_stride_t * elt;
  a.out_sh = out_stride_h * elt;
  a.sblk = pool_stride_block * elt;
  a.shead = pool_stride_head * elt;
  a.num_blocks = num_blocks;
  a.tables = block_tables;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.starts = starts;
  a.lens = context_lens;
  a.tokens = tokens;
  a.batch = batch;
  a.max_new = max_new;
  a.max_len = max_context_len;
  a.kv_heads = num_kv_heads;
  a.scale = softcap > 0.f ? 2.f * kLog2e * scale / softcap : scale * kLog2e;
  a.cap = softcap * kLog2e;
  a.cap_ratio = softcap > 0.f ? scale / softcap : 0.f;
  a.slopes = slopes;
  a.window = window > 1 << 30 ? 0 : window;  // no length reaches farther; positions less the window stay in 31 bits
  a.prefix = prefix_lens;
  a.whole_blocks = block_size % 16 == 0;
  a.tiles = static_cast<int32_t>(plan.tiles);
  a.parts = plan.parts;
  a.part_keys = plan.part_keys;
  a.ws_acc = static_cast<float*>(workspace);
  a.ws_ml = a.ws_acc + plan.tiles * num_kv_heads * plan.parts * plan.rows * head_dim;
  a.group = mie::FastDiv::make(static_cast<uint32_t>(group));
  a.bs = mie::FastDiv::make(static_cast<uint32_t>(block_size));
  mie::clear_error();
  if (dtype == MIE_DTYPE_F32)
    launch_dim<float>(a, plan, head_dim, static_cast<hipStream_t>(stream));
  else
    launch_dim<uint16_t>(a, plan, head_dim, static_cast<hipStream_t>(stream));
  return mie::check_launch(what);
}
