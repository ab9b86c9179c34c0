// What the kernels of mie_paged_extend share: the call, a workgroup's place in
// it (sequence, rows, keys), scores and the softmax's steps.
//
// Rows.  The rows of one K/V head are its query heads' rows of every new token
// of a sequence, token after token: row r is token r / group, head r % group,
// group = num_heads / num_kv_heads.  Grouped heads thereby share every key
// that is read.
#pragma once

#include <limits.h>
#include <math.h>

#include "gemm_tile.h"
#include "mie_common.h"

namespace mie {
namespace extend {

using gemm::f32x4;
using gemm::u32x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMaxSoftcap = 1024.f;
constexpr int kFewRows = 16;    // rows per workgroup where a sequence has few (extend_rows_kernel)
constexpr int kTileRows = 128;  // and where it has many (extend_tile_kernel)

struct Args {
  const char* q;
  const char* k_pool;
  const char* v_pool;
  char* out;
  int64_t q_st, q_sh, out_st, out_sh, sblk, shead;  // bytes
  int32_t num_blocks;
  const int32_t* tables;
  int64_t table_stride;
  int32_t table_width;
  const int32_t* starts;
  const int32_t* lens;
  int32_t tokens, batch, max_new, max_len, kv_heads;
  float scale;      // log2(e) / sqrt(D), or as the caller gave it; with a cap 2 log2(e) scale / cap
  float cap;        // softcap * log2(e), or 0
  float cap_ratio;  // scale / softcap (float32's tanh)
  const float* slopes;
  int32_t window;
  const int32_t* prefix;
  int32_t tiles;             // row tiles of the launch, a bound
  int32_t parts, part_keys;  // a row tile's keys in at most `parts` pieces, of part_keys or more
  float* ws_acc;             // [tile, kv head, part, row, D]
  float* ws_ml;              // [tile, kv head, part, row, 2]
  int32_t whole_blocks;      // blocks hold a multiple of 16 keys
  FastDiv group, bs;
};

// A workgroup's rows and keys.
struct Place {
  int b;                // sequence; -1: none
  int start, count, len;  // first token in q, new tokens, context length
  int row0, rows;       // of the sequence's rows: this tile's first one, and how many the sequence has
  int p_first, p_last;  // positions of the tile's first and last row
  int prefix;
  int low, high;  // keys any row of the tile sees lie in [low, high); low is a multiple of 32
  bool bad;       // a length past the bound
};

__device__ __forceinline__ int new_tokens(const Args& a, int b, int& start) {
  const int s = min(max(a.starts[b], 0), a.tokens), e = min(max(a.starts[b + 1], s), a.tokens);
  start = s;
  return e - s;
}

// The place of row tile `tile` of the batch, ROWS rows per tile.  Every lane
// of the wave gets the same (wave-uniform) answer.
template <int ROWS>
__device__ __forceinline__ Place find_place(const Args& a, int tile) {
  Place p;
  p.b = -1;
  int in_seq = 0;
  const int group = a.group.d;
  const int lane = threadIdx.x & 63;
  if (a.max_new * group <= ROWS) {  // at most one tile per sequence
    p.b = tile < a.batch ? tile : -1;
  } else {
    int seen = 0;
    for (int base = 0; base < a.batch; base += 64) {
      int tiles = 0, unused;
      if (base + lane < a.batch)
        tiles = (min(new_tokens(a, base + lane, unused), a.max_new) * group + ROWS - 1) / ROWS;
      int upto = tiles;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(upto, off);
        if (lane >= off) upto += y;
      }
      const uint64_t past = __ballot(seen + upto > tile);
      if (past) {
        const int l = __builtin_ctzll(past);
        p.b = base + l;
        in_seq = tile - seen - __builtin_amdgcn_readlane(upto - tiles, l);
        break;
      }
      seen += __builtin_amdgcn_readlane(upto, 63);
    }
  }
  p.b = __builtin_amdgcn_readfirstlane(p.b);
  in_seq = __builtin_amdgcn_readfirstlane(in_seq);
  if (p.b < 0) return p;
  int n = new_tokens(a, p.b, p.start);
  p.count = n;
  p.len = max(a.lens[p.b], 0);
  p.bad = p.len > a.max_len;
  n = min(n, a.max_new);
  p.rows = n * group;
  p.row0 = in_seq * ROWS;
  if (p.row0 >= p.rows) {  // a sequence without new tokens
    p.b = -1;
    return p;
  }
  const int base = p.len - p.count;
  p.p_first = base + static_cast<int>(a.group.div(p.row0));
  p.p_last = base + static_cast<int>(a.group.div(min(p.row0 + ROWS, p.rows) - 1));
  p.prefix = a.prefix ? min(a.prefix[p.b], p.len) : 0;
  p.high = min(p.len, max(p.p_last + 1, p.prefix));
  p.low = a.window > 0 ? max(0, p.p_first - a.window + 1) & ~31 : 0;
  if (p.bad || p.high < p.low) p.high = p.low;
  return p;
}

// A workgroup's K/V head, row tile and part: heads side by side, then tiles,
// all first parts before the second ones.  Workgroups go to the XCDs and their
// shader engines in turn, and a short tile's later parts are empty: with a
// tile's parts side by side the engines at the places of the later ones had
// less to do (8 chunks of 100 to 500 float32 tokens behind 1000 to 4000 in two
// parts 1810 us, 945 this way; 64 decode tokens 222 and 212).  For the same
// reason the tiles of each part start one later.
struct Item {
  int kvh, tile, part;
};
__device__ __forceinline__ Item item_of(const Args& a) {
  const int kvh = blockIdx.x % a.kv_heads, item = blockIdx.x / a.kv_heads;
  const int part = item / a.tiles;
  return Item{kvh, (item + part) % a.tiles, part};
}

// Pieces the tile's keys come in: at least one (empty rows are written too), at
// most those the launch and the workspace have, each larger where these do not
// hold the keys (a prefix may end far beyond the window the host counted).
struct Split {
  int parts, keys;
};
__device__ __forceinline__ Split split_of(const Args& a, const Place& p) {
  if (a.parts == 1) return Split{1, INT_MAX};
  const int range = p.high - p.low;
  const int keys = max(a.part_keys, ((range + a.parts - 1) / a.parts + 127) & ~127);
  return Split{max(1, (range + keys - 1) / keys), keys};
}

// The keys a token sees are [low, high): those up to its own position or the
// prefix's end, from the window's first on.
struct Range {
  int low, high;
};
__device__ __forceinline__ Range keys_of(const Args& a, const Place& p, int position) {
  return Range{a.window > 0 ? max(0, position - a.window + 1) : 0, min(p.len, max(position + 1, p.prefix))};
}
// The keys every row of two positions and those between them sees.
__device__ __forceinline__ Range shared_keys(const Args& a, const Place& p, int first, int last) {
  return Range{keys_of(a, p, last).low, keys_of(a, p, first).high};
}
__device__ __forceinline__ bool holds(Range r, int k0, int k1) { return k0 >= r.low && k1 <= r.high; }
__device__ __forceinline__ bool holds(Range r, int key) {
  return static_cast<uint32_t>(key - r.low) < static_cast<uint32_t>(max(r.high - r.low, 0));
}

// cap tanh(q . k scale / softcap) in base 2 (Args: cap, scale, cap_ratio).
// tanh(x) = 1 - 2 / (exp(2 x) + 1) has an absolute error of 2^-23, times the
// cap a few 1e-6 of the exponent (at most 4e-4, kMaxSoftcap), which bfloat16
// does not show; float32 takes the library's.
template <typename T>
__device__ __forceinline__ float capped(float dot, float cap, float scale, float ratio) {
  if constexpr (sizeof(T) == 4) return cap * tanhf(dot * ratio);
  return fmaf(-2.f * cap, __builtin_amdgcn_rcpf(fast_exp2(dot * scale) + 1.f), cap);
}
// The score's base-2 exponent from q . k; `slope` is the head's times log2(e),
// `away` the position less the key's.
template <typename T>
__device__ __forceinline__ float exponent(const Args& a, float dot, float slope, float away) {
  const float x = a.cap > 0.f ? capped<T>(dot, a.cap, a.scale, a.cap_ratio) : dot * a.scale;
  return a.slopes ? fmaf(-slope, fabsf(away), x) : x;
}

// Byte offset of a key's row in one head of the pool, from its table entry;
// for an id outside the pool a row of block 0, and `bad`.
__device__ __forceinline__ int64_t row_offset(const Args& a, int key, int32_t id, int row_bytes, bool& bad) {
  bad = static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.num_blocks);
  const uint32_t blk = a.bs.div(static_cast<uint32_t>(key));
  const uint32_t slot = static_cast<uint32_t>(key) - blk * a.bs.d;
  return (bad ? 0 : id) * a.sblk + static_cast<int64_t>(slot) * row_bytes;
}
// The table entry of a key (which is below the sequence's length); -1 past the row.
__device__ __forceinline__ int32_t entry_of(const Args& a, int b, int key) {
  const int blk = static_cast<int>(a.bs.div(static_cast<uint32_t>(key)));
  const int32_t id = a.tables[b * a.table_stride + min(blk, a.table_width - 1)];
  return blk < a.table_width ? id : -1;
}

// x combined over the four 16-lane groups (lanes i, i + 16, i + 32, i + 48).
template <bool MAX>
__device__ __forceinline__ float across_groups(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float u = __uint_as_float(a[0]), v = __uint_as_float(a[1]);
  x = MAX ? fmaxf(u, v) : u + v;
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float s = __uint_as_float(a[0]), t = __uint_as_float(a[1]);
  return MAX ? fmaxf(s, t) : s + t;
}

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }
// The same for bfloat16: the largest magnitude in each half of the words taken.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void take_magnitudes(u16x2& most, uint32_t w) {
  most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w & 0x7fff7fffu));
}
__device__ __forceinline__ bool not_finite(u16x2 most) { return most.x >= 0x7f80u || most.y >= 0x7f80u; }

// Launches extend_tile_kernel (float32 or bfloat16, the head_dims checked).
void launch_tiles(const Args& a, int dtype, int head_dim, hipStream_t stream);

}  // namespace extend
}  // namespace mie
