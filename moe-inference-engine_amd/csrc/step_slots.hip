// A serving step's pages from lengths on the device (mie_step_reserve,
// mie_step_release): block ids off and onto a stack of free blocks, block
// tables, packed starts, slots and positions.
//
// Mathematics: two exclusive prefix sums over the batch, of the new tokens and
// of the new blocks.  A token's sequence is the last one whose start is not
// past it; its block is either one the sequence held (read from the table) or
// the j-th block the step takes, which is free_ids[count - 1 - j].
//
// One launch.  Every workgroup sums the whole batch itself (a few KB of
// lengths from the cache), so none waits for another, and then maps its share
// of the tokens; workgroup 0 also writes what there is one of per sequence.
// Nothing that is read is written in the same launch: the table entries
// written are those of blocks the step takes, the entries read those of blocks
// held before, and the counts and lengths go to other arrays.  Bound by
// latency (three dependent rounds and two scans): on MI355X 4.5 us for a decode
// step of 64 sequences, 10.6 us for a million tokens of 500 (13 MB, 2.6 us at
// the rate of a copy), 7.2 us for the release of 1000 sequences' 250 000 blocks.
#include <limits.h>

#include <algorithm>

#include "mie_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBatch = 8192;
constexpr int kMaxGroups = 1024;
constexpr int kMaxItems = 1 << 30;  // tokens or blocks of a step: the strided loops stay in 31 bits

enum StepStatus { kOk = 0, kNoBlocks = 1, kTableFull = 2, kTooManyTokens = 3, kBadLength = 4 };

__device__ __forceinline__ int wave_inclusive(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  return x;
}

// Exclusive prefix sums of (a, b) over the workgroup's threads.
__device__ __forceinline__ void block_exclusive(int& a, int& b, int (*s)[kThreads / 64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ia = wave_inclusive(a), ib = wave_inclusive(b);
  if (lane == 63) {
    s[0][wave] = ia;
    s[1][wave] = ib;
  }
  __syncthreads();
  int pa = 0, pb = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) {
      pa += s[0][w];
      pb += s[1][w];
    }
  }
  a = pa + ia - a;
  b = pb + ib - b;
}

// The largest i in [0, n) with first[i] <= x (first[0] = 0 <= x, ascending).
__device__ __forceinline__ int last_at_or_below(const int* first, int n, int x) {
  int low = 0, high = n;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (first[mid] <= x)
      low = mid;
    else
      high = mid;
  }
  return low;
}

// ceil(tokens / block_size): tokens + d - 1 stays below 2^31 where FastDiv is
// exact, because a length past its row of the table was refused.
__device__ __forceinline__ int blocks_of(mie::FastDiv bs, int tokens) {
  const uint32_t q = bs.div(static_cast<uint32_t>(tokens));
  return static_cast<int>(q) + (q * bs.d != static_cast<uint32_t>(tokens));
}

// What the workgroup's threads found, in every thread: the worst status and
// the 64-bit totals.
struct Totals {
  long long tokens, blocks;
  int bad, full;
};
__device__ __forceinline__ Totals block_totals(Totals t) {
  __shared__ long long s_tokens[kThreads / 64], s_blocks[kThreads / 64];
  __shared__ int s_bad[kThreads / 64], s_full[kThreads / 64];
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    t.tokens += __shfl_xor(t.tokens, off);
    t.blocks += __shfl_xor(t.blocks, off);
  }
  t.bad = __any(t.bad);
  t.full = __any(t.full);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    s_tokens[wave] = t.tokens;
    s_blocks[wave] = t.blocks;
    s_bad[wave] = t.bad;
    s_full[wave] = t.full;
  }
  __syncthreads();
  t = Totals{0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    t.tokens += s_tokens[w];
    t.blocks += s_blocks[w];
    t.bad |= s_bad[w];
    t.full |= s_full[w];
  }
  return t;
}

struct ReserveArgs {
  const int32_t* free_ids;
  int32_t capacity;
  const int32_t* free_count;
  int32_t* tables;
  int64_t table_stride;
  int32_t table_width;
  const int32_t* lens;
  const int32_t* news;
  int32_t batch;
  int32_t max_tokens;
  int32_t* starts;
  int64_t* slots;
  int32_t* positions;
  int32_t* lens_out;
  int32_t* count_out;
  int32_t* status;
  mie::FastDiv bs;
};

// LDS: s_start[batch], s_block[batch] (dynamic).  A thread maps kRun
// consecutive tokens: one search and 16-byte stores for four where there are
// many (a million tokens of 500 sequences 12.4 -> 10.6 us), one where a chain
// of four is longer than the launch needs (64 tokens 4.5 us, 5.7 with four).
template <int kRun>
__global__ __launch_bounds__(kThreads) void step_reserve_kernel(ReserveArgs a) {
  extern __shared__ int s_dyn[];
  __shared__ int s_scan[2][kThreads / 64];
  int* s_start = s_dyn;
  int* s_block = s_dyn + a.batch;
  const int tid = threadIdx.x;
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  const int count = *a.free_count;
  const long long row_tokens = static_cast<long long>(a.table_width) * a.bs.d;

  Totals t{0, 0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    const int c = a.lens[b], n = a.news[b];
    const bool bad = c < 0 || n < 0;
    const bool full = !bad && static_cast<long long>(c) + n > row_tokens;
    t.bad |= bad;
    t.full |= full;
    if (!bad && !full) {
      t.tokens += n;
      t.blocks += blocks_of(a.bs, c + n) - blocks_of(a.bs, c);
    }
  }
  const int my_tokens = static_cast<int>(t.tokens), my_blocks = static_cast<int>(t.blocks);
  t = block_totals(t);
  const int status = t.bad || count < 0 || count > a.capacity ? kBadLength
                     : t.full                                 ? kTableFull
                     : t.tokens > a.max_tokens                ? kTooManyTokens
                     : t.blocks > count                       ? kNoBlocks
                                                              : kOk;
  const bool first = blockIdx.x == 0;
  const int stride = gridDim.x * kThreads;
  const bool vectors = ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0;
  if (first && tid == 0) {
    *a.status = status;
    *a.count_out = status == kOk ? count - static_cast<int>(t.blocks) : count;
  }
  if (status != kOk) {
    if (first) {
      for (int b = tid; b < a.batch; b += kThreads) a.lens_out[b] = a.lens[b];
      for (int b = tid; b <= a.batch; b += kThreads) a.starts[b] = 0;
    }
    for (int i = blockIdx.x * kThreads + tid; i < a.max_tokens; i += stride) {
      a.slots[i] = -1;
      a.positions[i] = 0;
    }
    return;
  }

  // Exact from here on: every total fits 31 bits (tokens <= max_tokens, blocks <= count).
  int start = my_tokens, block = my_blocks;
  block_exclusive(start, block, s_scan);
  for (int b = b0; b < b1; ++b) {
    const int c = a.lens[b], n = a.news[b];
    s_start[b] = start;
    s_block[b] = block;
    if (first) {
      a.starts[b] = start;
      a.lens_out[b] = c + n;
    }
    start += n;
    block += blocks_of(a.bs, c + n) - blocks_of(a.bs, c);
  }
  const int total = static_cast<int>(t.tokens);
  if (first && tid == 0) a.starts[a.batch] = total;
  __syncthreads();

  for (int i0 = (blockIdx.x * kThreads + tid) * kRun; i0 < a.max_tokens; i0 += stride * kRun) {
    int64_t slot[kRun];
    int32_t position[kRun];
    if (i0 >= total) {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        slot[j] = -1;
        position[j] = 0;
      }
    } else {
      // Of the sequences that start here the last one has tokens, the others none.
      int b = last_at_or_below(s_start, a.batch, i0);
      int c = a.lens[b], from = s_start[b], until = b + 1 < a.batch ? s_start[b + 1] : total;
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        const int i = i0 + j;
        slot[j] = -1;
        position[j] = 0;
        if (i >= total) continue;
        while (i >= until) {  // on to the next sequence with tokens
          ++b;
          from = until;
          until = b + 1 < a.batch ? s_start[b + 1] : total;
          c = a.lens[b];
        }
        const int p = c + i - from;
        const int blk = static_cast<int>(a.bs.div(static_cast<uint32_t>(p)));
        const int offset = p - blk * static_cast<int>(a.bs.d);
        const int held = blocks_of(a.bs, c);
        int32_t* entry = a.tables + b * a.table_stride + blk;
        int id;
        if (blk >= held) {
          id = a.free_ids[count - 1 - (s_block[b] + blk - held)];
          if (offset == 0) *entry = id;  // a taken block's first token is a new one
        } else {
          id = *entry;
        }
        slot[j] = static_cast<int64_t>(id) * a.bs.d + offset;
        position[j] = p;
      }
    }
    if (kRun == 4 && vectors && i0 + kRun <= a.max_tokens) {
      typedef long long i64x2 __attribute__((ext_vector_type(2)));
      typedef int i32x4 __attribute__((ext_vector_type(4)));
      *reinterpret_cast<i64x2*>(a.slots + i0) = i64x2{slot[0], slot[1 % kRun]};
      *reinterpret_cast<i64x2*>(a.slots + i0 + 2) = i64x2{slot[2 % kRun], slot[3 % kRun]};
      *reinterpret_cast<i32x4*>(a.positions + i0) = i32x4{position[0], position[1 % kRun], position[2 % kRun], position[3 % kRun]};
    } else {
#pragma unroll
      for (int j = 0; j < kRun; ++j)
        if (i0 + j < a.max_tokens) {
          a.slots[i0 + j] = slot[j];
          a.positions[i0 + j] = position[j];
        }
    }
  }
}

struct ReleaseArgs {
  int32_t* free_ids;
  int32_t capacity;
  const int32_t* free_count;
  const int32_t* tables;
  int64_t table_stride;
  int32_t table_width;
  const int32_t* lens;
  const uint8_t* finished;
  int32_t batch;
  int32_t* lens_out;
  int32_t* count_out;
  int32_t* status;
  mie::FastDiv bs;
};

// LDS: s_block[batch] (dynamic).
__global__ __launch_bounds__(kThreads) void step_release_kernel(ReleaseArgs a) {
  extern __shared__ int s_dyn[];
  __shared__ int s_scan[2][kThreads / 64];
  int* s_block = s_dyn;
  const int tid = threadIdx.x;
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  const int count = *a.free_count;
  const long long row_tokens = static_cast<long long>(a.table_width) * a.bs.d;

  Totals t{0, 0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    if (!a.finished[b]) continue;
    const int c = a.lens[b];
    t.bad |= c < 0;
    t.full |= c > row_tokens;
    if (c >= 0 && c <= row_tokens) t.blocks += blocks_of(a.bs, c);
  }
  int block = static_cast<int>(t.blocks), unused = 0;
  t = block_totals(t);
  const int status = t.bad || count < 0 || count > a.capacity ? kBadLength
                     : t.full                                 ? kTableFull
                     : t.blocks > a.capacity - count          ? kNoBlocks
                                                              : kOk;
  const bool first = blockIdx.x == 0;
  if (first) {
    if (tid == 0) {
      *a.status = status;
      *a.count_out = status == kOk ? count + static_cast<int>(t.blocks) : count;
    }
    for (int b = tid; b < a.batch; b += kThreads) a.lens_out[b] = status == kOk && a.finished[b] ? 0 : a.lens[b];
  }
  if (status != kOk) return;

  block_exclusive(block, unused, s_scan);
  for (int b = b0; b < b1; ++b) {
    s_block[b] = block;
    if (a.finished[b]) block += blocks_of(a.bs, a.lens[b]);
  }
  __syncthreads();
  const int total = static_cast<int>(t.blocks);
  for (int i = blockIdx.x * kThreads + tid; i < total; i += gridDim.x * kThreads) {
    const int b = last_at_or_below(s_block, a.batch, i);
    a.free_ids[count + i] = a.tables[b * a.table_stride + (i - s_block[b])];
  }
}

int32_t check_step(const char* what, int32_t capacity, int64_t table_stride, int32_t table_width, int32_t batch,
                   int32_t block_size) {
  if (batch < 1 || batch > kMaxBatch)
    return mie::fail(MIE_ERR_INVALID, "%s: batch %d outside [1, %d]", what, batch, kMaxBatch);
  if (block_size < 1) return mie::fail(MIE_ERR_INVALID, "%s: block_size %d", what, block_size);
  if (capacity < 1 || capacity > kMaxItems)
    return mie::fail(MIE_ERR_INVALID, "%s: a free list of %d entries", what, capacity);
  if (table_width < 1 || table_stride < table_width)
    return mie::fail(MIE_ERR_INVALID, "%s: table rows of %d entries, %lld apart", what, table_width,
                     static_cast<long long>(table_stride));
  // Positions and lengths are 31-bit (FastDiv's range).
  if (static_cast<int64_t>(table_width) * block_size > INT32_MAX)
    return mie::fail(MIE_ERR_INVALID, "%s: a table row of %d blocks of %d holds more than 2^31 - 1 tokens", what,
                     table_width, block_size);
  return MIE_OK;
}

template <typename... P>
bool any_null(P... p) {
  return (... || (p == nullptr));
}

}  // namespace

extern "C" int32_t mie_step_reserve(const int32_t* free_ids, int32_t capacity, const int32_t* free_count,
                                    int32_t* block_tables, int64_t table_stride, int32_t table_width,
                                    const int32_t* context_lens, const int32_t* new_lens, int32_t batch,
                                    int32_t block_size, int32_t max_tokens, int32_t* starts, int64_t* slots,
                                    int32_t* positions, int32_t* context_lens_out, int32_t* free_count_out,
                                    int32_t* status, void* stream) {
  if (int32_t rc = check_step("mie_step_reserve", capacity, table_stride, table_width, batch, block_size)) return rc;
  if (max_tokens < 0 || max_tokens > kMaxItems) return mie::fail(MIE_ERR_INVALID, "mie_step_reserve: max_tokens %d", max_tokens);
  if (any_null(free_ids, free_count, block_tables, context_lens, new_lens, starts, context_lens_out, free_count_out,
               status) ||
      (max_tokens > 0 && any_null(slots, positions)))
    return mie::fail(MIE_ERR_INVALID, "mie_step_reserve: null pointer");
  if (context_lens_out == context_lens || context_lens_out == new_lens || free_count_out == free_count)
    return mie::fail(MIE_ERR_INVALID, "mie_step_reserve: the outputs must not alias the inputs");
  ReserveArgs a{free_ids, capacity, free_count, block_tables, table_stride, table_width, context_lens, new_lens, batch,
                max_tokens, starts, slots, positions, context_lens_out, free_count_out, status,
                mie::FastDiv::make(static_cast<uint32_t>(block_size))};
  const int run = max_tokens > kThreads * 256 ? 4 : 1;
  const int groups = std::clamp((max_tokens - 1) / (kThreads * run) + 1, 1, kMaxGroups);
  const size_t lds = 2 * sizeof(int) * batch;
  mie::clear_error();
  if (run == 4)
    step_reserve_kernel<4><<<groups, kThreads, lds, static_cast<hipStream_t>(stream)>>>(a);
  else
    step_reserve_kernel<1><<<groups, kThreads, lds, static_cast<hipStream_t>(stream)>>>(a);
  return mie::check_launch("mie_step_reserve");
}

extern "C" int32_t mie_step_release(int32_t* free_ids, int32_t capacity, const int32_t* free_count,
                                    const int32_t* block_tables, int64_t table_stride, int32_t table_width,
                                    const int32_t* context_lens, const uint8_t* finished, int32_t batch,
                                    int32_t block_size, int32_t* context_lens_out, int32_t* free_count_out,
                                    int32_t* status, void* stream) {
  if (int32_t rc = check_step("mie_step_release", capacity, table_stride, table_width, batch, block_size)) return rc;
  if (any_null(free_ids, free_count, block_tables, context_lens, finished, context_lens_out, free_count_out, status))
    return mie::fail(MIE_ERR_INVALID, "mie_step_release: null pointer");
  if (context_lens_out == context_lens || free_count_out == free_count)
    return mie::fail(MIE_ERR_INVALID, "mie_step_release: the outputs must not alias the inputs");
  ReleaseArgs a{free_ids, capacity, free_count, block_tables, table_stride, table_width, context_lens, finished, batch,
                context_lens_out, free_count_out, status, mie::FastDiv::make(static_cast<uint32_t>(block_size))};
  const int64_t most = std::min<int64_t>(static_cast<int64_t>(batch) * table_width, capacity);
  const int groups = static_cast<int>(std::clamp<int64_t>((most - 1) / kThreads + 1, 1, kMaxGroups));
  mie::clear_error();
  step_release_kernel<<<groups, kThreads, sizeof(int) * batch, static_cast<hipStream_t>(stream)>>>(a);
  return mie::check_launch("mie_step_release");
}
