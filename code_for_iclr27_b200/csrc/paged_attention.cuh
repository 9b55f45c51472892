// What the paged attention's kernels share: their parameters, the even split of
// all slots' tiles over a persistent grid, and the join of units that several
// blocks took a part of.
//
// The tiles of all units (a slot and a block of its query rows), laid end to
// end, are divided evenly over the blocks, so neither few slots nor ragged ones
// leave SMs idle.  A unit whose tiles fall to several blocks leaves partial
// results (maximum, sum, output) in the workspace; the block that arrives last
// joins them in a fixed order, so the result does not depend on the arrival.
#pragma once

#include <atomic>

#include "paged.cuh"
#include "tc.cuh"

namespace lrk {
namespace {

using namespace paged;

// cudaFuncSetAttribute once per kernel and device (it costs a microsecond a call).
template <typename K>
int allow_shared(K kernel, int bytes, std::atomic<uint64_t> &allowed) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && device < 64 && (allowed.load(std::memory_order_relaxed) >> device & 1)) return LRK_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(LRK_ERR_CUDA, cudaGetErrorString(e));
  if (device < 64) allowed.fetch_or(uint64_t{1} << device, std::memory_order_relaxed);
  return LRK_OK;
}

constexpr int kCounters = 4096;  // workspace: arrival counters (zero between calls), then partial results

// Division by a number that the host knows: n / d for n below 2^31 as a
// product (Granlund and Montgomery's round-up method).
struct Divider {
  uint32_t multiplier, shift;
  static Divider of(uint32_t d) {
    Divider r{0, 0};
    while ((uint64_t{1} << r.shift) < d) ++r.shift;
    r.multiplier = static_cast<uint32_t>(((((uint64_t{1} << r.shift) - d) << 32) / d) + 1);
    return r;
  }
  __device__ __forceinline__ int32_t operator()(int32_t n) const {
    return static_cast<int32_t>((__umulhi(static_cast<uint32_t>(n), multiplier) + static_cast<uint32_t>(n)) >> shift);
  }
};

struct AttentionParam {
  Pages pages;
  const int32_t *table;
  int64_t table_stride;
  int32_t capacity;  // rows that a slot's table entries can hold
  const int32_t *lengths;
  const int32_t *token_starts;
  int32_t slots, tokens;
  const void *queries;
  int64_t query_token, query_head;
  int heads, groups;
  Divider by_heads, by_groups;
  float scale_log2;
  bool causal;
  void *out;
  float *lse;
  uint32_t *counters;
  float *partials;
  uint32_t *flag;
};

__device__ __forceinline__ uint32_t shared_address(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 2^x to a relative 2^-22 or so; results below 2^-126 are 0.
// The weights are rounded to 11 or 8 bits after it.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void bulk_copy(uint32_t to, const void *from, uint32_t bytes, uint32_t barrier) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(to),
               "l"(from), "r"(bytes), "r"(barrier)
               : "memory");
}

__device__ __noinline__ bool wait_long(uint32_t barrier, uint32_t parity, volatile int *abort) {
  return tc::wait_phase(barrier, parity, abort);
}
// Bounded wait for an mbarrier phase; the clock is read only after some tries.
__device__ __forceinline__ bool wait(uint32_t barrier, uint32_t parity, volatile int *abort) {
  uint32_t done = 0;
#pragma unroll 1
  for (int i = 0; i < 64 && !done; ++i)
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(barrier), "r"(parity)
        : "memory");
  return done || wait_long(barrier, parity, abort);
}

// a / b for a >= 0, b > 0.  Out of line: the 64-bit division is some hundred
// instructions that hardly any call needs.
__device__ __noinline__ int64_t divide_long(int64_t a, int64_t b) { return a / b; }
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return divide_long(a, b);
}

// A stretch of one unit's tiles: a unit is a slot and a block of its query rows.
struct Segment {
  int64_t unit_start;                   // where the unit begins among all units' tiles
  int32_t unit_tiles;
  int32_t slot, sequence;
  int32_t tokens, first_token;          // of the sequence
  int32_t row0;                         // first query row (token * groups + head in group) of the unit
  int32_t length;                       // of the slot
  int32_t tile0, tile1;                 // tiles of the stretch, those beyond every query's rows left out
  int32_t seen_max, seen_min;           // rows seen by the unit's last and first query
  bool starts, ends;                    // the stretch holds the unit's first / last tile
};

static_assert(sizeof(Segment) <= 64, "the layout keeps 64 bytes for a segment");

// What a slot asks for: tiles per unit (at least one, so that a query without
// a visible row gets its zeros), and units.
template <int ROWS, int TILE>
__device__ __forceinline__ void slot_work(const AttentionParam &p, int32_t slot, Segment &s, int32_t &units) {
  s.slot = slot;
  s.sequence = p.by_heads(slot);
  s.first_token = min(max(p.token_starts[s.sequence], 0), p.tokens);
  s.tokens = max(min(p.token_starts[s.sequence + 1], p.tokens) - s.first_token, 0);
  s.length = min(max(p.lengths[slot], 0), p.capacity);
  s.unit_tiles = max((s.length + TILE - 1) / TILE, 1);
  units = (s.tokens * p.groups + ROWS - 1) / ROWS;
}

__device__ __forceinline__ int32_t rows_seen(const AttentionParam &p, const Segment &s, int32_t row) {
  return p.causal ? max(s.length - s.tokens + p.by_groups(row) + 1, 0) : s.length;
}

// Walks a block's share of all units' tiles, laid end to end with every unit
// rounded up to a multiple of `round` tiles.
template <int ROWS, int TILE>
struct Walk {
  int64_t position, end;
  int64_t slot_start;
  int32_t slot, round;

  __device__ __forceinline__ bool next(const AttentionParam &p, Segment &s) {
    if (position >= end) return false;
    int64_t span;
    for (;; ++slot) {
      if (slot >= p.slots) return false;
      int32_t units;
      slot_work<ROWS, TILE>(p, slot, s, units);
      span = round == 1 ? s.unit_tiles : static_cast<int64_t>((s.unit_tiles + round - 1) / round) * round;
      if (position < slot_start + span * units) break;
      slot_start += span * units;
    }
    const int64_t unit = divide(position - slot_start, span);
    s.unit_start = slot_start + unit * span;
    s.tile0 = static_cast<int32_t>(position - s.unit_start);
    const int64_t stop = lmin(end, s.unit_start + span);
    s.tile1 = min(static_cast<int32_t>(stop - s.unit_start), s.unit_tiles);
    s.starts = s.tile0 == 0;
    s.ends = s.tile1 == s.unit_tiles;
    position = stop;
    s.row0 = static_cast<int32_t>(unit * ROWS);
    s.seen_min = rows_seen(p, s, s.row0);
    s.seen_max = rows_seen(p, s, min(s.row0 + ROWS, s.tokens * p.groups) - 1);
    s.tile1 = min(s.tile1, (s.seen_max + TILE - 1) / TILE);
    return true;
  }
};

// Tokens of no sequence (before the first one's `start`, from the last one's
// `stop` on) see nothing: one block writes their outputs.  Out of line: hardly any
// call needs it, and every block would fetch its instructions.
template <int D, int THREADS>
__device__ __noinline__ void fill_lost(const AttentionParam &p, int32_t start, int32_t stop) {
  if (threadIdx.x == 0) atomicOr(p.flag, kFlagRow);
  const int32_t before = min(max(start, 0), p.tokens), after = min(max(stop, 0), p.tokens);
  const int64_t rows = static_cast<int64_t>(before + p.tokens - after) * p.heads * p.groups;
  for (int64_t i = threadIdx.x; i < rows * (D / 8); i += THREADS) {
    int64_t row = i / (D / 8);
    if (row >= static_cast<int64_t>(before) * p.heads * p.groups)
      row += static_cast<int64_t>(after - before) * p.heads * p.groups;
    static_cast<uint4 *>(p.out)[row * (D / 8) + i % (D / 8)] = make_uint4(0, 0, 0, 0);
    if (i % (D / 8) == 0) p.lse[row] = -INFINITY;
  }
}

// A block's share of the work and its first segment; false for a block without
// any.  sums: 2 x THREADS / 32 shared words.  Ends with a barrier.
template <int D, int THREADS, int MIN_TILES, int CROSSING, int ROWS, int TILE>
__device__ __forceinline__ bool begin(const AttentionParam &p, int64_t *sums, int64_t &share,
                                      Walk<ROWS, TILE> &of_block, Segment &segment) {
  constexpr int kWarps = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t each = (p.slots + THREADS - 1) / THREADS;
  const int32_t mine0 = min(static_cast<int32_t>(threadIdx.x) * each, p.slots), mine1 = min(mine0 + each, p.slots);
  Segment s;
  int64_t tiles_sum = 0, units_sum = 0;
  int32_t units = 0;
  for (int32_t i = mine0; i < mine1; ++i) {
    slot_work<ROWS, TILE>(p, i, s, units);
    units_sum += units;
    tiles_sum += static_cast<int64_t>(units) * s.unit_tiles;
    if (blockIdx.x == 0 && (p.lengths[i] != s.length || p.token_starts[s.sequence + 1] < p.token_starts[s.sequence]))
      atomicOr(p.flag, kFlagRow);  // a length that is negative or beyond the table, or starts that descend
  }
#pragma unroll
  for (int step = 16; step > 0; step >>= 1) {
    tiles_sum += __shfl_xor_sync(0xffffffffu, tiles_sum, step);
    units_sum += __shfl_xor_sync(0xffffffffu, units_sum, step);
  }
  if (lane == 0) {
    sums[warp] = tiles_sum;
    sums[kWarps + warp] = units_sum;
  }
  __syncthreads();
  if (blockIdx.x == gridDim.x - 1) {  // it has the least to do
    const int32_t start = p.token_starts[0], stop = p.token_starts[p.by_heads(p.slots)];
    if (start != 0 || stop != p.tokens) fill_lost<D, THREADS>(p, start, stop);
  }
  tiles_sum = units_sum = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    tiles_sum += sums[w];
    units_sum += sums[kWarps + w];
  }
  // Shares are equal and cross the units' ends, or, where that costs at most
  // CROSSING tiles more a block, every block takes a piece of one unit alone (a
  // unit rounded up to whole pieces: sum ceil(tiles / share) <= tiles_sum /
  // share + units <= grid).  CROSSING is what a second unit costs a block (its
  // queries, its end, its join: some 4 us) in tiles.
  const int64_t even = lmax(divide(tiles_sum + gridDim.x - 1, gridDim.x), MIN_TILES);
  const int64_t left = static_cast<int64_t>(gridDim.x) - units_sum;
  const int64_t apart = left > 0 ? lmax(divide(tiles_sum + left - 1, left), MIN_TILES) : 0;
  const bool pieces_apart = left > 0 && apart <= even + CROSSING;
  share = pieces_apart ? apart : even;
  const int32_t round = pieces_apart ? static_cast<int32_t>(share) : 1;
  int64_t mine = 0;
  for (int32_t i = mine0; i < mine1; ++i) {
    if (mine1 - mine0 > 1) slot_work<ROWS, TILE>(p, i, s, units);
    mine += units *
            (pieces_apart ? static_cast<int64_t>((s.unit_tiles + round - 1) / round) * round : s.unit_tiles);
  }
  int64_t before = mine;
#pragma unroll
  for (int step = 1; step < 32; step <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, before, step);
    if (lane >= step) before += x;
  }
  __syncthreads();  // the sums have been read
  if (lane == 31) sums[warp] = before;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  before -= mine;
  const int64_t start = share * blockIdx.x;
  if (start >= total) return false;
  if (start >= before && start < before + mine) {
    Walk<ROWS, TILE> walk{start, lmin(start + share, total), before, mine0, round};
    walk.next(p, s);
    segment = s;
    of_block = walk;
  }
  __syncthreads();
  return true;
}

// Adds a part's (maximum, sum) to another's.
__device__ __forceinline__ void add_part(float &best, float &sum, float m, float l) {
  const float next = max_nan(best, m);
  sum = (best == -INFINITY ? 0.0f : sum * exp2_fast(best - next)) + (m == -INFINITY ? 0.0f : l * exp2_fast(m - next));
  best = next;
}

// lse of weights exp2(s - top) that add up to sum.
__device__ __noinline__ float natural(float top, float sum) {
  return sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.693147180559945f;
}

// The output row of a unit's query row.
__device__ __forceinline__ int64_t out_row(const AttentionParam &p, const Segment &s, int32_t query_row) {
  const int32_t token = p.by_groups(query_row), head = s.slot - s.sequence * p.heads;
  return (static_cast<int64_t>(s.first_token + token) * p.heads + head) * p.groups + (query_row - token * p.groups);
}

// Joins the units that a block shares with others: `pieces` segments whose
// results lie in the workspace.  scratch: shared floats; tops, weight_sums:
// ROWS floats each.
template <typename T, int D, int ROWS, int THREADS>
__device__ __forceinline__ void join(const AttentionParam &p, const Segment *pending, int32_t *arrived, int pieces,
                                     int64_t share, float *scratch, int scratch_floats, float *stat_top,
                                     float *stat_sum) {
  const int kept = (scratch_floats - 2 * THREADS) / ROWS;  // parts whose maxima are kept
  // A block has at most two units that it shares, the first and the last of its
  // stretch.  Their results are announced together at the end: one release,
  // and no wait in between.  The block that arrives last at a unit joins it.
  __syncthreads();
  if (threadIdx.x < pieces) {
    const Segment &of = pending[threadIdx.x];
    const int64_t first = divide(of.unit_start, share), last = divide(of.unit_start + of.unit_tiles - 1, share);
    uint32_t before_me;
    // Releases this block's results (after the barrier) and acquires the others'.
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                 : "=r"(before_me)
                 : "l"(p.counters + first)
                 : "memory");
    const bool joins = before_me == static_cast<uint32_t>(last - first);
    if (joins) p.counters[first] = 0;  // as the next call expects it
    arrived[threadIdx.x] = joins;
  }
  __syncthreads();
  for (int piece = 0; piece < pieces; ++piece) {
    if (!arrived[piece]) continue;
    const Segment &s = pending[piece];
    const int64_t first = divide(s.unit_start, share), last = divide(s.unit_start + s.unit_tiles - 1, share);
    const int32_t parts = static_cast<int32_t>(last - first) + 1;
    const int32_t rows_here = min(ROWS, s.tokens * p.groups - s.row0);
    constexpr int64_t kPart = ROWS * (D + 2);
    // Part 0 is the first block's second result, part i > 0 the first result of
    // block first + i.
    const float *from = p.partials + (first * 2) * kPart;
    auto part_at = [&](int32_t i) { return from + (2 * static_cast<int64_t>(i) + (i == 0 ? 1 : 0)) * kPart; };
    // Maxima and sums: thread (row, every kAcrossth part), joined over shared memory.
    constexpr int kApart = THREADS / ROWS;
      float *joined = scratch + kept * ROWS;
    const int own_row = threadIdx.x % ROWS;
    float best = -INFINITY, weight_sum = 0.0f;
#pragma unroll 4
    for (int32_t i = threadIdx.x / ROWS; i < parts; i += kApart) {
      const float m = __ldcg(part_at(i) + ROWS * D + own_row), l = __ldcg(part_at(i) + ROWS * (D + 1) + own_row);
      if (i < kept) scratch[i * ROWS + own_row] = m;
      add_part(best, weight_sum, m, l);
    }
    joined[threadIdx.x] = best;
    joined[THREADS + threadIdx.x] = weight_sum;
    __syncthreads();
    best = -INFINITY, weight_sum = 0.0f;
    for (int i = own_row; i < THREADS; i += ROWS)
      add_part(best, weight_sum, joined[i], joined[THREADS + i]);
    if (threadIdx.x < ROWS) {
      stat_top[own_row] = best;
      stat_sum[own_row] = weight_sum;
      if (own_row < rows_here) p.lse[out_row(p, s, s.row0 + own_row)] = natural(best, weight_sum);
    }
    __syncthreads();
    // The outputs, four channels a thread at a time.
    for (int item = threadIdx.x; item < rows_here * (D / 4); item += THREADS) {
      const int row = item / (D / 4), channel = item % (D / 4) * 4;
      const float top = stat_top[row];
      float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
      for (int32_t i = 0; i < parts; ++i) {
        const float *part = part_at(i);
        const float4 x = __ldcg(reinterpret_cast<const float4 *>(part + row * D + channel));
        const float m = i < kept ? scratch[i * ROWS + row] : __ldcg(part + ROWS * D + row);
        const float w = m == -INFINITY ? 0.0f : exp2_fast(m - top);
        value.x = fmaf(w, x.x, value.x);
        value.y = fmaf(w, x.y, value.y);
        value.z = fmaf(w, x.z, value.z);
        value.w = fmaf(w, x.w, value.w);
      }
      const float inverse = stat_sum[row] == 0.0f ? 0.0f : 1.0f / stat_sum[row];
      __align__(8) const T result[4] = {from_float<T>(value.x * inverse), from_float<T>(value.y * inverse),
                                        from_float<T>(value.z * inverse), from_float<T>(value.w * inverse)};
      *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + out_row(p, s, s.row0 + row) * D + channel) =
          *reinterpret_cast<const uint2 *>(result);
    }
    __syncthreads();  // before the next piece writes over the statistics
  }
}

}  // namespace
}  // namespace lrk
