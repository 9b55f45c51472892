// Attention over the paged cache for many query rows a slot (chunks of tokens,
// the audit's query window): 128 query rows per block on tcgen05.
//
// Per tile of 64 rows of the cache (32 with four scales a row):
//     S = Q K^T (tensor memory)  ->  P = exp2(factor S - top) (tensor memory)
//     ->  O += P V (tensor memory).
// Many query rows use each cache row, so products and exponentials bound it,
// not memory: 4 D flops and one exponential per (query row, cache row).  The
// 4-bit rows are unpacked once per block and tile into shared memory:
// * keys as the whole numbers n - 8, exact in f16; one accumulator per group,
//   and scale_g S_g + offset_g sum(q)_g in float32 by the thread that holds the
//   row's scores, so scores are as exact as with unpacked float32 rows;
// * values as f16(2^-power (offset + scale (n - 8))), 11 bits like the weights'.
//   The power is the block's: it brings the largest value of a segment's first
//   tile below 2^11, and is raised (the output so far rescaled) where a later
//   tile passes 2^15.  f16 scales and offsets name values from 2^-24 to some
//   500,000; a fixed power would overflow or round off the ends of that.
// Within each 8 channels both operands take the order 0 4 1 5 2 6 3 7 in which
// a word's nibbles unpack in pairs; Q takes it too, and the output undoes it.
// The weights go back to tensor memory as the A operand; values are the B
// operand with channels contiguous (MN-major), so nothing is transposed.
//
// Measured (250 tokens of 32 query heads over 8 slots of 34,768 rows, group 64):
// 404 us, 352 TFLOP/s, 21 % of the matrix peak; the tensor pipe is busy a fifth
// of the time and 45 % of the issue slots are used, by unpacking, by the scales (two
// packed multiply-adds per pair of scores and group) and by the exponentials,
// between three barriers a tile.  (With a fixed power for the values, and rows
// without a page not told apart, 391 us.)  The same work on paged_attention.cu's
// matrix instructions took 765 us.
//
// Two blocks run on an SM (256 tensor-memory columns and at most 113 KB each)
// and fill one another's waits; within a block the value product of a tile runs
// under the next tile's unpacking of keys.
#include <cuda.h>

#include <algorithm>

#include "paged_attention.cuh"

namespace lrk {
namespace {

constexpr int kBlockThreads = 256;
constexpr int kBlockRows = 128;
constexpr int kBlocksOfSm = 2;
constexpr int kLeastTiles = 2;    // tiles per block, at least
constexpr int kUnitCrossing = 1;  // a second unit's cost in tiles, at 3 us a tile
constexpr uint32_t kColumns = 256;  // of tensor memory

template <typename T, int D, int GROUP>
struct TcLayout {
  static constexpr int kGroups = GROUP ? D / GROUP : 1;
  static constexpr int kTile = kGroups == 4 ? 32 : 64;
  static constexpr int kHalf = kTile / 2;  // columns of a thread: two threads a row
  static constexpr int kQuery = kBlockRows * D * 2;
  static constexpr int kOperand = kTile * D * 2;  // keys or values
  static constexpr int kCodes = GROUP ? kTile * D / 2 : 0, kScales = GROUP ? kTile * kGroups * 4 : 0;
  // What a tile's copies fill: the operands themselves (16-bit), or codes and scales.
  static constexpr int kStage = GROUP ? 2 * (kCodes + kScales) : 2 * kOperand;
  static constexpr int kStages = GROUP ? 3 : 2;
  static constexpr int kOperandAt = kQuery;  // 4-bit: unpacked keys, values
  static constexpr int kStageAt = kOperandAt + (GROUP ? 2 * kOperand : 0);
  static constexpr int kTableAt = kStageAt + kStages * kStage;  // float4 (scale, scale, offset, offset) of two rows
  static constexpr int kTable = GROUP ? kTile / 2 * kGroups * 16 : 0;
  static constexpr int kSumsAt = kTableAt + kTable;             // float [2][2][rows]: group sums by half and group
  static constexpr int kStatsAt = kSumsAt + 4 * kBlockRows * 4; // float [4][rows]: maxima, sums
  static constexpr int kFactorAt = kStatsAt + 4 * kBlockRows * 4;
  static constexpr int kControlAt = kFactorAt + kBlockRows * 4;
  static constexpr int kControl = 512;
  static constexpr int kBytes = kControlAt + kControl;
  static constexpr uint32_t kScoreColumn = D;  // after the output; the weights take the scores' place
  static_assert(D + kGroups * kTile <= static_cast<int>(kColumns), "tensor memory");
  static_assert(kBytes <= 232448 / kBlocksOfSm - 1024, "two blocks an SM");
};

template <int TILE>
struct TcControl {
  uint64_t landed[3], scored, added;
  // Of tile number n, at n % 4 (more than there are stages: a later tile is fed
  // before the scores are masked): a bit for each row that lies beyond every
  // query's rows, or in a page that does not exist.
  uint64_t absent[4];
  int64_t sums[2][kBlockThreads / 32];
  Walk<kBlockRows, TILE> walk;
  uint32_t columns;
  int32_t abort;
  int32_t arrived[2];
  Segment pending[2];
  Segment segment;
};

// B descriptor of the values: channels contiguous, 128-byte swizzle; 64-channel
// columns `leading` bytes apart, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t value_descriptor(uint32_t address, uint32_t leading) {
  return static_cast<uint64_t>((address >> 4) & 0x3FFFu) | (static_cast<uint64_t>(leading >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(instr), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t instr, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(instr), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}

__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }

// N fp32 (or packed) columns of this thread's lane, 16 at a time.
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t address, uint32_t *v) {
#pragma unroll
  for (int i = 0; i < N; i += 16) tc::tmem_load16(address + i, v + i);
#pragma unroll
  for (int i = 0; i < N; i += 16) tc::tmem_wait_load16(v + i);
}
__device__ __forceinline__ void tmem_store8(uint32_t address, const uint32_t *v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(address),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// a * b + c on two floats at once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n"
      " mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ uint32_t pack2(const __half *, float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(const __nv_bfloat16 *, float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// The codes of a word, less 8, as half2 (0, 4), (1, 5), (2, 6), (3, 7): a nibble
// under the exponent of 1024 is 1024 + n (or 1024 + 16 n), and what is taken
// off again leaves n - 8 exactly.
__device__ __forceinline__ void unpack8(uint32_t x, __half2 *n) {
  const uint32_t y = x >> 8;
  const uint32_t bits[4] = {(x & 0x000f000fu) | 0x64006400u, (x & 0x00f000f0u) | 0x64006400u,
                            (y & 0x000f000fu) | 0x64006400u, (y & 0x00f000f0u) | 0x64006400u};
  const __half2 low = __float2half2_rn(-1032.0f), high = __float2half2_rn(-72.0f);
  const __half2 sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = *reinterpret_cast<const __half2 *>(&bits[i]);
    n[i] = i & 1 ? __hfma2(h, sixteenth, high) : __hadd2(h, low);
  }
}

// Where the 8-channel chunk c of a row lies in an operand of `rows` rows.
__device__ __forceinline__ uint32_t chunk_at(int row, int c, int rows) {
  return static_cast<uint32_t>((c >> 3) * rows * 128 + row * 128 + (((c & 7) ^ (row & 7)) << 4));
}

template <typename T, int D, int GROUP>
__global__ __launch_bounds__(kBlockThreads, kBlocksOfSm)
void attention_tc_kernel(const __grid_constant__ AttentionParam p, const __grid_constant__ CUtensorMap key_map,
                         const __grid_constant__ CUtensorMap value_map) {
  using L = TcLayout<T, D, GROUP>;
  using W = std::conditional_t<GROUP == 0, T, __half>;  // operands' and weights' type
  constexpr bool kHalfWeights = std::is_same<W, __half>::value;
  // top is the running maximum less kHead, followed loosely (paged_attention.cu).
  constexpr float kHead = kHalfWeights ? 10.0f : 0.0f, kMost = kHalfWeights ? 14.0f : 8.0f;
  constexpr uint32_t kType = kHalfWeights ? 0u : (1u << 7) | (1u << 10);
  constexpr uint32_t kScoreInstr = (1u << 4) | kType | ((L::kTile >> 3) << 17) | ((kBlockRows >> 4) << 24);
  constexpr uint32_t kValueInstr = (1u << 4) | kType | (1u << 16) | ((D >> 3) << 17) | ((kBlockRows >> 4) << 24);
  static_assert(sizeof(TcControl<L::kTile>) <= L::kControl, "TcControl has grown");
  extern __shared__ __align__(1024) uint8_t shared[];
  const uint32_t base = shared_address(shared);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  TcControl<L::kTile> &control = *reinterpret_cast<TcControl<L::kTile> *>(shared + L::kControlAt);
  volatile int *abort = &control.abort;
  if (base & 1023) {
    if (threadIdx.x == 0) atomicOr(p.flag, kFlagShared);
    return;
  }
  const uint32_t scored = shared_address(&control.scored), added = shared_address(&control.added);
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) tc::init_barrier(shared_address(&control.landed[i]), 1);
    tc::init_barrier(scored, 1);
    tc::init_barrier(added, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    *abort = 0;
  }
  int64_t share;
  if (!begin<D, kBlockThreads, kLeastTiles, kUnitCrossing>(p, &control.sums[0][0], share, control.walk, control.segment)) return;
  // The instructions on tensor memory want their whole warp: lanes that a wait or
  // a branch held apart are brought together before each (__syncwarp).
  __syncwarp();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                     shared_address(&control.columns)),
                 "r"(kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = *const_cast<volatile uint32_t *>(&control.columns);

  float *group_sums = reinterpret_cast<float *>(shared + L::kSumsAt);
  float *stats = reinterpret_cast<float *>(shared + L::kStatsAt);
  float *factors = reinterpret_cast<float *>(shared + L::kFactorAt);
  // This thread's query row and which half of the row's columns it takes.
  const int row = (warp & 3) * 32 + lane, half = warp >> 2;
  const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);  // this warp's 32 lanes
  const uint32_t turn = p.scale_log2 < 0.0f ? 0x80008000u : 0u;           // a negative scale is taken by the queries
  constexpr float kLeastFactor = 1e-37f;
  uint32_t count = 0;  // tiles so far: their number gives stages and parities
  int pieces = 0;
  bool good = true;    // no wait has run out

  // Copies of tile `tile` of the segment into the stage of number n: by warp 1,
  // a lane per page and kind.
  const auto feed = [&](const Segment &s, int32_t tile, uint32_t n) {
    const uint32_t slot = n % L::kStages, barrier = shared_address(&control.landed[slot]);
    const uint32_t to = base + L::kStageAt + slot * L::kStage;
    const int rows = min(p.pages.page_size, L::kTile), first = tile * L::kTile;
    // Pages that hold visible rows of the tile; others may not exist.
    const int parts = min(L::kTile / rows, (s.seen_max - first + rows - 1) >> min(p.pages.page_shift, L::kTile == 64 ? 6 : 5));
    constexpr int kKinds = GROUP ? 4 : 2 * (D / 64);
    const int part = lane / kKinds, kind = lane % kKinds;
    const int32_t at = first + part * rows;
    int32_t page = -1;
    if (part < parts) page = p.table[static_cast<int64_t>(s.slot) * p.table_stride + (at >> p.pages.page_shift)];
    const bool there = page >= 0 && page < p.pages.pages;
    const uint32_t found = __ballot_sync(0xffffffffu, there && kind == 0);
    if (lane == 0) {
      uint64_t absent = s.seen_max - first < L::kTile ? ~uint64_t{0} << (s.seen_max - first) : 0;
      if (__popc(found) < parts) {
        for (int i = 0; i < parts; ++i)
          if (!(found >> (i * kKinds) & 1)) absent |= (~uint64_t{0} >> (64 - rows)) << (i * rows);
        atomicOr(p.flag, kFlagRow);
      }
      control.absent[n & 3] = absent;
      tc::expect_bytes(barrier, __popc(found) * rows * (L::kStage / L::kTile));
    }
    __syncwarp();
    if (there) {
      const int64_t y = static_cast<int64_t>(page) * p.pages.page_size + (at & (p.pages.page_size - 1));
      if constexpr (GROUP == 0) {
        const int side = kind / (D / 64), box = kind % (D / 64);
        tc::tma_box(to + side * L::kOperand + box * (L::kTile * 128) + part * rows * 128, side ? &value_map : &key_map,
                    box * 64, static_cast<int>(y), barrier);
      } else {
        constexpr int kRowBytes = D / 2, kScaleBytes = 4 * L::kGroups;
        const int side = kind >> 1;
        const uint32_t dst = to + side * (L::kCodes + L::kScales);
        if (kind & 1)
          bulk_copy(dst + L::kCodes + part * rows * kScaleBytes,
                    (side ? p.pages.value_scales : p.pages.key_scales) + y * L::kGroups, rows * kScaleBytes, barrier);
        else
          bulk_copy(dst + part * rows * kRowBytes, (side ? p.pages.values : p.pages.keys) + y * kRowBytes,
                    rows * kRowBytes, barrier);
      }
    }
    __syncwarp();
  };
  // Unpacking values: a thread keeps its chunk of 8 channels, and takes every
  // (threads / chunks)th row.  `absent` (a bit for each of the tile's rows): rows
  // beyond every query's, or without a page, may hold anything, and 0 NaN is NaN.
  constexpr int kChunks = D / 8, kStep = kBlockThreads / kChunks;
  const auto unpack_values = [&](const uint8_t *stage, uint64_t absent, int32_t power) {
    const int c = threadIdx.x % kChunks;
    const uint8_t *value_stage = stage + L::kCodes + L::kScales;
    const __half2 down = __half2half2(__ushort_as_half(static_cast<unsigned short>((15 - power) << 10)));
#pragma unroll
    for (int r = threadIdx.x / kChunks; r < L::kTile; r += kStep) {
      __align__(16) __half2 n[4];
      unpack8(*reinterpret_cast<const uint32_t *>(value_stage + r * (D / 2) + c * 4), n);
      const __half2 pair =
          __hmul2(reinterpret_cast<const __half2 *>(value_stage + L::kCodes)[r * L::kGroups + c * 8 / GROUP], down);
      const __half2 scale = __low2half2(pair), offset = __high2half2(pair);
#pragma unroll
      for (int k = 0; k < 4; ++k) n[k] = __hfma2(n[k], scale, offset);
      *reinterpret_cast<uint4 *>(shared + L::kOperandAt + L::kOperand + chunk_at(r, c, L::kTile)) =
          *reinterpret_cast<uint4 *>(n);
    }
    if (absent != 0) {
#pragma unroll 1
      for (int r = threadIdx.x / kChunks; r < L::kTile; r += kStep)
        if (absent >> r & 1)
          *reinterpret_cast<uint4 *>(shared + L::kOperandAt + L::kOperand + chunk_at(r, c, L::kTile)) =
              make_uint4(0, 0, 0, 0);
    }
  };
  // The power for a tile's values, found by every warp for itself: a lane holds a
  // 32nd of the tile's (scale, offset) pairs, signs left out.  A value is below
  // 2^(e - 13), e the larger of the offset's exponent field and the scale's plus 3;
  // the power stays while that is at most 2^(15 + power), and brings it below
  // 2^(11 + power) otherwise (as far as f16 holds 2^-power).  Pairs that are not
  // finite reach their own rows, whatever the power.  `room`: what the pairs' bits
  // lack to that limit, less than 2^15 each.  Returns the factor for the output so far.
  const auto tile_power = [&](const uint8_t *stage, uint64_t absent, int32_t &power, uint32_t &room, bool first) {
    constexpr int kWords = L::kTile * L::kGroups / 32;
    uint32_t w[kWords];
    const uint8_t *from = stage + 2 * L::kCodes + L::kScales + lane * kWords * 4;
    if constexpr (kWords == 4) {
      const uint4 x = *reinterpret_cast<const uint4 *>(from);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2 *>(from);
      w[0] = x.x, w[1] = x.y;
    }
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] &= 0x7fff7fffu;
    if (absent != 0)
#pragma unroll
      for (int k = 0; k < kWords; ++k)
        if (absent >> ((lane * kWords + k) / L::kGroups) & 1) w[k] = 0;
    uint32_t largest = w[0];
#pragma unroll
    for (int k = 1; k < kWords; ++k) largest = __vmaxu2(largest, w[k]);
    if (!first && !__any_sync(0xffffffffu, ((largest + room) & 0x80008000u) != 0)) return 1.0f;
    int32_t field = 0;
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const int32_t scale = w[k] >> 10 & 31, offset = w[k] >> 26;
      field = max(field, max(scale < 31 ? scale + 3 : 0, offset < 31 ? offset : 0));
    }
    field = __reduce_max_sync(0xffffffffu, field);
    const int32_t last = power;
    power = max(field - 24, first ? -15 : power);
    room = static_cast<uint32_t>(max(0x8000 - ((26 + power) << 10), 0)) |
           static_cast<uint32_t>(max(0x8000 - ((29 + power) << 10), 0)) << 16;
    return first ? 1.0f : __int_as_float((127 + last - power) << 23);
  };
  const auto waits = [&](uint32_t barrier, uint32_t parity) {
    if (!wait(barrier, parity, abort)) {
      if (good) atomicOr(p.flag, kFlagTimeout);
      good = false;
    }
    __syncwarp();  // lanes leave the wait one by one
  };

  while (true) {
    const Segment s = control.segment;
    if (s.slot < 0) break;
    const int32_t tiles = max(s.tile1 - s.tile0, 0);
    if (warp == 1)
      for (int32_t i = 0; i < min(tiles, GROUP ? L::kStages : 1); ++i) feed(s, s.tile0 + i, count + i);

    // The queries, as operand A: two threads a row, D / 2 channels each.
    const int32_t rows_total = s.tokens * p.groups, query_row = s.row0 + row;
    const bool live = query_row < rows_total;
    const int32_t seen = live ? rows_seen(p, s, query_row) : s.seen_max;
    float factor = fmaxf(fabsf(p.scale_log2), kLeastFactor);
    float sums[L::kGroups];
    {
      const int32_t token = p.by_groups(live ? query_row : s.row0), head = s.slot - s.sequence * p.heads;
      const int32_t in_group = (live ? query_row : s.row0) - token * p.groups;
      const T *from = static_cast<const T *>(p.queries) + static_cast<int64_t>(s.first_token + token) * p.query_token +
                      (static_cast<int64_t>(head) * p.groups + in_group) * p.query_head + half * (D / 2);
      if constexpr (GROUP == 0) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint4 x = live ? *reinterpret_cast<const uint4 *>(from + c * 8) : make_uint4(0, 0, 0, 0);
          x.x ^= turn, x.y ^= turn, x.z ^= turn, x.w ^= turn;
          *reinterpret_cast<uint4 *>(shared + chunk_at(row, half * (D / 16) + c, kBlockRows)) = x;
        }
        sums[0] = 0.0f;
      } else {
        float largest = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          float x[8];
          load8(from + c * 8, x);
#pragma unroll
          for (int i = 0; i < 8; ++i) largest = fmaxf(largest, live ? fabsf(x[i]) : 0.0f);
        }
        stats[half * kBlockRows + row] = largest;
        __syncthreads();
        largest = fmaxf(largest, stats[(half ^ 1) * kBlockRows + row]);
        // As in paged_attention.cu: a power of two brings the row into [1, 2).
        const int exponent = static_cast<int>(__float_as_uint(largest) >> 23);
        const bool plain = exponent == 255 || largest == 0.0f;
        const int shift = plain ? 0 : (exponent == 0 ? 1 : exponent) - 127;
        const float to_unit = __int_as_float(((127 - min(shift, 126)) << 23) | (turn & 0x80000000u));
        const float from_unit = __int_as_float((127 + min(shift, 126)) << 23);
        factor = fmaxf(fabsf(p.scale_log2) * from_unit, kLeastFactor);
        constexpr int kParts = L::kGroups > 1 ? L::kGroups / 2 : 1;  // groups, or the part of one, in half a row
        float part_sums[kParts];
#pragma unroll
        for (int k = 0; k < kParts; ++k) part_sums[k] = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          float x[8];
          load8(from + c * 8, x);
          __half h[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            h[i] = __float2half_rn(live ? x[i] * to_unit : 0.0f);
            part_sums[c * kParts / (D / 16)] += __half2float(h[i]);
          }
          __align__(16) const __half2 b[4] = {__halves2half2(h[0], h[4]), __halves2half2(h[1], h[5]),
                                              __halves2half2(h[2], h[6]), __halves2half2(h[3], h[7])};
          *reinterpret_cast<uint4 *>(shared + chunk_at(row, half * (D / 16) + c, kBlockRows)) =
              *reinterpret_cast<const uint4 *>(b);
        }
#pragma unroll
        for (int k = 0; k < kParts; ++k) group_sums[(half * 2 + k) * kBlockRows + row] = part_sums[k];
        __syncthreads();
#pragma unroll
        for (int g = 0; g < L::kGroups; ++g)
          sums[g] = L::kGroups == 1 ? group_sums[row] + group_sums[2 * kBlockRows + row]
                                    : group_sums[(g / kParts * 2 + g % kParts) * kBlockRows + row];
      }
    }
    float top = -INFINITY, sum = 0.0f;
    int32_t power = 0;  // 4-bit values are held as v 2^-power
    uint32_t room = 0;

    for (int32_t i = 0; i < tiles; ++i, ++count) {
      const uint32_t slot = count % L::kStages;
      const int32_t first_row = (s.tile0 + i) * L::kTile;
      uint8_t *const stage = shared + L::kStageAt + slot * L::kStage;
      float change = 1.0f;  // of the output so far, with the values' power
      const uint32_t keys_at = base + (GROUP ? L::kOperandAt : L::kStageAt + slot * L::kStage);
      const uint32_t values_at = keys_at + L::kOperand;
      waits(shared_address(&control.landed[slot]), (count / L::kStages) & 1);
      const auto absent_rows = [&] { return *const_cast<volatile uint64_t *>(&control.absent[count & 3]); };
      if constexpr (GROUP != 0) {
        const int c = threadIdx.x % kChunks;
        uint8_t *const operands = shared + L::kOperandAt;
#pragma unroll
        for (int r = threadIdx.x / kChunks; r < L::kTile; r += kStep) {
          __align__(16) __half2 n[4];
          unpack8(*reinterpret_cast<const uint32_t *>(stage + r * (D / 2) + c * 4), n);
          *reinterpret_cast<uint4 *>(operands + chunk_at(r, c, L::kTile)) = *reinterpret_cast<uint4 *>(n);
        }
        for (int k = threadIdx.x; k < L::kTile / 2 * L::kGroups; k += kBlockThreads) {
          const __half2 *scales = reinterpret_cast<const __half2 *>(stage + L::kCodes) + (k / L::kGroups) * 2 * L::kGroups +
                                  k % L::kGroups;
          const float2 a = __half22float2(scales[0]), b = __half22float2(scales[L::kGroups]);
          reinterpret_cast<float4 *>(shared + L::kTableAt)[k] = make_float4(a.x, b.x, a.y, b.y);
        }
        const uint64_t absent = absent_rows();
        change = tile_power(stage, absent, power, room, i == 0);
        if (i > 0) waits(added, (count - 1) & 1);  // the last tile's values have been used
        unpack_values(stage, absent, power);
      } else {
        if (i > 0) waits(added, (count - 1) & 1);
        if (warp == 1 && i + 1 < tiles) feed(s, s.tile0 + i + 1, count + 1);  // into the stage that is free now
        const uint64_t absent = absent_rows();
        if (absent != 0)
          for (int k = threadIdx.x; k < L::kTile * (D / 8); k += kBlockThreads)
            if (absent >> (k % L::kTile) & 1)
              *reinterpret_cast<uint4 *>(stage + L::kOperand + chunk_at(k % L::kTile, k / L::kTile, L::kTile)) =
                  make_uint4(0, 0, 0, 0);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      before_sync();
      __syncthreads();
      after_sync();
      if (threadIdx.x == 0) {
#pragma unroll
        for (int g = 0; g < L::kGroups; ++g)
#pragma unroll
          for (int k = 0; k < D / L::kGroups / 16; ++k) {
            const int channel = g * (D / L::kGroups) + k * 16;  // 64-channel columns, 32 bytes a k-step
            mma_shared(tmem + L::kScoreColumn + g * L::kTile,
                       tc::smem_descriptor(base + (channel >> 6) * (kBlockRows * 128) + (channel & 63) * 2),
                       tc::smem_descriptor(keys_at + (channel >> 6) * (L::kTile * 128) + (channel & 63) * 2), kScoreInstr,
                       k > 0);
          }
        tc::umma_commit(scored);
      }
      if constexpr (GROUP != 0) {
        if (warp == 1 && i + L::kStages < tiles) feed(s, s.tile0 + i + L::kStages, count + L::kStages);
      }
      waits(scored, count & 1);
      after_sync();

      // This thread's scores.
      float2 x[L::kHalf / 2];
      const uint32_t score_at = lanes + L::kScoreColumn + half * L::kHalf;
      if constexpr (GROUP == 0) {
        tmem_load<L::kHalf>(score_at, reinterpret_cast<uint32_t *>(x));
      } else {
        const float4 *table = reinterpret_cast<const float4 *>(shared + L::kTableAt) + half * (L::kHalf / 2) * L::kGroups;
#pragma unroll
        for (int g = 0; g < L::kGroups; ++g) {
          float2 raw[L::kHalf / 2];
          tmem_load<L::kHalf>(score_at + g * L::kTile, reinterpret_cast<uint32_t *>(raw));
          const float2 group_sum = make_float2(sums[g], sums[g]);
#pragma unroll
          for (int k = 0; k < L::kHalf / 2; ++k) {
            const float4 v = table[k * L::kGroups + g];
            const float2 rest = fma2(make_float2(v.z, v.w), group_sum, g == 0 ? make_float2(0.0f, 0.0f) : x[k]);
            x[k] = fma2(make_float2(v.x, v.y), raw[k], rest);
          }
        }
      }
      if (const uint64_t absent = absent_rows(); first_row + L::kTile > s.seen_min || absent != 0) {
        const int32_t visible = seen - first_row - half * L::kHalf;
        const uint32_t hidden = static_cast<uint32_t>(absent >> (half * L::kHalf));
#pragma unroll
        for (int k = 0; k < L::kHalf / 2; ++k) {
          if (2 * k >= visible || (hidden >> (2 * k) & 1)) x[k].x = -INFINITY;
          if (2 * k + 1 >= visible || (hidden >> (2 * k + 1) & 1)) x[k].y = -INFINITY;
        }
      }
      float best = max_nan(x[0].x, x[0].y);
#pragma unroll
      for (int k = 1; k < L::kHalf / 2; ++k) best = max_nan(best, x[k].x, x[k].y);
      // The barrier also keeps the weights from the scores that others still read.
      before_sync();
      // (Also where best is NaN: top has to become NaN, since -inf stands for no rows.)
      const bool raises = __syncthreads_or(!(fmaf(best, factor, -kMost) <= top) || (GROUP != 0 && change != 1.0f));
      after_sync();
      if (raises) {
        stats[half * kBlockRows + row] = best;
        __syncthreads();
        best = max_nan(best, stats[(half ^ 1) * kBlockRows + row]);
        const float next = max_nan(fmaf(best, factor, -kHead), top);
        const float keep = top == -INFINITY ? 0.0f : exp2_fast(top - next);
        top = next;
        sum *= keep;
        if (i > 0 && __any_sync(0xffffffffu, keep * change != 1.0f)) {
#pragma unroll
          for (int k = 0; k < D / 2; k += 16) {
            uint32_t o[16];
            tmem_load<16>(lanes + half * (D / 2) + k, o);
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * (keep * change));
            tc::tmem_store16(lanes + half * (D / 2) + k, o);
          }
          tc::tmem_wait_store();
        }
        __syncthreads();  // before the maxima are written over
      }
      const float shift = top == -INFINITY ? 0.0f : -top;
      uint32_t weights[L::kHalf / 2];
      float2 both = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < L::kHalf / 2; ++k) {
        const float2 e = fma2(x[k], make_float2(factor, factor), make_float2(shift, shift));
        const float a = exp2_fast(e.x), b = exp2_fast(e.y);
        both = add2(both, make_float2(a, b));
        weights[k] = pack2(static_cast<const W *>(nullptr), a, b);
      }
      sum += both.x + both.y;
      const uint32_t weights_at = lanes + L::kScoreColumn + half * (L::kHalf / 2);
      __syncwarp();
      if constexpr (L::kHalf == 32) tc::tmem_store16(weights_at, weights);
      else tmem_store8(weights_at, weights);
      tc::tmem_wait_store();
      before_sync();
      __syncthreads();
      after_sync();
      if (threadIdx.x == 0) {
#pragma unroll
        for (int k = 0; k < L::kTile / 16; ++k)
          mma_tensor(tmem, tmem + L::kScoreColumn + k * 8, value_descriptor(values_at + k * 16 * 128, L::kTile * 128),
                     kValueInstr, i > 0 || k > 0);
        tc::umma_commit(added);
      }
    }
    if (tiles > 0) waits(added, (count - 1) & 1);
    after_sync();

    // The segment's end: a thread has half the channels of its row.
    stats[(2 + half) * kBlockRows + row] = sum;
    __syncthreads();
    const float weight_sum = stats[2 * kBlockRows + row] + stats[3 * kBlockRows + row];
    const bool whole_unit = s.starts && s.ends;
    float *partial = p.partials + (static_cast<int64_t>(blockIdx.x) * 2 + (s.starts ? 1 : 0)) * kBlockRows * (D + 2);
    const float restore = GROUP ? __int_as_float((127 + power) << 23) : 1.0f;
    const float inverse = (weight_sum == 0.0f ? 0.0f : 1.0f / weight_sum) * restore;
    const int64_t index = out_row(p, s, live ? query_row : s.row0);
#pragma unroll
    for (int k = 0; k < D / 2; k += 16) {
      uint32_t o[16];
      __syncwarp();  // lanes without a query row store nothing below
      if (tiles > 0) {
        tmem_load<16>(lanes + half * (D / 2) + k, o);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = 0;
      }
      float value[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        // Column j of 8 holds channel 0 4 1 5 2 6 3 7 of them (4-bit rows).
        const int channel = GROUP ? (j & 8) + ((j & 1) ? 4 : 0) + ((j & 7) >> 1) : j;
        value[channel] = __uint_as_float(o[j]);
      }
      const int at = half * (D / 2) + k;
      if (!live) {
        // No row to write.
      } else if (whole_unit) {
#pragma unroll
        for (int j = 0; j < 16; ++j) value[j] *= inverse;
        store8(static_cast<T *>(p.out) + index * D + at, value);
        store8(static_cast<T *>(p.out) + index * D + at + 8, value + 8);
      } else {
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          *reinterpret_cast<float4 *>(partial + row * D + at + j) =
              make_float4(value[j] * restore, value[j + 1] * restore, value[j + 2] * restore, value[j + 3] * restore);
      }
    }
    if (live && half == 0) {
      if (whole_unit) {
        p.lse[index] = natural(top, weight_sum);
      } else {
        partial[kBlockRows * D + row] = top;
        partial[kBlockRows * (D + 1) + row] = weight_sum;
      }
    }
    if (!whole_unit) {
      if (threadIdx.x == 0) control.pending[pieces] = s;
      ++pieces;
    }
    before_sync();
    __syncthreads();  // everyone has read the segment
    after_sync();
    if (threadIdx.x == 0) {
      Segment next;
      if (!control.walk.next(p, next)) next.slot = -1;
      control.segment = next;
    }
    __syncthreads();
  }

  if (*abort) {  // given up: leave only after the copies in flight have had their time to land
    for (uint32_t n = count > L::kStages ? count - L::kStages : 0; n < count + L::kStages; ++n)
      tc::wait_phase(shared_address(&control.landed[n % L::kStages]), (n / L::kStages) & 1, nullptr);
  }
  before_sync();
  __syncthreads();
  __syncwarp();
  if (warp == 0) {
    after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kColumns) : "memory");
  }
  if (pieces == 0) return;
  join<T, D, kBlockRows, kBlockThreads>(p, control.pending, control.arrived, pieces, share,
                                        reinterpret_cast<float *>(shared), L::kQuery / 4, stats, stats + kBlockRows);
}

template <typename T, int D, int GROUP>
int launch_tc_format(const AttentionParam &p, const lrk_pages &pages, cudaStream_t stream) {
  using L = TcLayout<T, D, GROUP>;
  auto kernel = attention_tc_kernel<T, D, GROUP>;
  static std::atomic<uint64_t> allowed{0};  // devices, a bit each, that know the kernel's shared memory
  if (const int status = allow_shared(kernel, L::kBytes, allowed)) return status;
  CUtensorMap maps[2] = {};
  if (GROUP == 0 && pages.pages > 0) {
    const int64_t rows = pages.pages * pages.page_size;
    if (rows > INT32_MAX) return fail(LRK_ERR_UNSUPPORTED, "paged attention: too many 16-bit rows");
    const uint32_t box = static_cast<uint32_t>(std::min<int64_t>(pages.page_size, L::kTile));
    for (int side = 0; side < 2; ++side) {
      const int status = tc::make_map(&maps[side], side ? pages.values : pages.keys, rows, D, D, 64,
                                      CU_TENSOR_MAP_SWIZZLE_128B, box);
      if (status != LRK_OK) return status;
    }
  }
  kernel<<<static_cast<unsigned>(sm_count() * kBlocksOfSm), kBlockThreads, L::kBytes, stream>>>(p, maps[0], maps[1]);
  return launch_status("paged attention");
}

template <typename T, int D>
int launch_tc_rows(const AttentionParam &p, const lrk_pages &pages, cudaStream_t stream) {
  switch (pages.group) {
    case 0: return launch_tc_format<T, D, 0>(p, pages, stream);
    case 32: return launch_tc_format<T, D, 32>(p, pages, stream);
    case 64: return launch_tc_format<T, D, 64>(p, pages, stream);
    default:
      if constexpr (D == 128) return launch_tc_format<T, D, 128>(p, pages, stream);
      return LRK_ERR_UNSUPPORTED;
  }
}

}  // namespace

// `param`: the AttentionParam of paged_attention.cu, checked there.
int launch_paged_attention_tc(const void *param, const lrk_pages &pages, int dtype, cudaStream_t stream) {
  const AttentionParam &p = *static_cast<const AttentionParam *>(param);
  if (dtype == LRK_F16)
    return pages.dimension == 64 ? launch_tc_rows<__half, 64>(p, pages, stream)
                                 : launch_tc_rows<__half, 128>(p, pages, stream);
  return pages.dimension == 64 ? launch_tc_rows<__nv_bfloat16, 64>(p, pages, stream)
                               : launch_tc_rows<__nv_bfloat16, 128>(p, pages, stream);
}

}  // namespace lrk
