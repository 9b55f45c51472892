// Attention over the paged cache.
//
// Query i of a sequence's n new tokens sees rows r <= length - n + i of each
// of its slots (every row without `causal`):
//     o = sum_r p_r v_r,   p = softmax(scale q k_r),   lse = log sum_r exp(scale q k_r).
// One pass over the rows with a running maximum m and sum l: a new maximum m'
// multiplies l and the accumulated output by exp(m - m').
//
// What bounds it: a decode step reads every row once (144 bytes of keys and
// values per 4-bit row at D = 128, group 64; 512 in 16 bits) for 4 D flops per
// query head, so memory bounds it if the 4-bit codes can be unpacked as fast
// as they arrive: at the copy rate about 40 codes per SM and clock, three
// instructions per code.  Hence the shape of the arithmetic:
//
// * S^T = K Q^T and O^T = V^T P^T on m16n8k16 matrix instructions with the
//   cache as the 16-row operand A, straight from registers, and the (few)
//   query rows as B: every unpacked register is used once, by one instruction,
//   and nothing is staged through shared memory a second time (tcgen05 takes
//   its operands from shared or tensor memory, so that unpacked rows would be
//   written and read once more).
// * A nibble n needs no conversion: n in the low bits of a half is the
//   subnormal n * 2^-24 (in bits 4-7: n * 2^-20), exact in the matrix
//   instruction's products, so one AND gives a pair of operands.  The powers
//   of two are put right outside the inner loop (in Q, and once in O).
// * Scales and offsets stay out of the products:
//     q k   = sum_groups scale_g (q . n - 8 sum q)_g + offset_g (sum q)_g,
//     p v   = scale_g p (n - 8) + offset_g p   ->  B operand f16(p scale_g),
//   the subtraction of 8 sum f16(p scale_g) by one more matrix instruction per
//   group with ones as A, so that it cancels exactly what was rounded.
//
// Split: the tiles of 32 rows of all slots, laid end to end, are divided
// evenly over a persistent grid, so neither few slots nor ragged ones leave
// SMs idle.  A slot whose tiles fall to several blocks leaves partial results
// (maximum, sum, output) in the workspace; the block that arrives last joins
// them in a fixed order, so the result does not depend on the arrival.
#include <cuda.h>

#include <algorithm>

#include "paged.cuh"
#include "tc.cuh"

namespace lrk {
namespace {

using namespace paged;

constexpr int kTile = 32;   // rows per tile
constexpr int kWarps = 4;   // consumer warps; one more feeds them
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kMinTiles = kWarps;  // tiles per block, at least
constexpr int kCounters = 4096;    // workspace: arrival counters, then partial results

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
  float scale_log2;
  bool causal;
  void *out;
  float *lse;
  uint32_t *counters;
  float *partials;
  uint32_t *flag;
};

template <typename T, int D, int GROUP, int NT>
struct Layout {
  static constexpr int kRowBytes = GROUP ? D / 2 : D * 2;
  static constexpr int kGroups = GROUP ? D / GROUP : 1;
  static constexpr int kScaleBytes = GROUP ? kGroups * 4 : 0;
  static constexpr int kRows = 8 * NT;  // query rows per block
  static constexpr int kCodes = kTile * kRowBytes, kScales = kTile * kScaleBytes;
  static constexpr int kStage = 2 * (kCodes + kScales);  // key rows, key scales, value rows, value scales
  static constexpr int kStages = GROUP ? 10 : (D == 128 ? 4 : 8);
  static constexpr int kPitch = D + 4;
  static constexpr int kScratch = kWarps * 8 * kPitch * 4;
  static constexpr int kQuery = NT * (D / 16) * 32 * 8;
  // After the stages: scratch, query fragments, group sums, factors, maxima and sums, barriers.
  static constexpr int kScratchAt = kStages * kStage;
  static constexpr int kQueryAt = kScratchAt + kScratch;
  static constexpr int kSumsAt = kQueryAt + kQuery;
  static constexpr int kFactorAt = kSumsAt + kGroups * kRows * 4;
  static constexpr int kStatsAt = kFactorAt + kRows * 4;
  static constexpr int kBarriersAt = kStatsAt + 2 * kWarps * kRows * 4;
  static constexpr int kBytes = kBarriersAt + 2 * kStages * 8 + 64 + 1024;
  static constexpr int kBlocksPerSm = NT == 1 ? 3 : (NT == 2 ? 2 : 1);
};

__device__ __forceinline__ void mma(const __half *, float *d, const uint32_t *a, uint32_t b0, uint32_t b1,
                                    const float *c) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma(const __nv_bfloat16 *, float *d, const uint32_t *a, uint32_t b0, uint32_t b1,
                                    const float *c) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Transpose of an 8 x 8 matrix of 16-bit elements spread over the warp: the
// columns of S^T (query rows) become the rows that P's B operand wants.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack(const __half *, float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack(const __nv_bfloat16 *, float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int WORDS>
__device__ __forceinline__ void load_words(uint32_t address, uint32_t *w) {
  if constexpr (WORDS == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(address));
  else if constexpr (WORDS == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(address));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(address));
}
__device__ __forceinline__ uint32_t load_short(uint32_t address) {
  uint16_t w;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(address));
  return w;
}
__device__ __forceinline__ float2 load_pair(uint32_t address) {  // (scale, offset)
  uint32_t w;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(address));
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

__device__ __forceinline__ void bulk_copy(uint32_t to, const void *from, uint32_t bytes, uint32_t barrier) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(to),
               "l"(from), "r"(bytes), "r"(barrier)
               : "memory");
}

__device__ __forceinline__ bool wait(uint32_t barrier, uint32_t parity, volatile int *abort) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(barrier), "r"(parity)
      : "memory");
  return done || tc::wait_phase(barrier, parity, abort);
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }

// A stretch of one unit's tiles: a unit is a slot and a block of its query rows.
struct Segment {
  int32_t slot;
  int32_t length, tokens, first_token;  // of the slot, its sequence
  int32_t row0;                         // first query row (token * groups + head in group) of the unit
  int32_t tile0, tile1;                 // tiles of the stretch, those beyond every query's rows left out
  int32_t seen_max, seen_min;           // rows seen by the unit's last and first query
  bool starts, ends;                    // the stretch holds the unit's first / last tile
  int64_t unit_start;
  int32_t unit_tiles;
};

// The blocks' shares of all units' tiles, laid end to end.
template <int ROWS>
struct Walk {
  const AttentionParam &p;
  int64_t position, end;
  int64_t slot_start;
  int32_t slot;

  __device__ __forceinline__ static int32_t rows_held(const AttentionParam &p, int32_t slot) {
    return min(max(p.lengths[slot], 0), p.capacity);
  }
  // A sequence's first token and its tokens, within those that there are.
  __device__ __forceinline__ static int2 tokens_of(const AttentionParam &p, int32_t sequence) {
    const int32_t first = min(max(p.token_starts[sequence], 0), p.tokens);
    return make_int2(first, max(min(p.token_starts[sequence + 1], p.tokens) - first, 0));
  }
  __device__ __forceinline__ static int64_t cost(const AttentionParam &p, int32_t slot) {
    const int64_t tokens = tokens_of(p, slot / p.heads).y;
    const int64_t blocks = (tokens * p.groups + ROWS - 1) / ROWS;
    return blocks * max((rows_held(p, slot) + kTile - 1) / kTile, 1);
  }

  __device__ __forceinline__ bool next(Segment &s) {
    if (position >= end) return false;
    int64_t whole = cost(p, slot);
    while (position >= slot_start + whole) {
      slot_start += whole;
      if (++slot >= p.slots) return false;
      whole = cost(p, slot);
    }
    const int2 tokens = tokens_of(p, slot / p.heads);
    s.slot = slot;
    s.length = rows_held(p, slot);
    s.first_token = tokens.x;
    s.tokens = tokens.y;
    s.unit_tiles = max((s.length + kTile - 1) / kTile, 1);
    const int64_t offset = position - slot_start;
    const int64_t block = offset / s.unit_tiles;
    s.tile0 = static_cast<int32_t>(offset - block * s.unit_tiles);
    s.unit_start = slot_start + block * s.unit_tiles;
    const int64_t stop = lmin(end, s.unit_start + s.unit_tiles);
    s.tile1 = s.tile0 + static_cast<int32_t>(stop - position);
    s.starts = s.tile0 == 0;
    s.ends = s.tile1 == s.unit_tiles;
    position = stop;
    s.row0 = static_cast<int32_t>(block * ROWS);
    const int32_t last_row = min(s.row0 + ROWS, s.tokens * p.groups) - 1;
    s.seen_min = seen(p, s, s.row0);
    s.seen_max = seen(p, s, last_row);
    s.tile1 = min(s.tile1, (s.seen_max + kTile - 1) / kTile);
    return true;
  }
  __device__ __forceinline__ static int32_t seen(const AttentionParam &p, const Segment &s, int32_t row) {
    if (!p.causal) return s.length;
    const int64_t rows = static_cast<int64_t>(s.length) - s.tokens + row / p.groups + 1;
    return static_cast<int32_t>(rows < 0 ? 0 : rows);
  }
};

template <typename T, int D, int GROUP, int NT>
struct Consumer {
  using L = Layout<T, D, GROUP, NT>;
  static constexpr int kOut = D / 16;
  static constexpr int kNG = L::kGroups;
  using P = std::conditional_t<GROUP == 0, T, __half>;  // the weights' type, as the matrix instruction wants V's

  float out[kOut][NT][4];
  float top[NT][2], sum[NT][2];
  float offset_sum[NT][kNG][2], scaled_sum[NT][kNG][4];
  uint32_t query[NT <= 2 ? NT : 1][D / 16][2];
  float factor[NT][2];
  int32_t seen[NT][2];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int m = 0; m < kOut; ++m) out[m][nt][i] = 0.0f;
#pragma unroll
        for (int g = 0; g < kNG; ++g) scaled_sum[nt][g][i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[nt][i] = -INFINITY;
        sum[nt][i] = 0.0f;
#pragma unroll
        for (int g = 0; g < kNG; ++g) offset_sum[nt][g][i] = 0.0f;
      }
    }
  }

  __device__ __forceinline__ void query_fragment(uint32_t query_at, int nt, int ks, int lane, uint32_t *b) const {
    if constexpr (NT <= 2) {
      b[0] = query[nt][ks][0];
      b[1] = query[nt][ks][1];
    } else {
      load_words<2>(query_at + ((nt * (D / 16) + ks) * 32 + lane) * 8, b);
    }
  }

  // Scores of 16 rows (first row: row0 of the tile) against the block's query
  // rows: s[nt][0..1] of row pi(g), s[nt][2..3] of row 8 + pi(g).
  __device__ __forceinline__ void scores(uint32_t stage, uint32_t query_at, const float *group_sums, int half, int lane,
                                         float (*s)[4]) {
    const int g = lane >> 2, t = lane & 3;
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (GROUP == 0) {
      const int row = half * 16 + (lane & 15);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t a[4], b[2];
        const uint32_t address = stage + (ks >> 2) * (kTile * 128) + row * 128 +
                                 (((2 * (ks & 3) + (lane >> 4)) ^ (row & 7)) << 4);
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                     : "r"(address));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          query_fragment(query_at, nt, ks, lane, b);
          mma(static_cast<const P *>(nullptr), s[nt], a, b[0], b[1], ks == 0 ? zero : s[nt]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[nt][i] *= factor[nt][i & 1];
    } else {
      const int row = half * 16 + (g ^ ((g >> 1) & 1));
#pragma unroll
      for (int gi = 0; gi < kNG; ++gi) {
        uint32_t w[2][GROUP / 32];
        const uint32_t address = stage + row * L::kRowBytes + gi * (GROUP / 2) + t * (GROUP / 8);
        load_words<GROUP / 32>(address, w[0]);
        load_words<GROUP / 32>(address + 8 * L::kRowBytes, w[1]);
        float acc[NT][4], q[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 pair = *reinterpret_cast<const float2 *>(group_sums + gi * L::kRows + nt * 8 + 2 * t);
          q[nt][0] = pair.x;
          q[nt][1] = pair.y;
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][i] = -8.0f * q[nt][i & 1];
        }
#pragma unroll
        for (int j = 0; j < GROUP / 32; ++j) {
          const uint32_t x0 = w[0][j], x1 = w[1][j], y0 = x0 >> 8, y1 = x1 >> 8;
          const uint32_t low[4] = {x0 & 0x000f000fu, x1 & 0x000f000fu, y0 & 0x000f000fu, y1 & 0x000f000fu};
          const uint32_t high[4] = {x0 & 0x00f000f0u, x1 & 0x00f000f0u, y0 & 0x00f000f0u, y1 & 0x00f000f0u};
          const int ks = gi * (GROUP / 16) + 2 * j;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint32_t b[2];
            query_fragment(query_at, nt, ks, lane, b);
            mma(static_cast<const P *>(nullptr), acc[nt], low, b[0], b[1], acc[nt]);
            query_fragment(query_at, nt, ks + 1, lane, b);
            mma(static_cast<const P *>(nullptr), acc[nt], high, b[0], b[1], acc[nt]);
          }
        }
        const uint32_t scales = stage + L::kCodes + (row * kNG + gi) * 4;
        const float2 k0 = load_pair(scales), k1 = load_pair(scales + 8 * kNG * 4);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 k = i < 2 ? k0 : k1;
            const float x = gi == 0 ? k.y * q[nt][i & 1] : fmaf(k.y, q[nt][i & 1], s[nt][i]);
            s[nt][i] = fmaf(k.x, acc[nt][i], x);
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[nt][i] *= factor[nt][i & 1];
    }
  }

  // Adds 16 rows' weighted values to the output.  With MASKED, rows that a
  // query does not see add nothing, whatever their scales hold.
  template <bool MASKED>
  __device__ __forceinline__ void values(uint32_t stage, int half, int lane, const float (*w)[4], int32_t first_row) {
    const int g = lane >> 2, t = lane & 3;
    const uint32_t values_at = stage + L::kCodes + L::kScales;
    if constexpr (GROUP == 0) {
      uint32_t b[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        b[nt][0] = transpose8(pack(static_cast<const P *>(nullptr), w[nt][0], w[nt][1]));
        b[nt][1] = transpose8(pack(static_cast<const P *>(nullptr), w[nt][2], w[nt][3]));
      }
      const int row = half * 16 + (lane & 7) + 8 * (lane >> 4);
#pragma unroll
      for (int m = 0; m < kOut; ++m) {
        uint32_t a[4];
        const uint32_t address = values_at + (m >> 2) * (kTile * 128) + row * 128 +
                                 (((2 * (m & 3) + ((lane >> 3) & 1)) ^ (row & 7)) << 4);
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                     : "r"(address));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma(static_cast<const P *>(nullptr), out[m][nt], a, b[nt][0], b[nt][1], out[m][nt]);
      }
    } else {
      const int row = half * 16 + (g ^ ((g >> 1) & 1));      // the row of this lane's weights
      const int token = half * 16 + 2 * t + (t & 1);         // and the rows that its value registers hold:
      const int other = half * 16 + 2 * t + (1 ^ (t & 1));   // pi(2t), pi(2t + 1), and 8 later
#pragma unroll
      for (int gi = 0; gi < kNG; ++gi) {
        const uint32_t scales = values_at + L::kCodes + (row * kNG + gi) * 4;
        const float2 v0 = load_pair(scales), v1 = load_pair(scales + 8 * kNG * 4);
        uint32_t b[NT][2];
        const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float scaled[4], shift[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = i < 2 ? v0 : v1;
            const bool none = MASKED && first_row + row + (i < 2 ? 0 : 8) >= seen[nt][i & 1];
            scaled[i] = none ? 0.0f : w[nt][i] * v.x;
            shift[i] = none ? 0.0f : w[nt][i] * v.y;
          }
          b[nt][0] = transpose8(pack(static_cast<const P *>(nullptr), scaled[0], scaled[1]));
          b[nt][1] = transpose8(pack(static_cast<const P *>(nullptr), scaled[2], scaled[3]));
          offset_sum[nt][gi][0] += shift[0] + shift[2];
          offset_sum[nt][gi][1] += shift[1] + shift[3];
          mma(static_cast<const P *>(nullptr), scaled_sum[nt][gi], ones, b[nt][0], b[nt][1], scaled_sum[nt][gi]);
        }
        const uint32_t at = values_at + gi * (GROUP / 2) + g * (GROUP / 16);
        constexpr int kWords = GROUP == 128 ? 2 : 1;
        constexpr int kBytes = GROUP / 16 / kWords;  // of a word that are used
        uint32_t x[4][kWords];
        const uint32_t rows[4] = {at + token * L::kRowBytes, at + other * L::kRowBytes,
                                  at + (token + 8) * L::kRowBytes, at + (other + 8) * L::kRowBytes};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (GROUP == 32) x[r][0] = load_short(rows[r]);
          else load_words<kWords>(rows[r], x[r]);
        }
#pragma unroll
        for (int word = 0; word < kWords; ++word)
#pragma unroll
          for (int k = 0; k < kBytes; ++k) {
            const uint32_t select = k * 0x0011u + (4 + k) * 0x1100u;
            const uint32_t lo = __byte_perm(x[0][word], x[1][word], select);
            const uint32_t hi = __byte_perm(x[2][word], x[3][word], select);
            const uint32_t a[4] = {lo & 0x000f000fu, lo & 0x00f000f0u, hi & 0x000f000fu, hi & 0x00f000f0u};
            const int m = gi * (GROUP / 16) + word * kBytes + k;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma(static_cast<const P *>(nullptr), out[m][nt], a, b[nt][0], b[nt][1], out[m][nt]);
          }
      }
    }
  }

  template <bool MASKED>
  __device__ __forceinline__ void tile(uint32_t stage, uint32_t query_at, const float *group_sums, int lane,
                                       int32_t first_row, int32_t seen_max) {
    float s[2][NT][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) scores(stage, query_at, group_sums, half, lane, s[half]);
    if constexpr (MASKED) {
      const int g = lane >> 2;
      const int row = first_row + (GROUP == 0 ? g : g ^ ((g >> 1) & 1));
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row + half * 16 + (i < 2 ? 0 : 8) >= seen[nt][i & 1]) s[half][nt][i] = -INFINITY;
    }
    bool grows = false;
    float best[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // max_nan: a NaN score makes the maximum, and with it the result, NaN.
        float m = max_nan(max_nan(s[0][nt][i], s[0][nt][i + 2]), max_nan(s[1][nt][i], s[1][nt][i + 2]));
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 16));
        best[nt][i] = max_nan(m, top[nt][i]);
        grows |= best[nt][i] != top[nt][i];
      }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float keep = top[nt][i] == -INFINITY ? 0.0f : exp2_fast(top[nt][i] - best[nt][i]);
          top[nt][i] = best[nt][i];
          sum[nt][i] *= keep;
#pragma unroll
          for (int g = 0; g < kNG; ++g) {
            offset_sum[nt][g][i] *= keep;
            scaled_sum[nt][g][i] *= keep;
            scaled_sum[nt][g][i + 2] *= keep;
          }
#pragma unroll
          for (int m = 0; m < kOut; ++m) {
            out[m][nt][i] *= keep;
            out[m][nt][i + 2] *= keep;
          }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float m = top[nt][i] == -INFINITY ? 0.0f : top[nt][i];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          s[half][nt][i] = exp2_fast(s[half][nt][i] - m);
          s[half][nt][i + 2] = exp2_fast(s[half][nt][i + 2] - m);
        }
        sum[nt][i] += (s[0][nt][i] + s[0][nt][i + 2]) + (s[1][nt][i] + s[1][nt][i + 2]);
      }
    if constexpr (MASKED && GROUP == 0) {
      // What lies beyond every query's rows may be NaN, and 0 NaN is NaN.
      const uint32_t values_at = stage + L::kCodes;
      if (first_row + lane >= seen_max)
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(values_at + (c >> 3) * (kTile * 128) + lane * 128 +
                                                                    (c & 7) * 16),
                       "r"(0)
                       : "memory");
      __syncwarp();
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) values<MASKED>(stage, half, lane, s[half], first_row);
  }
};

template <typename T, int D, int GROUP, int NT>
__global__ __launch_bounds__(kThreads, (Layout<T, D, GROUP, NT>::kBlocksPerSm))
void attention_kernel(const AttentionParam p, const __grid_constant__ CUtensorMap key_map,
                      const __grid_constant__ CUtensorMap value_map) {
  using L = Layout<T, D, GROUP, NT>;
  extern __shared__ uint8_t shared_raw[];
  uint8_t *shared = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(shared_raw) + 1023) & ~uintptr_t{1023});
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(shared));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t full = base + L::kBarriersAt, empty = full + L::kStages * 8;
  int64_t *walk_start = reinterpret_cast<int64_t *>(shared + L::kBarriersAt + 2 * L::kStages * 8);  // slot_start, total
  int32_t *walk_slot = reinterpret_cast<int32_t *>(walk_start + 2);
  volatile int *abort = walk_slot + 1;
  int *arrived = const_cast<int *>(walk_slot) + 2;

  // This block's stretch: a scan of every slot's tiles.
  __shared__ int64_t warp_sums[kWarps + 1];
  const int32_t each = (p.slots + kThreads - 1) / kThreads;
  const int32_t mine0 = min(static_cast<int32_t>(threadIdx.x) * each, p.slots), mine1 = min(mine0 + each, p.slots);
  int64_t mine = 0;
  for (int32_t s = mine0; s < mine1; ++s) {
    mine += Walk<L::kRows>::cost(p, s);
    if (blockIdx.x == 0 && p.lengths[s] > p.capacity) atomicOr(p.flag, kFlagRow);
  }
  int64_t before = mine;
#pragma unroll
  for (int step = 1; step < 32; step <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, before, step);
    if (lane >= step) before += x;
  }
  if (lane == 31) warp_sums[warp] = before;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      tc::init_barrier(full + i * 8, 1);
      tc::init_barrier(empty + i * 8, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    *abort = 0;
  }
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w <= kWarps; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  before -= mine;
  const int64_t share = lmax((total + gridDim.x - 1) / gridDim.x, kMinTiles);
  const int64_t start = share * blockIdx.x;
  if (start >= total) return;
  if (start >= before && start < before + mine) {
    int32_t s = mine0;
    for (int64_t c; start >= before + (c = Walk<L::kRows>::cost(p, s)); ++s) before += c;
    walk_start[0] = before;
    *walk_slot = s;
  }
  __syncthreads();
  Walk<L::kRows> walk{p, start, lmin(start + share, total), walk_start[0], *walk_slot};
  Segment s;

  if (warp == kWarps) {
    // The feeding warp: every tile of the stretch in order, through the ring.
    int64_t count = 0;
    while (walk.next(s)) {
      const int32_t *entries = p.table + static_cast<int64_t>(s.slot) * p.table_stride;
      for (int32_t first = s.tile0; first < s.tile1; first += 32) {
        // Lane i looks up the page(s) of tile first + i.
        const int32_t ahead = first + lane;
        int32_t page[2] = {0, 0};
        constexpr int kParts = 2;
        const int parts = p.pages.page_size == 16 ? kParts : 1;
        if (ahead < s.tile1)
          for (int part = 0; part < parts; ++part) {
            const int32_t row = ahead * kTile + part * 16;
            if (row >= s.seen_max) break;
            page[part] = entries[row >> p.pages.page_shift];
            if (page[part] < 0 || page[part] >= p.pages.pages) {
              page[part] = 0;
              atomicOr(p.flag, kFlagRow);
            }
          }
        const int32_t last = min(first + 32, s.tile1);
        for (int32_t tile = first; tile < last; ++tile, ++count) {
          const int32_t page0 = __shfl_sync(0xffffffffu, page[0], tile - first);
          const int32_t page1 = __shfl_sync(0xffffffffu, page[1], tile - first);
          const int stage = static_cast<int>(count % L::kStages);
          const uint32_t phase = static_cast<uint32_t>(count / L::kStages) & 1;
          const uint32_t at = base + stage * L::kStage, barrier = full + stage * 8;
          if (count >= L::kStages && !wait(empty + stage * 8, phase ^ 1, abort)) {
            if (lane == 0) atomicOr(p.flag, kFlagTimeout);
            goto drained;
          }
          const int32_t row = tile * kTile;
          const int copies = parts == 1 || row + 16 >= s.seen_max ? 1 : 2;  // pages that the tile's rows lie in
          const int rows = parts == 1 ? kTile : 16;
          if (lane == 0) tc::expect_bytes(barrier, copies * rows * (L::kStage / kTile));
          __syncwarp();
          if constexpr (GROUP == 0) {
            constexpr int kBoxes = D / 64;  // 64 channels wide, per tensor and page
            if (lane < copies * 2 * kBoxes) {
              const int part = lane / (2 * kBoxes), side = (lane / kBoxes) & 1, box = lane % kBoxes;
              const int64_t y = static_cast<int64_t>(part ? page1 : page0) * p.pages.page_size +
                                (row & (p.pages.page_size - 1));
              tc::tma_box(at + side * L::kCodes + box * (kTile * 128) + part * 16 * 128, side ? &value_map : &key_map,
                          box * 64, static_cast<int>(y), barrier);
            }
          } else {
            if (lane < copies * 4) {
              const int part = lane >> 2, side = (lane >> 1) & 1;
              const bool scales = lane & 1;
              const int64_t y = static_cast<int64_t>(part ? page1 : page0) * p.pages.page_size +
                                (row & (p.pages.page_size - 1));
              const uint32_t to = at + side * (L::kCodes + L::kScales);
              if (scales) {
                const uint8_t *from = reinterpret_cast<const uint8_t *>(side ? p.pages.value_scales : p.pages.key_scales);
                bulk_copy(to + L::kCodes + part * 16 * L::kScaleBytes, from + y * L::kScaleBytes, rows * L::kScaleBytes,
                          barrier);
              } else {
                const uint8_t *from = side ? p.pages.values : p.pages.keys;
                bulk_copy(to + part * 16 * L::kRowBytes, from + y * L::kRowBytes, rows * L::kRowBytes, barrier);
              }
            }
          }
        }
      }
    }
    return;
  drained:
    // Given up: leave only after the copies in flight have landed.
    for (int64_t c = count > L::kStages ? count - L::kStages : 0; c < count; ++c)
      tc::wait_phase(full + static_cast<int>(c % L::kStages) * 8, static_cast<uint32_t>(c / L::kStages) & 1, nullptr);
    return;
  }

  Consumer<T, D, GROUP, NT> c;
  float *group_sums = reinterpret_cast<float *>(shared + L::kSumsAt);
  float *factors = reinterpret_cast<float *>(shared + L::kFactorAt);
  float *stat_top = reinterpret_cast<float *>(shared + L::kStatsAt), *stat_sum = stat_top + kWarps * L::kRows;
  float *scratch = reinterpret_cast<float *>(shared + L::kScratchAt);
  const uint32_t query_at = base + L::kQueryAt;
  const int g = lane >> 2, t = lane & 3;
  int64_t done = 0;  // tiles of the stretch before this segment
  while (walk.next(s)) {
    const int32_t sequence = s.slot / p.heads, head = s.slot - sequence * p.heads;
    const int32_t rows_total = s.tokens * p.groups;
    const int64_t query_heads = static_cast<int64_t>(p.heads) * p.groups;
    // Query fragments, one 8-row tile per warp: B operand of k-step ks holds,
    // for query row g, the channels of the matching A registers.
    for (int nt = warp; nt < NT; nt += kWarps) {
      const int32_t row = s.row0 + nt * 8 + g;
      const bool live = row < rows_total;
      const T *from = static_cast<const T *>(p.queries) +
                      static_cast<int64_t>(s.first_token + (live ? row / p.groups : 0)) * p.query_token +
                      (static_cast<int64_t>(head) * p.groups + (live ? row % p.groups : 0)) * p.query_head;
      uint2 *to = reinterpret_cast<uint2 *>(shared + L::kQueryAt) + nt * (D / 16) * 32 + lane;
      if constexpr (GROUP == 0) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t *pair = reinterpret_cast<const uint32_t *>(from + ks * 16 + 2 * t);
          to[ks * 32] = live ? make_uint2(pair[0], pair[4]) : make_uint2(0, 0);
        }
        if (t == 0) factors[nt * 8 + g] = p.scale_log2;
      } else {
        // This lane's D / 4 channels: GROUP / 4 of each group.
        float q[D / 4];
        float largest = 0.0f;
#pragma unroll
        for (int gi = 0; gi < L::kGroups; ++gi)
#pragma unroll
          for (int j = 0; j < GROUP / 32; ++j) {
            float *x = q + (gi * (GROUP / 32) + j) * 8;
            load8(from + gi * GROUP + t * (GROUP / 4) + j * 8, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (!live) x[i] = 0.0f;
              largest = fmaxf(largest, fabsf(x[i]));
            }
          }
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        // A power of two brings the row's largest value into [1, 2): f16 then
        // holds bf16 values exactly down to 2^-14 of the row's largest, and the
        // rest to 2^-25 of it.
        const int exponent = static_cast<int>(__float_as_uint(largest) >> 23);
        const bool plain = exponent == 255 || largest == 0.0f;
        const int shift = plain ? 0 : (exponent == 0 ? 1 : exponent) - 127;
        const float to_unit = __int_as_float((127 - min(shift, 126)) << 23);
        const float from_unit = __int_as_float((127 + min(shift, 127)) << 23);
#pragma unroll
        for (int gi = 0; gi < L::kGroups; ++gi) {
          float group_sum = 0.0f;
#pragma unroll
          for (int j = 0; j < GROUP / 32; ++j) {
            __half h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              h[i] = __float2half_rn(q[(gi * (GROUP / 32) + j) * 8 + i] * to_unit);
              group_sum += __half2float(h[i]);
            }
            const __half sixteen = __float2half_rn(16.0f);
            const int ks = gi * (GROUP / 16) + 2 * j;
            __half2 b[4] = {__halves2half2(__hmul(h[0], sixteen), __hmul(h[4], sixteen)),
                            __halves2half2(__hmul(h[2], sixteen), __hmul(h[6], sixteen)), __halves2half2(h[1], h[5]),
                            __halves2half2(h[3], h[7])};
            to[ks * 32] = *reinterpret_cast<uint2 *>(&b[0]);
            to[(ks + 1) * 32] = *reinterpret_cast<uint2 *>(&b[2]);
          }
          group_sum += __shfl_xor_sync(0xffffffffu, group_sum, 1);
          group_sum += __shfl_xor_sync(0xffffffffu, group_sum, 2);
          if (t == 0) group_sums[gi * L::kRows + nt * 8 + g] = group_sum * 0x1p-20f;
        }
        if (t == 0) factors[nt * 8 + g] = p.scale_log2 * 0x1p20f * from_unit;
      }
    }
    consumers_sync();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int32_t row = s.row0 + nt * 8 + 2 * t + i;
        c.factor[nt][i] = factors[nt * 8 + 2 * t + i];
        c.seen[nt][i] = row < rows_total ? Walk<L::kRows>::seen(p, s, row) : s.seen_max;
      }
    if constexpr (NT <= 2) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          load_words<2>(query_at + ((nt * (D / 16) + ks) * 32 + lane) * 8, c.query[nt][ks]);
    }
    c.clear();
    const int32_t tiles = max(s.tile1 - s.tile0, 0);
    // Tile number k of the whole stretch falls to warp k mod kWarps.
    for (int32_t i = static_cast<int32_t>((warp + kWarps - done % kWarps) % kWarps); i < tiles; i += kWarps) {
      const int64_t k = done + i;
      const int stage = static_cast<int>(k % L::kStages);
      const uint32_t phase = static_cast<uint32_t>(k / L::kStages) & 1;
      if (!wait(full + stage * 8, phase, abort)) {
        if (lane == 0) atomicOr(p.flag, kFlagTimeout);
        continue;  // every barrier below is still met
      }
      const int32_t first_row = (s.tile0 + i) * kTile;
      const uint32_t at = base + stage * L::kStage;
      if (first_row + kTile > s.seen_min) {
        c.template tile<true>(at, query_at, group_sums, lane, first_row, s.seen_max);
        if constexpr (GROUP == 0) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      } else {
        c.template tile<false>(at, query_at, group_sums, lane, first_row, s.seen_max);
      }
      __syncwarp();
      if (lane == 0) tc::arrive(empty + stage * 8);
    }
    done += tiles;

    // Join the warps.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int step = 4; step < 32; step <<= 1) {
          c.sum[nt][i] += __shfl_xor_sync(0xffffffffu, c.sum[nt][i], step);
#pragma unroll
          for (int gi = 0; gi < L::kGroups; ++gi)
            c.offset_sum[nt][gi][i] += __shfl_xor_sync(0xffffffffu, c.offset_sum[nt][gi][i], step);
        }
        if (g == 0) {
          stat_top[warp * L::kRows + nt * 8 + 2 * t + i] = c.top[nt][i];
          stat_sum[warp * L::kRows + nt * 8 + 2 * t + i] = c.sum[nt][i];
        }
      }
    consumers_sync();
    const bool whole = s.starts && s.ends;
    const bool whole_unit = whole || (s.starts && s.unit_start + s.unit_tiles <= walk.end);
    float *partial = p.partials + (static_cast<int64_t>(blockIdx.x) * 2 + (s.starts ? 1 : 0)) * L::kRows * (D + 2);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = nt * 8 + 2 * t + i;
        float best = stat_top[row];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) best = max_nan(best, stat_top[w * L::kRows + row]);
        const float weight = c.top[nt][i] == -INFINITY ? 0.0f : exp2_fast(c.top[nt][i] - best);
        float *to = scratch + (warp * 8 + 2 * t + i) * L::kPitch;
        if constexpr (GROUP == 0) {
#pragma unroll
          for (int m = 0; m < D / 16; ++m) {
            to[m * 16 + g] = weight * c.out[m][nt][i];
            to[m * 16 + 8 + g] = weight * c.out[m][nt][i + 2];
          }
        } else {
#pragma unroll
          for (int gi = 0; gi < L::kGroups; ++gi) {
            const float rest = fmaf(-8.0f, c.scaled_sum[nt][gi][i], c.offset_sum[nt][gi][i]);
#pragma unroll
            for (int k = 0; k < GROUP / 16; ++k) {
              const int m = gi * (GROUP / 16) + k;
              float2 pair = make_float2(weight * fmaf(c.out[m][nt][i], 0x1p24f, rest),
                                        weight * fmaf(c.out[m][nt][i + 2], 0x1p20f, rest));
              *reinterpret_cast<float2 *>(to + gi * GROUP + g * (GROUP / 8) + 2 * k) = pair;
            }
          }
        }
      }
      consumers_sync();
      constexpr int kEach = D / 16;  // channels per thread: 16 threads a row
      const int row = threadIdx.x >> 4, channel = (threadIdx.x & 15) * kEach;
      float best = stat_top[nt * 8 + row];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) best = max_nan(best, stat_top[w * L::kRows + nt * 8 + row]);
      float weight_sum = 0.0f;
      float value[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) value[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float m = stat_top[w * L::kRows + nt * 8 + row];
        weight_sum += m == -INFINITY ? 0.0f : exp2_fast(m - best) * stat_sum[w * L::kRows + nt * 8 + row];
#pragma unroll
        for (int i = 0; i < kEach; i += 4) {
          const float4 x = *reinterpret_cast<const float4 *>(scratch + (w * 8 + row) * L::kPitch + channel + i);
          value[i] += x.x;
          value[i + 1] += x.y;
          value[i + 2] += x.z;
          value[i + 3] += x.w;
        }
      }
      const int32_t query_row = s.row0 + nt * 8 + row;
      if (query_row < rows_total) {
        if (whole_unit) {
          const int64_t index = static_cast<int64_t>(s.first_token + query_row / p.groups) * query_heads +
                                static_cast<int64_t>(head) * p.groups + query_row % p.groups;
          const float inverse = weight_sum == 0.0f ? 0.0f : 1.0f / weight_sum;
          T result[kEach];
#pragma unroll
          for (int i = 0; i < kEach; ++i) result[i] = from_float<T>(value[i] * inverse);
          if constexpr (kEach == 8)
            *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + index * D + channel) = *reinterpret_cast<uint4 *>(result);
          else
            *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + index * D + channel) = *reinterpret_cast<uint2 *>(result);
          if (channel == 0)
            p.lse[index] = weight_sum == 0.0f ? -INFINITY : (best + log2f(weight_sum)) * 0.693147180559945f;
        } else {
#pragma unroll
          for (int i = 0; i < kEach; i += 4)
            *reinterpret_cast<float4 *>(partial + (nt * 8 + row) * D + channel + i) =
                make_float4(value[i], value[i + 1], value[i + 2], value[i + 3]);
          if (channel == 0) {
            partial[L::kRows * D + nt * 8 + row] = best;
            partial[L::kRows * (D + 1) + nt * 8 + row] = weight_sum;
          }
        }
      }
      consumers_sync();
    }
    if (whole_unit) continue;

    // The unit's blocks are first .. last; the one that arrives last joins.
    const int64_t first = s.unit_start / share, last = (s.unit_start + s.unit_tiles - 1) / share;
    __threadfence();
    consumers_sync();
    if (threadIdx.x == 0) {
      const uint32_t before_me = atomicAdd(p.counters + first, 1u);
      const bool joins = before_me == static_cast<uint32_t>(last - first);
      if (joins) p.counters[first] = 0;  // as the next call expects it
      *arrived = joins;
    }
    consumers_sync();
    if (!*arrived) continue;
    __threadfence();
    constexpr int kEach = D / 16;
    const int channel = (threadIdx.x & 15) * kEach;
    for (int row = threadIdx.x >> 4; row < L::kRows && s.row0 + row < rows_total; row += 8) {
      auto part_at = [&](int64_t block) {
        return p.partials + (block * 2 + (block == first ? 1 : 0)) * L::kRows * (D + 2);
      };
      float best = -INFINITY;
      for (int64_t b = first; b <= last; ++b) best = max_nan(best, __ldcg(part_at(b) + L::kRows * D + row));
      float weight_sum = 0.0f, value[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) value[i] = 0.0f;
#pragma unroll 4
      for (int64_t b = first; b <= last; ++b) {
        const float *from = part_at(b);
        const float m = __ldcg(from + L::kRows * D + row);
        const float weight = m == -INFINITY ? 0.0f : exp2_fast(m - best);
        weight_sum = fmaf(weight, __ldcg(from + L::kRows * (D + 1) + row), weight_sum);
#pragma unroll
        for (int i = 0; i < kEach; i += 4) {
          const float4 x = __ldcg(reinterpret_cast<const float4 *>(from + row * D + channel + i));
          value[i] = fmaf(weight, x.x, value[i]);
          value[i + 1] = fmaf(weight, x.y, value[i + 1]);
          value[i + 2] = fmaf(weight, x.z, value[i + 2]);
          value[i + 3] = fmaf(weight, x.w, value[i + 3]);
        }
      }
      const int32_t query_row = s.row0 + row;
      const int64_t index = static_cast<int64_t>(s.first_token + query_row / p.groups) * query_heads +
                            static_cast<int64_t>(head) * p.groups + query_row % p.groups;
      const float inverse = weight_sum == 0.0f ? 0.0f : 1.0f / weight_sum;
      T result[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) result[i] = from_float<T>(value[i] * inverse);
      if constexpr (kEach == 8)
        *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + index * D + channel) = *reinterpret_cast<uint4 *>(result);
      else
        *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + index * D + channel) = *reinterpret_cast<uint2 *>(result);
      if (channel == 0)
        p.lse[index] = weight_sum == 0.0f ? -INFINITY : (best + log2f(weight_sum)) * 0.693147180559945f;
    }
  }
}

template <typename T, int D, int GROUP, int NT>
int launch_rows(const AttentionParam &p, const lrk_pages &pages, cudaStream_t stream) {
  using L = Layout<T, D, GROUP, NT>;
  auto kernel = attention_kernel<T, D, GROUP, NT>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
  if (e != cudaSuccess) return fail(LRK_ERR_CUDA, cudaGetErrorString(e));
  CUtensorMap maps[2] = {};
  if (GROUP == 0 && pages.pages > 0) {
    const int64_t rows = pages.pages * pages.page_size;
    if (rows > INT32_MAX) return fail(LRK_ERR_UNSUPPORTED, "paged attention: too many 16-bit rows");
    const uint32_t box = static_cast<uint32_t>(std::min<int64_t>(pages.page_size, kTile));
    for (int side = 0; side < 2; ++side) {
      const int status = tc::make_map(&maps[side], side ? pages.values : pages.keys, rows, D, D, 64,
                                      CU_TENSOR_MAP_SWIZZLE_128B, box);
      if (status != LRK_OK) return status;
    }
  }
  const unsigned grid = static_cast<unsigned>(sm_count() * L::kBlocksPerSm);
  kernel<<<grid, kThreads, L::kBytes, stream>>>(p, maps[0], maps[1]);
  return launch_status("paged attention");
}

// Query rows per block by the rows that a slot has on average: 8, 16 or 32.
template <typename T, int D, int GROUP>
int launch_format(const AttentionParam &p, const lrk_pages &pages, int64_t tokens, int64_t sequences,
                  cudaStream_t stream) {
  const int64_t rows = ceil_div(tokens, sequences) * p.groups;
  if (rows <= 8) return launch_rows<T, D, GROUP, 1>(p, pages, stream);
  if (rows <= 16) return launch_rows<T, D, GROUP, 2>(p, pages, stream);
  return launch_rows<T, D, GROUP, 4>(p, pages, stream);
}

template <typename T, int D>
int launch_attention(const AttentionParam &p, const lrk_pages &pages, int64_t tokens, int64_t sequences,
                     cudaStream_t stream) {
  switch (pages.group) {
    case 0: return launch_format<T, D, 0>(p, pages, tokens, sequences, stream);
    case 32: return launch_format<T, D, 32>(p, pages, tokens, sequences, stream);
    case 64: return launch_format<T, D, 64>(p, pages, tokens, sequences, stream);
    default:
      if constexpr (D == 128) return launch_format<T, D, 128>(p, pages, tokens, sequences, stream);
      return LRK_ERR_UNSUPPORTED;
  }
}

}  // namespace
}  // namespace lrk

extern "C" size_t lrk_paged_attention_workspace_bytes(void) { return size_t{64} << 20; }

extern "C" int lrk_paged_attention(const lrk_pages *pages, const int32_t *table, int64_t table_stride,
                                   int64_t table_width, const int32_t *lengths, int64_t sequences, int64_t heads,
                                   const int32_t *token_starts, int64_t tokens, const lrk_rows *queries,
                                   int64_t query_heads, float scale, int causal, void *out, float *lse, int dtype,
                                   void *workspace, size_t workspace_bytes, unsigned int *flag, lrk_stream_t stream) {
  using namespace lrk;
  clear_error();
  if (int rc = paged::check_pages(pages)) return rc;
  LRK_REQUIRE(dtype == LRK_F16 || dtype == LRK_BF16, "paged attention: queries must be f16 or bf16");
  LRK_REQUIRE(pages->group != 0 || dtype == pages->dtype, "paged attention: queries must have the pages' type");
  LRK_REQUIRE(sequences >= 0 && heads >= 1 && tokens >= 0 && table_width >= 0, "paged attention: invalid sizes");
  LRK_REQUIRE(table_stride >= table_width, "paged attention: table rows overlap");
  LRK_REQUIRE(query_heads >= heads && query_heads % heads == 0 && query_heads < (1 << 20),
              "paged attention: query heads must be a multiple of the slots' heads");
  LRK_REQUIRE(scale == scale && scale - scale == 0.0f, "paged attention: scale must be finite");
  if (tokens == 0) return LRK_OK;
  LRK_REQUIRE(sequences >= 1, "paged attention: tokens without a sequence");
  LRK_REQUIRE((table != nullptr || table_width == 0) && lengths != nullptr && token_starts != nullptr &&
                  flag != nullptr && queries != nullptr && queries->data != nullptr && out != nullptr && lse != nullptr,
              "paged attention: null argument");
  LRK_REQUIRE(aligned(queries->data, 16) && queries->token_stride % 8 == 0 && queries->head_stride % 8 == 0 &&
                  aligned(out, 16),
              "paged attention: rows must be 16-byte aligned");
  LRK_REQUIRE(sequences * heads <= INT32_MAX && tokens * (query_heads / heads) <= INT32_MAX / 2,
              "paged attention: too many slots or query rows");
  if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < lrk_paged_attention_workspace_bytes())
    return fail(LRK_ERR_WORKSPACE, "paged attention: workspace too small");
  const int64_t capacity = pages->pages == 0 ? 0 : std::min<int64_t>(table_width * pages->page_size, INT32_MAX - 2 * kTile);
  AttentionParam p{};
  p.pages = paged::device_pages(*pages);
  p.table = table;
  p.table_stride = table_stride;
  p.capacity = static_cast<int32_t>(capacity);
  p.lengths = lengths;
  p.token_starts = token_starts;
  p.slots = static_cast<int32_t>(sequences * heads);
  p.tokens = static_cast<int32_t>(tokens);
  p.queries = queries->data;
  p.query_token = queries->token_stride;
  p.query_head = queries->head_stride;
  p.heads = static_cast<int>(heads);
  p.groups = static_cast<int>(query_heads / heads);
  p.scale_log2 = scale * 1.44269504088896f;
  p.causal = causal != 0;
  p.out = out;
  p.lse = lse;
  p.counters = static_cast<uint32_t *>(workspace);
  p.partials = reinterpret_cast<float *>(p.counters + kCounters);
  p.flag = flag;
  if (dtype == LRK_F16)
    return pages->dimension == 64 ? launch_attention<__half, 64>(p, *pages, tokens, sequences, stream)
                                  : launch_attention<__half, 128>(p, *pages, tokens, sequences, stream);
  return pages->dimension == 64 ? launch_attention<__nv_bfloat16, 64>(p, *pages, tokens, sequences, stream)
                                : launch_attention<__nv_bfloat16, 128>(p, *pages, tokens, sequences, stream);
}
