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
// instructions per code.  Measured (32 requests of 33,768 rows a head, 8 query
// heads a KV head, group 128): 268 to 285 us by machine, 4.1 to 4.4 TB/s, 63 to
// 67 % of the copy rate, at 58 % of the issue slots and 60 % of the integer pipe
// (four warps a scheduler wait for their own instructions); copies alone, with
// nothing computed, 203 us.  In 16 bits (8 ragged requests) 58 to 60 us, 5.4 TB/s.
// Hence the shape of the arithmetic:
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
// Tiles are 32 rows; every warp moves its own (bulk copies, or TMA boxes with a
// 128-byte swizzle for 16-bit rows) into one or two stages of its own, so the
// warps of a block meet only at a unit's ends.  How the tiles are split over the
// blocks: paged_attention.cuh.  Measured on the way, in short runs of the long
// case: a feeding warp per block (16 consumers and 4 feeders an SM) 296 us; twenty
// warps at 96 registers, with spills, 276; sixteen at 128 registers 257.
#include <cuda.h>

#include <algorithm>

#include "paged_attention.cuh"

namespace lrk {

// Many query rows a slot (paged_attention_tc.cu).
int launch_paged_attention_tc(const void *param, const lrk_pages &pages, int dtype, cudaStream_t stream);

namespace {

using namespace paged;

constexpr int kTile = 32;   // rows per tile
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
// More query rows a slot than this go to paged_attention_tc.cu.  At 64 rows this
// file's kernel takes 54, 84 and 41 us (one request of 16,384 rows a head,
// D = 128; 24 of 4,000, D = 64; two of 8,192 in 16 bits) and that one 62, 103 and
// 45; at 96 rows 68, 120 and 58 against 72, 112 and 52.
constexpr int kMatrixRows = 64;
constexpr int kMinTiles = kWarps;  // tiles per block, at least
constexpr int kCrossing = 10;      // a second unit's cost in tiles: its start, its end, its join

template <typename T, int D, int GROUP, int NT>
struct Layout {
  static constexpr int kRowBytes = GROUP ? D / 2 : D * 2;
  static constexpr int kGroups = GROUP ? D / GROUP : 1;
  static constexpr int kScaleBytes = GROUP ? kGroups * 4 : 0;
  static constexpr int kRows = 8 * NT;  // query rows per block
  static constexpr int kCodes = kTile * kRowBytes, kScales = kTile * kScaleBytes;
  static constexpr int kStage = 2 * (kCodes + kScales);  // key rows, key scales, value rows, value scales
  static constexpr int kPitch = D + 4;
  static constexpr int kScratch = kWarps * 8 * kPitch * 4;
  static constexpr int kQuery = NT * (D / 16) * 32 * 8;
  // Blocks on an SM, by registers (4-bit rows: 128, 168 and 255 a thread), and
  // one or two stages a warp, as their share of shared memory holds.  16-bit
  // rows: three blocks 57 us, two 59 (8 ragged requests).
  static constexpr int kBlocksPerSm = GROUP ? (NT == 1 ? 4 : NT == 2 ? 3 : 2) : (NT <= 2 ? 3 : 2);
  static constexpr int kControl = 416;  // bytes of Control
  static constexpr int kFixed = kQuery + kGroups * kRows * 8 + kRows * 8 + 2 * kWarps * kRows * 4 + kControl;
  static constexpr int kFit = ((232448 / kBlocksPerSm - 1024) / 128 * 128 - kFixed) / kStage / kWarps;
  static constexpr int kDepth = kFit > 2 ? 2 : kFit;  // stages of a warp
  static constexpr int kStages = kDepth * kWarps;
  // The stages, in their place the scratch of a segment's end; query
  // fragments, group sums, factors, maxima and sums, control.
  static constexpr int kQueryAt = kStages * kStage > kScratch ? kStages * kStage : kScratch;
  static constexpr int kSumsAt = kQueryAt + kQuery;
  static constexpr int kFactorAt = kSumsAt + kGroups * kRows * 8;
  static constexpr int kSeenAt = kFactorAt + kRows * 4;
  static constexpr int kStatsAt = kSeenAt + kRows * 4;
  static constexpr int kControlAt = kStatsAt + 2 * kWarps * kRows * 4;
  static constexpr int kBytes = kControlAt + kControl;
  static_assert(kDepth >= 1, "every warp needs a stage of its own");
};

__device__ __forceinline__ void mma(const __half *, float *d, const uint32_t *a, uint32_t b0, uint32_t b1,
                                    const float *c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma(const __nv_bfloat16 *, float *d, const uint32_t *a, uint32_t b0, uint32_t b1,
                                    const float *c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Transpose of an 8 x 8 matrix of 16-bit elements spread over the warp: the
// columns of S^T (query rows) become the rows that P's B operand wants.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
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

// Two halves, 65504 in the place of NaN and what is larger.
__device__ __forceinline__ uint32_t drop_nan(uint32_t x) {
  uint32_t y;
  asm("min.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x7bff7bffu));
  return y;
}

template <int WORDS>
__device__ __forceinline__ void load_words(const uint8_t *from, uint32_t *w) {
  if constexpr (WORDS == 4) {
    const uint4 x = *reinterpret_cast<const uint4 *>(from);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else if constexpr (WORDS == 2) {
    const uint2 x = *reinterpret_cast<const uint2 *>(from);
    w[0] = x.x, w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t *>(from);
  }
}
__device__ __forceinline__ float2 load_pair(const uint8_t *from) {  // (scale, offset)
  return __half22float2(*reinterpret_cast<const __half2 *>(from));
}

// A block's shared words beside the stages.
template <int ROWS>
struct Control {
  uint64_t landed[2 * kWarps];  // barriers of the stages
  int64_t sums[2][kWarps];
  Walk<ROWS, kTile> walk;
  int32_t abort;
  int32_t arrived[2];
  uint8_t gone[2 * kWarps];  // of a stage's tile: bit h set where the page of its rows 16 h .. does not exist
  Segment pending[2];
  Segment segments[2];  // this one and the next; slot -1 ends them
};

template <typename T, int D, int GROUP, int NT>
struct Consumer {
  using L = Layout<T, D, GROUP, NT>;
  static constexpr int kOut = D / 16;
  static constexpr int kNG = L::kGroups;
  using P = std::conditional_t<GROUP == 0, T, __half>;  // the weights' type, as the matrix instruction wants V's

  // Weights are exp2(s - top).  top follows the running maximum loosely: it is
  // set to the maximum less kHead, and set again only when a score passes it by
  // more than kMost.  So most tiles neither exchange maxima nor rescale (with
  // an exact maximum 11 of a warp's first 18 tiles did), and small weights stay
  // in f16's normal range (11 bits down to 2^-22 of the largest; with kHead = 0
  // it would be 2^-14, which cost a third of a bf16 output's precision over
  // 34,768 rows).  For 4-bit rows the operand is weight * scale: 2^12 * 8 = 2^15
  // while a value's scale is at most 8; `lift` (0 until then) raises top where
  // a larger one is met.  bf16 has float32's range and needs no head.
  static constexpr bool kHalfWeights = std::is_same<P, __half>::value;
  static constexpr float kHead = GROUP ? 8.0f : kHalfWeights ? 10.0f : 0.0f;
  static constexpr float kMost = GROUP ? 12.0f : kHalfWeights ? 14.0f : 8.0f;

  float out[kOut][NT][4];
  float top[NT][2], sum[NT][2];
  int32_t lift;
  float offset_sum[NT][kNG][2];
  float scaled_sum[NT][(kNG + 1) / 2][4];  // of group gi: elements 2 (gi mod 2) and after
  float factor[NT][2];

  __device__ __forceinline__ void clear() {
    lift = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int m = 0; m < kOut; ++m) out[m][nt][i] = 0.0f;
#pragma unroll
        for (int g = 0; g < (kNG + 1) / 2; ++g) scaled_sum[nt][g][i] = 0.0f;
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

  // B operands of k-steps 2 pair and 2 pair + 1.
  __device__ __forceinline__ static void query_fragments(const uint8_t *query_at, int nt, int pair, int lane,
                                                         uint32_t *b) {
    load_words<4>(query_at + ((nt * (D / 32) + pair) * 32 + lane) * 16, b);
  }

  // The largest of the value scales' bits, signs left out, in this lane's row of
  // the tile; with FINITE, of those that are finite.
  template <bool FINITE = false>
  __device__ __forceinline__ static uint32_t largest_scale(const uint8_t *stage, int lane) {
    uint32_t w[kNG], largest = 0;
    load_words<kNG>(stage + 2 * L::kCodes + L::kScales + lane * L::kScaleBytes, w);
#pragma unroll
    for (int gi = 0; gi < kNG; ++gi) {
      const uint32_t bits = w[gi] & 0x7fffu;
      largest = max(largest, FINITE && bits >= 0x7c00u ? 0u : bits);
    }
    return largest;
  }

  // The largest scale (in f16's bits) that the lift allows: 8 * 2^lift.
  __device__ __forceinline__ uint32_t plain_scale() const { return 0x4800u + (static_cast<uint32_t>(lift) << 10); }

  // Sets top anew for scores whose maxima in this lane are `best`.
  __device__ __forceinline__ void raise(const float (*best)[2], uint32_t largest) {
    const int32_t lifted = lift;
    if constexpr (GROUP != 0) {
      if (__any_sync(0xffffffffu, largest > plain_scale())) {
        const uint32_t exponent = __reduce_max_sync(0xffffffffu, largest >> 10);
        lift = max(lift, static_cast<int32_t>(exponent) - 17);  // scale < 2^(exponent - 14)
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // max_nan: a NaN score makes the result NaN.
        float m = best[nt][i];
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 16));
        const float next = max_nan(fmaf(m, factor[nt][i], static_cast<float>(lift) - kHead),
                                   top[nt][i] + static_cast<float>(lift - lifted));
        const float keep = top[nt][i] == -INFINITY ? 0.0f : exp2_fast(top[nt][i] - next);
        top[nt][i] = next;
        sum[nt][i] *= keep;
#pragma unroll
        for (int g = 0; g < kNG; ++g) {
          offset_sum[nt][g][i] *= keep;
          scaled_sum[nt][g / 2][i + 2 * (g & 1)] *= keep;
        }
#pragma unroll
        for (int m = 0; m < kOut; ++m) {
          out[m][nt][i] *= keep;
          out[m][nt][i + 2] *= keep;
        }
      }
  }

  // Scores of the tile's rows against the block's query rows, both halves of 16
  // rows side by side: s[half][nt][0..1] of row pi(g), [2..3] of row 8 + pi(g).
  // pi(g) = g ^ (g >> 1 & 1), so that keys (rows by g) and values (rows by t)
  // both spread over the banks; 16-bit rows are swizzled and take pi(g) = g.
  __device__ __forceinline__ void scores(const uint8_t *stage, const uint8_t *query_at, const float *group_sums, int lane,
                                         float (*s)[NT][4]) {
    const int g = lane >> 2, t = lane & 3;
    if constexpr (GROUP == 0) {
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[half][nt][i] = 0.0f;
#pragma unroll
      for (int pair = 0; pair < D / 32; ++pair) {
        uint32_t a[2][2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int row = half * 16 + (lane & 15), ks = 2 * pair + k;
            const uint32_t address = shared_address(stage) + (ks >> 2) * (kTile * 128) + row * 128 +
                                     (((2 * (ks & 3) + (lane >> 4)) ^ (row & 7)) << 4);
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(a[half][k][0]), "=r"(a[half][k][1]), "=r"(a[half][k][2]), "=r"(a[half][k][3])
                         : "r"(address)
                         : "memory");
          }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          uint32_t b[4];
          query_fragments(query_at, nt, pair, lane, b);
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int half = 0; half < 2; ++half)
              mma(static_cast<const P *>(nullptr), s[half][nt], a[half][k], b[2 * k], b[2 * k + 1], s[half][nt]);
        }
      }
    } else {
      const int row = g ^ ((g >> 1) & 1);
#pragma unroll
      for (int gi = 0; gi < kNG; ++gi) {
        uint32_t w[4][GROUP / 32];
        const uint8_t *address = stage + row * L::kRowBytes + gi * (GROUP / 2) + t * (GROUP / 8);
#pragma unroll
        for (int r = 0; r < 4; ++r) load_words<GROUP / 32>(address + 8 * r * L::kRowBytes, w[r]);
        float acc[2][NT][4], q[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float4 sums = *reinterpret_cast<const float4 *>(group_sums + 2 * (gi * L::kRows + nt * 8 + 2 * t));
          q[nt][0] = sums.x;
          q[nt][1] = sums.z;
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[0][nt][i] = acc[1][nt][i] = i & 1 ? sums.w : sums.y;
        }
#pragma unroll
        for (int j = 0; j < GROUP / 32; ++j) {
          uint32_t low[2][4], high[2][4];
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const uint32_t x = w[2 * half + r][j], y = x >> 8;
              low[half][r] = x & 0x000f000fu;
              low[half][r + 2] = y & 0x000f000fu;
              high[half][r] = x & 0x00f000f0u;
              high[half][r + 2] = y & 0x00f000f0u;
            }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint32_t b[4];
            query_fragments(query_at, nt, gi * (GROUP / 32) + j, lane, b);
#pragma unroll
            for (int half = 0; half < 2; ++half)
              mma(static_cast<const P *>(nullptr), acc[half][nt], low[half], b[0], b[1], acc[half][nt]);
#pragma unroll
            for (int half = 0; half < 2; ++half)
              mma(static_cast<const P *>(nullptr), acc[half][nt], high[half], b[2], b[3], acc[half][nt]);
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint8_t *scales = stage + L::kCodes + ((half * 16 + row) * kNG + gi) * 4;
          const float2 k0 = load_pair(scales), k1 = load_pair(scales + 8 * kNG * 4);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 k = i < 2 ? k0 : k1;
              const float x = gi == 0 ? k.y * q[nt][i & 1] : fmaf(k.y, q[nt][i & 1], s[half][nt][i]);
              s[half][nt][i] = fmaf(k.x, acc[half][nt][i], x);
            }
        }
      }
    }
  }

  // Adds 16 rows' weighted values to the output.  With MASKED, rows that a
  // query does not see add nothing, whatever their scales hold.
  template <bool MASKED>
  __device__ __forceinline__ void values(const uint8_t *stage, int half, int lane, const float (*w)[4], int32_t first_row,
                                         const int32_t *seen_by) {
    const int g = lane >> 2, t = lane & 3;
    const uint8_t *values_at = stage + L::kCodes + L::kScales;
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
        const uint32_t address = shared_address(values_at) + (m >> 2) * (kTile * 128) + row * 128 +
                                 (((2 * (m & 3) + ((lane >> 3) & 1)) ^ (row & 7)) << 4);
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                     : "r"(address)
                     : "memory");
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
        const uint8_t *scales = values_at + L::kCodes + (row * kNG + gi) * 4;
        const float2 v0 = load_pair(scales), v1 = load_pair(scales + 8 * kNG * 4);
        uint32_t b[NT][2];
        // Ones in the upper or the lower eight rows: two groups share an accumulator.
        const uint32_t up = gi & 1 ? 0u : 0x3c003c00u, down = gi & 1 ? 0x3c003c00u : 0u;
        const uint32_t ones[4] = {up, down, up, down};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float scaled[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = i < 2 ? v0 : v1;
            const bool none = MASKED && first_row + row + (i < 2 ? 0 : 8) >= seen_by[nt * 8 + 2 * t + (i & 1)];
            scaled[i] = none ? 0.0f : w[nt][i] * v.x;
            float &sum_of = offset_sum[nt][gi][i & 1];
            sum_of = none ? sum_of : fmaf(w[nt][i], v.y, sum_of);
          }
          b[nt][0] = transpose8(pack(static_cast<const P *>(nullptr), scaled[0], scaled[1]));
          b[nt][1] = transpose8(pack(static_cast<const P *>(nullptr), scaled[2], scaled[3]));
          // A NaN (whose own products reach the group's output) must not reach the other
          // group through the zeros of `ones`: the minimum drops it.
          const uint32_t summed[2] = {kNG > 1 ? drop_nan(b[nt][0]) : b[nt][0], kNG > 1 ? drop_nan(b[nt][1]) : b[nt][1]};
          mma(static_cast<const P *>(nullptr), scaled_sum[nt][gi / 2], ones, summed[0], summed[1], scaled_sum[nt][gi / 2]);
        }
        const uint8_t *at = values_at + gi * (GROUP / 2) + g * (GROUP / 16);
        constexpr int kWords = GROUP == 128 ? 2 : 1;
        constexpr int kBytes = GROUP / 16 / kWords;  // of a word that are used
        uint32_t x[4][kWords];
        const uint8_t *rows[4] = {at + token * L::kRowBytes, at + other * L::kRowBytes,
                                  at + (token + 8) * L::kRowBytes, at + (other + 8) * L::kRowBytes};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (GROUP == 32) x[r][0] = *reinterpret_cast<const uint16_t *>(rows[r]);
          else load_words<kWords>(rows[r], x[r]);
        }
#pragma unroll
        for (int word = 0; word < kWords; ++word)
#pragma unroll
          for (int k = 0; k < kBytes; ++k) {
            const uint32_t select = k * 0x0011u + (4 + k) * 0x1100u;
            const uint32_t lo = __byte_perm(x[0][word], x[1][word], select);
            const uint32_t hi = __byte_perm(x[2][word], x[3][word], select);
            // (A whole byte, low + 16 high, as the lower operand row would save a
            // mask, but its sixteen times larger sums lose the output's precision.)
            const uint32_t a[4] = {lo & 0x000f000fu, lo & 0x00f000f0u, hi & 0x000f000fu, hi & 0x00f000f0u};
            const int m = gi * (GROUP / 16) + word * kBytes + k;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma(static_cast<const P *>(nullptr), out[m][nt], a, b[nt][0], b[nt][1], out[m][nt]);
          }
      }
    }
  }

  // With MASKED, rows that a query does not see are left out, and so are the 16
  // rows of half h where bit h of `gone` is set.
  template <bool MASKED>
  __device__ __forceinline__ void tile(uint8_t *stage, const uint8_t *query_at, const float *group_sums, int lane,
                                       int32_t first_row, int32_t seen_max, const int32_t *seen_by, uint32_t gone) {
    float s[2][NT][4];
    scores(stage, query_at, group_sums, lane, s);
    // Rows that are gone count as rows beyond every slot's length.
    constexpr int32_t kFar = INT32_MAX - 2 * kTile;
    const int32_t first[2] = {gone & 1 ? kFar : first_row, gone & 2 ? kFar : first_row};
    if constexpr (MASKED) {
      const int g = lane >> 2;
      const int row = GROUP == 0 ? g : g ^ ((g >> 1) & 1);
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (first[half] + row + half * 16 + (i < 2 ? 0 : 8) >= seen_by[nt * 8 + 2 * (lane & 3) + (i & 1)])
              s[half][nt][i] = -INFINITY;
    }
    uint32_t largest = 0;
    if constexpr (GROUP != 0) {
      // What lies beyond every query's rows (or was never copied) may be anything,
      // and must not raise `lift`.
      if (!MASKED || (lane < 16 ? first[0] : first[1]) + lane < seen_max) largest = largest_scale(stage, lane);
    }
    bool raises = largest > plain_scale();
    float best[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        best[nt][i] = max_nan(max_nan(s[0][nt][i], s[0][nt][i + 2], s[1][nt][i]), s[1][nt][i + 2]);
        // Also where best is NaN: top has to become NaN, since -inf stands for no rows.
        raises |= !(fmaf(best[nt][i], factor[nt][i], static_cast<float>(lift) - kMost) <= top[nt][i]);
      }
    if (__any_sync(0xffffffffu, raises)) {
      // Scales that are not finite reach their own group, whatever the lift, and must
      // not cost the others their precision.
      if constexpr (GROUP != 0) {
        if (largest >= 0x7c00u) largest = largest_scale<true>(stage, lane);
        __syncwarp();
      }
      raise(best, largest);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float m = top[nt][i] == -INFINITY ? 0.0f : top[nt][i];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          s[half][nt][i] = exp2_fast(fmaf(s[half][nt][i], factor[nt][i], -m));
          s[half][nt][i + 2] = exp2_fast(fmaf(s[half][nt][i + 2], factor[nt][i], -m));
        }
        sum[nt][i] += (s[0][nt][i] + s[0][nt][i + 2]) + (s[1][nt][i] + s[1][nt][i + 2]);
      }
    if constexpr (MASKED && GROUP == 0) {
      // What lies beyond every query's rows may be NaN, and 0 NaN is NaN.
      if ((lane < 16 ? first[0] : first[1]) + lane >= seen_max)
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          *reinterpret_cast<uint4 *>(stage + L::kCodes + (c >> 3) * (kTile * 128) + lane * 128 + (c & 7) * 16) =
              make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) values<MASKED>(stage, half, lane, s[half], first[half], seen_by);
  }
};

template <typename T, int D, int GROUP, int NT>
__global__ __launch_bounds__(kThreads, (Layout<T, D, GROUP, NT>::kBlocksPerSm))
void attention_kernel(const __grid_constant__ AttentionParam p, const __grid_constant__ CUtensorMap key_map,
                      const __grid_constant__ CUtensorMap value_map) {
  using L = Layout<T, D, GROUP, NT>;
  static_assert(sizeof(Control<L::kRows>) <= L::kControl, "Control has grown");
  extern __shared__ __align__(1024) uint8_t shared[];
  const uint32_t base = shared_address(shared);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Control<L::kRows> &control = *reinterpret_cast<Control<L::kRows> *>(shared + L::kControlAt);
  volatile int *abort = &control.abort;
  if (base & 1023) {  // the 128-byte swizzle goes by address bits
    if (threadIdx.x == 0) atomicOr(p.flag, kFlagShared);
    return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) tc::init_barrier(shared_address(&control.landed[i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    *abort = 0;
    for (int i = 0; i < 2 * kWarps; ++i) control.gone[i] = 0;
  }
  int64_t share;
  if (!begin<D, kThreads, kMinTiles, kCrossing>(p, &control.sums[0][0], share, control.walk, control.segments[0])) return;

  Consumer<T, D, GROUP, NT> c;
  float *group_sums = reinterpret_cast<float *>(shared + L::kSumsAt);
  float *factors = reinterpret_cast<float *>(shared + L::kFactorAt);
  int32_t *seen_by = reinterpret_cast<int32_t *>(shared + L::kSeenAt);
  float *stat_top = reinterpret_cast<float *>(shared + L::kStatsAt), *stat_sum = stat_top + kWarps * L::kRows;
  float *scratch = reinterpret_cast<float *>(shared);
  const uint8_t *query_at = shared + L::kQueryAt;
  const int g = lane >> 2, t = lane & 3;
  // A negative scale is taken by the queries, so that the largest score is the
  // largest product; the factor stays above zero for the sake of -inf.
  const uint32_t turn = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
  constexpr float kLeastFactor = 1e-37f;
  int pieces = 0;
  uint32_t phases = 0;  // of this warp's stages, a bit each
  // Set where this warp has met a page that does not exist in the segment: only
  // then is control.gone read and written.
  constexpr uint32_t kLost = 0x100;

  for (int number = 0;; ++number) {
    const Segment &s = control.segments[number & 1];
    if (s.slot < 0) break;
    // Warp w takes tiles w, w + kWarps, .. of the stretch, and moves them into
    // its own stages.  Lane i knows the page(s) of its tile number 32 k + i; -1
    // where the table names none, whose rows are left out.
    const int32_t tile0 = s.tile0 + warp, seen_min = s.seen_min, seen_max = s.seen_max;
    const int32_t own = max((s.tile1 - tile0 + kWarps - 1) / kWarps, 0);
    int32_t page0 = 0, page1 = 0;
    if (phases & kLost) {
      if (lane < L::kDepth) control.gone[warp * L::kDepth + lane] = 0;
      phases &= ~kLost;
      __syncwarp();
    }
    const auto look_up = [&](int32_t n) {
      const int32_t *entries = p.table + static_cast<int64_t>(s.slot) * p.table_stride;
      const int32_t row = (tile0 + (n + lane) * kWarps) * kTile;
      if (n + lane < own) {
        page0 = entries[row >> p.pages.page_shift];
        if (p.pages.page_size == 16 && row + 16 < seen_max) page1 = entries[(row + 16) >> p.pages.page_shift];
        else page1 = 0;
        if (static_cast<uint32_t>(page0) >= static_cast<uint32_t>(p.pages.pages)) page0 = -1;
        if (static_cast<uint32_t>(page1) >= static_cast<uint32_t>(p.pages.pages)) page1 = -1;
        if ((page0 | page1) < 0) atomicOr(p.flag, kFlagRow);
      }
      if (__any_sync(0xffffffffu, n + lane < own && (page0 | page1) < 0)) phases |= kLost;
    };
    const auto feed = [&](int32_t n) {
      if ((n & 31) == 0) look_up(n);
      if (lane != (n & 31)) return;
      const int slot = warp * L::kDepth + (L::kDepth == 2 ? n & 1 : 0);
      const uint32_t to = base + slot * L::kStage, barrier = shared_address(&control.landed[slot]);
      const int32_t row = (tile0 + n * kWarps) * kTile;
      const bool halves = p.pages.page_size == 16;
      const int rows = halves ? 16 : kTile;
      const int copies = halves && row + 16 < seen_max ? 2 : 1;  // pages that the tile's visible rows lie in
      int there = copies;
      if (phases & kLost) {
        const int gone0 = page0 < 0, gone1 = copies == 2 && page1 < 0;
        control.gone[slot] = gone0 && !halves ? 3 : gone0 | gone1 << 1;
        there -= gone0 + gone1;
      }
      tc::expect_bytes(barrier, there * rows * (L::kStage / kTile));
      for (int part = 0; part < copies; ++part) {
        if ((part ? page1 : page0) < 0) continue;
        const int64_t y = static_cast<int64_t>(part ? page1 : page0) * p.pages.page_size +
                          (row & (p.pages.page_size - 1));
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const uint32_t at = to + side * (L::kCodes + L::kScales);
          if constexpr (GROUP == 0) {
#pragma unroll
            for (int box = 0; box < D / 64; ++box)  // 64 channels wide
              tc::tma_box(at + box * (kTile * 128) + part * 16 * 128, side ? &value_map : &key_map, box * 64,
                          static_cast<int>(y), barrier);
          } else {
            bulk_copy(at + part * 16 * L::kRowBytes, (side ? p.pages.values : p.pages.keys) + y * L::kRowBytes,
                      rows * L::kRowBytes, barrier);
            bulk_copy(at + L::kCodes + part * 16 * L::kScaleBytes,
                      (side ? p.pages.value_scales : p.pages.key_scales) + y * L::kGroups, rows * L::kScaleBytes, barrier);
          }
        }
      }
    };
    for (int32_t n = 0; n < min(own, L::kDepth); ++n) feed(n);
    __syncwarp();
    if (threadIdx.x == kThreads - 1) {  // a thread of the warp with the fewest tiles finds the next segment
      Walk<L::kRows, kTile> walk = control.walk;
      Segment next;
      if (!walk.next(p, next)) next.slot = -1;
      control.segments[(number + 1) & 1] = next;
      control.walk = walk;
    }
    __syncwarp();
    const int32_t head = s.slot - s.sequence * p.heads;
    const int32_t rows_total = s.tokens * p.groups;
    // Query fragments: the B operand of a k-step holds, for query row g, the
    // channels of the matching A registers.  D / 8 threads a row, 8 channels each.
    constexpr int kAcross = D / 8;
    const int column = threadIdx.x % kAcross;
    for (int row = threadIdx.x / kAcross; row < L::kRows; row += kWarps * 32 / kAcross) {
      const int32_t query_row = s.row0 + row;
      const bool live = query_row < rows_total;
      if (column == 0) seen_by[row] = live ? rows_seen(p, s, query_row) : s.seen_max;
      const T *from = static_cast<const T *>(p.queries) +
                      static_cast<int64_t>(s.first_token + (live ? p.by_groups(query_row) : 0)) * p.query_token +
                      (static_cast<int64_t>(head) * p.groups + (live ? query_row - p.by_groups(query_row) * p.groups : 0)) * p.query_head;
      uint8_t *to = shared + L::kQueryAt + ((row >> 3) * (D / 32) * 32 + (row & 7) * 4) * 16;
      if constexpr (GROUP == 0) {
        // Channels 8 column ..: the low or high 8 of k-step column / 2, whose
        // pairs go to the four lanes of the row.
        uint4 x = live ? *reinterpret_cast<const uint4 *>(from + column * 8) : make_uint4(0, 0, 0, 0);
        const uint32_t pairs[4] = {x.x ^ turn, x.y ^ turn, x.z ^ turn, x.w ^ turn};
        uint32_t *words = reinterpret_cast<uint32_t *>(to + (column >> 2) * 32 * 16) + (column & 3);
#pragma unroll
        for (int i = 0; i < 4; ++i) words[i * 4] = pairs[i];
        if (column == 0) factors[row] = fmaxf(fabsf(p.scale_log2), kLeastFactor);
      } else {
        float x[8];
        load8(from + column * 8, x);
        float largest = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!live) x[i] = 0.0f;
          largest = fmaxf(largest, fabsf(x[i]));
        }
#pragma unroll
        for (int step = 1; step < kAcross; step <<= 1)
          largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, step));
        // A power of two brings the row's largest value into [1, 2) ([2, 4) from
        // 2^127 on): f16 then holds bf16 values exactly down to 2^-14 of the row's
        // largest, and the rest to 2^-25 of it.
        const int exponent = static_cast<int>(__float_as_uint(largest) >> 23);
        const bool plain = exponent == 255 || largest == 0.0f;
        const int shift = plain ? 0 : (exponent == 0 ? 1 : exponent) - 127;
        const float to_unit = __int_as_float(((127 - min(shift, 126)) << 23) | (turn & 0x80000000u));
        const float from_unit = __int_as_float((127 + min(shift, 126)) << 23);
        __half h[8];
        float group_sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          h[i] = __float2half_rn(x[i] * to_unit);
          group_sum += __half2float(h[i]);
        }
        const __half sixteen = __float2half_rn(16.0f);  // nibbles in bits 0-3 stand for a sixteenth of those in 4-7
        __align__(16) __half2 b[4] = {__halves2half2(__hmul(h[0], sixteen), __hmul(h[4], sixteen)),
                                      __halves2half2(__hmul(h[2], sixteen), __hmul(h[6], sixteen)),
                                      __halves2half2(h[1], h[5]), __halves2half2(h[3], h[7])};
        const int gi = column / (GROUP / 8), within = column % (GROUP / 8);
        const int quarter = within / (GROUP / 32), j = within % (GROUP / 32);
        reinterpret_cast<uint4 *>(to)[(gi * (GROUP / 32) + j) * 32 + quarter] = *reinterpret_cast<uint4 *>(b);
#pragma unroll
        for (int step = 1; step < GROUP / 8; step <<= 1) group_sum += __shfl_xor_sync(0xffffffffu, group_sum, step);
        group_sum *= 0x1p-20f;
        if (within == 0)
          reinterpret_cast<float2 *>(group_sums)[gi * L::kRows + row] = make_float2(group_sum, -8.0f * group_sum);
        if (column == 0) factors[row] = fmaxf(fabsf(p.scale_log2) * 0x1p20f * from_unit, kLeastFactor);
      }
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        c.factor[nt][i] = factors[nt * 8 + 2 * t + i];
      }
    c.clear();
    for (int32_t n = 0; n < own; ++n) {
      const int slot = L::kDepth == 2 ? n & 1 : 0;
      const uint32_t barrier = shared_address(&control.landed[warp * L::kDepth + slot]);
      uint8_t *const at = shared + (warp * L::kDepth + slot) * L::kStage;
      const int32_t first_row = (tile0 + n * kWarps) * kTile;
      const bool landed = __all_sync(0xffffffffu, wait(barrier, (phases >> slot) & 1, abort));
      const uint32_t gone = phases & kLost ? control.gone[warp * L::kDepth + slot] : 0;
      if (!landed) {
        // Given up: nothing more is computed, but every barrier is still met,
        // and the copy in flight gets its time to land.
        if (lane == 0) atomicOr(p.flag, kFlagTimeout);
        *abort = 1;
        tc::wait_phase(barrier, (phases >> slot) & 1, nullptr);
      } else if (first_row + kTile > seen_min || gone) {
        c.template tile<true>(at, query_at, group_sums, lane, first_row, seen_max, seen_by, gone);
        if constexpr (GROUP == 0) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      } else {
        c.template tile<false>(at, query_at, group_sums, lane, first_row, seen_max, seen_by, 0);
      }
      phases ^= 1u << slot;
      __syncwarp();
      if (n + L::kDepth < own) feed(n + L::kDepth);
      __syncwarp();
    }

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
    __syncthreads();  // the stages turn into scratch
    const bool whole_unit = s.starts && s.ends;
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
            const float rest = fmaf(-8.0f, c.scaled_sum[nt][gi / 2][i + 2 * (gi & 1)], c.offset_sum[nt][gi][i]);
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
      __syncthreads();
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
          const int64_t index = out_row(p, s, query_row);
          const float inverse = weight_sum == 0.0f ? 0.0f : 1.0f / weight_sum;
          __align__(16) T result[kEach];
#pragma unroll
          for (int i = 0; i < kEach; ++i) result[i] = from_float<T>(value[i] * inverse);
          if constexpr (kEach == 8)
            *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + index * D + channel) = *reinterpret_cast<uint4 *>(result);
          else
            *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + index * D + channel) = *reinterpret_cast<uint2 *>(result);
          if (channel == 0)
            p.lse[index] = natural(best, weight_sum);
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
      __syncthreads();
    }
    if (!whole_unit) {
      if (threadIdx.x == 0) control.pending[pieces] = s;
      ++pieces;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the scratch turns into stages
    __syncthreads();
  }
  if (pieces == 0) return;

  join<T, D, L::kRows, kThreads>(p, control.pending, control.arrived, pieces, share, scratch, kWarps * 8 * L::kPitch,
                                 stat_top, stat_sum);
}

template <typename T, int D, int GROUP, int NT>
int launch_rows(const AttentionParam &p, const lrk_pages &pages, cudaStream_t stream) {
  using L = Layout<T, D, GROUP, NT>;
  auto kernel = attention_kernel<T, D, GROUP, NT>;
  static std::atomic<uint64_t> allowed{0};  // devices, a bit each, that know the kernel's shared memory
  if (const int status = allow_shared(kernel, L::kBytes, allowed)) return status;
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

// Query rows per block by the rows that a slot has on average: 8, 16 or 32, the
// columns of the matrix instructions' B; rows that there are not cost as much.
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
  // Positions among all units' tiles stay far inside 64 bits, shares inside 32.
  LRK_REQUIRE(static_cast<double>(tokens) * query_heads / 8 * (static_cast<double>(table_width) * pages->page_size / kTile + 1) < 1e12,
              "paged attention: too many query rows for the table's length");
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
  p.by_heads = Divider::of(static_cast<uint32_t>(heads));
  p.by_groups = Divider::of(static_cast<uint32_t>(p.groups));
  p.scale_log2 = scale * 1.44269504088896f;
  p.causal = causal != 0;
  p.out = out;
  p.lse = lse;
  p.counters = static_cast<uint32_t *>(workspace);
  p.partials = reinterpret_cast<float *>(p.counters + kCounters);
  p.flag = flag;
  if (ceil_div(tokens, sequences) * p.groups > kMatrixRows) return launch_paged_attention_tc(&p, *pages, dtype, stream);
  if (dtype == LRK_F16)
    return pages->dimension == 64 ? launch_attention<__half, 64>(p, *pages, tokens, sequences, stream)
                                  : launch_attention<__half, 128>(p, *pages, tokens, sequences, stream);
  return pages->dimension == 64 ? launch_attention<__nv_bfloat16, 64>(p, *pages, tokens, sequences, stream)
                                : launch_attention<__nv_bfloat16, 128>(p, *pages, tokens, sequences, stream);
}
