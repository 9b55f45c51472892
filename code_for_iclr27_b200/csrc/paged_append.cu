// Paged cache: appending rows with the position rotation on the way, and
// reading rows back.
//
// Append.  Token i of sequence s (n_s new tokens) becomes row lengths - n_s + i
// of the sequence's slots.  Its keys and queries are rotated by the token's
// row of the rotary table: for each pair (a, b) of channels with cosine c and
// sine s,
//     a' = a c - b s,    b' = b c + a s,
// in float32, every product and sum rounded once (no contraction, so that a
// 4-bit code never depends on how the compiler fuses).  Pairs are (j, j + R/2)
// or, interleaved, (2j, 2j + 1), over the first R channels.  Keys and values
// are then stored as they are held: rounded to 16 bits, or in 4 bits per
// group of channels:
//     scale  = f16((max - min) * (1/15)),   offset = f16(min + 8 scale),
//     code   = clamp(rint((x - offset) * (1 / scale)) + 8, 0, 15).
// f16 keeps 11 bits of scale and offset, an error below a tenth of a step;
// bf16's 8 bits would move the ends of the range by up to a third of one.
//
// Memory bounds both (every row read and written once), launches the small ones.
// Measured: 19,538 tokens of 8 + 8 + 32 heads into 16-bit pages 88 us, 5.6 TB/s
// of what has to move; 32,768 tokens into 4-bit pages and the rows back 207 us,
// 4.4 TB/s (the append at 58 % of the issue slots, waiting for its rows most; the
// quantiser costs some ten instructions a channel); one layer of 276,000 4-bit rows
// back in bf16 37.5 us, 4.9 TB/s, at 73 % of the integer pipe.  In short runs the
// three took 87, 199 and 34.6 us, and with 16 neighbouring channels a lane, so that
// half of every rotated pair was read twice and half a sector stored at a time, 109,
// 267 and 38 us.
#include "paged.cuh"

namespace lrk {
namespace {

using namespace paged;

constexpr int kThreads = 128;
// From here on append_kernel goes BY_TOKENS (8 KV, 32 query heads, D = 128, into
// 16-bit pages; into 4-bit pages and back): 512 tokens 5.4 and 11.4 us against 4.5
// and 9.7, 1,024 6.0 and 13.5 against 6.5 and 13.4, 2,048 10.3 and 17.5 against
// 11.8 and 21.4.
constexpr int kManyTokens = 1024;

struct AppendParam {
  Pages pages;
  const int32_t *table;
  int64_t table_stride, table_width;
  const int32_t *lengths;
  const int32_t *token_starts;
  int64_t sequences, tokens;
  const void *keys, *values, *queries;
  void *out_queries;
  int64_t key_token, key_head, value_token, value_head, query_token, query_head;
  int heads, query_heads;
  const int64_t *positions;
  const float *rotary;
  int64_t rotary_positions;
  int rotary_dim;
  bool interleaved;
  uint32_t *flag;
};

__device__ __forceinline__ int64_t find_sequence(const AppendParam &p, int64_t token) {
  // Decode steps have one token a sequence: try that before searching.
  int64_t guess = p.tokens == p.sequences ? token : 0;
  if (p.token_starts[guess] <= token && token < p.token_starts[guess + 1]) return guess;
  int64_t lo = 0, hi = p.sequences;  // the last sequence whose start is <= token
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (p.token_starts[mid] <= token) lo = mid; else hi = mid;
  }
  return lo;
}

// Eight floats from 16-byte aligned memory, four from as many.
__device__ __forceinline__ void load_floats(const float *from, float *x) {
  const float4 v = *reinterpret_cast<const float4 *>(from);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}

// The rotation of a lane's two chunks of 8 channels: x' = x cosine + other sine,
// where `other` is the pair's other channel and the sine carries the sign.
struct Turn {
  float cosine[16], sine[16];
  bool turns[2];  // whether each chunk is rotated
};

template <int D, int CHUNKS>
__device__ __forceinline__ void load_turn(const AppendParam &p, const float *table, int lane, Turn &turn) {
  const int pairs = p.rotary_dim >> 1;
#pragma unroll
  for (int part = 0; part < CHUNKS; ++part) {
    const int c = lane * 8 + part * (D / 2);
    float *cosine = turn.cosine + 8 * part, *sine = turn.sine + 8 * part;
    turn.turns[part] = table != nullptr && c < p.rotary_dim;
    if (!turn.turns[part]) continue;
    if (p.interleaved) {
      float a[4], b[4];
      load_floats(table + (c >> 1), a);
      load_floats(table + pairs + (c >> 1), b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cosine[2 * i] = cosine[2 * i + 1] = a[i];
        sine[2 * i] = -b[i];
        sine[2 * i + 1] = b[i];
      }
    } else {
      const bool low = c < pairs;
      const int at = low ? c : c - pairs;
      load_floats(table + at, cosine);
      load_floats(table + at + 4, cosine + 4);
      load_floats(table + pairs + at, sine);
      load_floats(table + pairs + at + 4, sine + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) sine[i] = low ? -sine[i] : sine[i];
    }
  }
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &raw, float *x) {
  const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_float<T>(e[i]);
}

// Code words of 8 channels: levels held to [-8, 7] and added to 1.5 * 2^23 + 8
// leave their codes, rounded to nearest even, in the sums' last bits; the word is
// sum code_i 16^i.
__device__ __forceinline__ uint32_t code_word(const float *x, float centre, float inverse) {
  constexpr float kMagic = 12582920.0f;
  constexpr uint32_t kMagicBits = 0x4B400000u;  // of 1.5 * 2^23
  uint32_t word = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    const float level = __fmul_rn(__fsub_rn(x[i], centre), inverse);
    word = word * 16 + __float_as_uint(__fadd_rn(fminf(fmaxf(level, -8.0f), 7.0f), kMagic));
  }
  return word - kMagicBits * 0x11111111u;
}

// Quantises a lane's two chunks of 8 channels (lane * 8 and D / 2 after that); a
// group is GROUP / 8 neighbouring lanes' chunks, or the whole row.  Stores the
// codes and, once per group, the scale and offset; a negative row stores nothing.
template <int D, int GROUP>
__device__ __forceinline__ void store_codes(uint8_t *codes, __half2 *scales, int64_t row, int lane, const float *x) {
  constexpr bool kWhole = GROUP == D;
  constexpr int kLanes = kWhole ? D / 16 : GROUP / 8;
  float lo[2], hi[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float *y = x + 8 * k;
    lo[k] = min_nan(min_nan(y[0], y[1], y[2]), min_nan(y[3], y[4], y[5]), min_nan(y[6], y[7]));
    hi[k] = max_nan(max_nan(y[0], y[1], y[2]), max_nan(y[3], y[4], y[5]), max_nan(y[6], y[7]));
  }
  if (kWhole) {
    lo[0] = min_nan(lo[0], lo[1]);
    hi[0] = max_nan(hi[0], hi[1]);
  }
  __half scale[2], offset[2];
  uint32_t word[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (kWhole && k == 1) {
      scale[1] = scale[0], offset[1] = offset[0];
    } else {
#pragma unroll
      for (int step = 1; step < kLanes; step <<= 1) {
        lo[k] = min_nan(lo[k], __shfl_xor_sync(0xffffffffu, lo[k], step));
        hi[k] = max_nan(hi[k], __shfl_xor_sync(0xffffffffu, hi[k], step));
      }
      scale[k] = __float2half_rn(__fmul_rn(__fsub_rn(hi[k], lo[k]), 1.0f / 15.0f));
      offset[k] = __float2half_rn(__fadd_rn(lo[k], 8.0f * __half2float(scale[k])));
    }
    const float step = __half2float(scale[k]);
    const bool fine = !__hisinf(scale[k]) && !__hisnan(scale[k]) && !__hisinf(offset[k]) && !__hisnan(offset[k]);
    word[k] = fine ? code_word(x + 8 * k, __half2float(offset[k]), step > 0.0f ? __frcp_rn(step) : 0.0f) : 0u;
    if (!fine && !(kWhole && k == 0)) scale[k] = offset[k] = __ushort_as_half(0x7fff);
    if (kWhole && k == 1 && !fine) scale[0] = offset[0] = __ushort_as_half(0x7fff);
  }
  if (row < 0) return;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    *reinterpret_cast<uint32_t *>(codes + row * (D / 2) + lane * 4 + k * (D / 4)) = word[k];
    if (lane % kLanes == 0 && !(kWhole && k == 1))
      scales[row * (D / GROUP) + (lane * 8 + k * (D / 2)) / GROUP] = __halves2half2(scale[k], offset[k]);
  }
}

// D / 16 neighbouring lanes take a row of keys, values or queries, two chunks of 8
// channels each, D / 2 apart: every load and store is contiguous over the lanes,
// and the pairs (j, j + D/2) of a full rotation meet in one lane (those of a
// shorter one are read once more, from L1).  BY_TOKENS: a block takes as many tokens as it has such lane groups and
// four rows (heads) of each, so that a token's cosines and sines are read once,
// all four rows are in flight at a time, and a head's appended rows are written
// side by side.  Otherwise (few tokens) a block takes one token's rows.
// INSIDE: pairs (j, j + D/2) over all channels, which lie in one lane and share
// their cosines; four rows then fit 96 registers, five blocks an SM.
template <typename T, int D, int GROUP, bool BY_TOKENS, bool INSIDE>
__global__ __launch_bounds__(kThreads, BY_TOKENS ? (INSIDE ? 5 : 4) : 1) void append_kernel(const AppendParam p) {
  constexpr int kLanes = D / 16, kTeams = kThreads / kLanes;
  constexpr int kRows = BY_TOKENS ? 4 : 1;
  const int lane = threadIdx.x % kLanes, team = threadIdx.x / kLanes, first = lane * 8;
  const int parts = 2 * p.heads + p.query_heads;
  // Blocks of the same tokens follow one another, so that the rows read (and
  // the queries written) at a time lie together.
  const uint32_t chunks = (parts + (BY_TOKENS ? kRows : kTeams) - 1) / (BY_TOKENS ? kRows : kTeams);
  const uint32_t number = blockIdx.x / chunks, chunk = blockIdx.x - number * chunks;
  const int64_t wanted = BY_TOKENS ? static_cast<int64_t>(number) * kTeams + team : number;
  const int part0 = BY_TOKENS ? chunk * kRows : chunk * kTeams + team;
  const bool live = wanted < p.tokens;
  const int64_t token = live ? wanted : 0;
  const int half = p.rotary_dim >> 1;

  uint4 raw[kRows][2], pair[kRows][2];
  int64_t place[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int part = min(part0 + r, parts - 1);
    const bool is_value = part >= p.heads && part < 2 * p.heads;
    const T *from = part < p.heads ? static_cast<const T *>(p.keys) + token * p.key_token + part * p.key_head
                    : is_value ? static_cast<const T *>(p.values) + token * p.value_token + (part - p.heads) * p.value_head
                               : static_cast<const T *>(p.queries) + token * p.query_token +
                                     (part - 2 * p.heads) * p.query_head;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = first + k * (D / 2);
      raw[r][k] = *reinterpret_cast<const uint4 *>(from + c);
      if (!INSIDE && !is_value && !p.interleaved && c < p.rotary_dim)
        pair[r][k] = *reinterpret_cast<const uint4 *>(from + (c < half ? c + half : c - half));
    }
  }
  const int64_t position = p.positions[token];
  bool turned = p.rotary_dim > 0, lost = false;  // lost: a position outside the table
  if (turned && (position < 0 || position >= p.rotary_positions)) {
    turned = false;
    lost = true;
  }
  Turn turn;
  load_turn<D, INSIDE ? 1 : 2>(p, turned ? p.rotary + position * p.rotary_dim : nullptr, lane, turn);
  if (part0 < 2 * p.heads) {
    const int64_t sequence = find_sequence(p, token);
    const int64_t start = p.token_starts[sequence], count = p.token_starts[sequence + 1] - start;
    const bool known = live && token >= start && token - start < count;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int part = part0 + r;
      place[r] = -1;
      if (part >= 2 * p.heads) continue;
      const int64_t slot = sequence * p.heads + (part < p.heads ? part : part - p.heads);
      if (known)
        place[r] = pool_row(p.pages, p.table, p.table_stride, p.table_width, slot,
                            p.lengths[slot] - count + (token - start));
      if (place[r] < 0 && live && lane == 0) atomicOr(p.flag, kFlagRow);
      if (lost && part < p.heads) place[r] = -1;
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int part = part0 + r;
    if (BY_TOKENS && part >= parts) break;  // the same for the whole block
    const bool is_key = part < p.heads, is_value = !is_key && part < 2 * p.heads;
    float x[16];
    unpack8<T>(raw[r][0], x);
    unpack8<T>(raw[r][1], x + 8);
    if (!is_value) {
      if (lost && live && lane == 0 && part < parts) atomicOr(p.flag, kFlagPosition);
      if constexpr (INSIDE) {
        if (turned)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float a = x[i], b = x[8 + i], cosine = turn.cosine[i], sine = turn.sine[i];  // the first one's: -sin
            x[i] = __fadd_rn(__fmul_rn(a, cosine), __fmul_rn(b, sine));
            x[8 + i] = __fsub_rn(__fmul_rn(b, cosine), __fmul_rn(a, sine));
          }
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (!turn.turns[k]) continue;
          float other[8], *own = x + 8 * k;
          if (p.interleaved) {
#pragma unroll
            for (int i = 0; i < 8; ++i) other[i] = own[i ^ 1];
          } else {
            unpack8<T>(pair[r][k], other);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            own[i] = __fadd_rn(__fmul_rn(own[i], turn.cosine[8 * k + i]), __fmul_rn(other[i], turn.sine[8 * k + i]));
        }
      }
    }
    if (is_key || is_value) {
      const int64_t row = place[r];
      uint8_t *pool = is_key ? p.pages.keys : p.pages.values;
      if constexpr (GROUP == 0) {
        if (row >= 0) {
          T *to = reinterpret_cast<T *>(pool) + row * D + first;
          store8(to, x);
          store8(to + D / 2, x + 8);
        }
      } else if constexpr (BY_TOKENS) {
        store_codes<D, GROUP>(pool, is_key ? p.pages.key_scales : p.pages.value_scales, row, lane, x);
      }
      if (is_key && row >= 0 && lane == 0) p.pages.positions[row] = static_cast<float>(position);
    } else if (live && part < parts) {
      if (lost)  // nothing else says which queries were not rotated
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __int_as_float(0x7fffffff);
      T *to = static_cast<T *>(p.out_queries) + (token * p.query_heads + (part - 2 * p.heads)) * D + first;
      store8(to, x);
      store8(to + D / 2, x + 8);
    }
    if constexpr (GROUP != 0 && !BY_TOKENS) {
      // The warp's rows differ, and every lane takes part in the groups'
      // shuffles: rows of queries, and rows without a place, store nothing.
      store_codes<D, GROUP>(is_value ? p.pages.values : p.pages.keys,
                            is_value ? p.pages.value_scales : p.pages.key_scales,
                            part < 2 * p.heads ? place[r] : -1, lane, x);
    }
  }
}

struct ReadParam {
  Pages pages;
  const int32_t *table;
  int64_t table_stride, table_width;
  const int32_t *first_rows;
  const int32_t *row_starts;
  int64_t slots, rows;
  void *keys, *values;
  float *positions;
  uint32_t *flag;
};

constexpr int kReadRows = 2;

// D / 16 lanes per row, keys and values of the row together; a lane group takes
// two neighbouring rows, which mostly share their slot's lookup.  Rows without a
// place read as NaN.
template <typename T, int D, int GROUP, typename S>
__global__ __launch_bounds__(kThreads) void read_kernel(const ReadParam p) {
  constexpr int kLanes = D / 16, kTeams = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int64_t row0 = (static_cast<int64_t>(blockIdx.x) * kTeams + threadIdx.x / kLanes) * kReadRows;
  if (row0 >= p.rows) return;
  int64_t slot = 0;  // the last slot whose start is <= row0
  for (int64_t hi = p.slots; hi - slot > 1;) {
    const int64_t mid = (slot + hi) >> 1;
    if (p.row_starts[mid] <= row0) slot = mid; else hi = mid;
  }
  int64_t rows[kReadRows];
#pragma unroll
  for (int k = 0; k < kReadRows; ++k) {
    const int64_t out_row = row0 + k;
    rows[k] = -1;
    if (out_row >= p.rows) continue;
    while (slot + 1 < p.slots && out_row >= p.row_starts[slot + 1]) ++slot;
    const int64_t place = out_row - p.row_starts[slot];
    if (place >= 0 && out_row < p.row_starts[slot + 1])
      rows[k] = pool_row(p.pages, p.table, p.table_stride, p.table_width, slot, p.first_rows[slot] + place);
    if (rows[k] < 0 && lane == 0) atomicOr(p.flag, kFlagRow);
  }
  if constexpr (GROUP == 0) {
#pragma unroll
    for (int k = 0; k < kReadRows; ++k) {
      if (row0 + k >= p.rows) continue;
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const S *from = reinterpret_cast<const S *>(side ? p.pages.values : p.pages.keys) + rows[k] * D + lane * 8;
        T *to = static_cast<T *>(side ? p.values : p.keys) + (row0 + k) * D + lane * 8;
        float x[16];
        if (rows[k] >= 0) {
          load8(from, x);
          load8(from + D / 2, x + 8);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = __int_as_float(0x7fffffff);
        }
        store8(to, x);
        store8(to + D / 2, x + 8);
      }
    }
  } else {
    uint32_t words[kReadRows][2][2];
    __half2 pairs[kReadRows][2][2];
#pragma unroll
    for (int k = 0; k < kReadRows; ++k) {
#pragma unroll
      for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int chunk = 0; chunk < 2; ++chunk) {
          words[k][side][chunk] = 0;
          pairs[k][side][chunk] = __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff));
        }
      if (rows[k] < 0) continue;
#pragma unroll
      for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int chunk = 0; chunk < 2; ++chunk) {
          words[k][side][chunk] = *reinterpret_cast<const uint32_t *>((side ? p.pages.values : p.pages.keys) +
                                                                      rows[k] * (D / 2) + lane * 4 + chunk * (D / 4));
          pairs[k][side][chunk] = (side ? p.pages.value_scales : p.pages.key_scales)[rows[k] * (D / GROUP) +
                                                                                     (lane * 8 + chunk * (D / 2)) / GROUP];
        }
    }
#pragma unroll
    for (int k = 0; k < kReadRows; ++k) {
      if (row0 + k >= p.rows) continue;
#pragma unroll
      for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int chunk = 0; chunk < 2; ++chunk) {
          T *to = static_cast<T *>(side ? p.values : p.keys) + (row0 + k) * D + lane * 8 + chunk * (D / 2);
          const float scale = __low2float(pairs[k][side][chunk]), offset = __high2float(pairs[k][side][chunk]);
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            // 2^23 + code, less 2^23 + 8: the code without a conversion.
            const uint32_t code = (words[k][side][chunk] >> (4 * i)) & 15u;
            x[i] = fmaf(scale, __uint_as_float(0x4B000000u | code) - 8388616.0f, offset);
          }
          store8(to, x);
        }
    }
  }
#pragma unroll
  for (int k = 0; k < kReadRows; ++k)
    if (lane == 0 && row0 + k < p.rows)
      p.positions[row0 + k] = rows[k] >= 0 ? p.pages.positions[rows[k]] : __int_as_float(0x7fffffff);
}

template <typename T, int D, int GROUP>
void launch_append_rows(const AppendParam &p, cudaStream_t stream) {
  constexpr int kTeams = kThreads / (D / 16);
  const int64_t parts = 2 * p.heads + p.query_heads;
  if (p.tokens >= kManyTokens) {
    const int64_t grid = ceil_div(p.tokens, kTeams) * ceil_div(parts, 4);
    if (p.rotary_dim == D && !p.interleaved)
      append_kernel<T, D, GROUP, true, true><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p);
    else
      append_kernel<T, D, GROUP, true, false><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p);
  } else {
    const int64_t grid = p.tokens * ceil_div(parts, kTeams);
    if (p.rotary_dim == D && !p.interleaved)
      append_kernel<T, D, GROUP, false, true><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p);
    else
      append_kernel<T, D, GROUP, false, false><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p);
  }
}

template <typename T, int D>
void launch_append(const AppendParam &p, int group, cudaStream_t stream) {
  switch (group) {
    case 0: launch_append_rows<T, D, 0>(p, stream); break;
    case 32: launch_append_rows<T, D, 32>(p, stream); break;
    case 64: launch_append_rows<T, D, 64>(p, stream); break;
    default:
      if constexpr (D == 128) launch_append_rows<T, D, 128>(p, stream);
  }
}

template <typename T, int D>
void launch_read(const ReadParam &p, int group, int held, unsigned grid, cudaStream_t stream) {
  switch (group) {
    case 0:
      if (held == LRK_F16) read_kernel<T, D, 0, __half><<<grid, kThreads, 0, stream>>>(p);
      else read_kernel<T, D, 0, __nv_bfloat16><<<grid, kThreads, 0, stream>>>(p);
      break;
    case 32: read_kernel<T, D, 32, __half><<<grid, kThreads, 0, stream>>>(p); break;
    case 64: read_kernel<T, D, 64, __half><<<grid, kThreads, 0, stream>>>(p); break;
    default:
      if constexpr (D == 128) read_kernel<T, D, 128, __half><<<grid, kThreads, 0, stream>>>(p);
  }
}

bool rows_fit(const lrk_rows &r) { return aligned(r.data, 16) && r.token_stride % 8 == 0 && r.head_stride % 8 == 0; }

}  // namespace
}  // namespace lrk

extern "C" int lrk_paged_append(const lrk_pages *pages, const int32_t *table, int64_t table_stride,
                                int64_t table_width, const int32_t *lengths, int64_t sequences, int64_t heads,
                                const int32_t *token_starts, int64_t tokens, const lrk_rows *keys,
                                const lrk_rows *values, const int64_t *positions, const float *rotary,
                                int64_t rotary_positions, int64_t rotary_dim, int interleaved,
                                const lrk_rows *queries, int64_t query_heads, void *out_queries, int dtype,
                                unsigned int *flag, lrk_stream_t stream) {
  using namespace lrk;
  clear_error();
  if (int rc = paged::check_pages(pages)) return rc;
  LRK_REQUIRE(dtype == LRK_F16 || dtype == LRK_BF16, "paged append: rows must be f16 or bf16");
  LRK_REQUIRE(pages->group != 0 || dtype == pages->dtype, "paged append: new rows must have the pages' type");
  LRK_REQUIRE(sequences >= 0 && heads >= 1 && tokens >= 0 && table_width >= 0, "paged append: invalid sizes");
  LRK_REQUIRE(table_stride >= table_width, "paged append: table rows overlap");
  LRK_REQUIRE(query_heads >= 0 && heads < (1 << 20) && query_heads < (1 << 20), "paged append: invalid head counts");
  LRK_REQUIRE(rotary_dim >= 0 && rotary_dim <= pages->dimension && rotary_dim % 16 == 0,
              "paged append: rotary dimension must be a multiple of 16, at most the head dimension");
  if (tokens == 0) return LRK_OK;
  LRK_REQUIRE(sequences >= 1, "paged append: tokens without a sequence");
  LRK_REQUIRE((table != nullptr || table_width == 0) && lengths != nullptr && token_starts != nullptr && positions != nullptr &&
                  flag != nullptr && keys != nullptr && values != nullptr && keys->data != nullptr &&
                  values->data != nullptr,
              "paged append: null argument");
  LRK_REQUIRE(rotary_dim == 0 || (rotary != nullptr && rotary_positions >= 1), "paged append: no rotary table");
  LRK_REQUIRE(query_heads == 0 || (queries != nullptr && queries->data != nullptr && out_queries != nullptr),
              "paged append: null queries");
  LRK_REQUIRE(rows_fit(*keys) && rows_fit(*values) && (query_heads == 0 || rows_fit(*queries)) &&
                  aligned(out_queries, 16) && aligned(rotary, 16),
              "paged append: rows must be 16-byte aligned");
  AppendParam p{};
  p.pages = paged::device_pages(*pages);
  p.table = table;
  p.table_stride = table_stride;
  p.table_width = table_width;
  p.lengths = lengths;
  p.token_starts = token_starts;
  p.sequences = sequences;
  p.tokens = tokens;
  p.keys = keys->data;
  p.key_token = keys->token_stride;
  p.key_head = keys->head_stride;
  p.values = values->data;
  p.value_token = values->token_stride;
  p.value_head = values->head_stride;
  if (query_heads > 0) {
    p.queries = queries->data;
    p.query_token = queries->token_stride;
    p.query_head = queries->head_stride;
  }
  p.out_queries = out_queries;
  p.heads = static_cast<int>(heads);
  p.query_heads = static_cast<int>(query_heads);
  p.positions = positions;
  p.rotary = rotary;
  p.rotary_positions = rotary_positions;
  p.rotary_dim = static_cast<int>(rotary_dim);
  p.interleaved = interleaved != 0;
  p.flag = flag;
  LRK_REQUIRE(tokens * (2 * heads + query_heads) < (int64_t{1} << 31), "paged append: too many rows");
  const int group = static_cast<int>(pages->group);
  if (dtype == LRK_F16) {
    if (pages->dimension == 64) launch_append<__half, 64>(p, group, stream);
    else launch_append<__half, 128>(p, group, stream);
  } else {
    if (pages->dimension == 64) launch_append<__nv_bfloat16, 64>(p, group, stream);
    else launch_append<__nv_bfloat16, 128>(p, group, stream);
  }
  return launch_status("paged append");
}

extern "C" int lrk_paged_read(const lrk_pages *pages, const int32_t *table, int64_t table_stride, int64_t table_width,
                              const int32_t *first_rows, const int32_t *row_starts, int64_t slots, int64_t rows,
                              void *keys, void *values, float *positions, int dtype, unsigned int *flag,
                              lrk_stream_t stream) {
  using namespace lrk;
  clear_error();
  if (int rc = paged::check_pages(pages)) return rc;
  LRK_REQUIRE(dtype == LRK_F16 || dtype == LRK_BF16 || dtype == LRK_F32, "paged read: rows must be f16, bf16 or f32");
  LRK_REQUIRE(slots >= 0 && rows >= 0 && table_width >= 0 && table_stride >= table_width, "paged read: invalid sizes");
  if (rows == 0) return LRK_OK;
  LRK_REQUIRE(slots >= 1, "paged read: rows without a slot");
  LRK_REQUIRE((table != nullptr || table_width == 0) && first_rows != nullptr && row_starts != nullptr && keys != nullptr &&
                  values != nullptr && positions != nullptr && flag != nullptr,
              "paged read: null argument");
  LRK_REQUIRE(aligned(keys, 16) && aligned(values, 16), "paged read: output rows must be 16-byte aligned");
  ReadParam p{paged::device_pages(*pages), table, table_stride, table_width, first_rows, row_starts, slots, rows,
              keys, values, positions, flag};
  const int64_t grid = ceil_div(rows, kThreads / (pages->dimension / 16) * kReadRows);
  LRK_REQUIRE(grid < (int64_t{1} << 31), "paged read: too many rows");
  const int group = static_cast<int>(pages->group);
  const unsigned blocks = static_cast<unsigned>(grid);
  const bool small = pages->dimension == 64;
  switch (dtype) {
    case LRK_F16:
      if (small) launch_read<__half, 64>(p, group, pages->dtype, blocks, stream);
      else launch_read<__half, 128>(p, group, pages->dtype, blocks, stream);
      break;
    case LRK_BF16:
      if (small) launch_read<__nv_bfloat16, 64>(p, group, pages->dtype, blocks, stream);
      else launch_read<__nv_bfloat16, 128>(p, group, pages->dtype, blocks, stream);
      break;
    default:
      if (small) launch_read<float, 64>(p, group, pages->dtype, blocks, stream);
      else launch_read<float, 128>(p, group, pages->dtype, blocks, stream);
  }
  return launch_status("paged read");
}
