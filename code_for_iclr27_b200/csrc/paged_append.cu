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
#include "paged.cuh"

namespace lrk {
namespace {

using namespace paged;

constexpr int kThreads = 128;

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

// x[0..15]: the rotated channels [first, first + 16) of a row.
template <typename T>
__device__ __forceinline__ void rotate16(const AppendParam &p, const T *row, const float *turn, int first, float *x) {
  const int half = p.rotary_dim >> 1;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int c = first + 8 * part;
    float *y = x + 8 * part;
    if (turn == nullptr || c >= p.rotary_dim) continue;
    if (p.interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float cosine = turn[(c >> 1) + i], sine = turn[half + (c >> 1) + i];
        const float a = y[2 * i], b = y[2 * i + 1];
        y[2 * i] = __fsub_rn(__fmul_rn(a, cosine), __fmul_rn(b, sine));
        y[2 * i + 1] = __fadd_rn(__fmul_rn(b, cosine), __fmul_rn(a, sine));
      }
      continue;
    }
    const bool low = c < half;
    const int at = low ? c : c - half;
    float other[8];
    load8(row + (low ? c + half : at), other);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float own = __fmul_rn(y[i], turn[at + i]), cross = __fmul_rn(other[i], turn[half + at + i]);
      y[i] = low ? __fsub_rn(own, cross) : __fadd_rn(own, cross);
    }
  }
}

// Quantises 16 channels per lane; the group / 16 lanes of a group are
// neighbours.  Stores the lane's 8 bytes of codes and, once per group, the
// scale and offset.
template <int D, int GROUP>
__device__ __forceinline__ void store_codes(uint8_t *codes, __half2 *scales, int64_t row, int lane, const float *x) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int step = 1; step < GROUP / 16; step <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, step));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, step));
  }
  __half scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  const float step = __half2float(scale);
  __half offset = __float2half_rn(__fadd_rn(lo, 8.0f * step));
  const bool fine = !__hisinf(scale) && !__hisnan(scale) && !__hisinf(offset) && !__hisnan(offset);
  const float inverse = step > 0.0f ? __frcp_rn(step) : 0.0f;
  const float centre = __half2float(offset);
  uint32_t word[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float level = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[i], centre), inverse)) + 8.0f, 0.0f), 15.0f);
    word[i >> 3] |= static_cast<uint32_t>(level) << (4 * (i & 7));
  }
  if (!fine) {
    word[0] = word[1] = 0;
    scale = offset = __ushort_as_half(0x7fff);
  }
  if (row < 0) return;
  *reinterpret_cast<uint2 *>(codes + row * (D / 2) + lane * 8) = make_uint2(word[0], word[1]);
  if (lane % (GROUP / 16) == 0) scales[row * (D / GROUP) + lane / (GROUP / 16)] = __halves2half2(scale, offset);
}

// D / 16 neighbouring lanes per (token, row of keys, values or queries), 16
// channels each; rows of a token are consecutive work items, so a warp reads
// consecutive rows of the projection's output.
template <typename T, int D, int GROUP>
__global__ __launch_bounds__(kThreads) void append_kernel(const AppendParam p) {
  constexpr int kLanes = D / 16;
  const int lane = threadIdx.x % kLanes;
  const int rows_per_token = 2 * p.heads + p.query_heads;
  const int64_t items = p.tokens * rows_per_token;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kLanes;
  const bool live = item < items;
  const int64_t token = live ? item / rows_per_token : 0;
  const int part = live ? static_cast<int>(item % rows_per_token) : 0;
  const bool is_key = part < p.heads, is_value = !is_key && part < 2 * p.heads;
  const int64_t position = p.positions[token];
  const float *turn = nullptr;
  bool skip = !live;
  if (p.rotary_dim > 0 && !is_value) {
    if (position >= 0 && position < p.rotary_positions) turn = p.rotary + position * p.rotary_dim;
    else skip = true;
    if (skip && live && lane == 0) atomicOr(p.flag, kFlagPosition);
  }
  const T *from;
  int64_t row = -1;
  if (is_key || is_value) {
    const int head = is_key ? part : part - p.heads;
    from = is_key ? static_cast<const T *>(p.keys) + token * p.key_token + head * p.key_head
                  : static_cast<const T *>(p.values) + token * p.value_token + head * p.value_head;
    const int64_t sequence = find_sequence(p, token);
    const int64_t first = p.token_starts[sequence], count = p.token_starts[sequence + 1] - first;
    const int64_t slot = sequence * p.heads + head;
    if (token >= first && token - first < count)
      row = pool_row(p.pages, p.table, p.table_stride, p.table_width, slot, p.lengths[slot] - count + (token - first));
    if (row < 0 && live && lane == 0) atomicOr(p.flag, kFlagRow);
  } else {
    from = static_cast<const T *>(p.queries) + token * p.query_token + (part - 2 * p.heads) * p.query_head;
  }
  float x[16];
  load8(from + lane * 16, x);
  load8(from + lane * 16 + 8, x + 8);
  if (!is_value) rotate16<T>(p, from, turn, lane * 16, x);
  if (is_key || is_value) {
    if (skip) row = -1;
    uint8_t *pool = is_key ? p.pages.keys : p.pages.values;
    if constexpr (GROUP == 0) {
      if (row >= 0) {
        T *to = reinterpret_cast<T *>(pool) + row * D + lane * 16;
        store8(to, x);
        store8(to + 8, x + 8);
      }
    }
    if (is_key && row >= 0 && lane == 0) p.pages.positions[row] = static_cast<float>(position);
  } else if (!skip) {
    T *to = static_cast<T *>(p.out_queries) + (token * p.query_heads + (part - 2 * p.heads)) * D + lane * 16;
    store8(to, x);
    store8(to + 8, x + 8);
  }
  if constexpr (GROUP != 0) {
    // Every lane of the warp takes part in the group's shuffles; rows of
    // queries, and rows without a place, store nothing.
    const bool key_row = is_key || !is_value;
    store_codes<D, GROUP>(key_row ? p.pages.keys : p.pages.values, key_row ? p.pages.key_scales : p.pages.value_scales,
                          is_key || is_value ? row : -1, lane, x);
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

// D / 16 lanes per row, keys and values of the row together.
template <typename T, int D, int GROUP, typename S>
__global__ __launch_bounds__(kThreads) void read_kernel(const ReadParam p) {
  constexpr int kLanes = D / 16;
  const int lane = threadIdx.x % kLanes;
  const int64_t out_row = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kLanes;
  if (out_row >= p.rows) return;
  int64_t lo = 0, hi = p.slots;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (p.row_starts[mid] <= out_row) lo = mid; else hi = mid;
  }
  const int64_t place = out_row - p.row_starts[lo];
  const int64_t row = place >= 0 && out_row < p.row_starts[lo + 1]
                          ? pool_row(p.pages, p.table, p.table_stride, p.table_width, lo, p.first_rows[lo] + place)
                          : -1;
  if (row < 0) {
    if (lane == 0) atomicOr(p.flag, kFlagRow);
    return;
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const uint8_t *pool = side ? p.pages.values : p.pages.keys;
    T *to = static_cast<T *>(side ? p.values : p.keys) + out_row * D + lane * 16;
    float x[16];
    if constexpr (GROUP == 0) {
      const S *from = reinterpret_cast<const S *>(pool) + row * D + lane * 16;
      load8(from, x);
      load8(from + 8, x + 8);
    } else {
      const uint2 word = *reinterpret_cast<const uint2 *>(pool + row * (D / 2) + lane * 8);
      const __half2 pair =
          (side ? p.pages.value_scales : p.pages.key_scales)[row * (D / GROUP) + lane / (GROUP / 16)];
      const float scale = __low2float(pair), offset = __high2float(pair);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t code = ((i < 8 ? word.x : word.y) >> (4 * (i & 7))) & 15u;
        x[i] = fmaf(scale, static_cast<float>(code) - 8.0f, offset);
      }
    }
    store8(to, x);
    store8(to + 8, x + 8);
  }
  if (lane == 0) p.positions[out_row] = p.pages.positions[row];
}

template <typename T, int D>
void launch_append(const AppendParam &p, int group, unsigned grid, cudaStream_t stream) {
  switch (group) {
    case 0: append_kernel<T, D, 0><<<grid, kThreads, 0, stream>>>(p); break;
    case 32: append_kernel<T, D, 32><<<grid, kThreads, 0, stream>>>(p); break;
    case 64: append_kernel<T, D, 64><<<grid, kThreads, 0, stream>>>(p); break;
    default:
      if constexpr (D == 128) append_kernel<T, D, 128><<<grid, kThreads, 0, stream>>>(p);
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
  const int64_t rows = kThreads / (pages->dimension / 16);
  const int64_t grid = ceil_div(tokens * (2 * heads + query_heads), rows);
  LRK_REQUIRE(grid < (int64_t{1} << 31), "paged append: too many rows");
  const int group = static_cast<int>(pages->group);
  const unsigned blocks = static_cast<unsigned>(grid);
  if (dtype == LRK_F16) {
    if (pages->dimension == 64) launch_append<__half, 64>(p, group, blocks, stream);
    else launch_append<__half, 128>(p, group, blocks, stream);
  } else {
    if (pages->dimension == 64) launch_append<__nv_bfloat16, 64>(p, group, blocks, stream);
    else launch_append<__nv_bfloat16, 128>(p, group, blocks, stream);
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
  const int64_t grid = ceil_div(rows, kThreads / (pages->dimension / 16));
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
