// Attention over the paged cache.
//
// Query i of a sequence's n new tokens sees rows r <= length - n + i of each
// of its slots (every row without `causal`):
//     o = sum_r p_r v_r,   p = softmax(scale q k_r),   lse = log sum_r exp(scale q k_r).
// One pass over the rows with a running maximum m and sum l: a new maximum m'
// multiplies l and the accumulated output by exp(m - m').
#include "paged.cuh"

namespace lrk {
namespace {

using namespace paged;

constexpr int kWarps = 4;

struct AttentionParam {
  Pages pages;
  const int32_t *table;
  int64_t table_stride, table_width;
  const int32_t *lengths;
  const int32_t *token_starts;
  int64_t sequences, tokens;
  const void *queries;
  int64_t query_token, query_head;
  int heads, groups;
  float scale_log2;
  bool causal;
  void *out;
  float *lse;
  uint32_t *flag;
};

template <typename T, int D, int GROUP>
__device__ __forceinline__ void load_row(const uint8_t *pool, const __half2 *scales, int64_t row, int lane, float *x) {
  constexpr int kEach = D / 32;
  if constexpr (GROUP == 0) {
    const T *from = reinterpret_cast<const T *>(pool) + row * D + lane * kEach;
#pragma unroll
    for (int i = 0; i < kEach; ++i) x[i] = to_float<T>(from[i]);
  } else {
    const __half2 pair = scales[row * (D / GROUP) + lane * kEach / GROUP];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const uint32_t code = (pool[row * (D / 2) + (lane * kEach + i) / 2] >> (4 * (i & 1))) & 15u;
      x[i] = fmaf(__low2float(pair), static_cast<float>(code) - 8.0f, __high2float(pair));
    }
  }
}

// One CTA per (token, query head): each warp takes every kWarps-th row, each
// lane D / 32 channels; the warps' states are joined in shared memory.
template <typename T, int D, int GROUP>
__global__ __launch_bounds__(kWarps * 32) void attention_kernel(const AttentionParam p) {
  constexpr int kEach = D / 32;
  __shared__ float s_out[kWarps][D];
  __shared__ float s_max[kWarps], s_sum[kWarps];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int query_heads = p.heads * p.groups;
  const int64_t token = blockIdx.x / query_heads;
  const int query_head = static_cast<int>(blockIdx.x % query_heads);
  int64_t lo = 0, hi = p.sequences;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (p.token_starts[mid] <= token) lo = mid; else hi = mid;
  }
  const int64_t first = p.token_starts[lo], count = p.token_starts[lo + 1] - first;
  const int64_t slot = lo * p.heads + query_head / p.groups;
  const int64_t length = p.lengths[slot];
  const int64_t visible = token < first || token - first >= count ? 0 : p.causal ? length - count + (token - first) + 1 : length;
  float q[kEach], o[kEach];
  const T *query = static_cast<const T *>(p.queries) + token * p.query_token + query_head * p.query_head + lane * kEach;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    q[i] = to_float<T>(query[i]);
    o[i] = 0.0f;
  }
  float top = -INFINITY, sum = 0.0f;
  for (int64_t r = warp; r < visible; r += kWarps) {
    const int64_t row = pool_row(p.pages, p.table, p.table_stride, p.table_width, slot, r);
    if (row < 0) {
      if (lane == 0) atomicOr(p.flag, kFlagRow);
      break;
    }
    float x[kEach], dot = 0.0f;
    load_row<T, D, GROUP>(p.pages.keys, p.pages.key_scales, row, lane, x);
#pragma unroll
    for (int i = 0; i < kEach; ++i) dot = fmaf(q[i], x[i], dot);
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, step);
    dot *= p.scale_log2;
    if (dot == -INFINITY) continue;
    const float next = dot > top ? dot : top;
    const float keep = exp2f(top - next), weight = exp2f(dot - next);
    top = next;
    sum = fmaf(sum, keep, weight);
    load_row<T, D, GROUP>(p.pages.values, p.pages.value_scales, row, lane, x);
#pragma unroll
    for (int i = 0; i < kEach; ++i) o[i] = fmaf(weight, x[i], o[i] * keep);
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) s_out[warp][lane * kEach + i] = o[i];
  if (lane == 0) {
    s_max[warp] = top;
    s_sum[warp] = sum;
  }
  __syncthreads();
  float whole = s_max[0];
  for (int w = 1; w < kWarps; ++w) whole = fmaxf(whole, s_max[w]);
  float total = 0.0f;
  float weights[kWarps];
  for (int w = 0; w < kWarps; ++w) {
    weights[w] = s_max[w] == -INFINITY ? 0.0f : exp2f(s_max[w] - whole);
    total = fmaf(weights[w], s_sum[w], total);
  }
  const int64_t index = token * query_heads + query_head;
  for (int c = threadIdx.x; c < D; c += kWarps * 32) {
    float value = 0.0f;
    for (int w = 0; w < kWarps; ++w) value = fmaf(weights[w], s_out[w][c], value);
    static_cast<T *>(p.out)[index * D + c] = from_float<T>(total == 0.0f ? 0.0f : value / total);
  }
  if (threadIdx.x == 0) p.lse[index] = total == 0.0f ? -INFINITY : (whole + log2f(total)) * 0.69314718f;
}

template <typename T, int D>
void launch_attention(const AttentionParam &p, int group, unsigned grid, cudaStream_t stream) {
  switch (group) {
    case 0: attention_kernel<T, D, 0><<<grid, kWarps * 32, 0, stream>>>(p); break;
    case 32: attention_kernel<T, D, 32><<<grid, kWarps * 32, 0, stream>>>(p); break;
    case 64: attention_kernel<T, D, 64><<<grid, kWarps * 32, 0, stream>>>(p); break;
    default:
      if constexpr (D == 128) attention_kernel<T, D, 128><<<grid, kWarps * 32, 0, stream>>>(p);
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
  LRK_REQUIRE((table != nullptr || table_width == 0) && lengths != nullptr && token_starts != nullptr && flag != nullptr &&
                  queries != nullptr && queries->data != nullptr && out != nullptr && lse != nullptr,
              "paged attention: null argument");
  LRK_REQUIRE(aligned(queries->data, 16) && queries->token_stride % 8 == 0 && queries->head_stride % 8 == 0 &&
                  aligned(out, 16),
              "paged attention: rows must be 16-byte aligned");
  if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < lrk_paged_attention_workspace_bytes())
    return fail(LRK_ERR_WORKSPACE, "paged attention: workspace too small");
  AttentionParam p{paged::device_pages(*pages), table, table_stride, table_width, lengths, token_starts, sequences,
                   tokens, queries->data, queries->token_stride, queries->head_stride, static_cast<int>(heads),
                   static_cast<int>(query_heads / heads), scale * 1.44269504f, causal != 0, out, lse, flag};
  const int64_t grid = tokens * query_heads;
  LRK_REQUIRE(grid < (int64_t{1} << 31), "paged attention: too many queries");
  const unsigned blocks = static_cast<unsigned>(grid);
  const int group = static_cast<int>(pages->group);
  if (dtype == LRK_F16) {
    if (pages->dimension == 64) launch_attention<__half, 64>(p, group, blocks, stream);
    else launch_attention<__half, 128>(p, group, blocks, stream);
  } else {
    if (pages->dimension == 64) launch_attention<__nv_bfloat16, 64>(p, group, blocks, stream);
    else launch_attention<__nv_bfloat16, 128>(p, group, blocks, stream);
  }
  return launch_status("paged attention");
}
