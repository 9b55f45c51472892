// What the paged cache's kernels share: the pages as kernel parameters, row
// lookup, and the 4-bit row format.
//
// A page holds page_size rows of one slot (one KV head of one sequence).  Row
// r of a slot lies in page table[slot][r / page_size], place r % page_size.
// 16-bit rows are [pages, page_size, D] of f16 or bf16.  4-bit rows are codes
// [pages, page_size, D / 2] (channel 2j in the low half of byte j) with f16
// (scale, offset) pairs [pages, page_size, D / group, 2]; a channel's value is
// offset + scale * (code - 8).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace lrk {
namespace paged {

// Bits of the device flag of the paged operators.
constexpr uint32_t kFlagRow = 1;       // a length, row or page id outside the table or the pages
constexpr uint32_t kFlagPosition = 2;  // a position outside the rotary table
constexpr uint32_t kFlagTimeout = 4;   // a bounded wait of a kernel ran out
constexpr uint32_t kFlagShared = 8;    // a kernel's shared memory was not aligned to 1 KB: nothing computed

struct Pages {
  uint8_t *keys;
  uint8_t *values;
  __half2 *key_scales;
  __half2 *value_scales;
  float *positions;
  int32_t pages;
  int32_t page_shift;  // log2(page_size)
  int32_t page_size;
};

inline Pages device_pages(const lrk_pages &p) {
  Pages out{};
  out.keys = static_cast<uint8_t *>(p.keys);
  out.values = static_cast<uint8_t *>(p.values);
  out.key_scales = static_cast<__half2 *>(p.key_scales);
  out.value_scales = static_cast<__half2 *>(p.value_scales);
  out.positions = p.positions;
  out.pages = static_cast<int32_t>(p.pages);
  out.page_size = static_cast<int32_t>(p.page_size);
  while ((1 << out.page_shift) < out.page_size) ++out.page_shift;
  return out;
}

// Checks shared by every entry point of the paged cache.
inline int check_pages(const lrk_pages *p) {
  LRK_REQUIRE(p != nullptr, "paged: no pages");
  LRK_REQUIRE(p->pages >= 0 && p->pages < (int64_t{1} << 31), "paged: page count out of range");
  LRK_REQUIRE(p->page_size == 16 || p->page_size == 32 || p->page_size == 64 || p->page_size == 128,
              "paged: page size must be 16, 32, 64 or 128");
  if (p->dimension != 64 && p->dimension != 128)
    return fail(LRK_ERR_UNSUPPORTED, "paged: head dimension must be 64 or 128");
  LRK_REQUIRE(p->group == 0 || ((p->group == 32 || p->group == 64 || p->group == 128) && p->group <= p->dimension),
              "paged: group must be 0 (16-bit rows), 32, 64 or 128, at most the head dimension");
  LRK_REQUIRE(p->group != 0 || p->dtype == LRK_F16 || p->dtype == LRK_BF16, "paged: 16-bit rows must be f16 or bf16");
  LRK_REQUIRE(p->pages == 0 || (p->keys != nullptr && p->values != nullptr && p->positions != nullptr),
              "paged: null page memory");
  LRK_REQUIRE(p->pages == 0 || p->group == 0 || (p->key_scales != nullptr && p->value_scales != nullptr),
              "paged: null scales");
  LRK_REQUIRE(aligned(p->keys, 16) && aligned(p->values, 16) && aligned(p->key_scales, 16) &&
                  aligned(p->value_scales, 16),
              "paged: page memory must be 16-byte aligned");
  return LRK_OK;
}

// The pool row (page * page_size + place) of a slot's row, or -1 when the
// table gives it no page.
__device__ __forceinline__ int64_t pool_row(const Pages &p, const int32_t *table, int64_t table_stride,
                                            int64_t table_width, int64_t slot, int64_t row) {
  if (row < 0) return -1;
  const int64_t column = row >> p.page_shift;
  if (column >= table_width) return -1;
  const int32_t page = table[slot * table_stride + column];
  if (page < 0 || page >= p.pages) return -1;
  return static_cast<int64_t>(page) * p.page_size + (row & (p.page_size - 1));
}

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_float(float x) { return x; }

template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ float from_float(float x) { return x; }

// Eight consecutive 16-bit elements from / to 16-byte aligned memory.
template <typename T>
__device__ __forceinline__ void load8(const T *from, float *x) {
  const uint4 raw = *reinterpret_cast<const uint4 *>(from);
  const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_float<T>(e[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T *to, const float *x) {
  uint4 raw;
  T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_float<T>(x[i]);
  *reinterpret_cast<uint4 *>(to) = raw;
}
template <>
__device__ __forceinline__ void store8(float *to, const float *x) {
  reinterpret_cast<float4 *>(to)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4 *>(to)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// Minimum and maximum that keep a NaN (fminf and fmaxf drop it).
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

}  // namespace paged
}  // namespace lrk
