// qwc_paged.cuh -- what the operators on a paged key/value cache share: the
// pool and the batch as a kernel takes them, and where a token's row lies.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/qwenscriber_cuda.h"
#include "qwc_internal.h"

namespace qwc {

// Division of a 32-bit number by one known at the launch, as a multiplication
// and two shifts (Granlund and Montgomery, 1994, figure 4.1, exact for all):
// with l = ceil(log2 d), mul is 2^32 (2^l - d) / d + 1, the shifts min(l, 1) and
// max(l - 1, 0).
struct Divisor {
  uint32_t mul, shift1, shift2;
#ifdef __CUDACC__
  __device__ __forceinline__ uint32_t of(uint32_t x) const {
    const uint32_t t = __umulhi(x, mul);
    return (t + ((x - t) >> shift1)) >> shift2;
  }
#endif
};
inline Divisor divisor(uint32_t d) {
  uint32_t l = 0;
  while ((uint64_t(1) << l) < d) ++l;
  return Divisor{static_cast<uint32_t>(((((uint64_t(1) << l) - d) << 32) / d) + 1), l > 0 ? 1u : 0u, l > 0 ? l - 1 : 0u};
}

// qwc_paged_cache and qwc_paged_batch as the kernels take them.
struct PagedArgs {
  const uint8_t* k_scales;
  const uint8_t* k_codes;
  const uint8_t* v_scales;
  const uint8_t* v_codes;
  const int32_t* query_starts;
  const int32_t* context_lens;
  const int32_t* page_table;
  uint32_t pages, page_size;
  Divisor by_page;
  uint32_t kv_heads, head_dim;
  uint32_t code_row;   // kv_heads * head_dim bytes
  uint32_t scale_row;  // code_row / 64 * 2 bytes
  uint32_t sequences, tokens, table_stride, max_query, max_context;
};

// A sequence's tokens in this step: packed rows first .. first + n - 1, which
// are positions base .. base + n - 1 of its context.
struct PagedSeq {
  uint32_t first, n;
  int32_t base;
  uint32_t context;
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, uint32_t s) {
  const int32_t limit = static_cast<int32_t>(a.tokens);
  const int32_t b = min(max(a.query_starts[s], 0), limit);
  const int32_t e = min(max(a.query_starts[s + 1], b), limit);
  const int32_t c = min(max(a.context_lens[s], 0), static_cast<int32_t>(a.max_context));
  return PagedSeq{static_cast<uint32_t>(b), min(static_cast<uint32_t>(e - b), a.max_query), c - (e - b),
                  static_cast<uint32_t>(c)};
}

__device__ __forceinline__ uint32_t page_of(const PagedArgs& a, uint32_t p) { return a.by_page.of(p); }

// Row of the pool that holds position p of sequence s, or -1 if its page
// is not one of the pool's.
__device__ __forceinline__ int64_t paged_row(const PagedArgs& a, uint32_t s, uint32_t p) {
  const uint32_t pg = page_of(a, p);
  const int32_t id = __ldg(a.page_table + size_t(s) * a.table_stride + pg);
  if (static_cast<uint32_t>(id) >= a.pages) return -1;
  return int64_t(id) * a.page_size + (p - pg * a.page_size);
}

// Rows of f32, f16 or bf16 values, 16 bytes at a time.
template <typename T>
struct Vec16 {
  static constexpr int kCount = 16 / sizeof(T);
};

__device__ __forceinline__ void unpack16(uint4 w, float (&v)[4]) {
  v[0] = __uint_as_float(w.x);
  v[1] = __uint_as_float(w.y);
  v[2] = __uint_as_float(w.z);
  v[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void unpack16(uint4 w, float (&v)[8], __half) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack16(uint4 w, float (&v)[8], __nv_bfloat16) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(u[i] << 16);
    v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack16(uint4 w, float (&v)[4], float) { unpack16(w, v); }

__device__ __forceinline__ uint32_t pair_bits(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pair_bits(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&v)[8]) {
  return make_uint4(pair_bits(v[0], v[1], T()), pair_bits(v[2], v[3], T()), pair_bits(v[4], v[5], T()),
                    pair_bits(v[6], v[7], T()));
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&v)[4]) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store_as(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_as(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_as(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// One attention call, as its kernels take it.
struct AttnArgs {
  uint64_t q_stride, out_stride;
  const void* q;
  void* out;
  float* partials;     // results of stretches that are not a whole segment, two for each CTA
  uint32_t* counters;  // [kMaxAttnCtas][kAttnCounterStride], zero between calls
  int32_t* error;      // set when a bounded wait gave up
  uint32_t wait_tries;  // its bound
  uint32_t heads, share;  // query heads, and those of a kv head
  Divisor by_share;
  uint32_t group;      // few rows: kv heads of a CTA
  uint32_t pb;         // few rows: position blocks of a step
  uint32_t rows;       // few rows: most rows of a kv head, max_query * share
  float scaling;
};

constexpr uint32_t kMaxAttnCtas = 1024;
constexpr uint32_t kAttnCounterStride = 8;  // a CTA's counters: one for each softmax warp
constexpr uint32_t kAttnCounters = kAttnCounterStride * kMaxAttnCtas;
constexpr uint64_t kAttnHeadBytes = 256 + kAttnCounters * 4;  // of the workspace: the error word, the counters
static_assert(kAttnHeadBytes == QWC_PAGED_WORKSPACE_HEAD);

// Many rows (qwc_paged_tile.cu): 128-row tiles that a CTA takes at once, its grid, its part of the workspace.
struct TilePlan {
  uint32_t tiles, grid;
  bool too_long;
  uint64_t partial_bytes;
};
TilePlan paged_tile_plan(const PagedArgs& a, uint32_t format, uint32_t heads, uint32_t sms);
int32_t paged_tile_launch(const PagedArgs& a, const AttnArgs& p, uint32_t format, const TilePlan& plan, cudaStream_t stream);

// ---- arithmetic of the attention kernels ----

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

template <uint32_t SEL>
__device__ __forceinline__ uint32_t codes_f16x2(uint32_t w) {
  const uint32_t h = __byte_perm(w, 0x64646464u, SEL);
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x64806480u));  // (1024 + u) - (1024 + 128)
  return r;
}

__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 f16x2_f32(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// A value scale that is no number (infinity, NaN) must not reach the rows that do not see its position: a weight of 0 times it
// is NaN. It enters the products as some number, and the rows that do see it are made NaN by themselves. With
// kOddStep added, a scale's exponent field is one more, that of one that is no number is 0, and its sign bit is set.
constexpr uint32_t kOddStep = 0x04000400u, kOddBits = 0x80008000u;

// The power of two that brings a row of queries near 1: their f16 parts then
// hold 11 (or 22) bits of every value that matters beside the largest.
__device__ __forceinline__ int row_exponent(float amax) {
  const int e = static_cast<int>((__float_as_uint(amax) >> 23) & 0xFFu) - 127;
  return min(max(e, -126), 126);
}

// Host side: the checks of the two descriptors, and the kernels' form of
// them. A refused descriptor is refused before any launch.
int32_t paged_args(const qwc_paged_cache* cache, const qwc_paged_batch* batch, PagedArgs* out);
// Rows of `width` values of `format`, `stride` elements apart: 16-byte pointer and stride, no overlap.
int32_t paged_rows_check(const void* p, uint64_t stride, uint64_t width, uint32_t format);
int32_t paged_status(cudaError_t e);

constexpr uint32_t kFormatF16 = 1;
constexpr uint32_t kFormatBF16 = 2;
constexpr uint32_t kPagedMaxSequences = 65535;  // a grid dimension counts them

inline uint32_t value_bytes(uint32_t format) { return format == kFormatF32 ? 4u : 2u; }
inline bool value_format_ok(uint32_t format) {
  return format == kFormatF32 || format == kFormatF16 || format == kFormatBF16;
}

}  // namespace qwc
