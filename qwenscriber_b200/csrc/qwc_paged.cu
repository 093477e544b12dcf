// qwc_paged.cu -- append and read of a paged q8 key/value cache.
//
// append does in one pass what stands between the QKV projection and
// attention (decoder.zig:177-216): per head
//   x' = x * (1 / sqrt(mean(x^2) + eps)) * w          queries and keys
//   (lo, hi) -> (lo cos - hi sin, hi cos + lo sin)    pairs (d, d + half)
// and for keys and values, per 64 of them, scale = f16(max |x| / 128) and
// code = round(x / scale) + 128 (quant.zig:197-288), into the row that the
// page table gives the token's position. read is the way back:
// (code - 128) * scale.
//
// Both move each byte once and are bound by HBM.

#include <cuda_runtime.h>

#include "qwc_device.cuh"
#include "qwc_paged.cuh"

namespace qwc {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct AppendArgs {
  const T* q;
  const T* k;
  const T* v;
  T* q_out;
  uint64_t q_stride, k_stride, v_stride, q_out_stride;
  const float* q_norm;
  const float* k_norm;
  const float* cos_table;
  const float* sin_table;
  uint32_t heads, rope_rows;
  float eps;
};

// A block takes one token: its heads + 2 kv_heads rows are dealt to groups
// of LANES lanes, each lane with 16 bytes of its row (4 or 8 values).
template <typename T, int DIM>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const PagedArgs a, const AppendArgs<T> p) {
  constexpr int V = Vec16<T>::kCount;
  constexpr int LANES = DIM / V;
  constexpr int GROUP_LANES = static_cast<int>(kGroup) / V;
  const PagedSeq seq = paged_seq(a, blockIdx.y);
  if (blockIdx.x >= seq.n) return;
  const uint32_t token = seq.first + blockIdx.x;
  const int32_t pos = seq.base + static_cast<int32_t>(blockIdx.x);
  int64_t row = -1;
  if (pos >= 0 && static_cast<uint32_t>(pos) < p.rope_rows) row = paged_row(a, blockIdx.y, static_cast<uint32_t>(pos));
  const uint32_t lane = threadIdx.x % LANES;
  const uint32_t d0 = lane * V;
  const uint32_t rows = p.heads + 2 * a.kv_heads;
  float cs[V], sn[V];
  const uint32_t pair0 = d0 % (DIM / 2);
  if (row >= 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      *reinterpret_cast<float4*>(cs + i) = *reinterpret_cast<const float4*>(p.cos_table + size_t(pos) * (DIM / 2) + pair0 + i);
      *reinterpret_cast<float4*>(sn + i) = *reinterpret_cast<const float4*>(p.sin_table + size_t(pos) * (DIM / 2) + pair0 + i);
    }
  }
  // Whole warps leave the loop together: the shuffles below are warp-wide.
  const uint32_t per_pass = kThreads / LANES;
  for (uint32_t r0 = 0; r0 < rows; r0 += per_pass) {
    const uint32_t r = r0 + threadIdx.x / LANES;
    const bool in = r < rows && (row >= 0 || r < p.heads);
    const bool is_q = r < p.heads, is_k = !is_q && r < p.heads + a.kv_heads;
    const uint32_t h = is_q ? r : is_k ? r - p.heads : r - p.heads - a.kv_heads;
    const T* src = (is_q ? p.q + size_t(token) * p.q_stride : is_k ? p.k + size_t(token) * p.k_stride
                                                                    : p.v + size_t(token) * p.v_stride) +
                   size_t(h) * DIM + d0;
    float x[V];
    unpack16(in ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0), x, T());
    const float* weight = is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (weight && in) {
      const float inv = rms_inverse(ss, DIM, p.eps);
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = x[i] * inv * weight[d0 + i];
    }
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, x[i], LANES / 2);
      y[i] = (is_q || is_k) && row >= 0 ? (d0 < DIM / 2 ? rope_rn(true, x[i], other, cs[i], sn[i])
                                                                  : rope_rn(false, other, x[i], cs[i], sn[i]))
                                        : x[i];
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) amax = fmaxf(amax, fabsf(y[i]));
#pragma unroll
    for (int o = GROUP_LANES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!in) continue;
    if (is_q) {
      if (row < 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = 0.0f;
      }
      *reinterpret_cast<uint4*>(p.q_out + size_t(token) * p.q_out_stride + size_t(h) * DIM + d0) = pack16<T>(y);
      continue;
    }
    const __half sh = __float2half_rn(amax / 128.0f);
    const float stored = __half2float(sh);
    uint8_t* codes = const_cast<uint8_t*>(is_k ? a.k_codes : a.v_codes) + size_t(row) * a.code_row + size_t(h) * DIM + d0;
    uint8_t* scales = const_cast<uint8_t*>(is_k ? a.k_scales : a.v_scales) + size_t(row) * a.scale_row;
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[i] |= uint32_t(q8_code(y[4 * i + e], stored)) << (8 * e);
    }
#pragma unroll
    for (int i = 0; i < V / 4; ++i) reinterpret_cast<uint32_t*>(codes)[i] = w[i];
    if (d0 % kGroup == 0) reinterpret_cast<__half*>(scales)[(size_t(h) * DIM + d0) / kGroup] = sh;
  }
}

// One thread per 16 codes of a row.
template <typename T>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(const PagedArgs a, T* k_out, uint64_t k_stride, T* v_out,
                                                              uint64_t v_stride) {
  constexpr int V = Vec16<T>::kCount;
  const PagedSeq seq = paged_seq(a, blockIdx.y);
  if (blockIdx.x >= seq.n) return;
  const uint32_t token = seq.first + blockIdx.x;
  const int32_t pos = seq.base + static_cast<int32_t>(blockIdx.x);
  const int64_t row = pos >= 0 ? paged_row(a, blockIdx.y, static_cast<uint32_t>(pos)) : -1;
  for (uint32_t c = threadIdx.x; c < 2 * a.code_row / V; c += kThreads) {
    const bool is_v = c >= a.code_row / V;
    const uint32_t d = (c - (is_v ? a.code_row / V : 0u)) * V;
    float x[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = 0.0f;
    if (row >= 0) {
      const uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + size_t(row) * a.code_row + d;
      const uint16_t* scales = reinterpret_cast<const uint16_t*>((is_v ? a.v_scales : a.k_scales) + size_t(row) * a.scale_row);
      const float s = f16_bits_to_f32(scales[d / kGroup]);
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = static_cast<float>(static_cast<int>(codes[i]) - 128) * s;
    }
    *reinterpret_cast<uint4*>((is_v ? v_out + size_t(token) * v_stride : k_out + size_t(token) * k_stride) + d) = pack16<T>(x);
  }
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace

int32_t paged_status(cudaError_t e) {
  if (e == cudaSuccess) return QWC_OK;
  if (e == cudaErrorMemoryAllocation) return QWC_OUT_OF_MEMORY;
  return QWC_INVALID_STATE;
}

int32_t paged_rows_check(const void* p, uint64_t stride, uint64_t width, uint32_t format) {
  if (!p || !aligned(p, 16) || stride * value_bytes(format) % 16 != 0) return QWC_INVALID_ARGUMENT;
  if (stride < width) return QWC_SHAPE_MISMATCH;
  if (stride > (uint64_t(1) << 31)) return QWC_LIMIT_EXCEEDED;
  return QWC_OK;
}

int32_t paged_args(const qwc_paged_cache* c, const qwc_paged_batch* b, PagedArgs* out) {
  if (!c || !b) return QWC_INVALID_ARGUMENT;
  if (!c->k_scales || !c->k_codes || !c->v_scales || !c->v_codes) return QWC_INVALID_ARGUMENT;
  if (!b->query_starts || !b->context_lens || !b->page_table) return QWC_INVALID_ARGUMENT;
  if (!aligned(c->k_scales, 16) || !aligned(c->k_codes, 16) || !aligned(c->v_scales, 16) || !aligned(c->v_codes, 16) ||
      !aligned(b->query_starts, 4) || !aligned(b->context_lens, 4) || !aligned(b->page_table, 4)) {
    return QWC_INVALID_ARGUMENT;
  }
  if (c->head_dim != 64 && c->head_dim != 128) return QWC_UNSUPPORTED;
  if (c->kv_heads == 0 || c->page_size == 0 || c->pages == 0) return QWC_SHAPE_MISMATCH;
  // Every position of a sequence has an entry in its row of the table.
  if (uint64_t(b->table_stride) * c->page_size < b->max_context) return QWC_SHAPE_MISMATCH;
  if (uint64_t(c->pages) * c->page_size > 0x7FFFFFFFu || b->max_context > 0x7FFFFFFFu || b->tokens > 0x7FFFFFFFu ||
      c->kv_heads > 1024 || b->sequences > kPagedMaxSequences) {
    return QWC_LIMIT_EXCEEDED;
  }
  PagedArgs a = {};
  a.k_scales = static_cast<const uint8_t*>(c->k_scales);
  a.k_codes = static_cast<const uint8_t*>(c->k_codes);
  a.v_scales = static_cast<const uint8_t*>(c->v_scales);
  a.v_codes = static_cast<const uint8_t*>(c->v_codes);
  a.query_starts = b->query_starts;
  a.context_lens = b->context_lens;
  a.page_table = b->page_table;
  a.pages = c->pages;
  a.page_size = c->page_size;
  a.by_page = divisor(c->page_size);
  a.kv_heads = c->kv_heads;
  a.head_dim = c->head_dim;
  a.code_row = c->kv_heads * c->head_dim;
  a.scale_row = a.code_row / kGroup * 2;
  a.sequences = b->sequences;
  a.tokens = b->tokens;
  a.table_stride = b->table_stride;
  a.max_query = b->max_query < b->tokens ? b->max_query : b->tokens;
  a.max_context = b->max_context;
  *out = a;
  return QWC_OK;
}

namespace {

template <typename T>
int32_t append_as(const PagedArgs& a, const void* q, uint64_t q_stride, const void* k, uint64_t k_stride, const void* v,
                  uint64_t v_stride, uint32_t heads, const float* q_norm, const float* k_norm, float eps,
                  const float* cos_table, const float* sin_table, uint32_t rope_rows, void* q_out,
                  uint64_t q_out_stride, cudaStream_t stream) {
  AppendArgs<T> p{static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), static_cast<T*>(q_out),
                  q_stride, k_stride, v_stride, q_out_stride, q_norm, k_norm, cos_table, sin_table, heads, rope_rows, eps};
  const dim3 grid(a.max_query, a.sequences);
  if (a.head_dim == 128) {
    paged_append_kernel<T, 128><<<grid, kThreads, 0, stream>>>(a, p);
  } else {
    paged_append_kernel<T, 64><<<grid, kThreads, 0, stream>>>(a, p);
  }
  return paged_status(cudaGetLastError());
}

}  // namespace
}  // namespace qwc

using namespace qwc;

extern "C" {

int32_t qwc_op_paged_append(const qwc_paged_cache* cache, const qwc_paged_batch* batch, uint32_t format, const void* q,
                            uint64_t q_stride, const void* k, uint64_t k_stride, const void* v, uint64_t v_stride,
                            uint32_t heads, const float* q_norm, const float* k_norm, float eps, const float* cos_table,
                            const float* sin_table, uint32_t rope_rows, void* q_out, uint64_t q_out_stride,
                            void* stream) {
  if (!value_format_ok(format)) return QWC_UNSUPPORTED;
  PagedArgs a;
  int32_t st = paged_args(cache, batch, &a);
  if (st != QWC_OK) return st;
  if (!cos_table || !sin_table || !aligned(cos_table, 16) || !aligned(sin_table, 16) || !aligned(q_norm, 16) ||
      !aligned(k_norm, 16)) {
    return QWC_INVALID_ARGUMENT;
  }
  if (heads == 0 || heads % a.kv_heads != 0) return QWC_SHAPE_MISMATCH;
  if (heads > 4096) return QWC_LIMIT_EXCEEDED;
  if (a.max_query == 0 || a.sequences == 0) return QWC_OK;
  const uint64_t qw = uint64_t(heads) * a.head_dim;
  if ((st = paged_rows_check(q, q_stride, qw, format)) != QWC_OK) return st;
  if ((st = paged_rows_check(k, k_stride, a.code_row, format)) != QWC_OK) return st;
  if ((st = paged_rows_check(v, v_stride, a.code_row, format)) != QWC_OK) return st;
  if ((st = paged_rows_check(q_out, q_out_stride, qw, format)) != QWC_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto run = format == kFormatF32 ? append_as<float> : format == kFormatF16 ? append_as<__half> : append_as<__nv_bfloat16>;
  return run(a, q, q_stride, k, k_stride, v, v_stride, heads, q_norm, k_norm, eps, cos_table, sin_table, rope_rows, q_out,
             q_out_stride, s);
}

int32_t qwc_op_paged_read(const qwc_paged_cache* cache, const qwc_paged_batch* batch, uint32_t format, void* k_out,
                          uint64_t k_stride, void* v_out, uint64_t v_stride, void* stream) {
  if (!value_format_ok(format)) return QWC_UNSUPPORTED;
  PagedArgs a;
  int32_t st = paged_args(cache, batch, &a);
  if (st != QWC_OK) return st;
  if (a.max_query == 0 || a.sequences == 0) return QWC_OK;
  if ((st = paged_rows_check(k_out, k_stride, a.code_row, format)) != QWC_OK) return st;
  if ((st = paged_rows_check(v_out, v_stride, a.code_row, format)) != QWC_OK) return st;
  const dim3 grid(a.max_query, a.sequences);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (format == kFormatF32) {
    paged_read_kernel<float><<<grid, kThreads, 0, s>>>(a, static_cast<float*>(k_out), k_stride, static_cast<float*>(v_out), v_stride);
  } else if (format == kFormatF16) {
    paged_read_kernel<__half><<<grid, kThreads, 0, s>>>(a, static_cast<__half*>(k_out), k_stride, static_cast<__half*>(v_out), v_stride);
  } else {
    paged_read_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a, static_cast<__nv_bfloat16*>(k_out), k_stride,
                                                               static_cast<__nv_bfloat16*>(v_out), v_stride);
  }
  return paged_status(cudaGetLastError());
}

}  // extern "C"
