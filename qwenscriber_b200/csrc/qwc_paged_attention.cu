// qwc_paged_attention.cu -- causal attention of a step's tokens over a paged
// q8 key/value cache.

#include <cuda_runtime.h>

#include "qwc_device.cuh"
#include "qwc_paged.cuh"

namespace qwc {
namespace {

constexpr int kWarps = 4;

// One warp for each (token, query head): lane l holds DIM / 32 values of the
// query and of the output and walks the positions with a running maximum and
// sum.
template <typename T, int DIM>
__global__ void __launch_bounds__(32 * kWarps) paged_attention_kernel(const PagedArgs a, const T* q, uint64_t q_stride,
                                                                      uint32_t heads, T* out, uint64_t out_stride,
                                                                      float scaling) {
  constexpr int V = DIM / 32;
  const PagedSeq seq = paged_seq(a, blockIdx.y);
  const uint32_t unit = blockIdx.x * kWarps + threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t i = unit / heads, h = unit % heads;
  if (i >= seq.n) return;
  const uint32_t token = seq.first + i;
  const uint32_t kvh = h / (heads / a.kv_heads);
  const int32_t last = seq.base + static_cast<int32_t>(i);
  float x[V], o[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    x[e] = to_f32(q[size_t(token) * q_stride + size_t(h) * DIM + lane * V + e]);
    o[e] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  const uint32_t d = kvh * DIM + lane * V;
  for (int32_t p = 0; p <= last; ++p) {
    const int64_t row = paged_row(a, blockIdx.y, static_cast<uint32_t>(p));
    if (row < 0) continue;
    const uint8_t* kc = a.k_codes + size_t(row) * a.code_row + d;
    const uint8_t* vc = a.v_codes + size_t(row) * a.code_row + d;
    const float ks = f16_bits_to_f32(reinterpret_cast<const uint16_t*>(a.k_scales + size_t(row) * a.scale_row)[d / kGroup]);
    const float vs = f16_bits_to_f32(reinterpret_cast<const uint16_t*>(a.v_scales + size_t(row) * a.scale_row)[d / kGroup]);
    float t = 0.0f;
#pragma unroll
    for (int e = 0; e < V; ++e) t = fmaf(x[e], static_cast<float>(static_cast<int>(kc[e]) - 128) * ks, t);
    const float s = warp_sum(t) * scaling;
    const float nm = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.0f : expf(m - nm), w = s == -INFINITY ? 0.0f : expf(s - nm);
    l = l * keep + w;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = o[e] * keep + w * (static_cast<float>(static_cast<int>(vc[e]) - 128) * vs);
    m = nm;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    store_as(&out[size_t(token) * out_stride + size_t(h) * DIM + lane * V + e], last < 0 || l == 0.0f ? 0.0f : o[e] / l);
  }
}

template <typename T>
int32_t attention_as(const PagedArgs& a, const void* q, uint64_t q_stride, uint32_t heads, void* out, uint64_t out_stride,
                     cudaStream_t stream) {
  const float scaling = 1.0f / sqrtf(static_cast<float>(a.head_dim));
  const dim3 grid(static_cast<uint32_t>((uint64_t(a.max_query) * heads + kWarps - 1) / kWarps), a.sequences);
  auto kernel = a.head_dim == 128 ? paged_attention_kernel<T, 128> : paged_attention_kernel<T, 64>;
  kernel<<<grid, 32 * kWarps, 0, stream>>>(a, static_cast<const T*>(q), q_stride, heads, static_cast<T*>(out), out_stride,
                                           scaling);
  return paged_status(cudaGetLastError());
}

}  // namespace
}  // namespace qwc

using namespace qwc;

extern "C" {

int32_t qwc_op_paged_attention_workspace(const qwc_paged_cache* cache, const qwc_paged_batch* batch, uint32_t format,
                                         uint32_t heads, uint64_t* bytes) {
  if (!bytes) return QWC_INVALID_ARGUMENT;
  if (!value_format_ok(format)) return QWC_UNSUPPORTED;
  PagedArgs a;
  const int32_t st = paged_args(cache, batch, &a);
  if (st != QWC_OK) return st;
  if (heads == 0 || heads % a.kv_heads != 0) return QWC_SHAPE_MISMATCH;
  *bytes = 16;
  return QWC_OK;
}

int32_t qwc_op_paged_attention(const qwc_paged_cache* cache, const qwc_paged_batch* batch, uint32_t format,
                               const void* q, uint64_t q_stride, uint32_t heads, void* out, uint64_t out_stride,
                               void* workspace, uint64_t workspace_bytes, void* stream) {
  if (!value_format_ok(format)) return QWC_UNSUPPORTED;
  PagedArgs a;
  int32_t st = paged_args(cache, batch, &a);
  if (st != QWC_OK) return st;
  if (heads == 0 || heads % a.kv_heads != 0) return QWC_SHAPE_MISMATCH;
  if (heads > 4096) return QWC_LIMIT_EXCEEDED;
  if (a.max_query == 0 || a.sequences == 0) return QWC_OK;
  const uint64_t qw = uint64_t(heads) * a.head_dim;
  if ((st = paged_rows_check(q, q_stride, qw, format)) != QWC_OK) return st;
  if ((st = paged_rows_check(out, out_stride, qw, format)) != QWC_OK) return st;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return QWC_INVALID_ARGUMENT;
  uint64_t need = 0;
  qwc_op_paged_attention_workspace(cache, batch, format, heads, &need);
  if (workspace_bytes < need) return QWC_LIMIT_EXCEEDED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto run = format == kFormatF32 ? attention_as<float> : format == kFormatF16 ? attention_as<__half> : attention_as<__nv_bfloat16>;
  return run(a, q, q_stride, heads, out, out_stride, s);
}

}  // extern "C"
