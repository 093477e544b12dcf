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

// 1 / sqrt(v): the hardware's estimate and one step of Newton's iteration, where that is of numbers (not of a sum that
// overflowed, whose root's inverse is 0, nor of 0): 0 < r < 1e30 in one comparison of bits (69 us for 70.4 with two of
// values, 64 x 391 tokens).
__device__ __forceinline__ float inverse_root(float v) {
  const float r = rsqrtf(v);
  return __float_as_uint(r) - 1u < 0x7149F2C9u ? r * fmaf(-0.5f * v * r, r, 1.5f) : r;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Two integers as signed bytes, saturated, in the low half of a word above `low`'s.
__device__ __forceinline__ uint32_t pack_s8(int hi, int lo, uint32_t low) {
  uint32_t r;
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(hi), "r"(lo), "r"(low));
  return r;
}

// V values (in pairs) as q8 codes of one scale, four to a word: q8_code (quant.zig:280-288) by way of the
// scale's reciprocal. The product is within 2^-22 of the rounded quotient's size, so both round alike unless it
// lies that close to a half (or is no number): a lane with such a value divides.
template <int V>
__device__ __forceinline__ void q8_codes(const uint64_t (&y)[V / 2], float stored, uint32_t (&w)[V / 4]) {
  const float inverse = stored > 0x1p-100f ? 1.0f / stored : __int_as_float(0x7FC00000);  // 0: q8_code decides
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: a sum's low bits are the nearest integer
  const uint64_t inv2 = pack2(inverse, inverse), up2 = pack2(kRound, kRound), down2 = pack2(-kRound, -kRound);
  float off = 0.0f;
  uint64_t number = 0;
  int c[V];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const uint64_t q = mul2(y[i], inv2);
    const uint64_t t = add2(q, up2);
    const uint64_t r = add2(t, down2);
    const float2 n = unpack2(r), f = unpack2(q), bits = unpack2(t);
    off = fmaxf(off, fmaxf(fabsf(f.x - n.x), fabsf(f.y - n.y)));
    number = fma2(q, 0ull, number);
    c[2 * i] = __float_as_int(bits.x) - 0x4B400000;
    c[2 * i + 1] = __float_as_int(bits.y) - 0x4B400000;
  }
  const float2 nf = unpack2(number);
  if (!(off + nf.x + nf.y <= 0.4999f)) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 f = unpack2(y[i]);
      c[2 * i] = static_cast<int>(q8_code(f.x, stored)) - 128;
      c[2 * i + 1] = static_cast<int>(q8_code(f.y, stored)) - 128;
    }
  }
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    w[i] = pack_s8(c[4 * i + 1], c[4 * i], pack_s8(c[4 * i + 3], c[4 * i + 2], 0u)) ^ 0x80808080u;
  }
}

// A block takes kAppendTokens tokens. Their heads + 2 kv_heads rows are dealt to groups of LANES lanes, each lane with
// 16 bytes of a row (4 or 8 values); a group takes the same head of every token, so the loads of all of them are
// in flight at once and what depends on the head alone is worked out once.
//
// 64 x 391 tokens at most, 14,281 in all (bf16, 16 + 2 x 8 heads of 128): 69 us, 3.0 TB/s (f16 67, f32 90). 235 warp
// instructions for 256 values, about a third of them the quantizer's, the others norms, rotation and maxima, take 70% of the
// issue slots; the rest is latency: 115 us with a division for each value, 79 with 78 registers and three
// blocks to an SM instead of 48 and five, 71 with two tokens to a block.
constexpr uint32_t kAppendTokens = 4;

// What a token that is not cached reads of the rotation (and does not use) where the tables have no row.
__device__ __align__(16) const float kNoRotation[64] = {};

template <typename T, int DIM>
__global__ void __launch_bounds__(kThreads, 5) paged_append_kernel(const PagedArgs a, const AppendArgs<T> p) {
  constexpr int V = Vec16<T>::kCount;
  constexpr int LANES = DIM / V;
  constexpr int GROUP_LANES = static_cast<int>(kGroup) / V;
  constexpr uint32_t AT_ONCE = kThreads / LANES;  // rows of a block's pass
  __shared__ int64_t row_s[kAppendTokens];
  const PagedSeq seq = paged_seq(a, blockIdx.y);
  const uint32_t i0 = blockIdx.x * kAppendTokens;
  if (i0 >= seq.n) return;
  const uint32_t tokens = min(kAppendTokens, seq.n - i0);
  if (threadIdx.x < kAppendTokens) {
    const int32_t pos = seq.base + static_cast<int32_t>(i0 + threadIdx.x);
    const bool cached = threadIdx.x < tokens && pos >= 0 && static_cast<uint32_t>(pos) < p.rope_rows;
    row_s[threadIdx.x] = cached ? paged_row(a, blockIdx.y, static_cast<uint32_t>(pos)) : -1;
  }
  const uint32_t d0 = threadIdx.x % LANES * V;
  const bool high = d0 >= DIM / 2;
  const uint32_t rows = p.heads + 2 * a.kv_heads;
  const size_t first = seq.first + i0;
  bool synced = false;
  for (uint32_t r0 = 0; r0 < rows; r0 += AT_ONCE) {  // (whole warps stay together: the shuffles are warp-wide)
    const uint32_t r = r0 + threadIdx.x / LANES;
    const bool in = r < rows;
    const bool is_q = r < p.heads, is_k = !is_q && r < p.heads + a.kv_heads, turns = is_q || is_k;
    const uint32_t head = is_q ? r : is_k ? r - p.heads : r - p.heads - a.kv_heads;
    const uint64_t stride = is_q ? p.q_stride : is_k ? p.k_stride : p.v_stride;
    const T* src = (is_q ? p.q : is_k ? p.k : p.v) + first * stride + size_t(head) * DIM + d0;
    uint4 raw[kAppendTokens];
#pragma unroll
    for (uint32_t tk = 0; tk < kAppendTokens; ++tk) {
      // (Plain loads: q_out may be q.)
      raw[tk] = in && tk < tokens ? *reinterpret_cast<const uint4*>(src + tk * stride) : make_uint4(0, 0, 0, 0);
    }
    const float* weight = is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
    uint64_t w2[V / 2];
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 w = weight ? __ldg(reinterpret_cast<const float4*>(weight + d0 + i)) : make_float4(1, 1, 1, 1);
      w2[i / 2] = pack2(w.x, w.y);
      w2[i / 2 + 1] = pack2(w.z, w.w);
    }
    const bool any_turns = __any_sync(0xffffffffu, in && turns), any_kv = __any_sync(0xffffffffu, in && !is_q);
    if (!synced) __syncthreads();
    synced = true;
#pragma unroll
    for (uint32_t tk = 0; tk < kAppendTokens; ++tk) {
      if (tk >= tokens) break;
      const int64_t row = row_s[tk];
      float f[V];
      unpack16(raw[tk], f, T());
      uint64_t x[V / 2];
#pragma unroll
      for (int i = 0; i < V / 2; ++i) x[i] = pack2(f[2 * i], f[2 * i + 1]);
      if (any_turns) {
        uint64_t ss2 = 0;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) ss2 = fma2(x[i], x[i], ss2);
        const float2 sf = unpack2(ss2);
        float ss = sf.x + sf.y;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = weight ? inverse_root(ss * (1.0f / DIM) + p.eps) : 1.0f;
        const uint64_t inv2 = pack2(inv, inv);
        const size_t at = size_t(row < 0 ? 0 : seq.base + static_cast<int32_t>(i0 + tk)) * (DIM / 2) + d0 % (DIM / 2);
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          const float4 cs = __ldg(reinterpret_cast<const float4*>(p.cos_table + at + i));
          float4 sn = __ldg(reinterpret_cast<const float4*>(p.sin_table + at + i));
          if (!high) sn = make_float4(-sn.x, -sn.y, -sn.z, -sn.w);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // (lo, hi) -> (lo cos - hi sin, hi cos + lo sin), the second product rounded first
            const uint64_t y = weight ? mul2(mul2(x[i / 2 + e], inv2), w2[i / 2 + e]) : x[i / 2 + e];
            const float2 yf = unpack2(y);
            const uint64_t other = pack2(__shfl_xor_sync(0xffffffffu, yf.x, LANES / 2), __shfl_xor_sync(0xffffffffu, yf.y, LANES / 2));
            const uint64_t c2 = e ? pack2(cs.z, cs.w) : pack2(cs.x, cs.y), s2 = e ? pack2(sn.z, sn.w) : pack2(sn.x, sn.y);
            const uint64_t z = fma2(y, c2, mul2(other, s2));
            if (turns) x[i / 2 + e] = z;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 v = unpack2(x[i]);
        f[2 * i] = v.x, f[2 * i + 1] = v.y;
      }
      if (in && is_q) {
        *reinterpret_cast<uint4*>(p.q_out + (first + tk) * p.q_out_stride + size_t(head) * DIM + d0) =
            row < 0 ? make_uint4(0, 0, 0, 0) : pack16<T>(f);
      }
      if (any_kv) {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i += 2) amax = fmaxf(amax, fmaxf(fabsf(f[i]), fabsf(f[i + 1])));
#pragma unroll
        for (int o = GROUP_LANES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (in && !is_q && row >= 0) {
          const __half sh = __float2half_rn(amax * (1.0f / 128.0f));
          uint8_t* codes = const_cast<uint8_t*>(is_k ? a.k_codes : a.v_codes) + size_t(row) * a.code_row + size_t(head) * DIM + d0;
          uint8_t* scales = const_cast<uint8_t*>(is_k ? a.k_scales : a.v_scales) + size_t(row) * a.scale_row;
          uint32_t w[V / 4];
          q8_codes<V>(x, __half2float(sh), w);
          if constexpr (V == 8) {
            *reinterpret_cast<uint2*>(codes) = make_uint2(w[0], w[1]);
          } else {
            *reinterpret_cast<uint32_t*>(codes) = w[0];
          }
          if (d0 % kGroup == 0) reinterpret_cast<__half*>(scales)[(size_t(head) * DIM + d0) / kGroup] = sh;
        }
      }
    }
  }
}

// A block takes `block_rows` tokens; each lane writes 16 bytes of values at a time, from V codes. The loads of a
// thread are independent: four of them are in flight. Bound by HBM: 64 x 2850 tokens at most, 109,000 in all (bf16),
// 127 us, 5.3 TB/s. Eight tokens to a block: four 134 us, two 167; sixteen 126, but a single sequence then has too
// few blocks (391 tokens, f32: one token to a block 3 us, two 3.4, four 4.3, eight 6.7).
constexpr uint32_t kReadRows = 8;

template <typename T>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(const PagedArgs a, uint32_t block_rows, T* k_out,
                                                              uint64_t k_stride, T* v_out, uint64_t v_stride) {
  constexpr int V = Vec16<T>::kCount;
  __shared__ int64_t row_s[kReadRows];
  const PagedSeq seq = paged_seq(a, blockIdx.y);
  const uint32_t i0 = blockIdx.x * block_rows;
  if (i0 >= seq.n) return;
  const uint32_t rows = min(block_rows, seq.n - i0);
  if (threadIdx.x < rows) {
    const int32_t pos = seq.base + static_cast<int32_t>(i0 + threadIdx.x);
    row_s[threadIdx.x] = pos >= 0 ? paged_row(a, blockIdx.y, static_cast<uint32_t>(pos)) : -1;
  }
  __syncthreads();
  const uint32_t chunks = a.code_row / V;  // of a key or value row
  const uint32_t total = rows * 2 * chunks;
  constexpr uint32_t UNROLL = 4;
  for (uint32_t c0 = threadIdx.x; c0 < total; c0 += UNROLL * kThreads) {
    uint2 code[UNROLL];
    uint16_t scale[UNROLL];
#pragma unroll
    for (uint32_t u = 0; u < UNROLL; ++u) {
      const uint32_t c = c0 + u * kThreads;
      code[u] = make_uint2(0x80808080u, 0x80808080u);
      scale[u] = 0;
      if (c < total) {
        const uint32_t r = c / (2 * chunks), rest = c - r * 2 * chunks;
        const bool is_v = rest >= chunks;
        const uint32_t d = (rest - (is_v ? chunks : 0u)) * V;
        const int64_t row = row_s[r];
        if (row >= 0) {
          const uint8_t* from = (is_v ? a.v_codes : a.k_codes) + size_t(row) * a.code_row + d;
          if constexpr (V == 8) {
            code[u] = *reinterpret_cast<const uint2*>(from);
          } else {
            code[u].x = *reinterpret_cast<const uint32_t*>(from);
          }
          scale[u] = reinterpret_cast<const uint16_t*>((is_v ? a.v_scales : a.k_scales) + size_t(row) * a.scale_row)[d / kGroup];
        }
      }
    }
#pragma unroll
    for (uint32_t u = 0; u < UNROLL; ++u) {
      const uint32_t c = c0 + u * kThreads;
      if (c >= total) break;
      const uint32_t r = c / (2 * chunks), rest = c - r * 2 * chunks;
      const bool is_v = rest >= chunks;
      const uint32_t d = (rest - (is_v ? chunks : 0u)) * V;
      const float s = f16_bits_to_f32(scale[u]);
      float x[V];
      const uint32_t w[2] = {code[u].x, code[u].y};
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // 2^23 + code is exact in f32, so is the difference.
        x[e] = (bits_f32(__byte_perm(w[e / 4], kMagic, 0x7440 + e % 4)) + kNegQ8) * s;
      }
      const size_t token = seq.first + i0 + r;
      *reinterpret_cast<uint4*>((is_v ? v_out + token * v_stride : k_out + token * k_stride) + d) = pack16<T>(x);
    }
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
  if (b->sequences && (!b->query_starts || !b->context_lens || !b->page_table)) return QWC_INVALID_ARGUMENT;
  if (!aligned(c->k_scales, 16) || !aligned(c->k_codes, 16) || !aligned(c->v_scales, 16) || !aligned(c->v_codes, 16) ||
      !aligned(b->query_starts, 4) || !aligned(b->context_lens, 4) || !aligned(b->page_table, 4)) {
    return QWC_INVALID_ARGUMENT;
  }
  if (c->head_dim != 64 && c->head_dim != 128) return QWC_UNSUPPORTED;
  if (c->kv_heads == 0 || c->page_size == 0 || c->pages == 0) return QWC_SHAPE_MISMATCH;
  // Every position of a sequence has an entry in its row of the table, whatever lies between two rows.
  const uint32_t entries = b->table_entries ? b->table_entries : b->table_stride;
  if (b->sequences && uint64_t(entries) * c->page_size < b->max_context) return QWC_SHAPE_MISMATCH;
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
  const dim3 grid((a.max_query + kAppendTokens - 1) / kAppendTokens, a.sequences);
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
  if (rope_rows == 0) {
    void* none = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&none, kNoRotation);
    if (e != cudaSuccess) return paged_status(e);
    cos_table = sin_table = static_cast<const float*>(none);
  }
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
  const uint32_t rows = a.tokens >= 4 * 148 * kReadRows ? kReadRows : 1;
  const dim3 grid((a.max_query + rows - 1) / rows, a.sequences);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (format == kFormatF32) {
    paged_read_kernel<float><<<grid, kThreads, 0, s>>>(a, rows, static_cast<float*>(k_out), k_stride, static_cast<float*>(v_out), v_stride);
  } else if (format == kFormatF16) {
    paged_read_kernel<__half><<<grid, kThreads, 0, s>>>(a, rows, static_cast<__half*>(k_out), k_stride, static_cast<__half*>(v_out), v_stride);
  } else {
    paged_read_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a, rows, static_cast<__nv_bfloat16*>(k_out), k_stride,
                                                               static_cast<__nv_bfloat16*>(v_out), v_stride);
  }
  return paged_status(cudaGetLastError());
}

}  // extern "C"
