// qwc_sample.cu -- one token of each row of logits, from a given number.
//
// With x the row, m its maximum and T the temperature, w_i = exp((x_i - m) / T).
// The tokens kept are a prefix of the order (falling logit, rising index):
// top_k cuts it by count, top_p by the sum of w, min_p by w itself. So the
// kept set is one threshold logit t and a number of tokens that equal it:
// everything above t, and the first of those at t. The threshold comes from a
// radix selection on the logits' order-preserving bits; no sort. The token is
// the first in index order whose running sum of the kept w passes u times their
// total.
//
// Sums are of integers, w in units of 2^-42: they are exact, so neither the
// order of the atomics nor the split over threads changes a result.

#include <cuda_runtime.h>

#include "qwc_device.cuh"
#include "qwc_paged.cuh"

namespace qwc {
namespace {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kBins = 2048;
constexpr float kUnits = 4398046511104.0f;  // 2^42: 2^20 tokens of weight 1 stay below 2^63

struct SampleArgs {
  const void* logits;
  uint64_t row_stride;
  uint32_t vocab;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniforms;
  uint32_t* tokens;
  float* logprobs;
};

// A logit as the operator sees it: NaN is -inf, and -0 is 0 so that the two tie.
template <typename T>
__device__ __forceinline__ float logit(const T* row, uint32_t i) {
  const float x = to_f32(row[i]);
  return x != x ? -INFINITY : x + 0.0f;
}

// Bits in the order of the values.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float weight_of(float x, float best, float heat) {
  return x == best ? 1.0f : expf((x - best) / heat);
}

__device__ __forceinline__ uint64_t units_of(float w) { return __float2ull_rn(w * kUnits); }

__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ uint64_t warp_scan_u64(uint64_t v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31u) >= static_cast<uint32_t>(o)) v += u;
  }
  return v;
}

struct SampleSmem {
  uint64_t mass[kBins];
  uint32_t count[kBins];
  uint64_t sums[kSampleWarps];
  uint32_t keys[kSampleWarps];
  uint64_t above;
  uint32_t bin;
};

__device__ __forceinline__ uint64_t block_sum(SampleSmem* s, uint64_t v) {
  v = warp_sum_u64(v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s->sums[threadIdx.x / 32] = v;
  __syncthreads();
  uint64_t t = 0;
  for (int i = 0; i < kSampleWarps; ++i) t += s->sums[i];
  return t;
}

// The key where the prefix of (falling key) reaches `target`, counted in
// tokens (by_mass false) or in units of w, and what lies above that key.
template <typename T>
__device__ void select(SampleSmem* s, const T* row, uint32_t vocab, float best, float heat, bool by_mass, uint64_t target,
                       uint32_t* key, uint64_t* above_out) {
  uint32_t prefix = 0, mask = 0;
  uint64_t above = 0;
  const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
  for (int d = 0; d < 3; ++d) {
    const uint32_t bins = 1u << bits[d];
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kSampleThreads) {
      s->mass[i] = 0;
      s->count[i] = 0;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < vocab; i += kSampleThreads) {
      const float x = logit(row, i);
      const uint32_t k = order_key(x);
      if ((k & mask) != prefix) continue;
      const uint32_t b = (k >> shifts[d]) & (bins - 1);
      if (by_mass) {
        atomicAdd(reinterpret_cast<unsigned long long*>(&s->mass[b]),
                  static_cast<unsigned long long>(units_of(weight_of(x, best, heat))));
      } else {
        atomicAdd(&s->count[b], 1u);
      }
    }
    __syncthreads();
    // Bins from the top, two for each thread.
    const int b1 = static_cast<int>(bins) - 1 - 2 * static_cast<int>(threadIdx.x), b0 = b1 - 1;
    const uint64_t v1 = b1 >= 0 ? (by_mass ? s->mass[b1] : s->count[b1]) : 0;
    const uint64_t v0 = b0 >= 0 ? (by_mass ? s->mass[b0] : s->count[b0]) : 0;
    const uint64_t inc = warp_scan_u64(v0 + v1);
    if (threadIdx.x % 32 == 31) s->sums[threadIdx.x / 32] = inc;
    __syncthreads();
    uint64_t base = above;
    for (uint32_t w = 0; w < threadIdx.x / 32; ++w) base += s->sums[w];
    const uint64_t before1 = base + inc - v0 - v1, before0 = base + inc - v0;
    if (before1 < target && target <= before1 + v1) {
      s->bin = static_cast<uint32_t>(b1);
      s->above = before1;
    }
    if (before0 < target && target <= before0 + v0) {
      s->bin = static_cast<uint32_t>(b0);
      s->above = before0;
    }
    __syncthreads();
    prefix |= s->bin << shifts[d];
    mask |= (bins - 1) << shifts[d];
    above = s->above;
  }
  *key = prefix;
  *above_out = above;
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t sample_smem[];
  SampleSmem* s = reinterpret_cast<SampleSmem*>(sample_smem);
  const uint32_t r = blockIdx.x;
  const T* row = static_cast<const T*>(a.logits) + size_t(r) * a.row_stride;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const float heat_given = a.temperature ? a.temperature[r] : 1.0f;
  const bool greedy = !(heat_given > 0.0f);
  const float heat = greedy ? 1.0f : heat_given;
  const int32_t k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.0f;
  const float least = a.min_p ? fminf(a.min_p[r], 1.0f) : 0.0f;

  // The largest logit, and its first index.
  float best = -INFINITY;
  uint32_t at = 0xFFFFFFFFu;
  for (uint32_t i = threadIdx.x; i < a.vocab; i += kSampleThreads) {
    const float x = logit(row, i);
    if (x > best) {
      best = x;
      at = i;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ob = __shfl_xor_sync(0xffffffffu, best, o);
    const uint32_t oa = __shfl_xor_sync(0xffffffffu, at, o);
    if (ob > best || (ob == best && oa < at)) {
      best = ob;
      at = oa;
    }
  }
  if (lane == 0) {
    s->sums[warp] = at;
    s->keys[warp] = __float_as_uint(best);
  }
  __syncthreads();
  for (int w = 0; w < kSampleWarps; ++w) {
    const float ob = __uint_as_float(s->keys[w]);
    const uint32_t oa = static_cast<uint32_t>(s->sums[w]);
    if (ob > best || (ob == best && oa < at)) {
      best = ob;
      at = oa;
    }
  }
  if (best == -INFINITY) {
    if (threadIdx.x == 0) {
      a.tokens[r] = 0;
      if (a.logprobs) a.logprobs[r] = -INFINITY;
    }
    return;
  }
  uint64_t part = 0;
  for (uint32_t i = threadIdx.x; i < a.vocab; i += kSampleThreads) part += units_of(weight_of(logit(row, i), best, heat));
  const uint64_t all = block_sum(s, part);
  const float log_all = logf(static_cast<float>(all) / kUnits);
  if (greedy) {
    if (threadIdx.x == 0) {
      a.tokens[r] = at;
      if (a.logprobs) a.logprobs[r] = -log_all;
    }
    return;
  }

  // The kept set: keys above `cut`, and the first `ties` of those at it.
  uint32_t cut = 0, ties = 0xFFFFFFFFu;
  uint64_t mass = all;
  if (k > 0 && static_cast<uint32_t>(k) < a.vocab) {
    uint64_t above;
    select(s, row, a.vocab, best, heat, false, static_cast<uint64_t>(k), &cut, &above);
    ties = static_cast<uint32_t>(k - above);
    part = 0;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kSampleThreads) {
      const float x = logit(row, i);
      if (order_key(x) > cut) part += units_of(weight_of(x, best, heat));
    }
    mass = block_sum(s, part);
    const uint32_t bits = (cut & 0x80000000u) ? cut ^ 0x80000000u : ~cut;
    mass += ties * units_of(weight_of(__uint_as_float(bits), best, heat));
  }
  if (top_p < 1.0f) {
    const double want = ceil(static_cast<double>(fmaxf(top_p, 0.0f)) * static_cast<double>(mass));
    uint64_t target = static_cast<uint64_t>(want);
    if (target < 1) target = 1;
    if (target > mass) target = mass;
    uint64_t above;
    select(s, row, a.vocab, best, heat, true, target, &cut, &above);
    const uint32_t bits = (cut & 0x80000000u) ? cut ^ 0x80000000u : ~cut;
    const uint64_t each = units_of(weight_of(__uint_as_float(bits), best, heat));
    ties = each ? static_cast<uint32_t>((target - above + each - 1) / each) : 0xFFFFFFFFu;
  }

  // Each warp takes a run of the row. Tokens at the cut in its run, then the
  // mass that it keeps, then the walk of the one run that holds the token.
  const uint32_t run = (a.vocab + kSampleThreads - 1) / kSampleThreads * 32;
  const uint32_t i0 = min(warp * run, a.vocab), i1 = min(i0 + run, a.vocab);
  uint32_t tie_base = 0;
  if (ties != 0xFFFFFFFFu) {
    uint32_t n = 0;
    for (uint32_t i = i0 + lane; i < i1; i += 32) n += order_key(logit(row, i)) == cut ? 1u : 0u;
    const uint64_t sum = warp_sum_u64(n);
    __syncthreads();
    if (lane == 0) s->sums[warp] = sum;
    __syncthreads();
    for (uint32_t w = 0; w < warp; ++w) tie_base += static_cast<uint32_t>(s->sums[w]);
    __syncthreads();
  }
  auto kept_units = [&](uint32_t i, uint32_t& tie_at) -> uint64_t {
    const bool in = i < i1;
    const float x = in ? logit(row, i) : -INFINITY;
    const uint32_t key = order_key(x);
    const bool tie = in && key == cut;
    const uint32_t votes = __ballot_sync(0xffffffffu, tie);
    const uint32_t rank = tie_at + __popc(votes & ((1u << lane) - 1u));
    tie_at += __popc(votes);
    const float w = weight_of(x, best, heat);
    const bool keep = in && w >= least && (key > cut || (tie && rank < ties));
    return keep ? units_of(w) : 0;
  };
  part = 0;
  uint32_t tie_at = tie_base;
  for (uint32_t i = i0; i < i1; i += 32) part += kept_units(i + lane, tie_at);
  part = warp_sum_u64(part);
  __syncthreads();
  if (lane == 0) s->sums[warp] = part;
  __syncthreads();
  uint64_t total = 0, before = 0;
  for (uint32_t w = 0; w < kSampleWarps; ++w) {
    if (w == warp) before = total;
    total += s->sums[w];
  }
  const float u = fminf(fmaxf(a.uniforms[r], 0.0f), 1.0f);
  uint64_t goal = static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(total));
  if (goal >= total) goal = total - 1;
  if (before <= goal && goal < before + part) {
    uint64_t sum = before;
    tie_at = tie_base;
    for (uint32_t i = i0; i < i1; i += 32) {
      const uint64_t v = kept_units(i + lane, tie_at);
      const uint64_t inc = sum + warp_scan_u64(v);
      const uint32_t past = __ballot_sync(0xffffffffu, inc > goal);
      if (past) {
        if (lane == static_cast<uint32_t>(__ffs(past)) - 1) {
          const float x = logit(row, i + lane);
          a.tokens[r] = i + lane;
          if (a.logprobs) a.logprobs[r] = (x == best ? 0.0f : (x - best) / heat) - log_all;
        }
        break;
      }
      sum = __shfl_sync(0xffffffffu, inc, 31);
    }
  }
}

template <typename T>
int32_t sample_as(const SampleArgs& a, uint32_t rows, cudaStream_t stream) {
  sample_kernel<T><<<rows, kSampleThreads, sizeof(SampleSmem), stream>>>(a);
  return paged_status(cudaGetLastError());
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace qwc

using namespace qwc;

extern "C" {

int32_t qwc_op_sample(uint32_t format, const void* logits, uint64_t row_stride, uint32_t rows, uint32_t vocab,
                      const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                      const float* uniforms, uint32_t* tokens_out, float* logprobs_out, void* stream) {
  if (!value_format_ok(format)) return QWC_UNSUPPORTED;
  if (rows == 0) return QWC_OK;
  if (!logits || !uniforms || !tokens_out || vocab == 0) return QWC_INVALID_ARGUMENT;
  if (!aligned(logits, value_bytes(format)) || !aligned(temperature, 4) || !aligned(top_k, 4) || !aligned(top_p, 4) ||
      !aligned(min_p, 4) || !aligned(uniforms, 4) || !aligned(tokens_out, 4) || !aligned(logprobs_out, 4)) {
    return QWC_INVALID_ARGUMENT;
  }
  if (rows > 1 && row_stride < vocab) return QWC_SHAPE_MISMATCH;
  if (vocab > QWC_SAMPLE_MAX_VOCAB || rows > 0x7FFFFFFFu || row_stride > (uint64_t(1) << 31)) return QWC_LIMIT_EXCEEDED;
  const SampleArgs a{logits, row_stride, vocab, temperature, top_k, top_p, min_p, uniforms, tokens_out, logprobs_out};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return format == kFormatF32 ? sample_as<float>(a, rows, s)
         : format == kFormatF16 ? sample_as<__half>(a, rows, s)
                                : sample_as<__nv_bfloat16>(a, rows, s);
}

}  // extern "C"
