// qwc_sample.cu -- one token of each row of logits, from a given number.
//
// With x the row, m its maximum and T the temperature, w_i = exp((x_i - m) / T).
// The tokens kept are a prefix of the order (falling logit, rising index):
// top_k cuts it by count, top_p by the sum of w, min_p by w itself. So the
// kept set is one threshold logit and a number of tokens that equal it:
// everything above, and the first of those at it. No sort: the threshold is
// found by narrowing. A histogram of (m - x) / T in steps of 1/23 of a power of two says how far down the kept set can
// reach. Where that is 1024 tokens or fewer, as a rule, they go to the first CTA of the row, which compares them pair by
// pair or narrows by the logits' order-preserving bits (count or mass against its target) and then by the index
// (mass against u times the total) among them alone. top_p alone over more: the counts bound the mass above each bin
// from both sides, and only the few bins that can hold the cut go there. What is left (top_k above 1024, heaps of ties)
// is narrowed by all CTAs together. The token is the first in index order whose running sum passes.
//
// Bound by the chain of passes over the row's slices in shared memory (load and maximum 5.4 us, sums and histogram 6,
// list 4, cut and token 2, of 64 x 151936) and the exchanges between them, not by HBM: 1 x 151936, f32, 16 us; 64 x 151936,
// f32, 49 to 67 us, two waves of rows; 16 x 32003, bf16, 18 to 28 us. Of 24 inputs each, three had a row with a large kept
// set that takes longer: 25 to 27, 95 to 115 and 38 to 44 us.
//
// Sums are of integers, w in units of 2^-42: they are exact, so neither the
// order of the atomics nor the split over threads changes a result.
//
// A cluster of CTAs takes a row, each CTA a slice that it reads once and keeps in
// shared memory; histograms and totals meet in the first CTA's.

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "qwc_device.cuh"
#include "qwc_paged.cuh"

namespace qwc {
namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 1024;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr uint32_t kBins = kSampleThreads;  // a scan takes one bin for each thread
constexpr uint32_t kBinBits = 10;
constexpr uint32_t kListed = kSampleThreads;  // tokens that the first CTA takes by itself, one for each thread
// Up to this many of them are compared pair by pair, each token by as many lanes as there are: two passes over the
// list, where narrowing takes a histogram and more for each cut. 1 x 151936 16.5 us, by narrowing 23; 64 x 151936 55 and 59;
// 16 x 32003 17.7 and 19.5. (With 1024 in place of 256: 64 x 151936 148 us, 16 x 32003 61.)
constexpr uint32_t kPairs = 256;
constexpr uint32_t kLimbBits = 14;          // 2^17 tokens of a slice times 2^14 stay below 2^32
constexpr float kBinScale = 23.0f;      // coarse bins in a power of two; the last bin takes all below 2^-44, whose units are 0
constexpr int kUnitBits = 42;               // a weight of 1 in units: 2^20 tokens of it stay below 2^63
constexpr float kUnits = 4398046511104.0f;  // 2^42

struct SampleArgs {
  const void* logits;
  uint64_t row_stride;
  uint32_t vocab;
  uint32_t run;   // values of a warp, a multiple of 32
  uint32_t held;  // values of a slice that fit shared memory; the others are read again from global memory
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniforms;
  uint32_t* tokens;
  float* logprobs;
};

// A logit as the operator sees it: NaN is -inf, and -0 is 0 so that the two tie.
__device__ __forceinline__ float logit(float x) { return x != x ? -INFINITY : x + 0.0f; }

// Bits in the order of the values, without those that a value of type T leaves the same.
template <typename T>
__device__ __forceinline__ uint32_t order_key(float x) {
  constexpr int kIdle = std::is_same<T, float>::value ? 0 : std::is_same<T, __half>::value ? 13 : 16;
  const uint32_t b = __float_as_uint(x);
  return ((b & 0x80000000u) ? ~b : b | 0x80000000u) >> kIdle;
}
template <typename T>
__device__ __forceinline__ float key_value(uint32_t key) {
  constexpr int kIdle = std::is_same<T, float>::value ? 0 : std::is_same<T, __half>::value ? 13 : 16;
  const uint32_t k = key << kIdle;
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~(k | ((1u << kIdle) - 1u)));
}

// How far a logit lies below the best, at the row's temperature and in powers of two: t = (best - x) log2(e) / T,
// so w = 2^-t. One rounding of t: a relative 2^-24 t of w, below 2e-6 for every w that counts. best - x is 0 for two
// infinities; a temperature below 1e-37 counts as that, one above 3e38 as that (0 times -inf is no weight).
struct Fall {
  float best, scale;
  __device__ __forceinline__ float of(float x) const { return fmaxf(best - x, 0.0f) * scale; }
};
__device__ __forceinline__ float weight_of(float t) { return ex2(-t); }
// (Moving the mantissa to its place by 64-bit shifts instead: 1 x 151936 17.0 us, this 15.9.)
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

struct Histogram {
  uint64_t mass[kBins];
  uint32_t count[kBins];
};

// Where a prefix of the order ends: at the tokens whose key is `key`, with `count` tokens and `mass` above
// them and `here` tokens (of mass `here_mass`) at it.
struct Cut {
  uint64_t mass, here_mass;
  uint32_t count, here;
  uint32_t bin;
};

struct SampleSmem {
  // The first CTA's are the row's.
  uint32_t coarse_count[kBins];
  union {
    uint64_t coarse_mass[kBins];
    struct {
      uint64_t units[kListed];
      uint32_t key[kListed];
      uint32_t index[kListed];  // the top bit: less than min_p
    } list;
  };
  union {
    uint32_t limb[3][kBins];  // the slice's masses by bin, in limbs: 32-bit additions are native, 64-bit ones are not
    Histogram fine;
  };
  uint32_t listed;
  uint32_t reach, reached;  // the last coarse bin that the kept set can touch, and the tokens down to it
  uint64_t sums[kSampleWarps];
  uint64_t scan[kSampleWarps];
  uint32_t scan_count[kSampleWarps];
  uint64_t total;      // the row's (first CTA) sum of all units
  uint64_t mass_above; // the row's (first CTA) sum of the units above the bins in question; the units before the holder
  uint64_t slice_sum;  // this slice's sum of kept units
  uint32_t slice_ties;
  uint32_t holder;  // the run that holds the token
  uint32_t few, few_key[32];  // a bin's tokens
  uint64_t few_units[32];
  float best;
  uint32_t best_at;
  Cut cut;
  Cut answer;  // the first CTA's to the others
  float values[];
};

__device__ __forceinline__ void clear(Histogram& h) {
  h.mass[threadIdx.x] = 0;
  h.count[threadIdx.x] = 0;
}

__device__ __forceinline__ void add_to(uint32_t* counts, uint64_t* masses, uint32_t bin, uint32_t count, uint64_t mass) {
  atomicAdd(&counts[bin], count);
  if (mass) atomicAdd(reinterpret_cast<unsigned long long*>(&masses[bin]), static_cast<unsigned long long>(mass));
}

// Sums over the bins above (bins 0 .. threadIdx.x - 1) of a value for each thread of a CTA.
template <typename V>
__device__ V sum_above(SampleSmem* s, V v) {
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  V inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= static_cast<uint32_t>(o)) inc += u;
  }
  if (lane == 31) s->scan[warp] = inc;
  __syncthreads();
  V before = lane < warp ? static_cast<V>(s->scan[lane]) : V(0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  return before + inc - v;
}

// The bin (bin 0 on top) where what lies above it, added to `from`, reaches the target: `target` tokens, or
// units if by_mass. All threads of a CTA, each with the n tokens and the mass m of its bin; the answer is in
// s->cut after the next barrier.
__device__ void find_bin(SampleSmem* s, uint32_t n, uint64_t m, bool by_mass, uint64_t target, uint32_t from_count, uint64_t from_mass) {
  const uint64_t above_mass = from_mass + sum_above(s, m);
  __syncthreads();
  const uint32_t above_count = from_count + sum_above(s, n);
  const uint64_t above = by_mass ? above_mass : above_count, here = by_mass ? m : n;
  if (above < target && target <= above + here) s->cut = Cut{above_mass, m, above_count, n, threadIdx.x};
}

// Narrowing within one CTA: of the tokens that take part, one to a thread, with keys lo .. hi, the key at which
// the falling order reaches the target, in s->cut.bin, and what lies above and at it. False if it is not reached.
// Ten bits at a time, until a warp can compare the tokens of a bin with one another. (One copy of its code: a row's
// first call finds it in the instruction cache.)
__device__ __noinline__ bool narrow(SampleSmem* s, bool part, uint32_t key, uint64_t units, uint32_t lo, uint32_t hi, bool by_mass,
                                    uint64_t target, uint32_t from_count, uint64_t from_mass) {
  const uint32_t lane = threadIdx.x % 32;
  for (;;) {
    clear(s->fine);
    __syncthreads();
    if (threadIdx.x == 0) {
      s->cut.bin = 0xFFFFFFFFu;
      s->few = 0;
    }
    const uint32_t bits = 32 - __clz((hi - lo) | 1u);
    const uint32_t shift = bits > kBinBits ? bits - kBinBits : 0u;
    const bool mine = part && key >= lo && key <= hi;
    const uint32_t bin = (hi - key) >> shift;
    if (mine) add_to(s->fine.count, s->fine.mass, bin, 1, units);
    __syncthreads();
    find_bin(s, s->fine.count[threadIdx.x], s->fine.mass[threadIdx.x], by_mass, target, from_count, from_mass);
    __syncthreads();
    const Cut cut = s->cut;
    if (cut.bin == 0xFFFFFFFFu) return false;
    from_count = cut.count;
    from_mass = cut.mass;
    hi -= cut.bin << shift;
    if (shift == 0) break;
    if (cut.here <= 32) {
      if (mine && bin == cut.bin) {
        const uint32_t at = atomicAdd(&s->few, 1u);
        s->few_key[at] = key;
        s->few_units[at] = units;
      }
      __syncthreads();
      if (threadIdx.x < 32) {
        const bool in = lane < cut.here;
        const uint32_t k = in ? s->few_key[lane] : 0u;
        const uint64_t u = in ? s->few_units[lane] : 0;
        uint32_t above = 0, here = 0;
        uint64_t above_mass = 0, here_mass = 0;
        for (uint32_t j = 0; j < cut.here; ++j) {
          const uint32_t kj = __shfl_sync(0xffffffffu, k, j);
          const uint64_t uj = __shfl_sync(0xffffffffu, u, j);
          above += kj > k ? 1u : 0u;
          above_mass += kj > k ? uj : 0;
          here += kj == k ? 1u : 0u;
          here_mass += kj == k ? uj : 0;
        }
        above += cut.count;
        above_mass += cut.mass;
        const uint64_t before = by_mass ? above_mass : above, at_it = by_mass ? here_mass : here;
        if (in && before < target && target <= before + at_it) s->cut = Cut{above_mass, here_mass, above, here, k};
      }
      __syncthreads();
      return true;
    }
    lo = hi - min(hi - lo, (1u << shift) - 1u);
  }
  __syncthreads();
  if (threadIdx.x == 0) s->cut.bin = hi;
  __syncthreads();
  return true;
}

template <typename T, bool HELD>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t sample_smem[];
  SampleSmem* s = reinterpret_cast<SampleSmem*>(sample_smem);
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t size = cluster.num_blocks(), rank = cluster.block_rank();
  SampleSmem* s0 = cluster.map_shared_rank(s, 0);
  const uint32_t r = blockIdx.x / size;
  const T* row = static_cast<const T*>(a.logits) + size_t(r) * a.row_stride;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const float heat_given = a.temperature ? a.temperature[r] : 1.0f;
  const bool greedy = !(heat_given > 0.0f);
  const float heat = greedy ? 1.0f : fminf(fmaxf(heat_given, 1e-37f), 3e38f);
  const int32_t k_given = a.top_k ? a.top_k[r] : 0;
  const float p_given = a.top_p ? a.top_p[r] : 1.0f;
  const float least = a.min_p ? fminf(a.min_p[r], 1.0f) : 0.0f;
  const bool by_count = !greedy && k_given > 0 && static_cast<uint32_t>(k_given) < a.vocab;
  const bool by_mass = !greedy && p_given < 1.0f;

  // This CTA's slice, and this warp's run of it.
  const uint32_t slice0 = min(rank * a.run * kSampleWarps, a.vocab), slice1 = min(slice0 + a.run * kSampleWarps, a.vocab);
  const uint32_t i0 = min(slice0 + warp * a.run, slice1), i1 = min(i0 + a.run, slice1);
  auto value = [&](uint32_t i) {
    return HELD || i - slice0 < a.held ? s->values[i - slice0] : logit(to_f32(row[i]));
  };
  // The largest logit, and its first index.
  float best = -INFINITY;
  uint32_t at = 0xFFFFFFFFu;
  auto take = [&](uint32_t i, float x) {
    x = logit(x);
    if (HELD || i - slice0 < a.held) s->values[i - slice0] = x;
    if (x > best) {
      best = x;
      at = i;
    }
  };
  constexpr uint32_t V = 16 / sizeof(T);
  // 16-byte loads between the first and the last aligned value of the slice.
  const uint32_t skew = static_cast<uint32_t>((reinterpret_cast<uintptr_t>(row + slice0) % 16) / sizeof(T));
  const uint32_t v0 = min(slice0 + (skew ? V - skew : 0u), slice1), nv = (slice1 - v0) / V;
  if (threadIdx.x < v0 - slice0) take(slice0 + threadIdx.x, to_f32(row[slice0 + threadIdx.x]));
  for (uint32_t c = threadIdx.x; c < nv; c += 4 * kSampleThreads) {
    uint4 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (c + j * kSampleThreads < nv) w[j] = ld_nc4(row + v0 + (c + j * kSampleThreads) * V);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (c + j * kSampleThreads < nv) {
        float x[V];
        unpack16(w[j], x, T());
#pragma unroll
        for (uint32_t e = 0; e < V; ++e) take(v0 + (c + j * kSampleThreads) * V + e, x[e]);
      }
    }
  }
  if (threadIdx.x < slice1 - v0 - nv * V) take(v0 + nv * V + threadIdx.x, to_f32(row[v0 + nv * V + threadIdx.x]));
  auto better = [&](float ob, uint32_t oa) {
    if (ob > best || (ob == best && oa < at)) {
      best = ob;
      at = oa;
    }
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, at, o));
  if (lane == 0) s->sums[warp] = uint64_t(__float_as_uint(best)) << 32 | at;
  s->coarse_count[threadIdx.x] = 0;
  if (threadIdx.x == 0) s->total = 0, s->mass_above = 0, s->listed = 0, s->holder = kSampleWarps;
  __syncthreads();
  better(__uint_as_float(static_cast<uint32_t>(s->sums[lane] >> 32)), static_cast<uint32_t>(s->sums[lane]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, at, o));
  if (threadIdx.x == 0) {
    s->best = best;
    s->best_at = at;
  }
  cluster.sync();
  if (lane < size) better(cluster.map_shared_rank(s, lane)->best, cluster.map_shared_rank(s, lane)->best_at);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, at, o));
  if (best == -INFINITY) {
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[r] = 0;
      if (a.logprobs) a.logprobs[r] = -INFINITY;
    }
    cluster.sync();  // (the others may still be reading this CTA's maximum)
    return;
  }

  // All units, and how many tokens lie how far below the best.
  const Fall scaled{best, 1.4426950408889634f / heat};
  auto fall_of = [&](float x) { return scaled.of(x); };
  auto coarse_bin = [&](float t) { return static_cast<uint32_t>(fminf(t * kBinScale, static_cast<float>(kBins - 1))); };
  const bool cuts = by_count || by_mass, any_cut = cuts || (!greedy && least > 0.0f);
  uint64_t run_sum = 0;
  // (The last bin, which can hold most of a row, is not counted: it has the rest.)
  constexpr float kLastBin = static_cast<float>(kBins - 1);
  const uint32_t whole = i0 + (i1 - i0) / 32 * 32;
#pragma unroll 4
  for (uint32_t i = i0; i < whole; i += 32) {
    const float t = fall_of(value(i + lane));
    run_sum += units_of(weight_of(t));
    const float place = t * kBinScale;
    if (any_cut && place < kLastBin) atomicAdd(&s->coarse_count[static_cast<uint32_t>(place)], 1u);
  }
  if (whole + lane < i1) {
    const float t = fall_of(value(whole + lane));
    run_sum += units_of(weight_of(t));
    const float place = t * kBinScale;
    if (any_cut && place < kLastBin) atomicAdd(&s->coarse_count[static_cast<uint32_t>(place)], 1u);
  }
  run_sum = warp_sum_u64(run_sum);
  if (lane == 0) {
    s->sums[warp] = run_sum;
    atomicAdd(reinterpret_cast<unsigned long long*>(&s0->total), static_cast<unsigned long long>(run_sum));
  }
  __syncthreads();
  if (any_cut && rank != 0 && s->coarse_count[threadIdx.x]) atomicAdd(&s0->coarse_count[threadIdx.x], s->coarse_count[threadIdx.x]);
  cluster.sync();
  const uint64_t all = s0->total;
  // Of the sum 1 + rest, the largest token's unit taken off exactly: near 1 the logarithm keeps the bits of the rest.
  const float log_all = log1pf(static_cast<float>(all - (uint64_t(1) << kUnitBits)) / kUnits);
  auto log_of = [&](float x) { return (x == best ? 0.0f : (x - best) / heat) - log_all; };
  // The largest logit's token is the answer until another is found (each is written behind a barrier of the cluster):
  // whatever the row holds, the outputs are written.
  if (rank == 0 && threadIdx.x == 0) {
    a.tokens[r] = at;
    if (a.logprobs) a.logprobs[r] = -log_all;
  }
  if (greedy) {
    cluster.sync();
    return;
  }

  // The keys of coarse bins first .. last: their ends in logits, a little wider for their rounding.
  const float step_heat = heat * 0.6931471805599453f;  // of a power of two, in logits
  auto keys_of = [&](uint32_t first, uint32_t last, uint32_t& lo, uint32_t& hi) {
    const float slack = 4e-7f * (fabsf(best) + step_heat * (last + 2) / kBinScale);
    hi = order_key<T>(best - step_heat * first / kBinScale + slack);
    lo = last >= kBins - 1 ? 0u : order_key<T>(best - step_heat * (last + 1) / kBinScale - slack);
    if (!(best < INFINITY) || !(step_heat < INFINITY) || !(hi >= lo)) lo = 0, hi = 0xFFFFFFFFu;
  };

  const float draw = fminf(fmaxf(a.uniforms[r], 0.0f), 1.0f);
  auto goal_of = [&](uint64_t total) {
    const uint64_t goal = static_cast<uint64_t>(static_cast<double>(draw) * static_cast<double>(total));
    return goal >= total ? total - 1 : goal;
  };
  auto target_of = [&](uint64_t mass) {  // top_p's
    const uint64_t target = static_cast<uint64_t>(ceil(static_cast<double>(fmaxf(p_given, 0.0f)) * static_cast<double>(mass)));
    return !(p_given > 0.0f) || target < 1 ? uint64_t(1) : target > mass ? mass : target;
  };
  // A token for the first CTA's list, of each lane that has one.
  auto list_token = [&](bool mine, uint32_t k, uint32_t i, float w) {
    const uint32_t votes = __ballot_sync(0xffffffffu, mine);
    if (!votes) return;
    uint32_t at0 = 0;
    if (lane == 0) at0 = atomicAdd(&s0->listed, static_cast<uint32_t>(__popc(votes)));
    at0 = __shfl_sync(0xffffffffu, at0, 0) + __popc(votes & ((1u << lane) - 1u));
    if (mine && at0 < kListed) {
      s0->list.key[at0] = k;
      s0->list.index[at0] = i | (w < least ? 0x80000000u : 0u);
      s0->list.units[at0] = units_of(w);
    }
  };

  // The kept set, once it is known: keys above `key`, and at it the first `ties` of the `here` tokens, or those up to index `tie_last`.
  uint32_t key = 0, ties = 0xFFFFFFFFu, here = 0, tie_last = 0xFFFFFFFFu;
  bool summed = false;  // the sums of the runs are those of the kept set
  uint32_t bin_count = 0;  // of coarse bin threadIdx.x, over the row
  uint64_t bin_mass = 0;

  if (any_cut) {
    // How far down the kept set can reach. top_p's bin is bounded by the least that the bins' tokens can weigh; where
    // top_k cuts too, what top_k left has to be known first, and only top_k bounds.
    // (Every CTA works it out from the first one's counts.)
    uint32_t reach, reached;
    uint32_t n = s0->coarse_count[threadIdx.x];
    const uint32_t above = sum_above(s, n);
    if (threadIdx.x == kBins - 1) n = a.vocab - above;
    {
      __syncthreads();
      if (threadIdx.x == 0) s->reach = kBins - 1;
      const uint64_t want = static_cast<uint64_t>(ceil(static_cast<double>(fmaxf(p_given, 0.0f)) * static_cast<double>(all)));
      uint64_t floor_mass = 0, floor_above = 0;
      if (by_mass && !by_count) {
        floor_mass = threadIdx.x == kBins - 1 ? 0 : units_of(weight_of((threadIdx.x + 1) / kBinScale) * 0.99999f) * n;
        floor_above = sum_above(s, floor_mass);
      } else {
        __syncthreads();
      }
      bool last = false;
      if (by_count) last |= above < static_cast<uint32_t>(k_given) && static_cast<uint32_t>(k_given) <= above + n;
      if (by_mass && !by_count) last |= floor_above < want && want <= floor_above + floor_mass;
      if (!by_mass && least > 0.0f) last |= threadIdx.x == min(static_cast<uint32_t>(fmaxf(-log2f(least), 0.0f) * kBinScale) + 1u, kBins - 1);
      if (by_mass && !by_count && want == 0) last |= threadIdx.x == 0;
      __syncthreads();
      if (last) atomicMin(&s->reach, threadIdx.x);
      __syncthreads();
      reach = s->reach;
      if (threadIdx.x == reach) s->reached = above + n;
      __syncthreads();
      reached = s->reached;
    }
    bin_count = n;
    if (reached <= kListed) {
      // ---- few enough for the first CTA ----
      uint32_t lo, hi;
      keys_of(0, reach, lo, hi);
#pragma unroll 4
      for (uint32_t i = i0; i < i1; i += 32) {
        const bool in = i + lane < i1;
        const float x = in ? value(i + lane) : 0.0f;
        const uint32_t k = order_key<T>(x);
        bool mine = in && k >= lo;
        if (!__any_sync(0xffffffffu, mine)) continue;
        const float fall = fall_of(x);
        mine = mine && coarse_bin(fall) <= reach;
        list_token(mine, k, i + lane, weight_of(fall));
      }
      cluster.sync();
      if (rank != 0) return;  // nothing of this CTA is read from here on
      const uint32_t listed = min(s->listed, kListed);
      if (listed <= kPairs) {
        // Lanes of a token: a power of two, at most a warp.
        uint32_t lanes = 32;
        while (lanes * listed > kSampleThreads) lanes /= 2;
        const uint32_t me = threadIdx.x / lanes, part = threadIdx.x % lanes;
        const bool in = me < listed;
        const uint32_t k = in ? s->list.key[me] : 0u, index = in ? s->list.index[me] & 0x7FFFFFFFu : 0u;
        const bool low = in && (s->list.index[me] & 0x80000000u);
        const uint64_t u = in ? s->list.units[me] : 0;
        uint32_t place = 0;
        uint64_t above = 0;
        if (in) {
          for (uint32_t j = part; j < listed; j += lanes) {
            const uint32_t kj = s->list.key[j];
            if (kj > k || (kj == k && (s->list.index[j] & 0x7FFFFFFFu) < index)) {
              ++place;
              above += s->list.units[j];
            }
          }
        }
        for (uint32_t o = lanes / 2; o > 0; o /= 2) {
          place += __shfl_xor_sync(0xffffffffu, place, o);
          above += __shfl_xor_sync(0xffffffffu, above, o);
        }
        bool kept = in && !(by_count && place >= static_cast<uint32_t>(k_given));
        uint64_t mass = all;
        if (by_count) {
          // The last token that top_k keeps has all of their mass behind it.
          const uint32_t last = min(static_cast<uint32_t>(k_given), listed) - 1;
          if (in && place == last && part == 0) s->slice_sum = above + u;
          __syncthreads();
          mass = s->slice_sum;
        }
        if (by_mass) kept = kept && above < target_of(mass);
        kept = kept && !low;
        __syncthreads();
        if (in && part == 0 && !kept) s->list.units[me] = 0;
        __syncthreads();
        uint64_t before = 0, total = 0;
        for (uint32_t j = part; j < listed; j += lanes) {
          const uint64_t uj = s->list.units[j];
          total += uj;
          if ((s->list.index[j] & 0x7FFFFFFFu) < index) before += uj;
        }
        for (uint32_t o = lanes / 2; o > 0; o /= 2) {
          before += __shfl_xor_sync(0xffffffffu, before, o);
          total += __shfl_xor_sync(0xffffffffu, total, o);
        }
        const uint64_t goal = goal_of(total);
        if (kept && part == 0 && before <= goal && goal < before + u) {
          a.tokens[r] = index;
          if (a.logprobs) a.logprobs[r] = log_of(key_value<T>(k));
        }
        return;
      }
      bool kept = threadIdx.x < listed;
      const uint32_t k = kept ? s->list.key[threadIdx.x] : 0u, index = kept ? s->list.index[threadIdx.x] : 0u;
      const uint32_t place = ~index & 0x7FFFFFFFu;  // falling in the index
      const uint64_t u = kept ? s->list.units[threadIdx.x] : 0;
      const uint32_t place_lo = 0x7FFFFFFFu - (a.vocab - 1), place_hi = 0x7FFFFFFFu;
      Cut cut = {};
      // Keeps the tokens down to the cut, and `ties` of those at it, the lowest indices first.
      auto keep_to = [&](uint32_t ties) {
        const uint32_t key = cut.bin;
        if (ties < cut.here) {
          const bool tie = kept && k == key;
          const bool found = narrow(s, tie, place, u, place_lo, place_hi, false, ties, 0, 0);
          if (tie && found && place < s->cut.bin) kept = false;
        }
        kept = kept && k >= key;
      };
      uint64_t mass = all;
      if (by_count) {
        uint32_t bin_lo, bin_hi;
        keys_of(0, reach, bin_lo, bin_hi);
        if (narrow(s, kept, k, u, bin_lo, bin_hi, false, static_cast<uint32_t>(k_given), 0, 0)) {
          cut = s->cut;
          keep_to(static_cast<uint32_t>(k_given) - cut.count);
        }
        if (by_mass) {
          const uint64_t above = sum_above(s, kept ? u : 0);
          if (threadIdx.x == kSampleThreads - 1) s->slice_sum = above + (kept ? u : 0);
          __syncthreads();
          mass = s->slice_sum;
          __syncthreads();
        }
      }
      if (by_mass) {
        const uint64_t target = target_of(mass);
        if (narrow(s, kept, k, u, lo, hi, true, target, 0, 0)) {
          cut = s->cut;
          const uint64_t each = cut.here_mass / cut.here;
          keep_to(static_cast<uint32_t>((target - cut.mass + each - 1) / each));
        }
      }
      kept = kept && !(index & 0x80000000u);
      const uint64_t above = sum_above(s, kept ? u : 0);
      if (threadIdx.x == kSampleThreads - 1) s->slice_sum = above + (kept ? u : 0);
      __syncthreads();
      const uint64_t goal = goal_of(s->slice_sum);
      if (narrow(s, kept, place, u, place_lo, place_hi, true, goal + 1, 0, 0) && kept && place == s->cut.bin) {
        a.tokens[r] = index;
        if (a.logprobs) a.logprobs[r] = log_of(key_value<T>(k));
      }
      return;
    }
    if (by_mass && !by_count) {
      // ---- top_p alone, many tokens: the few bins that can hold the cut ----
      // The counts bound the mass above a bin from both sides, by what its tokens weigh at least and at most (a bin is 3%
      // wide) and by the same of what lies below, taken from the total: near the end of the row, where top_p as a rule
      // cuts, to a small part of a bin.
      uint64_t n_least = n * units_of(weight_of((threadIdx.x + 1) / kBinScale) * 0.99999f);
      uint64_t n_most = n * (units_of(weight_of(threadIdx.x / kBinScale) * 1.00001f) + 1);
      if (threadIdx.x == kBins - 1) n_least = n_most = 0;  // (its units are 0)
      const uint64_t above_least = sum_above(s, n_least);
      __syncthreads();
      const uint64_t above_most = sum_above(s, n_most);
      if (threadIdx.x == kBins - 1) {
        s->cut.mass = above_least;
        s->cut.here_mass = above_most;
      }
      if (threadIdx.x == 0) s->reach = 0, s->reached = kBins - 1;
      __syncthreads();
      const uint64_t target = target_of(all);
      const uint64_t below_least = s->cut.mass - above_least, below_most = s->cut.here_mass - above_most;  // this bin and all below
      const uint64_t at_most = min(above_most, all - below_least);
      const uint64_t next_most = below_most - n_most;
      const uint64_t next_least = max(above_least + n_least, next_most < all ? all - next_most : uint64_t(0));
      if (at_most < target) atomicMax(&s->reach, threadIdx.x);
      if (next_least >= target) atomicMin(&s->reached, threadIdx.x);
      __syncthreads();
      const uint32_t b0 = s->reach, b1 = s->reached;
      if (threadIdx.x == b0) s->cut.count = above;
      if (threadIdx.x == b1) s->cut.here = above + n;
      __syncthreads();
      const uint32_t over = s->cut.count, in_question = s->cut.here - over;
      if (in_question <= kListed) {
        // One pass: the exact mass above them, kept by run, and their tokens to the first CTA's list.
        const float t0 = static_cast<float>(b0), t1 = static_cast<float>(b1 + 1);
        uint64_t over_mass = 0, kept_mass = 0;
#pragma unroll 4
        for (uint32_t i = i0; i < i1; i += 32) {
          const bool in = i + lane < i1;
          const float x = in ? value(i + lane) : -INFINITY;
          const float t = fall_of(x), w = weight_of(t), place = t * kBinScale;
          if (place < t0) {
            const uint64_t u = units_of(w);
            over_mass += u;
            if (least > 0.0f && w >= least) kept_mass += u;
          }
          list_token(in && place >= t0 && place < t1, order_key<T>(x), i + lane, w);
        }
        over_mass = warp_sum_u64(over_mass);
        if (least > 0.0f) kept_mass = warp_sum_u64(kept_mass);
        if (lane == 0) {
          s->sums[warp] = least > 0.0f ? kept_mass : over_mass;
          atomicAdd(reinterpret_cast<unsigned long long*>(&s0->mass_above), static_cast<unsigned long long>(over_mass));
        }
        cluster.sync();
        if (rank == 0) {
          const bool have = threadIdx.x < min(s->listed, kListed);
          const uint32_t k = have ? s->list.key[threadIdx.x] : 0u, flagged = have ? s->list.index[threadIdx.x] : 0u;
          const uint32_t index = flagged & 0x7FFFFFFFu;
          const uint64_t u = have ? s->list.units[threadIdx.x] : 0;
          uint32_t lo, hi;
          keys_of(b0, b1, lo, hi);
          narrow(s, have, k, u, lo, hi, true, target, over, s->mass_above);
          const Cut cut = s->cut;
          const uint64_t each = cut.here_mass / cut.here;
          const uint32_t stay = static_cast<uint32_t>((target - cut.mass + each - 1) / each);
          uint32_t last = 0xFFFFFFFFu;
          if (stay < cut.here) {
            narrow(s, have && k == cut.bin, ~index & 0x7FFFFFFFu, u, 0x7FFFFFFFu - (a.vocab - 1), 0x7FFFFFFFu, false, stay, 0, 0);
            last = ~s->cut.bin & 0x7FFFFFFFu;
          }
          if (have && flagged == index && (k > cut.bin || (k == cut.bin && index <= last))) {
            const uint32_t slice = index / (a.run * kSampleWarps);
            atomicAdd(reinterpret_cast<unsigned long long*>(
                          &cluster.map_shared_rank(s, slice)->sums[(index - slice * a.run * kSampleWarps) / a.run]),
                      static_cast<unsigned long long>(u));
          }
          if (threadIdx.x == 0) s->answer = Cut{0, 0, last, 0, cut.bin};
        }
        cluster.sync();
        key = s0->answer.bin;
        tie_last = s0->answer.count;
        run_sum = s->sums[warp];
        summed = true;
      }
    }
  }

  if (cuts && !summed) {
    // ---- a large kept set: the masses of the coarse bins, then the one that holds the cut ----
#pragma unroll
    for (int i = 0; i < 3; ++i) s->limb[i][threadIdx.x] = 0;
    s->coarse_mass[threadIdx.x] = 0;
    cluster.sync();
#pragma unroll 4
    for (uint32_t i = i0; i < i1; i += 32) {
      if (i + lane >= i1) continue;
      const float fall = fall_of(value(i + lane));
      const uint32_t bin = coarse_bin(fall);
      if (bin == kBins - 1) continue;  // (its units are 0)
      const uint64_t u = units_of(weight_of(fall));
      constexpr uint32_t kLimb = (1u << kLimbBits) - 1u;
      const uint32_t l0 = static_cast<uint32_t>(u) & kLimb, l1 = static_cast<uint32_t>(u >> kLimbBits) & kLimb;
      const uint32_t l2 = static_cast<uint32_t>(u >> (2 * kLimbBits));
      atomicAdd(&s->limb[0][bin], l0);
      if (l1) atomicAdd(&s->limb[1][bin], l1);
      if (l2) atomicAdd(&s->limb[2][bin], l2);
    }
    __syncthreads();
    const uint64_t u = s->limb[0][threadIdx.x] + (uint64_t(s->limb[1][threadIdx.x]) << kLimbBits) +
                       (uint64_t(s->limb[2][threadIdx.x]) << (2 * kLimbBits));
    if (u) atomicAdd(reinterpret_cast<unsigned long long*>(&s0->coarse_mass[threadIdx.x]), static_cast<unsigned long long>(u));
    __syncthreads();
    clear(s->fine);
    cluster.sync();
    bin_mass = s0->coarse_mass[threadIdx.x];
    cluster.sync();  // (the list takes the masses' room)
  }

  // The key at which a prefix reaches the target. Every CTA comes here or none.
  auto find_cut = [&](bool mass, uint64_t target, uint32_t& key, Cut& cut) {
    __syncthreads();
    find_bin(s, bin_count, bin_mass, mass, target, 0, 0);
    __syncthreads();
    cut = s->cut;
    const uint32_t bin = cut.bin;
    uint32_t lo, hi;
    keys_of(bin, bin, lo, hi);
    const bool by_list = cut.here <= kListed;
    auto each_of_bin = [&](auto use) {  // the bin's tokens of this slice, those with keys lo .. hi
#pragma unroll 4
      for (uint32_t i = i0; i < i1; i += 32) {
        const bool in = i + lane < i1;
        const float x = in ? value(i + lane) : 0.0f;
        const uint32_t k = order_key<T>(x);
        bool mine = in && k <= hi && k >= lo;
        if (!__any_sync(0xffffffffu, mine)) continue;
        const float fall = fall_of(x);
        mine = mine && coarse_bin(fall) == bin;
        use(mine, k, units_of(weight_of(fall)));
      }
    };
    if (by_list) {
      each_of_bin([&](bool mine, uint32_t k, uint64_t u) {
        const uint32_t votes = __ballot_sync(0xffffffffu, mine);
        if (!votes) return;
        uint32_t at0 = 0;
        if (lane == 0) at0 = atomicAdd(&s0->listed, static_cast<uint32_t>(__popc(votes)));
        at0 = __shfl_sync(0xffffffffu, at0, 0) + __popc(votes & ((1u << lane) - 1u));
        if (mine && at0 < kListed) {
          s0->list.key[at0] = k;
          s0->list.units[at0] = u;
        }
      });
      cluster.sync();
      if (rank == 0) {
        const bool have = threadIdx.x < min(s->listed, kListed);
        const uint32_t k = have ? s->list.key[threadIdx.x] : 0u;
        const uint64_t u = have ? s->list.units[threadIdx.x] : 0;
        narrow(s, have, k, u, lo, hi, mass, target, cut.count, cut.mass);
        clear(s->fine);  // (the next cut may be narrowed by all CTAs, which add to it)
        if (threadIdx.x == 0) {
          s->answer = s->cut;
          s->listed = 0;
        }
        __syncthreads();
      }
      cluster.sync();
      cut = s0->answer;
      hi = cut.bin;
    } else {
      for (;;) {
        const uint32_t bits = 32 - __clz((hi - lo) | 1u);
        const uint32_t shift = bits > kBinBits ? bits - kBinBits : 0u;
        each_of_bin([&](bool mine, uint32_t k, uint64_t u) {
          if (mine) add_to(s0->fine.count, s0->fine.mass, (hi - k) >> shift, 1, u);
        });
        cluster.sync();
        if (rank == 0) {
          find_bin(s, s->fine.count[threadIdx.x], s->fine.mass[threadIdx.x], mass, target, cut.count, cut.mass);
          __syncthreads();
          clear(s->fine);
          if (threadIdx.x == 0) s->answer = s->cut;
        }
        cluster.sync();
        cut = s0->answer;
        hi -= cut.bin << shift;
        cluster.sync();  // (the first CTA does not answer again before all have read it)
        if (shift == 0) break;
        lo = hi - min(hi - lo, (1u << shift) - 1u);
      }
    }
    key = hi;
  };

  uint64_t mass = all;
  if (by_count && !summed) {
    Cut cut;
    find_cut(false, static_cast<uint64_t>(k_given), key, cut);
    ties = static_cast<uint32_t>(k_given) - cut.count;
    here = cut.here;
    mass = cut.mass + cut.here_mass / cut.here * ties;
  }
  if (by_mass && !summed) {
    if (by_count) cluster.sync();  // (all have read the first answer)
    const uint64_t target = target_of(mass);
    Cut cut;
    find_cut(true, target, key, cut);
    const uint64_t each = cut.here_mass / cut.here;
    ties = static_cast<uint32_t>((target - cut.mass + each - 1) / each);
    here = cut.here;
  }

  // Tokens at the cut in the runs before this one, where not all of them stay.
  uint32_t tie_base = 0;
  const bool rank_ties = ties < here;
  if (rank_ties) {
    uint32_t n = 0;
#pragma unroll 4
    for (uint32_t i = i0 + lane; i < i1; i += 32) n += order_key<T>(value(i)) == key ? 1u : 0u;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) s->scan_count[warp] = n;
    __syncthreads();
    const uint32_t mine = s->scan_count[lane];
    tie_base = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0u);
    const uint32_t sum = __reduce_add_sync(0xffffffffu, mine);
    if (threadIdx.x == 0) s->slice_ties = sum;
    cluster.sync();
    tie_base += __reduce_add_sync(0xffffffffu, lane < rank ? cluster.map_shared_rank(s, lane)->slice_ties : 0u);
  }
  auto kept_units = [&](uint32_t i, uint32_t& tie_at) -> uint64_t {
    const bool in = i < i1;
    const float x = in ? value(i) : -INFINITY;
    const uint32_t k = order_key<T>(x);
    bool keep = in && (k > key || (k == key && i <= tie_last));
    if (rank_ties) {
      const bool tie = in && k == key;
      const uint32_t votes = __ballot_sync(0xffffffffu, tie);
      if (tie && tie_at + __popc(votes & ((1u << lane) - 1u)) >= ties) keep = false;
      tie_at += __popc(votes);
    }
    if (!__any_sync(0xffffffffu, keep)) return 0;
    if (!keep) return 0;
    const float w = weight_of(fall_of(x));
    return w >= least ? units_of(w) : 0;
  };
  // The sum of each run, then the walk of the one that holds the token.
  const bool every = !cuts && !(least > 0.0f);
  if (!every && !summed) {
    uint32_t tie_at = tie_base;
    run_sum = 0;
#pragma unroll 4
    for (uint32_t i = i0; i < i1; i += 32) run_sum += kept_units(i + lane, tie_at);
    run_sum = warp_sum_u64(run_sum);
    if (lane == 0) s->sums[warp] = run_sum;
    __syncthreads();
  }
  const uint64_t other = s->sums[lane];
  uint64_t before = warp_sum_u64(lane < warp ? other : 0);
  if (warp == 0) {
    const uint64_t sum = warp_sum_u64(other);
    if (lane == 0) s->slice_sum = sum;
  }
  cluster.sync();
  const uint64_t slice = lane < size ? cluster.map_shared_rank(s, lane)->slice_sum : 0;
  before += warp_sum_u64(lane < rank ? slice : 0);
  const uint64_t kept = warp_sum_u64(slice);
  const uint64_t goal = goal_of(kept);
  auto answer_with = [&](uint32_t i) {
    a.tokens[r] = i;
    if (a.logprobs) a.logprobs[r] = log_of(value(i));
  };
  auto units_if_kept = [&](uint32_t i) -> uint64_t {
    const float x = value(i);
    const uint32_t k = order_key<T>(x);
    if (!(k > key || (k == key && i <= tie_last))) return 0;
    const float w = weight_of(fall_of(x));
    return w >= least ? units_of(w) : 0;
  };
  if (before <= goal && goal < before + run_sum) {
    if (rank_ties) {
      uint64_t sum = before;
      uint32_t tie_at = tie_base;
      for (uint32_t i = i0; i < i1; i += 32) {
        const uint64_t inc = sum + warp_scan_u64(kept_units(i + lane, tie_at));
        const uint32_t past = __ballot_sync(0xffffffffu, inc > goal);
        if (past) {
          if (lane == static_cast<uint32_t>(__ffs(past)) - 1) answer_with(i + lane);
          break;
        }
        sum = __shfl_sync(0xffffffffu, inc, 31);
      }
    } else if (lane == 0) {
      s->holder = warp;
      s->mass_above = before;
    }
  }
  __syncthreads();
  if (s->holder < kSampleWarps) {
    // All warps walk the run that holds the token, 32 tokens of it to a warp at a time.
    const uint32_t h0 = slice0 + s->holder * a.run, h1 = min(h0 + a.run, slice1);
    uint64_t from = s->mass_above;
    for (uint32_t h = h0; h < h1; h += 32 * kSampleWarps) {
      const uint32_t i = h + threadIdx.x;
      const uint64_t u = i < h1 ? units_if_kept(i) : 0, inc = warp_scan_u64(u);
      if (lane == 31) s->scan[warp] = inc;
      __syncthreads();
      const uint64_t group = s->scan[lane];
      const uint64_t mine = from + warp_sum_u64(lane < warp ? group : 0) + inc;
      if (mine > goal && mine - u <= goal) answer_with(i);
      from += warp_sum_u64(group);
      if (from > goal) break;
      __syncthreads();  // (before the next sums)
    }
  }
  cluster.sync();  // no CTA leaves while another reads its sums
}

template <typename T>
int32_t sample_as(SampleArgs a, uint32_t rows, cudaStream_t stream) {
  // CTAs to a row: as few as hold it in their shared memory, then twice as many while there are SMs for all rows, at
  // most 8. One row of 151936: eight CTAs 16.5 us, four 21, two 55 (sixteen as eight, on an earlier build); 64 rows: four 55 us,
  // eight 69 (more waves, each with a row's dozen exchanges), two 105 (slices that do not fit are read again and again).
  const uint32_t most = (227 * 1024 - 1024 - static_cast<uint32_t>(sizeof(SampleSmem))) / 4;
  uint32_t size = 1;
  while (size < 8 && (uint64_t(size) * most < a.vocab || rows * size * 2 <= 148)) size *= 2;
  a.run = ((a.vocab + size * kSampleWarps - 1) / (size * kSampleWarps) + 31) / 32 * 32;
  a.held = a.run * kSampleWarps < most ? a.run * kSampleWarps : most;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * size);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = sizeof(SampleSmem) + size_t(a.held) * 4;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = a.run * kSampleWarps <= most ? sample_kernel<T, true> : sample_kernel<T, false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(cfg.dynamicSmemBytes));
  if (e != cudaSuccess) return paged_status(e);
  return paged_status(cudaLaunchKernelEx(&cfg, kernel, a));
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
  if (vocab > QWC_SAMPLE_MAX_VOCAB || rows > (1u << 24) || row_stride > (uint64_t(1) << 31)) return QWC_LIMIT_EXCEEDED;
  const SampleArgs a{logits, row_stride, vocab, 0, 0, temperature, top_k, top_p, min_p, uniforms, tokens_out, logprobs_out};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return format == kFormatF32 ? sample_as<float>(a, rows, s)
         : format == kFormatF16 ? sample_as<__half>(a, rows, s)
                                : sample_as<__nv_bfloat16>(a, rows, s);
}

}  // extern "C"
