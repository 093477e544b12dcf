// qwc_paged_tile.cu -- attention over a paged q8 cache for tokens that give a
// kv head more rows than mma.sync's tiles are worth: 128-row tiles on the
// 5th-generation tensor cores.
//
// A tile is 128 rows of one (sequence, kv head): row i is token i / share,
// query head i % share of the kv head's. It walks the positions that its last
// token sees, 64 at a time:
//
//   warps 0-3  softmax: one row to a thread. Scores from tensor memory, the
//              key scales, the causal limit, the running maximum and sum;
//              the weights go back to tensor memory in place of the scores.
//   warps 4-7  convert: the step's code rows, fetched through the page table
//              into registers a step ahead, become f16 integers in shared memory
//              (keys and values alike, 128-byte swizzled rows of 64 dims).
//   warp 8     issues the MMAs: scores S_g = Q_g K_g^T for each group g of 64
//              dims (its own accumulator, as each position has a scale for each
//              group), output O_g += (P . vs_g) V_g with the weights read from tensor memory.
//
// Codes are exact in f16. A query row enters as f16 at its own power of two
// (f32 rows as two parts, hi and lo), a weight times its value scale likewise;
// everything else is f32. Tensor memory: 256 columns a CTA (scores 128, output
// 128), so two CTAs share an SM and one's softmax covers the other's MMAs.
//
// The output is rescaled only when a row's maximum has grown by more than
// 2^8: until then the old maximum serves, and the weights stay below 2^8.
//
// Work is dealt as in qwc_paged_attention.cu: the steps of all tiles stand in
// one line, each CTA takes an equal stretch, a tile that is cut is joined by
// the CTA that comes last, in the order of the stretches.

#include <cuda_runtime.h>

#include "qwc_device.cuh"
#include "qwc_paged.cuh"
#include "qwc_tcgen05.cuh"

namespace qwc {
namespace {

constexpr uint32_t kRows = 128;   // rows of a tile
constexpr uint32_t kStep = 64;    // positions of a step
constexpr uint32_t kTileThreads = 288;
constexpr uint32_t kGrowth = 8;   // log2 of how far a maximum may run ahead of the one in use

template <int DIM, bool SPLIT>
struct __align__(1024) TileSmem {
  static constexpr int G = DIM / 64;
  static constexpr int PARTS = SPLIT ? 2 : 1;
  uint8_t q[PARTS][G][kRows * 128];  // f16, 128-byte swizzled rows of 64 dims
  uint8_t k[G][kStep * 128];
  uint8_t v[G][kStep * 128];
  float ks[2][G][kStep];  // the step's key scales; by the step's parity
  float vs[2][G][kStep];  // its value scales, times 2^(21 - vexp)
  uint32_t valid[2][2];   // one bit for each position that is cached
  uint32_t vexp[2];
  uint64_t q_full, k_full, k_empty, s_full, p_full, v_full, v_empty, o_full;
  uint64_t scales_full[2];  // by the step's parity, like the scales
  uint64_t sums[9];
  uint64_t found_base;
  uint32_t found_s;
  uint32_t tmem;
};

// A tile of the line, and the tiles after it.
struct TileWalk {
  uint32_t s, h, qt;
  uint32_t tiles, steps;  // of the sequence's kv head; of this tile
  uint64_t first;         // its first step in the line
  PagedSeq seq;
};

__device__ __forceinline__ uint32_t tiles_of(const PagedSeq& q, uint32_t share) {
  return (q.n * share + kRows - 1) / kRows;
}
__device__ __forceinline__ uint32_t tile_steps(const PagedSeq& q, uint32_t share, uint32_t qt) {
  const uint32_t last = min((qt * kRows + kRows - 1) / share, q.n - 1);
  const int32_t seen = min(q.base + static_cast<int32_t>(last) + 1, static_cast<int32_t>(q.context));
  return seen > 0 ? (static_cast<uint32_t>(seen) + kStep - 1) / kStep : 1u;
}
__device__ __forceinline__ uint64_t head_steps(const PagedSeq& q, uint32_t share) {
  const uint32_t t = tiles_of(q, share);
  uint64_t sum = 0;
  for (uint32_t i = 0; i < t; ++i) sum += tile_steps(q, share, i);
  return sum;
}

__device__ __forceinline__ void next_tile(const PagedArgs& a, uint32_t share, TileWalk& w) {
  w.first += w.steps;
  if (++w.qt == w.tiles) {
    w.qt = 0;
    if (++w.h == a.kv_heads) {
      w.h = 0;
      do {
        w.seq = paged_seq(a, ++w.s);
      } while (w.seq.n == 0 && w.s + 1 < a.sequences);
      w.tiles = tiles_of(w.seq, share);
    }
  }
  w.steps = tile_steps(w.seq, share, w.qt);
}

// 16 columns of each of two places in tensor memory (lane quarter of this warp).
__device__ __forceinline__ void tmem_ld16x2(uint32_t t0, uint32_t t1, float (&x)[16], float (&y)[16]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=&r"(r[0]), "=&r"(r[1]), "=&r"(r[2]), "=&r"(r[3]), "=&r"(r[4]), "=&r"(r[5]), "=&r"(r[6]), "=&r"(r[7]), "=&r"(r[8]),
        "=&r"(r[9]), "=&r"(r[10]), "=&r"(r[11]), "=&r"(r[12]), "=&r"(r[13]), "=&r"(r[14]), "=&r"(r[15]), "=&r"(r[16]),
        "=&r"(r[17]), "=&r"(r[18]), "=&r"(r[19]), "=&r"(r[20]), "=&r"(r[21]), "=&r"(r[22]), "=&r"(r[23]), "=&r"(r[24]),
        "=&r"(r[25]), "=&r"(r[26]), "=&r"(r[27]), "=&r"(r[28]), "=&r"(r[29]), "=&r"(r[30]), "=&r"(r[31])
      : "r"(t0), "r"(t1)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] = __uint_as_float(r[i]);
    y[i] = __uint_as_float(r[16 + i]);
  }
}

__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(t),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st16f(uint32_t t, const float (&f)[16]) {
  uint32_t v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(f[i]);
  tmem_st16(t, v);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void fence_proxy_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// D = f32, A and B f16, M = 128, N = 64; B with the dims along its rows (keys)
// or along its columns (values).
constexpr uint32_t kIdescScores = (1u << 4) | ((kStep >> 3) << 17) | ((kRows >> 4) << 24);
constexpr uint32_t kIdescOutput = (1u << 4) | (1u << 16) | ((64u >> 3) << 17) | ((kRows >> 4) << 24);

template <typename T, int DIM>
__global__ void __launch_bounds__(kTileThreads, 2) paged_attention_tile_kernel(const PagedArgs a, const AttnArgs p) {
  constexpr bool SPLIT = sizeof(T) == 4;
  constexpr int G = DIM / 64;
  constexpr int PARTS = SPLIT ? 2 : 1;
  constexpr uint32_t kTmemScores = 0, kTmemOutput = G * kStep, kTmemCols = G * kStep + DIM;
  using Smem = TileSmem<DIM, SPLIT>;
  extern __shared__ __align__(1024) uint8_t tile_smem_raw[];
  const uint32_t pad = (1024u - (smem_addr(tile_smem_raw) & 1023u)) & 1023u;
  Smem* sm = reinterpret_cast<Smem*>(tile_smem_raw + pad);
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;

  // ---- this CTA's stretch of the line ----
  uint64_t part = 0;
  for (uint32_t s = tid; s < a.sequences; s += kTileThreads) part += head_steps(paged_seq(a, s), p.share) * a.kv_heads;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if (lane == 0) sm->sums[warp] = part;
  __syncthreads();
  uint64_t total = 0;
  for (int w = 0; w < 9; ++w) total += sm->sums[w];
  const uint64_t grid = total < gridDim.x ? total : gridDim.x;
  if (blockIdx.x >= grid) return;
  const uint64_t u0 = total * blockIdx.x / grid, u1 = total * (blockIdx.x + 1) / grid;
  uint64_t running = 0;
  for (uint32_t base = 0; base < a.sequences; base += kTileThreads) {
    const uint32_t s = base + tid;
    const uint64_t v = s < a.sequences ? head_steps(paged_seq(a, s), p.share) * a.kv_heads : 0;
    uint64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= static_cast<uint32_t>(o)) inc += t;
    }
    __syncthreads();
    if (lane == 31) sm->sums[warp] = inc;
    __syncthreads();
    uint64_t before = running, all = running;
    for (uint32_t w = 0; w < 9; ++w) {
      if (w < warp) before += sm->sums[w];
      all += sm->sums[w];
    }
    if (v && before + inc - v <= u0 && u0 < before + inc) {
      sm->found_s = s;
      sm->found_base = before + inc - v;
    }
    running = all;
    if (running > u0) break;
  }
  if (tid == 0) {
    mbar_init(&sm->q_full, 4);
    mbar_init(&sm->k_full, 4);
    mbar_init(&sm->k_empty, 1);
    mbar_init(&sm->s_full, 1);
    mbar_init(&sm->p_full, 4);
    mbar_init(&sm->v_full, 4);
    mbar_init(&sm->v_empty, 1);
    mbar_init(&sm->o_full, 1);
    mbar_init(&sm->scales_full[0], 4);
    mbar_init(&sm->scales_full[1], 4);
    fence_mbar_init();
  }
  if (warp == 8) tmem_alloc(&sm->tmem, kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm->tmem;
  TileWalk walk;
  {
    walk.s = sm->found_s;
    walk.seq = paged_seq(a, walk.s);
    walk.tiles = tiles_of(walk.seq, p.share);
    const uint64_t per_head = head_steps(walk.seq, p.share);
    uint64_t off = u0 - sm->found_base;
    walk.h = static_cast<uint32_t>(off / per_head);
    off -= walk.h * per_head;
    walk.first = u0 - off;
    walk.qt = 0;
    walk.steps = tile_steps(walk.seq, p.share, 0);
    while (off >= walk.steps) {
      off -= walk.steps;
      walk.first += walk.steps;
      walk.steps = tile_steps(walk.seq, p.share, ++walk.qt);
    }
  }
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t n, int32_t code) {  // phase n of a barrier
    return mbar_wait_bounded(bar, n & 1u, p.error, p.timeout_ns, code);
  };

  if (warp < 4) {
    // ---- softmax: row tid of the tile ----
    const uint32_t taddr = tmem + ((warp * 32u) << 16);
    uint32_t it = 0, seg = 0;
    for (uint64_t cur = u0; cur < u1 && ok; ++seg) {
      const uint32_t j0 = static_cast<uint32_t>(cur - walk.first);
      const uint32_t j1 = static_cast<uint32_t>((u1 < walk.first + walk.steps ? u1 : walk.first + walk.steps) - walk.first);
      const uint32_t row = walk.qt * kRows + tid;
      const bool in = row < walk.seq.n * p.share;
      const uint32_t tok = in ? row / p.share : 0u, head = walk.h * p.share + (in ? row % p.share : 0u);
      // The row's queries: its largest value gives the power of two, then the f16 parts.
      const T* src = static_cast<const T*>(p.q) + size_t(walk.seq.first + tok) * p.q_stride + size_t(head) * DIM;
      constexpr int V = Vec16<T>::kCount;
      float amax = 0.0f;
      if (in) {
#pragma unroll 4
        for (int d = 0; d < DIM; d += V) {
          float x[V];
          unpack16(*reinterpret_cast<const uint4*>(src + d), x, T());
#pragma unroll
          for (int e = 0; e < V; ++e) amax = fmaxf(amax, fabsf(x[e]));
        }
      }
      const int e2 = row_exponent(amax);
      const float down = pow2i(-e2);
      const float factor = p.scaling * 1.4426950408889634f * pow2i(e2);
      const int32_t limit = in ? walk.seq.base + static_cast<int32_t>(tok) : -1;
#pragma unroll 2
      for (int d = 0; d < DIM; d += 8) {
        float x[8];
        if (!in) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = 0.0f;
        } else if constexpr (SPLIT) {
          const float4 f0 = *reinterpret_cast<const float4*>(src + d), f1 = *reinterpret_cast<const float4*>(src + d + 4);
          x[0] = f0.x, x[1] = f0.y, x[2] = f0.z, x[3] = f0.w, x[4] = f1.x, x[5] = f1.y, x[6] = f1.z, x[7] = f1.w;
        } else {
          unpack16(*reinterpret_cast<const uint4*>(src + d), x, T());
        }
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y0 = fmaf(x[2 * e], down, x[2 * e] - x[2 * e]);  // an infinity is NaN from here on
          const float y1 = fmaf(x[2 * e + 1], down, x[2 * e + 1] - x[2 * e + 1]);
          hi[e] = f16x2(y0, y1);
          const float2 f = f16x2_f32(hi[e]);
          lo[e] = f16x2(y0 - f.x, y1 - f.y);
        }
        const uint32_t at = tid * 128u + ((((d % 64) / 8) ^ (tid & 7u)) << 4);
        *reinterpret_cast<uint4*>(&sm->q[0][d / 64][at]) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if constexpr (SPLIT) *reinterpret_cast<uint4*>(&sm->q[PARTS - 1][d / 64][at]) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm->q_full);

      float m = -INFINITY, l = 0.0f;
      uint32_t vexp = 0;
      for (uint32_t j = j0; j < j1; ++j, ++it) {
        const uint32_t b = it & 1u;
        ok = __all_sync(0xffffffffu, wait(&sm->scales_full[b], it >> 1, 210) && wait(&sm->s_full, it, 201));
        if (!ok) break;
        tc_fence_after();
        float x[kStep];
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < static_cast<int>(kStep); i += 32 / G) {
          // Both groups' sums of 16 positions, or the one group's of 32.
          float s0[16], s1[16];
          tmem_ld16x2(taddr + kTmemScores + i, taddr + kTmemScores + i + (G == 2 ? kStep : 16u), s0, s1);
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 k0 = *reinterpret_cast<const float4*>(&sm->ks[b][0][i + e]);
            const float4 k1 = *reinterpret_cast<const float4*>(G == 2 ? &sm->ks[b][G - 1][i + e] : &sm->ks[b][0][i + 16 + e]);
            const float f0[4] = {k0.x, k0.y, k0.z, k0.w}, f1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if constexpr (G == 2) {
                x[i + e + q] = fmaf(s1[e + q], f1[q], s0[e + q] * f0[q]);
              } else {
                x[i + e + q] = s0[e + q] * f0[q];
                x[i + 16 + e + q] = s1[e + q] * f1[q];
              }
            }
          }
        }
        const int32_t pos0 = static_cast<int32_t>(j * kStep);
        const uint32_t v0 = sm->valid[b][0], v1 = sm->valid[b][1];
        if (pos0 + static_cast<int32_t>(kStep) - 1 > limit || (v0 & v1) != 0xFFFFFFFFu) {
#pragma unroll
          for (int i = 0; i < static_cast<int>(kStep); ++i) {
            if (pos0 + i > limit || !(((i < 32 ? v0 : v1) >> (i % 32)) & 1u)) x[i] = -INFINITY;
          }
        }
#pragma unroll
        for (int i = 0; i < static_cast<int>(kStep); ++i) mx = fmaxf(mx, x[i]);
        float rescale = 1.0f;
        bool grew = false;
        if ((mx - m) * factor > static_cast<float>(kGrowth) || (m == -INFINITY && mx > m)) {
          rescale = m == -INFINITY ? 0.0f : ex2((m - mx) * factor);
          l *= rescale;
          m = mx;
          grew = true;
        }
        const uint32_t top = sm->vexp[b];
        if (top > vexp) {
          rescale *= pow2i(static_cast<int>(vexp) - static_cast<int>(top));
          vexp = top;
          grew = true;
        }
        if (j > j0 && __any_sync(0xffffffffu, grew)) {
          // The MMAs behind s_full are the last step's too: its output is complete.
#pragma unroll
          for (int i = 0; i < DIM; i += 32) {
            float o0[16], o1[16];
            tmem_ld16x2(taddr + kTmemOutput + i, taddr + kTmemOutput + i + 16, o0, o1);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              o0[e] *= rescale;
              o1[e] *= rescale;
            }
            tmem_st16f(taddr + kTmemOutput + i, o0);
            tmem_st16f(taddr + kTmemOutput + i + 16, o1);
          }
        }
        const float mf = m == -INFINITY ? 0.0f : m * factor;
#pragma unroll
        for (int i = 0; i < static_cast<int>(kStep); ++i) {
          x[i] = ex2(fmaf(x[i], factor, -mf));
          l += x[i];
        }
        // Weights over the scores' columns: part q of group g at columns 32 (q G + g).
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
          for (int i = 0; i < static_cast<int>(kStep); i += 32) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 f = *reinterpret_cast<const float4*>(&sm->vs[b][g][i + e]);
              const float w0 = x[i + e] * f.x, w1 = x[i + e + 1] * f.y, w2 = x[i + e + 2] * f.z, w3 = x[i + e + 3] * f.w;
              hi[e / 2] = f16x2(w0, w1);
              hi[e / 2 + 1] = f16x2(w2, w3);
              if constexpr (SPLIT) {
                const float2 r0 = f16x2_f32(hi[e / 2]), r1 = f16x2_f32(hi[e / 2 + 1]);
                lo[e / 2] = f16x2(w0 - r0.x, w1 - r0.y);
                lo[e / 2 + 1] = f16x2(w2 - r1.x, w3 - r1.y);
              }
            }
            tmem_st16(taddr + kTmemScores + 32 * g + i / 2, hi);
            if constexpr (SPLIT) tmem_st16(taddr + kTmemScores + 32 * (G + g) + i / 2, lo);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm->p_full);
      }
      if (!ok) break;

      // ---- the tile's output, or this stretch's part of it ----
      ok = __all_sync(0xffffffffu, wait(&sm->o_full, seg, 202));
      if (!ok) break;
      tc_fence_after();
      const float back = pow2i(static_cast<int>(vexp) - 21);
      T* dst = static_cast<T*>(p.out) + size_t(walk.seq.first + tok) * p.out_stride + size_t(head) * DIM;
      const bool whole = j0 == 0 && j1 == walk.steps;
      const uint32_t slot = 2 * blockIdx.x + (walk.first > u0 ? 1u : 0u);
      float* mine = p.partials + size_t(slot) * (DIM + 2) * kRows + tid;
      const float inv = whole ? (l == 0.0f ? 0.0f : back / l) : back;
#pragma unroll
      for (int i = 0; i < DIM; i += 32) {
        float o[32];
        tmem_ld32(taddr + kTmemOutput + i, o);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = l == 0.0f ? 0.0f : o[e] * inv;
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 32; ++e) mine[size_t(i + e) * kRows] = o[e];
        } else if (in) {
          constexpr int W = Vec16<T>::kCount;
#pragma unroll
          for (int e = 0; e < 32; e += W) {
            float y[W];
#pragma unroll
            for (int q = 0; q < W; ++q) y[q] = o[e + q];
            *reinterpret_cast<uint4*>(dst + i + e) = pack16<T>(y);
          }
        }
      }
      if (!whole) {
        mine[size_t(DIM) * kRows] = m == -INFINITY ? m : m * factor;
        mine[size_t(DIM + 1) * kRows] = l;
        // The stretches that hold this tile: c0 .. c1 (stretch x starts at
        // floor(x * total / grid)). Each warp joins its 32 rows by itself.
        const uint64_t seg0 = walk.first, seg1 = walk.first + walk.steps;
        const uint32_t c0 = static_cast<uint32_t>(((seg0 + 1) * grid - 1) / total);
        const uint32_t c1 = static_cast<uint32_t>((seg1 * grid - 1) / total);
        __threadfence();
        __syncwarp();
        uint32_t last = 0;
        if (lane == 0) {
          uint32_t* counter = &p.counters[4 * c0 + warp];
          const uint32_t before = atomicAdd(counter, 1u);
          last = before == c1 - c0;
          if (last) *counter = 0;
        }
        last = __shfl_sync(0xffffffffu, last, 0);
        if (last) {
          __threadfence();
          auto piece = [&](uint32_t x) {
            const uint32_t sl = 2 * x + (seg0 > total * x / grid ? 1u : 0u);
            return p.partials + size_t(sl) * (DIM + 2) * kRows + tid;
          };
          float best = -INFINITY, sum = 0.0f;
          for (uint32_t x = c0; x <= c1; ++x) best = fmaxf(best, __ldcg(piece(x) + size_t(DIM) * kRows));
          for (uint32_t x = c0; x <= c1; ++x) {
            const float pm = __ldcg(piece(x) + size_t(DIM) * kRows);
            sum = fmaf(__ldcg(piece(x) + size_t(DIM + 1) * kRows), best == -INFINITY ? 1.0f : ex2(pm - best), sum);
          }
          const float norm = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll 1
          for (int i = 0; i < DIM; i += 16) {
            float o[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0.0f;
            for (uint32_t x = c0; x <= c1; ++x) {
              const float* from = piece(x);
              const float pm = __ldcg(from + size_t(DIM) * kRows);
              const float f = (best == -INFINITY ? 1.0f : ex2(pm - best)) * norm;
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = fmaf(__ldcg(from + size_t(i + e) * kRows), f, o[e]);
            }
            if (in) {
              constexpr int W = Vec16<T>::kCount;
#pragma unroll
              for (int e = 0; e < 16; e += W) {
                float y[W];
#pragma unroll
                for (int q = 0; q < W; ++q) y[q] = o[e + q];
                *reinterpret_cast<uint4*>(dst + i + e) = pack16<T>(y);
              }
            }
          }
        }
      }
      tc_fence_before();  // the output's columns may be written again once the next weights arrive
      cur = walk.first + j1;
      if (cur < u1) next_tile(a, p.share, walk);
    }
  } else if (warp < 8) {
    // ---- convert: keys, then values, of each step ----
    const uint32_t ct = tid - 128;
    constexpr uint32_t CH = DIM / 16;              // 16-byte chunks of a row of codes
    constexpr uint32_t ROWS_PASS = 128 / CH;       // rows that the 128 threads fetch at once
    constexpr uint32_t PASSES = kStep / ROWS_PASS;
    const uint32_t ch = ct % CH, r0 = ct / CH;
    uint32_t it = 0;
    uint32_t vexp = 0;
    // A step ahead: its code chunks, and its scales (lane l: positions 2 l and 2 l + 1).
    uint4 kraw[PASSES], vraw[PASSES];
    TileWalk ahead = walk;
    uint32_t aj = static_cast<uint32_t>(u0 - walk.first);
    auto row_at = [&](uint32_t pos) -> int32_t {
      if (pos >= ahead.seq.context) return -1;
      return static_cast<int32_t>(paged_row(a, ahead.s, pos));
    };
    auto fetch = [&](uint4 (&raw)[PASSES], const uint8_t* plane) {
#pragma unroll
      for (uint32_t i = 0; i < PASSES; ++i) {
        const int32_t row = row_at(aj * kStep + r0 + i * ROWS_PASS);
        raw[i] = row >= 0 ? ld_nc4(plane + uint64_t(static_cast<uint32_t>(row)) * a.code_row + ahead.h * DIM + 16u * ch)
                          : make_uint4(0, 0, 0, 0);
      }
    };
    uint32_t scale_raw[2][2];  // [key, value][position 2 lane + e]: both groups
    uint32_t valid_bits[2];
    auto fetch_scales = [&]() {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int32_t row = row_at(aj * kStep + 32u * e + lane);
        valid_bits[e] = __ballot_sync(0xffffffffu, row >= 0);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          scale_raw[n][e] = 0;
          if (row >= 0) {
            const uint8_t* from = (n ? a.v_scales : a.k_scales) + uint64_t(static_cast<uint32_t>(row)) * a.scale_row + ahead.h * (2 * G);
            scale_raw[n][e] = G == 2 ? *reinterpret_cast<const uint32_t*>(from) : *reinterpret_cast<const uint16_t*>(from);
          }
        }
      }
    };
    auto put = [&](uint8_t* tile, const uint4 (&raw)[PASSES]) {
      // Chunk ch is dims 16 ch .. + 15: two 16-byte chunks of f16 in group ch / 4's tile.
      uint8_t* base = tile + (ch / 4) * (kStep * 128);
#pragma unroll
      for (uint32_t i = 0; i < PASSES; ++i) {
        const uint32_t r = r0 + i * ROWS_PASS;
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint4 o[2];
        o[0] = make_uint4(codes_f16x2<0x4140>(w[0]), codes_f16x2<0x4342>(w[0]), codes_f16x2<0x4140>(w[1]), codes_f16x2<0x4342>(w[1]));
        o[1] = make_uint4(codes_f16x2<0x4140>(w[2]), codes_f16x2<0x4342>(w[2]), codes_f16x2<0x4140>(w[3]), codes_f16x2<0x4342>(w[3]));
        const uint32_t c2 = 2 * (ch % 4), flip = ch / 4;  // the two groups' lanes on different banks
        *reinterpret_cast<uint4*>(base + r * 128u + (((c2 + flip) ^ (r & 7u)) << 4)) = flip ? o[1] : o[0];
        *reinterpret_cast<uint4*>(base + r * 128u + (((c2 + 1 - flip) ^ (r & 7u)) << 4)) = flip ? o[0] : o[1];
      }
    };
    fetch(kraw, a.k_codes);
    fetch_scales();
    fetch(vraw, a.v_codes);
    for (uint64_t cur = u0; cur < u1; ++cur, ++it) {
      const uint32_t b = it & 1u;
      if (cur >= walk.first + walk.steps) next_tile(a, p.share, walk);
      if (cur == walk.first || it == 0) vexp = 0;
      // The place of the step after this one.
      const bool more = cur + 1 < u1;
      if (more) {
        if (++aj == ahead.steps) {
          next_tile(a, p.share, ahead);
          aj = 0;
        }
      }
      if (it > 0) ok = __all_sync(0xffffffffu, wait(&sm->k_empty, it - 1, 203));
      if (!ok) break;
      put(&sm->k[0][0], kraw);
      {
        // Every warp finds the largest exponent of the step's value scales; each writes 16 positions' scales.
        uint32_t e = 0;
#pragma unroll
        for (int n = 0; n < 2; ++n) e = max(e, max((scale_raw[1][n] >> 10) & 31u, (scale_raw[1][n] >> 26) & 31u));
        vexp = max(vexp, min(__reduce_max_sync(0xffffffffu, e), 30u));
        const float up = pow2i(21 - static_cast<int>(vexp));
        const uint32_t half = (warp - 4) / 2;
        if (lane / 16 == (warp & 1u)) {
          const float2 kf = f16x2_f32(scale_raw[0][half]), vf = f16x2_f32(scale_raw[1][half]);
          const uint32_t at = 32u * half + lane;
          sm->ks[b][0][at] = kf.x;
          sm->vs[b][0][at] = vf.x * up;
          if constexpr (G == 2) {
            sm->ks[b][G - 1][at] = kf.y;
            sm->vs[b][G - 1][at] = vf.y * up;
          }
        }
        if (warp == 4 && lane == 0) {
          sm->valid[b][0] = valid_bits[0];
          sm->valid[b][1] = valid_bits[1];
          sm->vexp[b] = vexp;
        }
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm->k_full);
        mbar_arrive(&sm->scales_full[b]);
      }
      if (more) {
        fetch(kraw, a.k_codes);
        fetch_scales();
      }
      if (it > 0) ok = __all_sync(0xffffffffu, wait(&sm->v_empty, it - 1, 204));
      if (!ok) break;
      put(&sm->v[0][0], vraw);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm->v_full);
      if (more) fetch(vraw, a.v_codes);
    }
  } else if (lane == 0) {
    // ---- MMAs ----
    uint32_t it = 0, seg = 0;
    bool waiting = false;  // a commit to o_full is due before this thread may leave
    for (uint64_t cur = u0; cur < u1 && ok; ++seg) {
      const uint32_t j0 = static_cast<uint32_t>(cur - walk.first);
      const uint32_t j1 = static_cast<uint32_t>((u1 < walk.first + walk.steps ? u1 : walk.first + walk.steps) - walk.first);
      ok = wait(&sm->q_full, seg, 205);
      for (uint32_t j = j0; j < j1 && ok; ++j, ++it) {
        ok = wait(&sm->k_full, it, 206);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint64_t kd = umma_desc(smem_addr(sm->k[g]), 16, 1024, kLayoutSw128);
#pragma unroll
          for (int q = 0; q < PARTS; ++q) {
            const uint64_t qd = umma_desc(smem_addr(sm->q[q][g]), 16, 1024, kLayoutSw128);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {  // 16 dims: 32 bytes of each row
              umma_f16_ss(tmem + kTmemScores + g * kStep, qd + 2 * kk, kd + 2 * kk, kIdescScores, q > 0 || kk > 0);
            }
          }
        }
        umma_commit(&sm->k_empty);
        umma_commit(&sm->s_full);
        waiting = true;
        ok = wait(&sm->v_full, it, 207) && wait(&sm->p_full, it, 208);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
          for (int q = 0; q < PARTS; ++q) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {  // 16 positions: 16 rows of 128 bytes
              const uint64_t vd = umma_desc(smem_addr(sm->v[g]) + kk * 2048u, 16, 1024, kLayoutSw128);
              umma_f16_ts(tmem + kTmemOutput + 64 * g, tmem + kTmemScores + 32 * (q * G + g) + 8 * kk, vd, kIdescOutput,
                          j > j0 || q > 0 || kk > 0);
            }
          }
        }
        umma_commit(&sm->v_empty);
      }
      if (ok) {
        umma_commit(&sm->o_full);
        cur = walk.first + j1;
        if (cur < u1) next_tile(a, p.share, walk);
      }
    }
    if (!ok && waiting) {  // MMAs in flight end before tensor memory is freed
      umma_commit(&sm->o_full);
      mbar_wait_bounded(&sm->o_full, seg & 1u, p.error, p.timeout_ns, 209);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T, int DIM>
int32_t launch_tile(const PagedArgs& a, const AttnArgs& p, uint32_t grid, cudaStream_t stream) {
  const size_t smem = sizeof(TileSmem<DIM, sizeof(T) == 4>) + 1024;  // + alignment of the dynamic window
  const cudaError_t e = cudaFuncSetAttribute(paged_attention_tile_kernel<T, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(smem));
  if (e != cudaSuccess) return paged_status(e);
  paged_attention_tile_kernel<T, DIM><<<grid, kTileThreads, smem, stream>>>(a, p);
  return paged_status(cudaGetLastError());
}

}  // namespace

uint32_t paged_tile_grid(const PagedArgs& a, uint32_t heads, uint32_t sms) {
  const uint64_t tiles = (uint64_t(a.max_query) * (heads / a.kv_heads) + kRows - 1) / kRows;
  const uint64_t steps = uint64_t(a.sequences) * a.kv_heads * tiles * (a.max_context ? (a.max_context + kStep - 1) / kStep : 1);
  return static_cast<uint32_t>(steps < 2 * sms ? steps : 2 * sms);
}

uint64_t paged_tile_partial_bytes(const PagedArgs& a, uint32_t grid) {
  return uint64_t(2) * grid * (a.head_dim + 2) * kRows * 4;
}

int32_t paged_tile_launch(const PagedArgs& a, const AttnArgs& p, uint32_t format, uint32_t grid, cudaStream_t stream) {
  if (a.head_dim == 128) {
    return format == kFormatF32   ? launch_tile<float, 128>(a, p, grid, stream)
           : format == kFormatF16 ? launch_tile<__half, 128>(a, p, grid, stream)
                                  : launch_tile<__nv_bfloat16, 128>(a, p, grid, stream);
  }
  return format == kFormatF32   ? launch_tile<float, 64>(a, p, grid, stream)
         : format == kFormatF16 ? launch_tile<__half, 64>(a, p, grid, stream)
                                : launch_tile<__nv_bfloat16, 64>(a, p, grid, stream);
}

}  // namespace qwc
