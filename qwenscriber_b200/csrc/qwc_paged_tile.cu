// qwc_paged_tile.cu -- attention over a paged q8 cache for tokens that give a
// kv head more rows than mma.sync's tiles are worth: 128-row tiles on the
// 5th-generation tensor cores.
//
// A tile is 128 rows of one (sequence, kv head): row i is token i / share,
// query head i % share of the kv head's. A CTA walks one or two tiles (TILES)
// over the positions that their last token sees, 64 at a time:
//
//   softmax  four warps a tile, one row to a thread: scores from tensor
//            memory, the causal limit, the running maximum and sum; the weights
//            go back to tensor memory in place of the scores.
//   convert  the step's code rows, fetched through the page table into registers
//            a step ahead, become f16 in shared memory (128-byte swizzled rows of
//            64 dims); half of these warps take the keys, half the values.
//   MMA      one thread: scores S = Q K^T, output O += P V with the weights
//            read from tensor memory.
//
// How the scales enter depends on the rows' type.
// f32 and f16 rows (exact): the codes are f16 integers. Each group of 64 dims has
// its own scores, which the softmax threads multiply by the key scales, and its
// own weights, the softmax weight times the group's value scale. f32 queries and
// weights enter as two f16 parts, hi and lo (22 bits), f16 rows as one.
// bf16 rows (scaled): code times scale is rounded to f16 as it is converted, at a
// power of two of the step. That adds up to 2^-11 to each factor of a sum that is
// rounded to 2^-9 in the end (4 x 1500 over 4096: 1.71e-3 from 64 bits, the rounding
// alone 1.66e-3), and leaves the softmax threads a third of the work: f16 rows, which
// keep codes exact, take 190 us there and bf16 148. A scale 2^14 below the largest of its
// step (keys) or of the tile so far (values) loses bits.
//
// Each row of queries has its own power of two, so f16 holds its values whatever
// their size; sums, maxima and the output are f32. The output is rescaled only when a
// row's maximum has grown by more than 2^8: until then the old maximum serves,
// and the weights stay below 2^8.
//
// Tensor memory: G x 64 columns of scores and DIM of output for a tile. With one
// tile two CTAs share an SM, with two one CTA has it: either way one tile's
// softmax covers the other's MMAs. Two tiles convert each step once for 256 rows, so
// they are taken where a kv head has more than 128: 4 x 1500 over 4096, bf16, one tile 218 us, two 148;
// 2 x 391 over 2047, f32, one 69, two 66.
//
// What bounds it: the softmax and convert warps' instructions, not the tensor cores. 4 x 1500 over 4096, bf16:
// 148 us, 520 TFLOP/s (f16 190, f32 366); 24 x 64 over 1237, bf16: 50 to 53 us, many tiles with few
// rows (16 to 128) that cost as much as a full one, converting the cache; 2 x 391 over 2047, f32: 68 us,
// four times the scores' instructions of bf16 and four MMAs for one. With 54% of the issue slots and 29% of the tensor
// pipe in use neither is at its limit: much of it is the wait from scores to weights, one step of 64 positions at a time.
//
// Work is dealt as in qwc_paged_attention.cu: the steps of all tiles stand in
// one line, each CTA takes an equal stretch, a tile that is cut is joined by
// the CTA that comes last, in the order of the stretches.

#include <cuda_runtime.h>

#include <cmath>
#include <type_traits>

#include "qwc_device.cuh"
#include "qwc_paged.cuh"
#include "qwc_tcgen05.cuh"

namespace qwc {
namespace {

constexpr uint32_t kRows = 128;   // rows of a tile
constexpr uint32_t kStep = 64;    // positions of a step
constexpr uint32_t kGrowth = 8;   // log2 of how far a maximum may run ahead of the one in use
// What setting up and finishing a tile takes, in steps, when the work is dealt: these places of the line are
// paid for but empty. With 0, 1, 2, 3, 5 and 8 places: 4 x 1500 rows over 4096, bf16, 174, 164, 160, 154, 154 and 155 us;
// 24 x 64 over 1237, bf16, 58, 57.5, 55.5, 56.5 (0 to 3); 2 x 391 over 2047, f32, 69.5, 66, -, 66, 68 and 71 us.
constexpr uint32_t kTileCost = 3;
// What joining one more piece of a cut tile takes, in steps. A stretch is no shorter than the square root of this times
// the longest tile, where a tile's own steps and the joining of its pieces take equally long, unless a tile is shorter.
// With 0, 0.3, 0.8, 2 and 4, bf16: 1 x 64 over 4096 84, 50, 44, 45 and 54 us; over 1237 47, 33, 30, 32, 37; 2 x 64 over 4096
// 61, 54, 44, 46, 54; f32 (steps twice as long): 1 x 100 over 4096 69, 62, 65, 73, 93, 1 x 64 over 1237 52, 38, 40, 46, 54.
constexpr double kJoinCost = 0.8, kJoinCostF32 = 0.4;

template <typename T, int DIM_, int TILES_>
struct TileConfig {
  static constexpr int DIM = DIM_, TILES = TILES_;
  static constexpr bool SPLIT = sizeof(T) == 4;
  static constexpr bool SCALED = std::is_same<T, __nv_bfloat16>::value;
  static constexpr int G = DIM / 64;
  static constexpr int PARTS = SPLIT ? 2 : 1;
  static constexpr int SCORES = SCALED ? 1 : G;              // accumulators of 64 columns
  static constexpr int STAGES = TILES == 2 || !SPLIT ? 2 : 1;  // steps of converted keys and values
  static constexpr int CONVERT_WARPS = 4;                    // for the keys, and as many for the values
  static constexpr int WARPS = 4 * TILES + 2 * CONVERT_WARPS + 1;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr uint32_t SCORE_COLS = SCALED ? 2 * kStep : G * kStep;  // scaled: two steps' scores in turn
  static constexpr uint32_t TMEM_TILE = SCORE_COLS + DIM;    // columns of a tile: scores, output
  static constexpr uint32_t TMEM_COLS = TMEM_TILE * TILES <= 128 ? 128 : TMEM_TILE * TILES <= 256 ? 256 : 512;
  // Registers a thread: at launch what fits (65,536 over the resident warps, by quarters of an SM), then the
  // softmax warps take what the convert warps give back.
  static constexpr int LAUNCH_REGS = TILES == 2 ? 96 : 72;
  static constexpr int SOFTMAX_REGS = TILES == 2 ? 128 : 120;
  static constexpr int CONVERT_REGS = TILES == 2 ? 64 : 48;
  static_assert(4 * TILES * SOFTMAX_REGS + 2 * CONVERT_WARPS * CONVERT_REGS + LAUNCH_REGS <= WARPS * LAUNCH_REGS,
                "a split cannot exceed the launch");
  // The tensor cores cut off what an addition to an f32 sum leaves over, always towards zero: over n additions the
  // output loses about n times 8e-9 of its size (2048 positions in two parts, 256 additions: 2e-6). f32 rows therefore
  // start a new sum every FLUSH steps, and the sums are added in f32 in global memory. Of 2 x 391 rows over 2047
  // positions, f32: a sum over 2 steps 73 us, 4 steps 69, 8 steps 65; the largest error at length 2048 0.48e-6, 0.74e-6
  // and 1.1e-6 of the output, where f32 arithmetic throughout has 0.9e-6.
  static constexpr uint32_t FLUSH = SPLIT ? 4 : 1u << 31;
  // The weights' power of two, 2^(UP - vexp): weight times value scale below 2^15 (exact), value below 2^7 (scaled).
  static constexpr int UP = SCALED ? 14 : 21;
};

template <typename C>
struct __align__(1024) TileSmem {
  uint8_t q[C::TILES][C::PARTS][C::G][kRows * 128];  // f16, 128-byte swizzled rows of 64 dims
  uint8_t k[C::STAGES][C::G][kStep * 128];
  uint8_t v[C::STAGES][C::G][kStep * 128];
  // What the softmax needs to know of a step, for the four steps that may be in hand at once (step n + 4's
  // keys are converted only after step n's weights are made).
  float ks[4][C::G][kStep];  // exact: the key scales
  float vs[4][C::G][kStep];  // and the value scales, times 2^(UP - vexp)
  uint64_t valid[4];         // one bit for each position that is cached
  uint64_t odd[4];           // and for each whose values are no numbers
  uint32_t kexp[4], vexp[4];
  // Scores and weights by the step's parity: with scores a step ahead, a barrier of one phase could pass two
  // phases before a late warp looks.
  uint64_t s_full[2][C::TILES], p_full[2][C::TILES];
  uint64_t q_full[C::TILES], pv_done[C::TILES], o_full[C::TILES];
  uint64_t k_full[C::STAGES], k_empty[C::STAGES], v_full[C::STAGES], v_empty[C::STAGES];
  uint64_t ks_full[4], vs_full[4];
  uint64_t sums[C::WARPS];
  uint64_t found_base;
  uint32_t found_s;
  uint32_t tmem;
};

// A tile of the line (HEIGHT rows: all of a CTA's tiles), and the tiles after it. It takes kTileCost places,
// then one for each step.
struct TileWalk {
  uint32_t s, h, qt;
  uint32_t tiles, steps;  // of the sequence's kv head; of this tile
  int32_t first;          // its first place, counted from the start of the CTA's stretch
  PagedSeq seq;
};

template <uint32_t HEIGHT>
__device__ __forceinline__ uint32_t tiles_of(const PagedSeq& q, const AttnArgs& p) {
  return (q.n * p.share + HEIGHT - 1) / HEIGHT;
}
template <uint32_t HEIGHT>
__device__ __forceinline__ uint32_t tile_steps(const PagedSeq& q, const AttnArgs& p, uint32_t qt) {
  const uint32_t last = min(p.by_share.of(qt * HEIGHT + HEIGHT - 1), q.n - 1);
  const int32_t seen = min(q.base + static_cast<int32_t>(last) + 1, static_cast<int32_t>(q.context));
  return seen > 0 ? (static_cast<uint32_t>(seen) + kStep - 1) / kStep : 1u;
}
template <uint32_t HEIGHT>
__device__ __forceinline__ uint64_t head_places(const PagedSeq& q, const AttnArgs& p) {
  const uint32_t t = tiles_of<HEIGHT>(q, p);
  uint64_t sum = 0;
  for (uint32_t i = 0; i < t; ++i) sum += kTileCost + tile_steps<HEIGHT>(q, p, i);
  return sum;
}

template <uint32_t HEIGHT>
__device__ __forceinline__ void next_tile(const PagedArgs& a, const AttnArgs& p, TileWalk& w) {
  w.first += static_cast<int32_t>(kTileCost + w.steps);
  if (++w.qt == w.tiles) {
    w.qt = 0;
    if (++w.h == a.kv_heads) {
      w.h = 0;
      do {
        w.seq = paged_seq(a, ++w.s);
      } while (w.seq.n == 0 && w.s + 1 < a.sequences);
      w.tiles = tiles_of<HEIGHT>(w.seq, p);
    }
  }
  w.steps = tile_steps<HEIGHT>(w.seq, p, w.qt);
}

// The steps j0 .. j1 - 1 of a tile that a stretch of `len` places holds; false if none.
__device__ __forceinline__ bool piece_of(const TileWalk& w, int32_t len, uint32_t& j0, uint32_t& j1) {
  const int32_t f = w.first + static_cast<int32_t>(kTileCost);
  j0 = static_cast<uint32_t>(max(0, -f));
  j1 = static_cast<uint32_t>(max(0, min(static_cast<int32_t>(w.steps), len - f)));
  return j1 > j0;
}
template <uint32_t HEIGHT>
__device__ __forceinline__ bool next_piece(const PagedArgs& a, const AttnArgs& p, TileWalk& w, int32_t len, uint32_t& j0, uint32_t& j1) {
  do {
    if (w.first + static_cast<int32_t>(kTileCost + w.steps) >= len) return false;
    next_tile<HEIGHT>(a, p, w);
  } while (!piece_of(w, len, j0, j1));
  return true;
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

// The MMAs and commits of a warp whose lanes all come here: one elected lane (always the same one)
// issues. The operands then stay warp-uniform, which the instruction wants.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void fence_proxy_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// D = f32, A and B f16, M = 128, N = 64; B with the dims along its rows (keys)
// or along its columns (values).
constexpr uint32_t kIdescScores = (1u << 4) | ((kStep >> 3) << 17) | ((kRows >> 4) << 24);
constexpr uint32_t kIdescOutput = (1u << 4) | (1u << 16) | ((64u >> 3) << 17) | ((kRows >> 4) << 24);

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 32 columns (16 pairs) of tensor memory, or 16 columns at each of two places.
__device__ __forceinline__ void tmem_ld_pairs(uint32_t t0, uint32_t t1, uint64_t (&x)[8], uint64_t (&y)[8]) {
  float f0[16], f1[16];
  tmem_ld16x2(t0, t1, f0, f1);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = pack2(f0[2 * i], f0[2 * i + 1]);
    y[i] = pack2(f1[2 * i], f1[2 * i + 1]);
  }
}

template <typename T, int DIM, int TILES>
__global__ void __launch_bounds__(TileConfig<T, DIM, TILES>::THREADS, TILES == 1 ? 2 : 1)
    paged_attention_tile_kernel(const PagedArgs a, const AttnArgs p) {
  using C = TileConfig<T, DIM, TILES>;
  constexpr bool SPLIT = C::SPLIT, SCALED = C::SCALED;
  constexpr int G = C::G, PARTS = C::PARTS, STAGES = C::STAGES, WARPS = C::WARPS;
  constexpr uint32_t HEIGHT = kRows * TILES;
  constexpr uint32_t kOutput = C::SCORE_COLS;  // columns of a tile: scores, then output
  constexpr uint32_t CONVERT = 4 * TILES;  // first convert warp
  using Smem = TileSmem<C>;
  extern __shared__ __align__(1024) uint8_t tile_smem_raw[];
  const uint32_t pad = (1024u - (smem_addr(tile_smem_raw) & 1023u)) & 1023u;
  Smem* sm = reinterpret_cast<Smem*>(tile_smem_raw + pad);
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;

  // ---- this CTA's stretch of the line ----
  uint64_t part = 0, mine_steps = 0;  // (of sequence tid: all there is to look up in a batch of fewer sequences than threads)
  for (uint32_t s = tid; s < a.sequences; s += C::THREADS) {
    const uint64_t v = head_places<HEIGHT>(paged_seq(a, s), p) * a.kv_heads;
    if (s == tid) mine_steps = v;
    part += v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if (lane == 0) sm->sums[warp] = part;
  __syncthreads();
  uint64_t total = 0;
  for (int w = 0; w < WARPS; ++w) total += sm->sums[w];
  const uint64_t grid = total < gridDim.x ? total : gridDim.x;
  if (blockIdx.x >= grid) return;
  const uint64_t u0 = total * blockIdx.x / grid, u1 = total * (blockIdx.x + 1) / grid;
  uint64_t running = 0;
  for (uint32_t base = 0; base < a.sequences; base += C::THREADS) {
    const uint32_t s = base + tid;
    const uint64_t v = base == 0 ? mine_steps : s < a.sequences ? head_places<HEIGHT>(paged_seq(a, s), p) * a.kv_heads : 0;
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
    for (uint32_t w = 0; w < WARPS; ++w) {
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
    for (int t = 0; t < TILES; ++t) {
      mbar_init(&sm->q_full[t], 4);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sm->s_full[i][t], 1);
        mbar_init(&sm->p_full[i][t], 4);
      }
      mbar_init(&sm->pv_done[t], 1);
      mbar_init(&sm->o_full[t], 1);
    }
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&sm->k_full[i], C::CONVERT_WARPS);
      mbar_init(&sm->k_empty[i], 1);
      mbar_init(&sm->v_full[i], C::CONVERT_WARPS);
      mbar_init(&sm->v_empty[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sm->ks_full[i], C::CONVERT_WARPS);
      mbar_init(&sm->vs_full[i], C::CONVERT_WARPS);
    }
    fence_mbar_init();
  }
  if (warp == WARPS - 1) tmem_alloc(&sm->tmem, C::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm->tmem;
  TileWalk walk;
  {
    walk.s = sm->found_s;
    walk.seq = paged_seq(a, walk.s);
    walk.tiles = tiles_of<HEIGHT>(walk.seq, p);
    const uint64_t per_head = head_places<HEIGHT>(walk.seq, p);
    uint64_t off = u0 - sm->found_base;
    walk.h = static_cast<uint32_t>(off / per_head);
    off -= walk.h * per_head;
    walk.qt = 0;
    walk.steps = tile_steps<HEIGHT>(walk.seq, p, 0);
    while (off >= kTileCost + walk.steps) {
      off -= kTileCost + walk.steps;
      walk.steps = tile_steps<HEIGHT>(walk.seq, p, ++walk.qt);
    }
    walk.first = -static_cast<int32_t>(off);
  }
  const int32_t len = static_cast<int32_t>(u1 - u0);  // places of the stretch
  uint32_t first_j0, first_j1;
  const bool any = piece_of(walk, len, first_j0, first_j1) || next_piece<HEIGHT>(a, p, walk, len, first_j0, first_j1);
  bool ok = true;
  // Phase n of a barrier, bounded: each try sleeps up to 20 us, so the limit of tries is also one of time. (Few
  // instructions on purpose: there are twenty such waits, and the loops around them have to stay in the
  // instruction cache.)
  auto wait = [&](uint64_t* bar, uint32_t n, int32_t code) {
    uint32_t left = p.wait_tries;
    while (!mbar_try_wait_sleep(bar, n & 1u, 20000u)) {
      if (--left == 0) {
        atomicCAS(p.error, 0, code);
        return false;
      }
    }
    return true;
  };

  if (warp < CONVERT) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
    // ---- softmax: row tid of the CTA's tiles ----
    const uint32_t t = warp / 4, trow = tid % kRows;
    const uint32_t taddr = tmem + ((warp % 4 * 32u) << 16) + t * C::TMEM_TILE;
    uint32_t it = 0, seg = 0;
    uint32_t j0 = first_j0, j1 = first_j1;
    for (bool more_pieces = any; more_pieces && ok; more_pieces = next_piece<HEIGHT>(a, p, walk, len, j0, j1), ++seg) {
      const uint32_t rows = walk.seq.n * p.share;
      const uint32_t row = walk.qt * HEIGHT + tid;
      const bool in = row < rows;
      const uint32_t tok = in ? p.by_share.of(row) : 0u;
      const int32_t limit = in ? walk.seq.base + static_cast<int32_t>(tok) : -1;
      auto row_at = [&](uint32_t rr) -> size_t {  // of a tensor of rows: the token (times a stride) and the head
        return walk.seq.first + p.by_share.of(rr);
      };
      auto head_at = [&](uint32_t rr) { return walk.h * p.share + (rr - p.by_share.of(rr) * p.share); };
      // The warp's 32 rows of queries, eight lanes to a row: the largest value gives the row's power of two,
      // then the f16 parts go to shared memory.
      constexpr int PER = DIM / 8;                      // values of a lane
      constexpr int LOADS = PER / Vec16<T>::kCount;     // 16-byte loads of a lane
      constexpr int AHEAD = 16 / LOADS < 4 ? 16 / LOADS : 4;  // rows of eight lanes in flight
      float factor = 0.0f;
#pragma unroll 1
      for (uint32_t r0 = 0; r0 < 32; r0 += 4 * AHEAD) {
        uint4 raw[AHEAD][LOADS];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const uint32_t rr = row - lane + r0 + 4 * i + lane / 8;  // (row - lane: the warp's first row)
          const T* src = static_cast<const T*>(p.q) + row_at(rr) * p.q_stride + size_t(head_at(rr)) * DIM + PER * (lane % 8);
#pragma unroll
          for (int e = 0; e < LOADS; ++e) {
            raw[i][e] = rr < rows ? reinterpret_cast<const uint4*>(src)[e] : make_uint4(0, 0, 0, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          float x[LOADS][Vec16<T>::kCount];
          float top = 0.0f;
#pragma unroll
          for (int e = 0; e < LOADS; ++e) {
            unpack16(raw[i][e], x[e], T());
#pragma unroll
            for (int k = 0; k < Vec16<T>::kCount; ++k) top = fmaxf(top, fabsf(x[e][k]));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          const int e2 = row_exponent(top);
          const float down = pow2i(-e2);
          // The thread that owns the row takes its factor.
          const float f = __shfl_sync(0xffffffffu, p.scaling * 1.4426950408889634f * pow2i(e2), (lane % 4) * 8);
          if (lane / 4 == r0 / 4 + i) factor = f;
          const uint32_t r = trow - lane + r0 + 4 * i + lane / 8, d = PER * (lane % 8);
          uint8_t* dst = &sm->q[t][0][d / 64][r * 128u];
          uint8_t* dst_lo = &sm->q[t][PARTS - 1][d / 64][r * 128u];
#pragma unroll
          for (int e = 0; e < PER; e += 8) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float a0 = (&x[0][0])[e + 2 * k], a1 = (&x[0][0])[e + 2 * k + 1];
              const float y0 = fmaf(a0, down, a0 - a0), y1 = fmaf(a1, down, a1 - a1);  // an infinity is NaN from here on
              hi[k] = f16x2(y0, y1);
              const float2 h = f16x2_f32(hi[k]);
              lo[k] = f16x2(y0 - h.x, y1 - h.y);
            }
            const uint32_t at = (((d % 64 + e) / 8) ^ (r & 7u)) << 4;
            *reinterpret_cast<uint4*>(dst + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (SPLIT) *reinterpret_cast<uint4*>(dst_lo + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
        }
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm->q_full[t]);

      // Maxima and sums are those of scores in powers of two.
      float m = -INFINITY, l = 0.0f;
      uint32_t vexp = 0;
      // f32: the sums so far, in units of the maximum flushed_m: [DIM / 4][HEIGHT] of four dims.
      float4* const flushed = reinterpret_cast<float4*>(p.partials + (size_t(2) * gridDim.x * (DIM + 2) + size_t(blockIdx.x) * DIM) * HEIGHT);
      float flushed_m = -INFINITY;
      bool any_flushed = false;
      for (uint32_t j = j0; j < j1; ++j, ++it) {
        const uint32_t b = it & 3u;
        if (SPLIT && j > j0 && (j - j0) % C::FLUSH == 0) {
          ok = __all_sync(0xffffffffu, wait(&sm->pv_done[t], it - 1, 213));
          if (!ok) break;
          tc_fence_after();
          // (m == -inf: this row has seen nothing, and its columns are sums of zeros.)
          const float old = any_flushed && flushed_m != -INFINITY ? ex2(flushed_m - m) : 0.0f;
          const float unit = pow2i(static_cast<int>(vexp) - (C::UP + 1));
#pragma unroll 1
          for (int i = 0; i < DIM; i += 32) {
            float4 f[8];
            if (any_flushed) {
#pragma unroll
              for (int e = 0; e < 8; ++e) f[e] = flushed[size_t(i / 4 + e) * HEIGHT + tid];
            }
            float o[32];
            tmem_ld32(taddr + kOutput + i, o);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (!any_flushed) f[e] = make_float4(0, 0, 0, 0);
              flushed[size_t(i / 4 + e) * HEIGHT + tid] =
                  make_float4(fmaf(f[e].x, old, o[4 * e] * unit), fmaf(f[e].y, old, o[4 * e + 1] * unit),
                              fmaf(f[e].z, old, o[4 * e + 2] * unit), fmaf(f[e].w, old, o[4 * e + 3] * unit));
            }
          }
          tc_fence_before();
          flushed_m = m;
          any_flushed = true;
        }
        ok = __all_sync(0xffffffffu, wait(&sm->ks_full[b], it >> 2, 210) && wait(&sm->s_full[it & 1u][t], it >> 1, 201) &&
                                            wait(&sm->vs_full[b], it >> 2, 211));
        if (!ok) break;
        tc_fence_after();
        const uint32_t scol = taddr + (SCALED ? (it & 1u) * kStep : 0u);
        uint64_t seen = sm->valid[b];
        const uint32_t top = sm->vexp[b];
        const float step_factor = SCALED ? factor * pow2i(static_cast<int>(sm->kexp[b]) - 15) : factor;
        uint64_t x[kStep / 2];
#pragma unroll
        for (int i = 0; i < static_cast<int>(kStep); i += 32 / C::SCORES) {
          // Both groups' sums of 16 positions, or the one sum of 32.
          uint64_t s0[8], s1[8];
          tmem_ld_pairs(scol + i, scol + i + (C::SCORES == 2 ? kStep : 16u), s0, s1);
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            if constexpr (SCALED) {
              x[i / 2 + e] = s0[e], x[i / 2 + e + 1] = s0[e + 1];
              x[i / 2 + 8 + e] = s1[e], x[i / 2 + 8 + e + 1] = s1[e + 1];
            } else {
              const ulonglong2 k0 = *reinterpret_cast<const ulonglong2*>(&sm->ks[b][0][i + 2 * e]);
              const ulonglong2 k1 = *reinterpret_cast<const ulonglong2*>(G == 2 ? &sm->ks[b][G - 1][i + 2 * e] : &sm->ks[b][0][i + 16 + 2 * e]);
              if constexpr (G == 2) {
                x[i / 2 + e] = fma2(s1[e], k1.x, mul2(s0[e], k0.x));
                x[i / 2 + e + 1] = fma2(s1[e + 1], k1.y, mul2(s0[e + 1], k0.y));
              } else {
                x[i / 2 + e] = mul2(s0[e], k0.x), x[i / 2 + e + 1] = mul2(s0[e + 1], k0.y);
                x[i / 2 + 8 + e] = mul2(s1[e], k1.x), x[i / 2 + 8 + e + 1] = mul2(s1[e + 1], k1.y);
              }
            }
          }
        }
        const int32_t pos0 = static_cast<int32_t>(j * kStep);
        if (pos0 + static_cast<int32_t>(kStep) - 1 > limit) seen &= limit < pos0 ? 0ull : (2ull << (limit - pos0)) - 1;
        if (seen != ~0ull) {
#pragma unroll
          for (int i = 0; i < static_cast<int>(kStep); i += 2) {
            const uint32_t bits = static_cast<uint32_t>(i < 32 ? seen : seen >> 32);
            const float2 f = unpack2(x[i / 2]);
            x[i / 2] = pack2((bits & (1u << (i % 32))) ? f.x : -INFINITY, (bits & (2u << (i % 32))) ? f.y : -INFINITY);
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < static_cast<int>(kStep) / 2; ++i) {
          const float2 f = unpack2(x[i]);
          mx4[i % 4] = fmaxf(fmaxf(mx4[i % 4], f.x), f.y);
        }
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * step_factor;
        float rescale = 1.0f;
        bool grew = false;
        if (mx - m > static_cast<float>(kGrowth) || (m == -INFINITY && mx > m)) {
          rescale = m == -INFINITY ? 0.0f : ex2(m - mx);
          l *= rescale;
          m = mx;
          grew = true;
        }
        if (top > vexp) {
          rescale *= pow2i(static_cast<int>(vexp) - static_cast<int>(top));
          vexp = top;
          grew = true;
        }
        const bool fresh = (j - j0) % C::FLUSH == 0;  // nothing in the output's columns
        if (!fresh && __any_sync(0xffffffffu, grew)) {
          // The last step's output must be complete. (The one before it is: its MMAs came before this step's scores.)
          ok = __all_sync(0xffffffffu, wait(&sm->pv_done[t], it - 1, 212));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int i = 0; i < DIM; i += 32) {
            float o0[16], o1[16];
            tmem_ld16x2(taddr + kOutput + i, taddr + kOutput + i + 16, o0, o1);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              o0[e] *= rescale;
              o1[e] *= rescale;
            }
            tmem_st16f(taddr + kOutput + i, o0);
            tmem_st16f(taddr + kOutput + i + 16, o1);
          }
        }
        const float base = m == -INFINITY ? 0.0f : -m;
        const uint64_t f2 = pack2(step_factor, step_factor), b2 = pack2(base, base);
        uint64_t l0 = 0, l1 = 0;
#pragma unroll
        for (int i = 0; i < static_cast<int>(kStep) / 2; i += 2) {
          const float2 e0 = unpack2(fma2(x[i], f2, b2)), e1 = unpack2(fma2(x[i + 1], f2, b2));
          x[i] = pack2(ex2(e0.x), ex2(e0.y));
          x[i + 1] = pack2(ex2(e1.x), ex2(e1.y));
          l0 = add2(l0, x[i]);
          l1 = add2(l1, x[i + 1]);
        }
        const float2 lf = unpack2(add2(l0, l1));
        l += lf.x + lf.y;
        // Weights over the scores' columns: part q of group g at columns 32 (q G + g).
#pragma unroll
        for (int g = 0; g < C::SCORES; ++g) {
#pragma unroll
          for (int i = 0; i < static_cast<int>(kStep); i += 32) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              uint64_t w0 = x[(i + e) / 2], w1 = x[(i + e) / 2 + 1];
              if constexpr (!SCALED) {
                const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(&sm->vs[b][g][i + e]);
                w0 = mul2(w0, f.x);
                w1 = mul2(w1, f.y);
              }
              const float2 a0 = unpack2(w0), a1 = unpack2(w1);
              hi[e / 2] = f16x2(a0.x, a0.y);
              hi[e / 2 + 1] = f16x2(a1.x, a1.y);
              if constexpr (SPLIT) {
                const float2 r0 = f16x2_f32(hi[e / 2]), r1 = f16x2_f32(hi[e / 2 + 1]);
                lo[e / 2] = f16x2(a0.x - r0.x, a0.y - r0.y);
                lo[e / 2 + 1] = f16x2(a1.x - r1.x, a1.y - r1.y);
              }
            }
            tmem_st16(scol + 32 * g + i / 2, hi);
            if constexpr (SPLIT) tmem_st16(scol + 32 * (G + g) + i / 2, lo);
          }
        }
        if (const uint64_t odd = sm->odd[b]) {  // (looked at here, where few registers are in use: 6 us of 190 beside the mask)
          const uint64_t sees = limit < pos0 ? 0ull : limit - pos0 > 62 ? ~0ull : (2ull << (limit - pos0)) - 1;
          if (odd & sees) l = __int_as_float(0x7FC00000);  // and so is all that it divides
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm->p_full[it & 1u][t]);
      }
      if (!ok) break;

      // ---- the tile's output, or this stretch's part of it ----
      ok = __all_sync(0xffffffffu, wait(&sm->o_full[t], seg, 202));
      if (!ok) break;
      tc_fence_after();
      const float back = pow2i(static_cast<int>(vexp) - (C::UP + 1));
      const bool whole = j0 == 0 && j1 == walk.steps;
      // Finished rows go through shared memory (the tile's queries are done with) and leave a row at a time.
      constexpr int W = Vec16<T>::kCount;
      constexpr int ROW_CHUNKS = DIM / W;
      uint8_t* const stage = &sm->q[t][0][0][0];
      static_assert(sizeof(sm->q[0]) == size_t(kRows) * DIM * sizeof(T), "the queries' room holds the tile's output");
      auto put_row = [&](int i, const float (&o)[32]) {
#pragma unroll
        for (int e = 0; e < 32; e += W) {
          float y[W];
#pragma unroll
          for (int q = 0; q < W; ++q) y[q] = o[e + q];
          const uint32_t chunk = (i + e) / W;
          *reinterpret_cast<uint4*>(stage + (chunk / 8) * (kRows * 128) + trow * 128u + (((chunk % 8) ^ (trow & 7u)) << 4)) = pack16<T>(y);
        }
      };
      auto write_rows = [&]() {
        __syncwarp();
        constexpr uint32_t AT_ONCE = 32 / ROW_CHUNKS;  // rows of an instruction
#pragma unroll 4
        for (uint32_t r0 = 0; r0 < 32; r0 += AT_ONCE) {
          const uint32_t r = r0 + lane / ROW_CHUNKS, chunk = lane % ROW_CHUNKS;
          const uint32_t rr = row - lane + r, tr = trow - lane + r;
          const uint4 v = *reinterpret_cast<const uint4*>(stage + (chunk / 8) * (kRows * 128) + tr * 128u + (((chunk % 8) ^ (tr & 7u)) << 4));
          if (rr < rows) {
            *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row_at(rr) * p.out_stride + size_t(head_at(rr)) * DIM + W * chunk) = v;
          }
        }
        __syncwarp();
      };
      // 32 dims of the row's sum, in true units.
      const float old = any_flushed && flushed_m != -INFINITY ? ex2(flushed_m - m) : 0.0f;
      auto row_sum = [&](int i, float (&o)[32]) {
        tmem_ld32(taddr + kOutput + i, o);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = l == 0.0f ? 0.0f : o[e] * back;  // (nothing seen: the columns may hold anything)
        if (SPLIT && any_flushed) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 f = flushed[size_t((i + e) / 4) * HEIGHT + tid];
            o[e] = fmaf(f.x, old, o[e]), o[e + 1] = fmaf(f.y, old, o[e + 1]);
            o[e + 2] = fmaf(f.z, old, o[e + 2]), o[e + 3] = fmaf(f.w, old, o[e + 3]);
          }
        }
      };
      if (whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
        for (int i = 0; i < DIM; i += 32) {
          float o[32];
          row_sum(i, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= inv;
          put_row(i, o);
        }
        write_rows();
      } else {
        // A partial: [DIM / 4][HEIGHT] of four dims, then maxima and sums. In the slots of stretch x: 2 x for the tile
        // that the stretch begins with, 2 x + 1 for the one that it ends with.
        auto slot = [&](uint32_t i) { return p.partials + size_t(i) * (DIM + 2) * HEIGHT; };
        const uint64_t seg0 = u0 + static_cast<int64_t>(walk.first) + kTileCost, seg1 = seg0 + walk.steps;
        // The stretches that hold this tile: c0 .. c1 (stretch x starts at floor(x * total / grid)). Each warp joins its
        // 32 rows by itself. One that finds all others done has no need to write its own part.
        const uint32_t c0 = static_cast<uint32_t>(((seg0 + 1) * grid - 1) / total);
        const uint32_t c1 = static_cast<uint32_t>((seg1 * grid - 1) / total);
        uint32_t* counter = &p.counters[kAttnCounterStride * c0 + warp];
        bool last = __shfl_sync(0xffffffffu, lane == 0 ? ld_acquire(counter) : 0u, 0) == c1 - c0;
        if (!last) {
          float* mine = slot(2 * blockIdx.x + (walk.first + static_cast<int32_t>(kTileCost) > 0 ? 1u : 0u));
#pragma unroll 1
          for (int i = 0; i < DIM; i += 32) {
            float o[32];
            row_sum(i, o);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              reinterpret_cast<float4*>(mine)[size_t((i + e) / 4) * HEIGHT + tid] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
          mine[size_t(DIM) * HEIGHT + tid] = m;
          mine[size_t(DIM + 1) * HEIGHT + tid] = l;
          __threadfence();
          __syncwarp();
          last = __shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(counter, 1u) : 0u, 0) == c1 - c0;
        }
        if (last) {
          if (lane == 0) *counter = 0;
          __threadfence();
          __syncwarp();  // what lane 0 has acquired, the others may read
          const float* first = slot(2 * c0 + (seg0 > total * c0 / grid ? 1u : 0u));
          auto piece = [&](uint32_t x) -> const float* { return x == c0 ? first : slot(2 * x); };
          constexpr uint32_t kMax = DIM * HEIGHT, kSum = (DIM + 1) * HEIGHT;
          // The pieces in order, this one's own from where it is: maxima, then the sum of the sums.
          float best = m, sum = 0.0f;
#pragma unroll 4
          for (uint32_t x = c0; x <= c1; ++x) {
            if (x != blockIdx.x) best = fmaxf(best, __ldcg(piece(x) + kMax + tid));
          }
          auto share_of = [&](float pm) { return best == -INFINITY ? 1.0f : ex2(pm - best); };
#pragma unroll 4
          for (uint32_t x = c0; x <= c1; ++x) {
            const float pl = x == blockIdx.x ? l : __ldcg(piece(x) + kSum + tid);
            const float pm = x == blockIdx.x ? m : __ldcg(piece(x) + kMax + tid);
            sum = fmaf(pl, share_of(pm), sum);
          }
          const float norm = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll 1
          for (int i = 0; i < DIM; i += 32) {
            float o[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.0f;
#pragma unroll 1
            for (uint32_t x = c0; x <= c1; ++x) {
              float v[32];
              float pm = m;
              if (x == blockIdx.x) {
                row_sum(i, v);
              } else {
                const float* from = piece(x);
                pm = __ldcg(from + kMax + tid);
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                  const float4 f = __ldcg(reinterpret_cast<const float4*>(from) + size_t((i + e) / 4) * HEIGHT + tid);
                  v[e] = f.x, v[e + 1] = f.y, v[e + 2] = f.z, v[e + 3] = f.w;
                }
              }
              const float k = share_of(pm) * norm;
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = fmaf(v[e], k, o[e]);
            }
            put_row(i, o);
          }
          write_rows();
        }
      }
      tc_fence_before();  // the output's columns may be written again once the next weights arrive
    }
  } else if (warp < WARPS - 1) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::CONVERT_REGS));
    // ---- convert: half of these warps the keys of each step, half the values ----
    auto convert = [&](auto is_v) {
      constexpr bool VALUES = decltype(is_v)::value;
      constexpr uint32_t CW = C::CONVERT_WARPS;
      const uint32_t cw = (warp - CONVERT) % CW, ct = cw * 32 + lane;
      constexpr uint32_t CH = DIM / 16;              // 16-byte chunks of a row of codes
      constexpr uint32_t ROWS_PASS = 32 * CW / CH;   // rows that the warps fetch at once
      constexpr uint32_t PASSES = kStep / ROWS_PASS;
      const uint32_t ch = ct % CH, r0 = ct / CH;
      const uint8_t* code_plane = VALUES ? a.v_codes : a.k_codes;
      const uint8_t* scale_plane = VALUES ? a.v_scales : a.k_scales;
      uint64_t* full = VALUES ? sm->v_full : sm->k_full;
      uint64_t* empty = VALUES ? sm->v_empty : sm->k_empty;
      uint8_t* tiles = VALUES ? &sm->v[0][0][0] : &sm->k[0][0][0];
      // A step ahead: its code chunks and its scales.
      uint4 raw[PASSES];
      TileWalk ahead = walk;
      uint32_t aj = first_j0, aj1 = first_j1;
      // Rows of the pool of that step's positions 32 e + lane (-1: not cached): the page table is read
      // before the step in hand is converted, its answers are used after.
      int32_t page_id[2], page_at[2], rows[2];
      auto look_up = [&]() {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t pos = aj * kStep + 32u * e + lane;
          const uint32_t pg = page_of(a, pos);
          page_at[e] = static_cast<int32_t>(pos - pg * a.page_size);
          page_id[e] = pos < ahead.seq.context ? __ldg(a.page_table + size_t(ahead.s) * a.table_stride + pg) : -1;
        }
      };
      uint32_t scale_raw[2];  // position 32 e + lane: both groups
      uint32_t valid_bits[2];
      auto fetch = [&]() {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          rows[e] = static_cast<uint32_t>(page_id[e]) < a.pages ? page_id[e] * static_cast<int32_t>(a.page_size) + page_at[e] : -1;
        }
        const uint8_t* from = code_plane + ahead.h * DIM + 16u * ch;
#pragma unroll
        for (uint32_t i = 0; i < PASSES; ++i) {
          const int32_t row = __shfl_sync(0xffffffffu, rows[i * ROWS_PASS / 32], (r0 + i * ROWS_PASS) % 32);
          raw[i] = row >= 0 ? ld_nc4(from + uint64_t(static_cast<uint32_t>(row)) * a.code_row) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          valid_bits[e] = __ballot_sync(0xffffffffu, rows[e] >= 0);
          scale_raw[e] = 0;
          if (rows[e] >= 0) {
            const uint8_t* at = scale_plane + uint64_t(static_cast<uint32_t>(rows[e])) * a.scale_row + ahead.h * (2 * G);
            scale_raw[e] = G == 2 ? *reinterpret_cast<const uint32_t*>(at) : *reinterpret_cast<const uint16_t*>(at);
          }
        }
      };
      bool have = any;
      if (have) {
        look_up();
        fetch();
      }
      uint32_t top = 0;  // values: the largest exponent field of a scale of the tile so far; keys: of the step
      uint32_t it = 0;
      for (; have; ++it) {
        const uint32_t b = it & 3u, st = it % STAGES, use = it / STAGES;
        if (!VALUES || aj == 0) top = 0;  // (aj: still the step in hand)
        // The place of the step after this one.
        if (++aj == aj1) have = next_piece<HEIGHT>(a, p, ahead, len, aj, aj1);
        if (have) look_up();
        if (it >= STAGES) ok = __all_sync(0xffffffffu, wait(&empty[st], use - 1, VALUES ? 204 : 203));
        if (!ok) break;
        // Every warp finds the largest exponent for itself.
        int up = 0;
        uint32_t odd[2] = {0, 0};
        if (VALUES || SCALED) {
          // (One more: the fields that kOddStep gives.)
          uint32_t e = 0;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint32_t f = scale_raw[n] + kOddStep;
            if (VALUES) odd[n] = __ballot_sync(0xffffffffu, f & kOddBits);
            e = max(e, max((f >> 10) & 31u, (f >> 26) & 31u));
          }
          top = max(top, __reduce_max_sync(0xffffffffu, e));
          up = (VALUES ? C::UP : 14) + 1 - static_cast<int>(top);
        }
        const float up2 = pow2i(up);
        // Chunk ch is dims 16 ch .. + 15: two 16-byte chunks of f16 in group ch / 4's tile.
        uint8_t* base = tiles + (st * G + ch / 4) * (kStep * 128);
        const uint32_t c2 = 2 * (ch % 4), flip = ch / 4;  // the two groups' lanes on different banks
#pragma unroll
        for (uint32_t i = 0; i < PASSES; ++i) {
          const uint32_t r = r0 + i * ROWS_PASS;
          const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            h[2 * e] = codes_f16x2<0x4140>(w[e]);
            h[2 * e + 1] = codes_f16x2<0x4342>(w[e]);
          }
          if constexpr (SCALED) {
            const uint32_t both = __shfl_sync(0xffffffffu, scale_raw[i * ROWS_PASS / 32], r % 32);
            float f = f16_bits_to_f32(ch >= 4 ? both >> 16 : both & 0xFFFFu) * up2;
            if (VALUES) f = fminf(f, 1.0f);  // (more is no number)
            const uint32_t f2 = f16x2(f, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(h[e]) : "r"(f2));
          }
          const uint4 o0 = make_uint4(h[0], h[1], h[2], h[3]), o1 = make_uint4(h[4], h[5], h[6], h[7]);
          *reinterpret_cast<uint4*>(base + r * 128u + (((c2 + flip) ^ (r & 7u)) << 4)) = flip ? o1 : o0;
          *reinterpret_cast<uint4*>(base + r * 128u + (((c2 + 1 - flip) ^ (r & 7u)) << 4)) = flip ? o0 : o1;
        }
        if constexpr (!SCALED) {
          // Each warp writes its share of the positions' scales.
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t pos = 32u * e + lane;
            if (pos / (kStep / CW) != cw) continue;
            const float2 f = f16x2_f32(scale_raw[e]);
            float* dst = VALUES ? &sm->vs[b][0][pos] : &sm->ks[b][0][pos];
            // (Values' are below 128; more is no number.)
            dst[0] = VALUES ? fminf(f.x * up2, 128.0f) : f.x * up2;
            if constexpr (G == 2) dst[kStep] = VALUES ? fminf(f.y * up2, 128.0f) : f.y * up2;
          }
        }
        if (cw == 0 && lane == 0) {
          if constexpr (VALUES) {
            sm->odd[b] = odd[0] | uint64_t(odd[1]) << 32;
            sm->vexp[b] = top;
          } else {
            sm->valid[b] = valid_bits[0] | uint64_t(valid_bits[1]) << 32;
            sm->kexp[b] = top;
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&full[st]);
          mbar_arrive(VALUES ? &sm->vs_full[b] : &sm->ks_full[b]);
        }
        if (have) fetch();
      }
    };
    if (warp < CONVERT + C::CONVERT_WARPS) {
      convert(std::false_type());
    } else {
      convert(std::true_type());
    }
  } else {
    // ---- MMAs: the whole warp walks, one lane issues ----
    uint32_t it = 0, seg = 0;
    bool waiting = false;  // MMAs may be in flight
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t q0 = umma_desc(smem_addr(sm->q[0][0][0]), 16, 1024, kLayoutSw128);
    const uint64_t k0 = umma_desc(smem_addr(sm->k[0][0]), 16, 1024, kLayoutSw128);
    const uint64_t v0 = umma_desc(smem_addr(sm->v[0][0]), 16, 1024, kLayoutSw128);
    constexpr uint32_t kQTile = kRows * 128 / 16, kKvTile = kStep * 128 / 16;  // in a descriptor's units
    auto wait_all = [&](uint64_t* bar, uint32_t n, int32_t code) { return __all_sync(0xffffffffu, wait(bar, n, code)) != 0; };
    auto scores = [&](uint32_t t, uint32_t n) {  // of step n
      const uint32_t st = n % STAGES;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint64_t kd = k0 + (st * G + g) * kKvTile;
#pragma unroll
        for (int q = PARTS - 1; q >= 0; --q) {  // lo before hi: while the sum is small, so is what an addition rounds off
          const uint64_t qd = q0 + ((t * PARTS + q) * G + g) * kQTile;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {  // 16 dims: 32 bytes of each row
            mma_ss(base + t * C::TMEM_TILE + (SCALED ? (n & 1u) * kStep : g * kStep), qd + 2 * kk, kd + 2 * kk, kIdescScores,
                   (SCALED && g > 0) || q < PARTS - 1 || kk > 0);
          }
        }
      }
    };
    auto output = [&](uint32_t t, uint32_t n, bool first) {
      const uint32_t st = n % STAGES;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint64_t vd = v0 + (st * G + g) * kKvTile;
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {  // 16 positions: 16 rows of 128 bytes
            mma_ts(base + t * C::TMEM_TILE + kOutput + 64 * g,
                   base + t * C::TMEM_TILE + (SCALED ? (n & 1u) * kStep : 32 * (q * G + g)) + 8 * kk, vd + 128 * kk, kIdescOutput,
                   !first || q > 0 || kk > 0);
          }
        }
      }
    };
    uint32_t j0 = first_j0, j1 = first_j1;
    for (bool more_pieces = any; more_pieces && ok; more_pieces = next_piece<HEIGHT>(a, p, walk, len, j0, j1), ++seg) {
      for (int t = 0; t < TILES && ok; ++t) ok = wait_all(&sm->q_full[t], seg, 205);
      // Exact: step n's scores are issued behind step n - 1's output, tile by tile, as the weights lie in the
      // scores' columns. Scaled: they have columns of their own, and are issued before step n - 1's
      // weights are made. MMAs of one thread run in order.
      auto issue_scores = [&](uint32_t t, uint32_t n) {
        tc_fence_after();
        scores(t, n);
        mma_commit(&sm->s_full[n & 1u][t]);
        waiting = true;
        if (t == TILES - 1) mma_commit(&sm->k_empty[n % STAGES]);
      };
      ok = ok && wait_all(&sm->k_full[it % STAGES], it / STAGES, 206);
      for (int t = 0; t < TILES && ok; ++t) issue_scores(t, it);
      for (uint32_t j = j0; j < j1 && ok; ++j, ++it) {
        const bool more = j + 1 < j1;
        if (more) ok = wait_all(&sm->k_full[(it + 1) % STAGES], (it + 1) / STAGES, 206);
        if (SCALED && more && ok) {
          for (int t = 0; t < TILES; ++t) issue_scores(t, it + 1);
        }
        if (ok) ok = wait_all(&sm->v_full[it % STAGES], it / STAGES, 207);
        for (int t = 0; t < TILES && ok; ++t) {
          ok = wait_all(&sm->p_full[it & 1u][t], it >> 1, 208);
          if (!ok) break;
          tc_fence_after();
          output(t, it, (j - j0) % C::FLUSH == 0);
          mma_commit(&sm->pv_done[t]);
          if (!more) mma_commit(&sm->o_full[t]);
          if (t == TILES - 1) mma_commit(&sm->v_empty[it % STAGES]);
          if (!SCALED && more) issue_scores(t, it + 1);
        }
      }
    }
    if (!ok && waiting) {  // MMAs in flight end before tensor memory is freed
      mma_commit(&sm->o_full[0]);
      wait(&sm->o_full[0], seg, 209);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == WARPS - 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

template <typename T, int DIM, int TILES>
int32_t launch_tile(const PagedArgs& a, const AttnArgs& p, uint32_t grid, cudaStream_t stream) {
  using C = TileConfig<T, DIM, TILES>;
  const size_t smem = sizeof(TileSmem<C>) + 1024;  // + alignment of the dynamic window
  const cudaError_t e = cudaFuncSetAttribute(paged_attention_tile_kernel<T, DIM, TILES>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return paged_status(e);
  paged_attention_tile_kernel<T, DIM, TILES><<<grid, C::THREADS, smem, stream>>>(a, p);
  return paged_status(cudaGetLastError());
}

template <typename T>
int32_t launch_tile_as(const PagedArgs& a, const AttnArgs& p, const TilePlan& plan, cudaStream_t stream) {
  if (a.head_dim == 128) {
    return plan.tiles == 2 ? launch_tile<T, 128, 2>(a, p, plan.grid, stream) : launch_tile<T, 128, 1>(a, p, plan.grid, stream);
  }
  return plan.tiles == 2 ? launch_tile<T, 64, 2>(a, p, plan.grid, stream) : launch_tile<T, 64, 1>(a, p, plan.grid, stream);
}

}  // namespace

TilePlan paged_tile_plan(const PagedArgs& a, uint32_t format, uint32_t heads, uint32_t sms) {
  TilePlan plan;
  const uint64_t rows = uint64_t(a.max_query) * (heads / a.kv_heads);
  plan.tiles = rows > kRows ? 2 : 1;
  const uint64_t height = uint64_t(kRows) * plan.tiles;
  const uint64_t most = plan.tiles == 2 ? sms : 2 * sms;  // what is resident at once
  const uint64_t length = (a.max_context ? (a.max_context + kStep - 1) / kStep : 1);
  const uint64_t tiles = uint64_t(a.sequences) * a.kv_heads * ((rows + height - 1) / height), steps = tiles * length;
  const double join = format == kFormatF32 ? kJoinCostF32 : kJoinCost;
  const double stretch = sqrt(1.0 + join * static_cast<double>(length));
  uint64_t grid = static_cast<uint64_t>(static_cast<double>(steps) / stretch);
  if (grid < tiles) grid = tiles;
  plan.grid = static_cast<uint32_t>(grid < most ? grid : most);
  plan.too_long = plan.grid && tiles * (length + kTileCost) / plan.grid >= 0x7FFFFFFFu;  // a stretch's places are counted in 31 bits
  // Two partial tiles a CTA, and its sums (f32 rows).
  plan.partial_bytes = uint64_t(plan.grid) * (2 * (a.head_dim + 2) + a.head_dim) * height * 4;
  return plan;
}

int32_t paged_tile_launch(const PagedArgs& a, const AttnArgs& p, uint32_t format, const TilePlan& plan, cudaStream_t stream) {
  return format == kFormatF32   ? launch_tile_as<float>(a, p, plan, stream)
         : format == kFormatF16 ? launch_tile_as<__half>(a, p, plan, stream)
                                : launch_tile_as<__nv_bfloat16>(a, p, plan, stream);
}

}  // namespace qwc
