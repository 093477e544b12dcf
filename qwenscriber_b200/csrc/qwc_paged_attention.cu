// qwc_paged_attention.cu -- causal attention of a step's tokens over a paged
// q8 key/value cache.

#include <cuda_runtime.h>

#include <type_traits>

#include "qwc_device.cuh"
#include "qwc_paged.cuh"

namespace qwc {
namespace {

// ---- few query rows ----
//
// A sequence whose tokens give at most kRows rows to a kv head (a row is one
// token's query head) is bound by its cache: every code byte is read once and
// used by a handful of rows. The products run on mma.sync m16n8k16 (f16
// operands, f32 sums), whose rate is ample here; tcgen05's 128-row tiles
// would be nearly empty.
//
// Work is dealt evenly whatever the lengths: the steps of all (sequence, group
// of kv heads) pairs, 16 * PB positions each, stand in one line and each CTA
// takes an equal stretch of it. In a step warp (pb, h) takes head h's 16
// positions number pb. A (sequence, group) that lies in one stretch is finished there; one that is
// cut leaves a partial result (maximum, sum, unnormalised output) for each stretch, and the CTA that
// comes last adds them up in the order of the stretches, so the result does
// not depend on who was last.
//
// Scores: A rows are 16 positions, the codes as exact f16 integers; B columns are query rows, an f32
// row as two columns (its f16 parts hi and lo, 22 bits), a 16-bit row as one, so NCT column tiles of 8
// hold 4 NCT or 8 NCT rows. Each group of 64 dims has its own sum, which the key scale multiplies. Values:
// A rows are 16 dims, the codes transposed between registers, B the weights times the value scale of
// the group, again in one or two f16 parts; movmatrix turns the score layout
// into that operand. The weights carry a factor 2^(28 - e) with e the largest exponent field of a value
// scale so far, which keeps them in f16's normal range whatever the scales.
//
// Both products have the cache on the 16-row side: with the query rows there instead, twice as many
// MMAs and twice the output registers were spent on mostly empty rows (64 x 1 over 4096, f32: 95 us).
//
// 64 x 1 over up to 4096 (361 MB of cache), f32: 73 us, 4.9 TB/s; the copies and the conversions of codes share the
// issue slots (66% taken), and two CTAs of eight warps leave them partly idle behind the chain of a block: scores,
// maximum, exponential, transpose. 1 x 1 over 301: 9.7 us, of which the launch and the chain of dependent loads
// (lengths, page table, codes, the joined pieces) are nearly all.

constexpr int kFewWarps = 8;
constexpr int kFewThreads = 32 * kFewWarps;
constexpr int kFewBlock = 16;   // positions a warp takes at a time
constexpr int kFewStages = 2;   // blocks of codes in a warp's ring

template <int DIM>
struct FewTile {
  uint8_t k[kFewBlock][DIM];
  uint8_t v[kFewBlock][DIM];
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The transpose of an 8 x 8 matrix of f16 held two to a lane (row lane / 4, columns 2 (lane % 4) + 0, 1).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename T, int DIM, int NCT>
__global__ void __launch_bounds__(kFewThreads, 2) paged_attention_few_kernel(const PagedArgs a, const AttnArgs p) {
  constexpr bool SPLIT = sizeof(T) == 4;  // f32 rows enter as two f16 parts
  constexpr int G = DIM / 64;             // scale groups of a head
  constexpr int CHUNKS = DIM / 16;        // 16-byte chunks of a row of codes
  constexpr int PARTS = SPLIT ? 2 : 1;    // columns of a query row
  constexpr int RPL = SPLIT ? 1 : 2;      // rows of a column tile whose scores a lane holds
  constexpr uint32_t kValueSwizzle = DIM == 128 ? 6u : 2u;  // chunks of the rows that a half warp reads at once: apart
  constexpr bool kComparesFields = SPLIT && NCT == 2;
  constexpr int kUp = kComparesFields ? 28 : 29;  // the weights' power of two, and 1 where the fields are one more
  constexpr int STATE = DIM + 4;          // a row's state in shared memory or a partial: output, maximum, sum
  extern __shared__ __align__(128) uint8_t few_smem[];
  FewTile<DIM>* ring = reinterpret_cast<FewTile<DIM>*>(few_smem);                                  // [warp][stage]
  float2* scales = reinterpret_cast<float2*>(few_smem + sizeof(FewTile<DIM>) * kFewWarps * kFewStages);  // [warp][keys, values][16]
  float* states = reinterpret_cast<float*>(scales + kFewWarps * 32);  // [warp][rows][STATE]
  __shared__ uint64_t sums[kFewWarps];
  __shared__ uint64_t found_base;
  __shared__ uint32_t found_s, last_flag;

  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t r = lane >> 2, c = lane & 3u;
  const uint32_t ngroups = a.kv_heads / p.group;
  const uint32_t span = kFewBlock * p.pb;
  const uint32_t wh = warp % p.group, wpb = warp / p.group;
  const bool works = warp < p.group * p.pb;

  // ---- this CTA's stretch of the line of steps ----
  auto steps_of = [&](const PagedSeq& q) -> uint32_t { return q.n ? max(1u, (q.context + span - 1) / span) : 0u; };
  uint64_t part = 0;
  for (uint32_t s = tid; s < a.sequences; s += kFewThreads) part += uint64_t(steps_of(paged_seq(a, s))) * ngroups;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if (lane == 0) sums[warp] = part;
  __syncthreads();
  uint64_t total = 0;
#pragma unroll
  for (int w = 0; w < kFewWarps; ++w) total += sums[w];
  const uint64_t grid = total < gridDim.x ? total : gridDim.x;
  if (blockIdx.x >= grid) return;
  const uint64_t u0 = total * blockIdx.x / grid, u1 = total * (blockIdx.x + 1) / grid;
  uint64_t running = 0;
  for (uint32_t base = 0; base < a.sequences; base += kFewThreads) {
    const uint32_t s = base + tid;
    const uint64_t v = s < a.sequences ? uint64_t(steps_of(paged_seq(a, s))) * ngroups : 0;
    uint64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= static_cast<uint32_t>(o)) inc += t;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    uint64_t before = running, all = running;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      if (w < static_cast<int>(warp)) before += sums[w];
      all += sums[w];
    }
    if (v && before + inc - v <= u0 && u0 < before + inc) {
      found_s = s;
      found_base = before + inc - v;
    }
    running = all;
    if (running > u0) break;
  }
  __syncthreads();
  uint32_t s = found_s;
  uint64_t seq_base = found_base;
  PagedSeq seq = paged_seq(a, s);
  uint32_t sp = steps_of(seq);

  FewTile<DIM>* my_ring = ring + warp * kFewStages;
  float2* my_scales = scales + warp * 32;  // both groups' scales of the block in hand: [0..15] keys, [16..31] values times `up`

  for (uint64_t cur = u0; cur < u1;) {
    while (cur >= seq_base + uint64_t(sp) * ngroups) {
      seq_base += uint64_t(sp) * ngroups;
      seq = paged_seq(a, ++s);
      sp = steps_of(seq);
    }
    const uint32_t gi = static_cast<uint32_t>((cur - seq_base) / sp);
    const uint64_t seg0 = seq_base + uint64_t(gi) * sp, seg1 = seg0 + sp;
    const uint64_t stop = u1 < seg1 ? u1 : seg1;
    const uint32_t j0 = static_cast<uint32_t>(cur - seg0), j1 = static_cast<uint32_t>(stop - seg0);
    const uint32_t h = gi * p.group + wh;
    const uint32_t rows = min(seq.n * p.share, p.rows);

    if (works) {
      // ---- queries ----
      // Lane (r, c) holds column r of each tile: dims 64 g + 16 c + 4 t + 0..3 of its row, for every (g, t).
      // Of the scores it holds rows (tile, c) or (tile, 2 c), (tile, 2 c + 1).
      uint32_t qb[NCT][G * 4][2];
      float factor[NCT][RPL];   // log2(e) / sqrt(d) * 2^e: from a difference of sums to a power of two
      int32_t limit[NCT][RPL];  // last position that the row sees
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        const uint32_t row = ct * (8 / PARTS) + r / PARTS;
        const bool in = row < rows;
        const uint32_t tok = in ? p.by_share.of(row) : 0, hq = h * p.share + (in ? row - tok * p.share : 0);
        const T* src = static_cast<const T*>(p.q) + size_t(seq.first + tok) * p.q_stride + size_t(hq) * DIM;
        float x[G * 4][4];
        float amax = 0.0f;
#pragma unroll
        for (int kk = 0; kk < G * 4; ++kk) {
          const uint32_t d = 64u * (kk / 4) + 16u * c + 4u * (kk % 4);
          if constexpr (SPLIT) {
            const float4 f = in ? *reinterpret_cast<const float4*>(src + d) : make_float4(0, 0, 0, 0);
            x[kk][0] = f.x, x[kk][1] = f.y, x[kk][2] = f.z, x[kk][3] = f.w;
          } else {
            const uint2 f = in ? *reinterpret_cast<const uint2*>(src + d) : make_uint2(0, 0);
            float y[8];
            unpack16(make_uint4(f.x, f.y, 0, 0), y, T());
#pragma unroll
            for (int e = 0; e < 4; ++e) x[kk][e] = y[e];
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(x[kk][e]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int e2 = row_exponent(amax);
        const float down = pow2i(-e2);
        const float my_factor = p.scaling * 1.4426950408889634f * pow2i(e2);
        const int32_t my_limit = in ? seq.base + static_cast<int32_t>(tok) : -1;
#pragma unroll
        for (int e = 0; e < RPL; ++e) {
          const int from = static_cast<int>((SPLIT ? 2 * c : 2 * c + e) * 4);
          factor[ct][e] = __shfl_sync(0xffffffffu, my_factor, from);
          limit[ct][e] = __shfl_sync(0xffffffffu, my_limit, from);
        }
#pragma unroll
        for (int kk = 0; kk < G * 4; ++kk) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = fmaf(x[kk][e], down, x[kk][e] - x[kk][e]);  // an infinity is NaN from here on
          uint32_t h01 = f16x2(y[0], y[1]), h23 = f16x2(y[2], y[3]);
          if (SPLIT && (r & 1u)) {
            const float2 f01 = f16x2_f32(h01), f23 = f16x2_f32(h23);
            h01 = f16x2(y[0] - f01.x, y[1] - f01.y);
            h23 = f16x2(y[2] - f23.x, y[3] - f23.y);
          }
          qb[ct][kk][0] = h01;
          qb[ct][kk][1] = h23;
        }
      }

      // ---- the loads: positions of block j, one row for each lane of a half warp ----
      const uint32_t context = seq.context;
      const int32_t* table = a.page_table + size_t(s) * a.table_stride;
      struct Place {
        int32_t page, at;  // a position's page, and its row there
      };
      auto place_of = [&](uint32_t j) -> Place {
        const uint32_t pos = j * span + wpb * kFewBlock + (lane & 15u);
        if (j >= j1 || pos >= context) return Place{-1, 0};
        const uint32_t pg = page_of(a, pos);
        return Place{__ldg(table + pg), static_cast<int32_t>(pos - pg * a.page_size)};
      };
      const uint32_t lane_row = lane / CHUNKS, lane_chunk = lane % CHUNKS;
      const uint8_t* k_src = a.k_codes + size_t(h) * DIM + 16u * lane_chunk;
      const uint8_t* v_src = a.v_codes + size_t(h) * DIM + 16u * lane_chunk;
      const uint8_t* s_src = (lane < 16 ? a.k_scales : a.v_scales) + size_t(h) * (2 * G);
      uint32_t scale_next = 0, valid_next = 0;
      auto load = [&](uint32_t j, Place at) {  // block j's codes into its stage; its scales into a register
        const int32_t row = static_cast<uint32_t>(at.page) < a.pages ? at.page * static_cast<int32_t>(a.page_size) + at.at : -1;
        valid_next = __ballot_sync(0xffffffffu, row >= 0) & 0xFFFFu;
        FewTile<DIM>* t = my_ring + j % kFewStages;
#pragma unroll
        for (int i = 0; i < CHUNKS / 2; ++i) {
          const uint32_t tr = lane_row + i * (32 / CHUNKS);
          const int32_t src = __shfl_sync(0xffffffffu, row, tr);
          const uint64_t off = uint64_t(static_cast<uint32_t>(max(src, 0))) * a.code_row;
          cp_async16(&t->k[tr][16u * (lane_chunk ^ ((tr & 1u) * (CHUNKS / 2)))], k_src + off, src >= 0);
          cp_async16(&t->v[tr][16u * (lane_chunk ^ (tr & kValueSwizzle))], v_src + off, src >= 0);
        }
        cp_async_commit();
        scale_next = 0;
        if (row >= 0) {
          const uint8_t* from = s_src + uint64_t(static_cast<uint32_t>(row)) * a.scale_row;
          scale_next = G == 2 ? *reinterpret_cast<const uint32_t*>(from) : *reinterpret_cast<const uint16_t*>(from);
        }
      };

      // Output tile (g, i) has row n at dim 64 g + 8 n + 2 i and row n + 8 at the next dim.
      float acc[NCT][G * 4][4];
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
#pragma unroll
        for (int i = 0; i < G * 4; ++i) acc[ct][i][0] = acc[ct][i][1] = acc[ct][i][2] = acc[ct][i][3] = 0.0f;
      }
      // Maxima are of the bare sums; `factor` (positive) turns a difference into a power of two.
      float m[NCT][RPL], l[NCT][RPL];
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
#pragma unroll
        for (int e = 0; e < RPL; ++e) m[ct][e] = -INFINITY, l[ct][e] = 0.0f;
      }
      uint32_t vexp = 0;  // the largest exponent field of a value scale so far

      load(j0, place_of(j0));
      Place ahead = place_of(j0 + 1);
      for (uint32_t j = j0; j < j1; ++j) {
        const uint32_t valid = valid_next;
        // Value scales: the largest exponent so far decides the weights' factor.
        bool grew = false;
        float down = 1.0f;
        {
          const uint32_t f = scale_next, next = f + kOddStep;
          const uint32_t odd = __shfl_xor_sync(0xffffffffu, next & kOddBits, 16);  // keys: of the position's values
          // The fields without those of 31, which are no numbers: by comparing them for two column tiles of f32 rows, whose
          // registers come out better that way (64 x 4 over 4096 146 us for 155), else by kOddStep (74.4 us for 76.2 of
          // 64 x 1, f16).
          uint32_t e;
          if constexpr (kComparesFields) {
            const uint32_t e0 = (f >> 10) & 31u, e1 = (f >> 26) & 31u;
            e = lane < 16 ? 0u : max(e0 == 31u ? 0u : e0, e1 == 31u ? 0u : e1);
          } else {
            e = lane < 16 ? 0u : max((next >> 10) & 31u, (next >> 26) & 31u);
          }
          const uint32_t top = __reduce_max_sync(0xffffffffu, e);
          if (top > vexp) {
            down = pow2i(static_cast<int>(vexp) - static_cast<int>(top));
            vexp = top;
            grew = true;
          }
          const float up = lane >= 16 ? pow2i(kUp - static_cast<int>(vexp)) : odd ? __int_as_float(0x7FC00000) : 1.0f;  // (NaN: its scores)
          const float2 both = f16x2_f32(f);
          my_scales[lane] = make_float2(both.x * up, both.y * up);  // (the last block's reads lie before the loop's end)
        }
        if (j + 1 < j1) {
          load(j + 1, ahead);
          ahead = place_of(j + 2);
          cp_async_wait<1>();
        } else {
          cp_async_wait<0>();
        }
        __syncwarp();
        const FewTile<DIM>* t = my_ring + j % kFewStages;

        // ---- sums of positions r and r + 8 ----
        float sc[NCT][2][RPL];  // [tile][position half][row]
        {
          float d[NCT][G][4];
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const uint32_t at = 16u * ((4u * g + c) ^ ((r & 1u) * (CHUNKS / 2)));
            const uint4 k0 = *reinterpret_cast<const uint4*>(&t->k[r][at]);
            const uint4 k1 = *reinterpret_cast<const uint4*>(&t->k[r + 8][at]);
            const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) d[ct][g][0] = d[ct][g][1] = d[ct][g][2] = d[ct][g][3] = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t a0 = codes_f16x2<0x4140>(w0[e]), a1 = codes_f16x2<0x4140>(w1[e]);
              const uint32_t a2 = codes_f16x2<0x4342>(w0[e]), a3 = codes_f16x2<0x4342>(w1[e]);
#pragma unroll
              for (int ct = 0; ct < NCT; ++ct) mma16816(d[ct][g], a0, a1, a2, a3, qb[ct][4 * g + e][0], qb[ct][4 * g + e][1]);
            }
          }
          const float2 ks[2] = {my_scales[r], my_scales[r + 8]};
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) {
#pragma unroll
            for (int hp = 0; hp < 2; ++hp) {
#pragma unroll
              for (int e = 0; e < RPL; ++e) {
                float x[G];
#pragma unroll
                for (int g = 0; g < G; ++g) x[g] = SPLIT ? d[ct][g][2 * hp] + d[ct][g][2 * hp + 1] : d[ct][g][2 * hp + e];
                float v = x[0] * ks[hp].x;
                if constexpr (G == 2) v = fmaf(x[G - 1], ks[hp].y, v);
                sc[ct][hp][e] = v;
              }
            }
          }
        }
        // ---- what a row does not see: only in the blocks at the end of the context, or with rows missing ----
        const int32_t pos0 = static_cast<int32_t>(j * span + wpb * kFewBlock);
        if (valid != 0xFFFFu || pos0 + kFewBlock - 1 > seq.base) {
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) {
#pragma unroll
            for (int hp = 0; hp < 2; ++hp) {
              const uint32_t key = r + 8u * hp;
#pragma unroll
              for (int e = 0; e < RPL; ++e) {
                if (!((valid >> key) & 1u) || pos0 + static_cast<int32_t>(key) > limit[ct][e]) sc[ct][hp][e] = -INFINITY;
              }
            }
          }
        }
        float rescale[NCT][RPL];
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
#pragma unroll
          for (int e = 0; e < RPL; ++e) {
            float mx = fmaxf(sc[ct][0][e], sc[ct][1][e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            rescale[ct][e] = 1.0f;
            if (mx > m[ct][e]) {
              rescale[ct][e] = m[ct][e] == -INFINITY ? 0.0f : ex2((m[ct][e] - mx) * factor[ct][e]);
              m[ct][e] = mx;
              grew = true;
            }
            const float base = m[ct][e] == -INFINITY ? 0.0f : m[ct][e];
            sc[ct][0][e] = ex2((sc[ct][0][e] - base) * factor[ct][e]);
            sc[ct][1][e] = ex2((sc[ct][1][e] - base) * factor[ct][e]);
            l[ct][e] = fmaf(l[ct][e], rescale[ct][e], sc[ct][0][e] + sc[ct][1][e]);
          }
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) {
            const float f0 = rescale[ct][0] * down, f1 = rescale[ct][RPL - 1] * down;
#pragma unroll
            for (int i = 0; i < G * 4; ++i) {
              acc[ct][i][0] *= f0;
              acc[ct][i][1] *= f1;
              acc[ct][i][2] *= f0;
              acc[ct][i][3] *= f1;
            }
          }
        }
        // ---- weights: B fragments for each group ----
        uint32_t wb[NCT][G][2];
#pragma unroll
        for (int hp = 0; hp < 2; ++hp) {
          const float2 vs = my_scales[16 + r + 8 * hp];
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const float v = fminf(g ? vs.y : vs.x, 32768.0f);  // (more is no number)
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
              if constexpr (SPLIT) {
                const float w = sc[ct][hp][0] * v;
                const float hi = __half2float(__float2half_rn(w));
                wb[ct][g][hp] = transpose8x8(f16x2(hi, w - hi));
              } else {
                wb[ct][g][hp] = transpose8x8(f16x2(sc[ct][hp][0] * v, sc[ct][hp][RPL - 1] * v));
              }
            }
          }
        }
        // ---- values ----
#pragma unroll
        for (int g = 0; g < G; ++g) {
          uint2 vw[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t vr = 8u * (i / 2) + 2u * c + (i % 2);
            const uint32_t ch = (4u * g + r / 2) ^ (vr & kValueSwizzle);
            vw[i] = *reinterpret_cast<const uint2*>(&t->v[vr][16u * ch + 8u * (r & 1u)]);
          }
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t x0 = w ? vw[0].y : vw[0].x, x1 = w ? vw[1].y : vw[1].x;
            const uint32_t x2 = w ? vw[2].y : vw[2].x, x3 = w ? vw[3].y : vw[3].x;
            const uint32_t a01 = __byte_perm(x0, x1, 0x5140), a23 = __byte_perm(x0, x1, 0x7362);
            const uint32_t b01 = __byte_perm(x2, x3, 0x5140), b23 = __byte_perm(x2, x3, 0x7362);
            const uint32_t e0 = codes_f16x2<0x4140>(a01), e1 = codes_f16x2<0x4342>(a01);
            const uint32_t e2 = codes_f16x2<0x4140>(b01), e3 = codes_f16x2<0x4342>(b01);
            const uint32_t o0 = codes_f16x2<0x4140>(a23), o1 = codes_f16x2<0x4342>(a23);
            const uint32_t o2 = codes_f16x2<0x4140>(b23), o3 = codes_f16x2<0x4342>(b23);
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
              mma16816(acc[ct][4 * g + 2 * w], e0, e1, e2, e3, wb[ct][g][0], wb[ct][g][1]);
              mma16816(acc[ct][4 * g + 2 * w + 1], o0, o1, o2, o3, wb[ct][g][0], wb[ct][g][1]);
            }
          }
        }
        __syncwarp();  // the block's stage and scales are free
      }

      // ---- this warp's state: lane (r, c) has dims 64 g + 8 r + 0..7 of its rows ----
      const float back = pow2i(static_cast<int>(vexp) - kUp);
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
#pragma unroll
        for (int e = 0; e < RPL; ++e) {
          const uint32_t row = ct * (8 / PARTS) + RPL * c + e;
          float lsum = l[ct][e];
          lsum += __shfl_xor_sync(0xffffffffu, lsum, 4);
          lsum += __shfl_xor_sync(0xffffffffu, lsum, 8);
          lsum += __shfl_xor_sync(0xffffffffu, lsum, 16);
          if (row < rows) {
            float* st = states + (size_t(warp) * p.rows + row) * STATE;
#pragma unroll
            for (int g = 0; g < G; ++g) {
              float o[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float(&f)[4] = acc[ct][4 * g + i];
                o[2 * i] = (SPLIT ? f[0] + f[1] : f[e]) * back;
                o[2 * i + 1] = (SPLIT ? f[2] + f[3] : f[2 + e]) * back;
              }
              *reinterpret_cast<float4*>(st + 64 * g + 8 * r) = make_float4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<float4*>(st + 64 * g + 8 * r + 4) = make_float4(o[4], o[5], o[6], o[7]);
            }
            if (r == 0) {
              st[DIM] = m[ct][e] * factor[ct][e];
              st[DIM + 1] = lsum;
            }
          }
        }
      }
    }
    __syncthreads();

    // ---- the segment's rows: merge the position blocks, then finish or leave a partial ----
    const bool whole = j0 == 0 && j1 == sp;
    const uint32_t tasks = p.group * rows;
    constexpr int PER = DIM / 32;
    const uint32_t slot = 2 * blockIdx.x + (seg0 > u0 ? 1u : 0u);
    auto finish = [&](uint32_t hh, uint32_t row, const float (&o)[PER], float lsum) {
      T* dst = static_cast<T*>(p.out) + size_t(seq.first + row / p.share) * p.out_stride +
               size_t((gi * p.group + hh) * p.share + row % p.share) * DIM + PER * lane;
      const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
#pragma unroll
      for (int e = 0; e < PER; ++e) store_as(dst + e, o[e] * inv);
    };
    for (uint32_t task = warp; task < tasks; task += kFewWarps) {
      const uint32_t hh = task / rows, row = task % rows;
      float mx = -INFINITY;
      for (uint32_t b = 0; b < p.pb; ++b) {
        const float* st = states + (size_t(b * p.group + hh) * p.rows + row) * STATE;
        mx = fmaxf(mx, st[DIM]);
      }
      float o[PER], lsum = 0.0f;
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] = 0.0f;
      for (uint32_t b = 0; b < p.pb; ++b) {
        const float* st = states + (size_t(b * p.group + hh) * p.rows + row) * STATE;
        const float f = mx == -INFINITY ? 1.0f : ex2(st[DIM] - mx);
        lsum = fmaf(st[DIM + 1], f, lsum);
#pragma unroll
        for (int e = 0; e < PER; ++e) o[e] = fmaf(st[PER * lane + e], f, o[e]);
      }
      if (whole) {
        finish(hh, row, o, lsum);
      } else {
        float* dst = p.partials + (size_t(slot * p.group + hh) * p.rows + row) * STATE;
#pragma unroll
        for (int e = 0; e < PER; ++e) dst[PER * lane + e] = o[e];
        if (lane == 0) {
          dst[DIM] = mx;
          dst[DIM + 1] = lsum;
        }
      }
    }
    if (!whole) {
      // The stretches that hold this segment: c0 .. c1 (stretch x starts at floor(x * total / grid)).
      const uint32_t c0 = static_cast<uint32_t>(((seg0 + 1) * grid - 1) / total);
      const uint32_t c1 = static_cast<uint32_t>((seg1 * grid - 1) / total);
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const uint32_t before = atomicAdd(&p.counters[kAttnCounterStride * c0], 1u);
        last_flag = before == c1 - c0;
        if (before == c1 - c0) p.counters[kAttnCounterStride * c0] = 0;
      }
      __syncthreads();
      if (last_flag) {
        __threadfence();
        for (uint32_t task = warp; task < tasks; task += kFewWarps) {
          const uint32_t hh = task / rows, row = task % rows;
          auto piece = [&](uint32_t x) {
            const uint32_t sl = 2 * x + (seg0 > total * x / grid ? 1u : 0u);
            return p.partials + (size_t(sl * p.group + hh) * p.rows + row) * STATE;
          };
          float mx = -INFINITY;
          for (uint32_t x = c0 + lane; x <= c1; x += 32) mx = fmaxf(mx, __ldcg(piece(x) + DIM));
          mx = warp_max(mx);
          float o[PER], lsum = 0.0f;
#pragma unroll
          for (int e = 0; e < PER; ++e) o[e] = 0.0f;
          for (uint32_t x0 = c0; x0 <= c1; x0 += 8) {
            float v[8][PER], pm[8], pl[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const bool in = x0 + i <= c1;
              const float* src = piece(in ? x0 + i : c1);
              pm[i] = in ? __ldcg(src + DIM) : -INFINITY;
              pl[i] = in ? __ldcg(src + DIM + 1) : 0.0f;
              if constexpr (PER == 4) {
                const float4 f = __ldcg(reinterpret_cast<const float4*>(src) + lane);
                v[i][0] = f.x, v[i][1] = f.y, v[i][2] = f.z, v[i][3] = f.w;
              } else {
                const float2 f = __ldcg(reinterpret_cast<const float2*>(src) + lane);
                v[i][0] = f.x, v[i][1] = f.y;
              }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (x0 + i > c1) break;
              const float f = mx == -INFINITY ? 1.0f : ex2(pm[i] - mx);
              lsum = fmaf(pl[i], f, lsum);
#pragma unroll
              for (int e = 0; e < PER; ++e) o[e] = fmaf(v[i][e], f, o[e]);
            }
          }
          finish(hh, row, o, lsum);
        }
      }
    }
    __syncthreads();  // the states are free again
    cur = stop;
  }
}

template <int DIM>
size_t few_smem_bytes(uint32_t rows) {
  return sizeof(FewTile<DIM>) * kFewWarps * kFewStages + kFewWarps * 32 * 8 + size_t(kFewWarps) * rows * (DIM + 4) * 4;
}

constexpr uint32_t kWaitTries = 100000;  // tries that sleep up to 20 us each: at most 2 s

// How a call is run: which kernel, its grid, and its part of the workspace.
struct AttnPlan {
  bool few;
  uint32_t grid, group, pb, rows;
  TilePlan tile;
  uint64_t partial_bytes;
};

AttnPlan attention_plan(const PagedArgs& a, uint32_t format, uint32_t heads) {
  AttnPlan p = {};
  const uint64_t rows = uint64_t(a.max_query) * (heads / a.kv_heads);
  const uint64_t sms = 148;
  // As many rows as the few-row kernel has columns for. 64 sequences of up to 4096 positions, 8 kv heads: f32, 8 rows,
  // 147 us here and 387 on 128-row tiles; bf16, 16 rows, 193 and 229; 2 sequences up to 2047, f32, 8 rows, 21 and 43;
  // 64 of one token, f32, 75 and 418. (One kernel for the whole call: single tokens beside a chunk pay the latter.)
  p.few = rows <= (format == kFormatF32 ? 8u : 16u);
  if (!p.few) {
    p.tile = paged_tile_plan(a, format, heads, sms);
    p.partial_bytes = p.tile.partial_bytes;
    return p;
  }
  p.rows = static_cast<uint32_t>(rows);
  // Heads to a CTA. More of them read wider rows and leave fewer warps' states to merge, but a sequence then lies in
  // more stretches, each with more rows to join. 64 x 1 over 4096, f32: one head 82 us, two 74, four 73, eight 78;
  // 64 x 4 over 4096 one 165, two 153, four 150; 8 x 1 over 4096 one 24, two 25, four 29; 2 x 4 over 2047 one 18,
  // two 31, four 78. Two for a good number of short single tokens: 64 x 1 over 512 one 29, two 25; over 64 one 12, two
  // 8; 16 x 1 over 4096 one 34.7, two 33.8; but 64 x 4 over 256 one 34, two 39.
  p.group = 1;
  const uint64_t pairs = uint64_t(a.sequences) * a.kv_heads;
  const uint32_t most = pairs * a.max_context >= 8ull * 2 * sms * 512 ? 4 : pairs >= 128 && rows <= 2 ? 2 : 1;
  for (uint32_t g = 2; g <= most; ++g) {
    if (a.kv_heads % g == 0) p.group = g;
  }
  p.pb = kFewWarps / p.group;
  const uint64_t span = uint64_t(kFewBlock) * p.pb;
  const uint64_t steps = uint64_t(a.sequences) * (a.kv_heads / p.group) * (a.max_context ? (a.max_context + span - 1) / span : 1);
  p.grid = static_cast<uint32_t>(steps < 2 * sms ? steps : 2 * sms);
  p.partial_bytes = uint64_t(2) * p.grid * p.group * p.rows * (a.head_dim + 4) * 4;
  return p;
}

template <typename T, int DIM, int NCT>
int32_t launch_few(const PagedArgs& a, AttnArgs p, const AttnPlan& plan, cudaStream_t stream) {
  const size_t smem = few_smem_bytes<DIM>(plan.rows);
  cudaError_t e = cudaFuncSetAttribute(paged_attention_few_kernel<T, DIM, NCT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem));
  if (e != cudaSuccess) return paged_status(e);
  p.group = plan.group;
  p.pb = plan.pb;
  p.rows = plan.rows;
  paged_attention_few_kernel<T, DIM, NCT><<<plan.grid, kFewThreads, smem, stream>>>(a, p);
  return paged_status(cudaGetLastError());
}

template <typename T>
int32_t attention_as(const PagedArgs& a, AttnArgs p, const AttnPlan& plan, cudaStream_t stream) {
  if (plan.few) {
    const bool one = plan.rows <= (sizeof(T) == 4 ? 4u : 8u);  // column tiles
    if (a.head_dim == 128) return one ? launch_few<T, 128, 1>(a, p, plan, stream) : launch_few<T, 128, 2>(a, p, plan, stream);
    return one ? launch_few<T, 64, 1>(a, p, plan, stream) : launch_few<T, 64, 2>(a, p, plan, stream);
  }
  return paged_tile_launch(a, p, sizeof(T) == 4 ? kFormatF32 : std::is_same<T, __half>::value ? kFormatF16 : kFormatBF16,
                           plan.tile, stream);
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
  *bytes = kAttnHeadBytes + attention_plan(a, format, heads).partial_bytes;
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
  const AttnPlan plan = attention_plan(a, format, heads);
  if (!plan.few && plan.tile.too_long) return QWC_LIMIT_EXCEEDED;
  if (workspace_bytes < kAttnHeadBytes + plan.partial_bytes) return QWC_LIMIT_EXCEEDED;
  AttnArgs p = {};
  p.q = q;
  p.q_stride = q_stride;
  p.out = out;
  p.out_stride = out_stride;
  p.error = static_cast<int32_t*>(workspace);
  p.wait_tries = kWaitTries;
  p.counters = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + 256);
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kAttnHeadBytes);
  p.heads = heads;
  p.share = heads / a.kv_heads;
  p.by_share = divisor(p.share);
  p.scaling = 1.0f / sqrtf(static_cast<float>(a.head_dim));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return format == kFormatF32   ? attention_as<float>(a, p, plan, s)
         : format == kFormatF16 ? attention_as<__half>(a, p, plan, s)
                                : attention_as<__nv_bfloat16>(a, p, plan, s);
}

}  // extern "C"
