// The block-scaled product on the tensor cores: D[M, N] = sum over k of (a_scale A)[m, k] (b_scale B)[n, k]  (+ bias)
// with e4m3 operands, both with the contraction contiguous in memory, and one power-of-two scale per block of 128 along
// the contraction (hapx_block8.h).
//
// The scales are applied by the tensor cores (tcgen05.mma kind::mxf8f6f4, which multiplies every 32 products by the two
// scales of their row and column before adding them): the four 32-deep instructions of a block of 128 name the same
// scale bytes.  So an accumulator runs over the whole contraction, as in the bfloat16 product (hapx_gemm_sm100.cu),
// whose structure this kernel has: persistent, warp-specialised, accumulators in tensor memory.
//   warp 0      : TMA producer (128 x 128 byte tiles, 128-byte swizzle; every fourth block also the scales of four blocks)
//   warp 1      : allocates TMEM; one thread copies scales to tensor memory (tcgen05.cp) and issues tcgen05.mma
//   the others  : epilogue, a warp per 32 rows x 64 columns (or two such pieces): bias, one rounding, bulk stores through a staging tile
// (An earlier form kept one accumulator per block and the running sums in registers, adding block products with their
// scales in the epilogue warps; it was bound by the chain commit -> wait -> read -> arrive of its two accumulators.)
//
// Pair kernel (M > 128): clusters of two CTAs, cta_group::2; each CTA stages its 128 rows of A and half of B's rows.  Tiles
// of 256 x 192 with two accumulators (which leave tensor memory for the scales, and divide widths of 768 and 2304), or of
// 256 x 256 with one: unit_us chooses.  Single kernel (M <= 128): 128 x 64 tiles, so that a narrow product still spreads
// over the SMs.
//
// 8192 x 8192 x 8192: 380 us = 2.9 PFLOP/s (the library's bfloat16 product 690 us), the tensor pipe 90 % of the time active: bound
// by it and by the clock that power leaves.  8192 x 33280 from 768: 205 us, of which 138 are what filling the 545 MB of
// output takes.  8192 x 768 -> 2304 and back: 16, 15 and 20 us (forward, to the input, to the weight).
//
// Single kernel with X (a float type): the first operand comes as it is, bfloat16 or float32, and eight more warps make its
// 8-bit tiles and scales in shared memory as the blocks go by, for themselves in every thread block: one launch for a few
// rows (16 x 768 -> 2304: 7.2 us).
//
// Every mbarrier wait is bounded; on expiry a role raises the error word and leaves, the others follow as their own
// waits run out, TMEM is freed and the kernel returns.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>
#include <mutex>
#include <string>
#include <type_traits>

#include "hapx_block8.h"
#include "hapx_internal.h"
#include "hapx_tc.h"

namespace hapx {
namespace gemm8 {

using namespace tc;

constexpr int BM = 128;      // rows of the tile per CTA
constexpr int BK = 128;      // one block of the contraction: one 128-byte swizzle row
constexpr int UMMA_K = 32;
constexpr unsigned kAtom = 512;      // scales of 128 rows x 4 blocks

// One product of a launch.
struct Problem {
  int M, N, k_blocks;
  void* D; long long ldd;
  const void* bias;          // N values of D's type, or null
  int out_f32, tma_store, bias_vec;
  int m_tiles, n_tiles, band;
  int splits, kb_per_split;  // > 1: the blocks are cut into ranges; each writes a float32 partial tile to rows [split * m_pad, ...)
  long long m_pad;
  const float* colsum;       // null, or colsum_tiles x M floats whose column sums go to colsum_out (the bias gradient that
  int colsum_tiles;          // belongs to a weight gradient: see the epilogue)
  int colsum_f32;
  void* colsum_out;
};
// One or two products; units (tile, range of blocks) of the first, which has the longer ones, are dealt out first.
struct Params {
  Problem pr[2];
  int units[2];
  int rounds;                // of the second product's units that every worker takes part in: see the kernel
  unsigned* error;
  const void* x; long long ldx;   // the first operand as it is, M x K, for the kernel that converts it
  int K;
};
struct Maps { CUtensorMap a[2], b[2], sa[2], sb[2], d[2]; };

template <bool PAIR>
__device__ __forceinline__ void umma8(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned sfa, unsigned sfb,
                                      unsigned accumulate) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// One atom of scales (32 lanes x 16 bytes, lane by lane in shared memory) to 4 columns of tensor memory, in all four
// lane quarters; with a pair, in each CTA from its own shared memory.
template <bool PAIR>
__device__ __forceinline__ void copy_scales(unsigned taddr, unsigned smem) {
  // no swizzle; 8 lanes x 16 bytes are a core matrix, the next 8 lanes follow 128 bytes later
  const unsigned long long desc = (unsigned long long)((smem & 0x3ffffu) >> 4) | (8ull << 16) | (8ull << 32) | (1ull << 46);
  if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// BN: columns of the tile - 192 or 256 for the pair kernel, 64 for the single one.
template <int BN_, bool CONVERT = false>
struct Cfg {
  static constexpr int BN = BN_;
  static constexpr bool PAIR = BN > 64;
  static constexpr int ACCS = 2 * BN + 64 <= 512 ? 2 : 1;    // accumulators in tensor memory, next to the scales
  static constexpr int PIECES = BN / 64;                     // 64 columns: 128 bytes of a bfloat16 row
  static constexpr int PARTS = BN == 256 ? 2 : PIECES;       // pieces that are worked on at a time, one of 32 rows per warp
  static constexpr int EPI_WARPS = 4 * PARTS;
  static constexpr int CONVERT_WARPS = CONVERT ? 8 : 0;      // every eighth block each
  static constexpr int THREADS = 64 + 32 * (EPI_WARPS + CONVERT_WARPS);
  static constexpr int STAGES = BN == 256 ? 5 : PAIR ? 6 : 8;
  // A wait for a stage tells apart its last use and the one before, no more.  A converting warp that has seen block j - STAGES
  // consumed knows nothing of the next one: its following turn may come a whole round of the stages later, not more.
  static_assert(CONVERT_WARPS <= STAGES, "a converting warp's wait would take an older use of the stage for the last");
  static constexpr int B_ATOMS = PAIR ? 2 : 1;               // 192 columns from a multiple of 64 on lie in two groups of 128
  static constexpr unsigned A_BYTES = BM * BK;
  static constexpr unsigned B_BYTES = (PAIR ? BN / 2 : BN) * BK;
  static constexpr unsigned STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr unsigned SCALE_BYTES = (1 + B_ATOMS) * kAtom;
  static constexpr unsigned STORE_BYTES = EPI_WARPS * 32 * 128;  // one 32-row x 128-byte staging tile per epilogue warp
  static constexpr unsigned SF_COL = ACCS * BN;              // scales behind the accumulators, one set per stage
  static constexpr unsigned SF_SET = 4 * (1 + B_ATOMS);
  static constexpr unsigned TMEM_COLS = PAIR ? 512 : 256;
  static_assert(SF_COL + STAGES * SF_SET <= TMEM_COLS, "tensor memory");
  static constexpr unsigned SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + STORE_BYTES + STAGES * SCALE_BYTES + 256;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
  // e4m3 x e4m3 (format 0), K-major operands, N >> 3 at bit 17, scales of type ue8m0 (bit 23), M >> 7 at bit 27; the
  // bytes of the scale words that an instruction uses at bits 4 (B) and 29 (A)
  static constexpr unsigned IDESC = ((unsigned)(BN >> 3) << 17) | (1u << 23) | ((unsigned)((PAIR ? 2 * BM : BM) >> 7) << 27);
};

// One 128-byte row piece per thread, swizzled within the warp's staging tile (chunk ^ row % 8).
__device__ __forceinline__ void stage_row(unsigned char* row, int sw, const unsigned (&w)[32]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(row + ((j ^ sw) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}

// v[j] += bias[n + j] (float32) for the columns inside the matrix; `vec`: all are, and the bias lies on 16 bytes.
__device__ __forceinline__ void add_bias(const Problem& p, int n, bool vec, unsigned (&v)[32]) {
  const float* bias = static_cast<const float*>(p.bias) + n;
  auto add = [&](int j, float x) { v[j] = __float_as_uint(__uint_as_float(v[j]) + x); };
  if (vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(bias) + j);
      add(4 * j, x.x); add(4 * j + 1, x.y); add(4 * j + 2, x.z); add(4 * j + 3, x.w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (n + j < p.N) add(j, bias[j]);
  }
}

// JOIN: the output is float32, and the accumulator runs over kChunk blocks at a time; the epilogue warps add the chunks in
// registers, rounding to nearest.  The tensor cores cut what an addition shifts out, so an accumulator drifts towards zero
// with every step: a float32 weight gradient over 12232 tokens of uneven size was off by 5e-6 where float32 sums of the
// library are off by 5e-7, and is by 3e-7 now.  One chunk is added while the next runs (8192 x 8192 x 8192: 400 us without,
// 426 in chunks of 8, 443 of 4; 8192 x 4096 from 1024: 45 us either way).  A bfloat16 output rounds by a thousand times as
// much and does not pay for it.
constexpr int kChunk = 4;

template <int BN, typename X, bool JOIN>
__global__ void __launch_bounds__(Cfg<BN, !std::is_void<X>::value>::THREADS, 1)
gemm8_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params params) {
  constexpr bool CONVERT = !std::is_void<X>::value;
  using C = Cfg<BN, CONVERT>;
  constexpr bool PAIR = C::PAIR;
  extern __shared__ unsigned char smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* gen_base = smem_raw + (base - smem_u32(smem_raw));
  constexpr unsigned kStore = C::STAGES * C::STAGE_BYTES, kScales = kStore + C::STORE_BYTES, kBars = kScales + C::STAGES * C::SCALE_BYTES;
  const unsigned bars = base + kBars;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (C::STAGES + s); };
  auto tfull_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + a); };
  auto tempty_bar = [&](int a) { return bars + 8u * (2 * C::STAGES + 2 + a); };
  const unsigned tmem_slot = bars + 8u * (2 * C::STAGES + 4);
  volatile unsigned* tmem_slot_gen = reinterpret_cast<volatile unsigned*>(gen_base + kBars + 8 * (2 * C::STAGES + 4));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = PAIR ? (int)cluster_ctarank() : 0;       // 0 leads the pair
  const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, workers = PAIR ? gridDim.x >> 1 : gridDim.x;
  // A worker's units in order: its share of the first product's, dealt round by round; then of the second's - `rounds`
  // rounds over all workers, and what is left over the workers that had no unit in the first product's last, partly
  // filled round.  So the longer units of one product and the shorter ones of the other even out without a counter in
  // memory.
  const int left = params.units[0] % workers, own0 = params.units[0] / workers + (worker < left ? 1 : 0);
  struct Unit { int which, m0, n0, split, kb0, kb1; };
  auto next_unit = [&](int step, Unit& u) {
    int unit = step * workers + worker;
    u.which = step >= own0;
    if (u.which) {
      const int t = step - own0;
      if (t < params.rounds) unit = t * workers + worker;
      else if (worker >= left) unit = params.rounds * workers + (t - params.rounds) * (workers - left) + worker - left;
      else return false;
      if (unit >= params.units[1]) return false;
    }
    const Problem& p = params.pr[u.which];
    const int tile = unit / p.splits;
    u.split = unit - tile * p.splits;
    int row = tile, column, row0 = 0, rows = p.m_tiles;
    if (p.band) {                                            // so many rows of tiles across all columns, then the next ones
      const int band = tile / (p.band * p.n_tiles);
      row0 = band * p.band;
      row = tile - row0 * p.n_tiles;
      rows = min(p.band, p.m_tiles - row0);
    }
    column = row / rows;
    u.m0 = (row0 + row - column * rows) * (PAIR ? 2 * BM : BM) + cta * BM;
    u.n0 = column * C::BN;
    u.kb0 = u.split * p.kb_per_split;
    u.kb1 = min(u.kb0 + p.kb_per_split, p.k_blocks);
    return true;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(full_bar(s), CONVERT ? 2 : 1); mbar_init(empty_bar(s), 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), (PAIR ? 2 : 1) * C::EPI_WARPS); }
    fence_barrier_init();
    const int which = own0 == 0;
    prefetch_tensormap(&maps.a[which]);
    prefetch_tensormap(&maps.b[which]);
    prefetch_tensormap(&maps.sa[which]);
    prefetch_tensormap(&maps.sb[which]);
  }
  if (warp == 1) {
    if (PAIR) { tmem_alloc2(tmem_slot, C::TMEM_COLS); tmem_relinquish2(); }
    else { tmem_alloc(tmem_slot, C::TMEM_COLS); tmem_relinquish(); }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();
  tc_fence_after();
  const unsigned tmem_base = *tmem_slot_gen;

  if (warp == 0) {
    // ---------------- TMA producer (one per CTA) ----------------
    int stage = 0;
    unsigned phase = 0;
    bool ok = true;
    Unit u;
    for (int step = 0; ok && next_unit(step, u); ++step) {
      for (int kb = u.kb0; kb < u.kb1; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(empty_bar(stage), phase ^ 1u));
        if (!ok) break;
        if (elect_one()) {
          const unsigned sa = base + stage * C::STAGE_BYTES, sb = sa + C::A_BYTES;
          // the scales of four blocks come with the first of them that the unit needs, in the stage's own slot
          const bool scales = CONVERT || kb == u.kb0 || (kb & 3) == 0;
          const unsigned ss = base + kScales + stage * C::SCALE_BYTES;
          const unsigned bytes = CONVERT ? C::B_BYTES + C::SCALE_BYTES - kAtom : C::STAGE_BYTES + (scales ? C::SCALE_BYTES : 0u);
          if (PAIR) {
            const unsigned bar = map_to_cta(full_bar(stage), 0);
            if (cta == 0) mbar_expect_tx(full_bar(stage), 2 * bytes);     // the bytes of both CTAs
            tma_load_4d_pair(sa, &maps.a[u.which], kb * BK, u.m0, 0, 0, bar);
            tma_load_4d_pair(sb, &maps.b[u.which], kb * BK, u.n0 + cta * (C::BN / 2), 0, 0, bar);
            if (scales) {
              tma_load_4d_pair(ss, &maps.sa[u.which], 0, u.m0 >> 7, kb >> 2, 0, bar);
              tma_load_4d_pair(ss + kAtom, &maps.sb[u.which], 0, u.n0 >> 7, kb >> 2, 0, bar);
            }
          } else {
            mbar_expect_tx(full_bar(stage), bytes);
            if (!CONVERT) tma_load_4d(sa, &maps.a[u.which], kb * BK, u.m0, 0, 0, full_bar(stage));
            tma_load_4d(sb, &maps.b[u.which], kb * BK, u.n0, 0, 0, full_bar(stage));
            if (scales) {
              if (!CONVERT) tma_load_4d(ss, &maps.sa[u.which], 0, u.m0 >> 7, kb >> 2, 0, full_bar(stage));
              tma_load_4d(ss + kAtom, &maps.sb[u.which], 0, u.n0 >> 7, kb >> 2, 0, full_bar(stage));
            }
          }
        }
        __syncwarp();
        if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok) {
      if (lane == 0) atomicCAS(params.error, 0u, 1u);
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);      // a millisecond for the copies in flight to land
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (leader CTA only) ----------------
    if (cta == 0) {
      int stage = 0, acc = 0;
      unsigned phase = 0, acc_phase = 0;
      bool ok = true;
      // descriptors of the first 32 bytes of a stage; a stage or a step of 32 further on is an addition to the address field
      const unsigned long long desc_a = make_desc(base, 16u, 1024u), desc_b = make_desc(base + C::A_BYTES, 16u, 1024u);
      Unit u;
      for (int step = 0; ok && next_unit(step, u); ++step) {
        const unsigned shift = (unsigned)(u.n0 >> 5) & 3u;   // B's rows start inside a group of 128
        unsigned sf = 0, d = 0;
        for (int kb = u.kb0; kb < u.kb1; ++kb) {
          const bool first = kb == u.kb0 || (JOIN && (kb - u.kb0) % kChunk == 0), last = kb + 1 == u.kb1 || (JOIN && (kb + 1 - u.kb0) % kChunk == 0);
          if (first) {
            ok = __all_sync(0xffffffffu, mbar_wait(tempty_bar(acc), acc_phase ^ 1u));
            if (!ok) break;
            d = tmem_base + (unsigned)(acc * C::BN);
          }
          ok = __all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase));
          if (!ok) break;
          tc_fence_after();
          const bool scales = CONVERT || kb == u.kb0 || (kb & 3) == 0;
          if (scales) sf = tmem_base + C::SF_COL + stage * C::SF_SET;
          if (elect_one()) {
            if (scales) {
              // tcgen05.cp and tcgen05.mma run in the order of their issue, and a set is not written again before the
              // stages have gone round
              const unsigned ss = base + kScales + stage * C::SCALE_BYTES;
#pragma unroll
              for (int i = 0; i <= C::B_ATOMS; ++i) copy_scales<PAIR>(sf + 4 * i, ss + i * kAtom);
            }
            const unsigned long long da = desc_a + (unsigned)(stage * (C::STAGE_BYTES >> 4)), db = desc_b + (unsigned)(stage * (C::STAGE_BYTES >> 4));
            const unsigned idesc = C::IDESC | ((unsigned)(kb & 3) << 4) | ((unsigned)(kb & 3) << 29);
#pragma unroll
            for (int k = 0; k < BK / UMMA_K; ++k) umma8<PAIR>(d, da + 2 * k, db + 2 * k, idesc, sf, sf + 4 + shift, !first || k != 0);
            if (PAIR) umma2_commit_both(empty_bar(stage));
            else umma_commit(empty_bar(stage));
            if (last) {                                      // the accumulator is complete
              if (PAIR) umma2_commit_both(tfull_bar(acc));
              else umma_commit(tfull_bar(acc));
            }
          }
          __syncwarp();
          if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
          if (last && ++acc == C::ACCS) { acc = 0; acc_phase ^= 1u; }
        }
      }
      if (!ok && lane == 0) atomicCAS(params.error, 0u, 2u);
    }
  } else if (CONVERT && warp >= 2 + C::EPI_WARPS) {
    // ---------------- 8-bit tiles of the first operand: a warp per block, R rows at a time ----------------
    // (A block's rows over all warps would put the loads' latency and the fence into every block: 2 us each.)
    if constexpr (CONVERT) {
      const int mine = warp - 2 - C::EPI_WARPS, M = params.pr[0].M, K = params.K;     // the rows are those of one tile: M <= 128
      const X* x = static_cast<const X*>(params.x) + 4 * lane;
      const bool vec = (params.ldx & 3) == 0 && (reinterpret_cast<uintptr_t>(params.x) & (4 * sizeof(X) - 1)) == 0;
      constexpr int R = 8;                                   // 16 for bfloat16 was no faster
      block8::Raw4<X> next[R];
      auto fetch = [&](int kb, int r0) {
        const int valid = max(0, min(4, K - kb * BK - 4 * lane));
        const X* src = x + (long long)kb * BK + r0 * params.ldx;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (r0 + i >= M || valid == 0) next[i].zero();
          else if (vec && valid == 4) next[i].load(src + i * params.ldx);
          else next[i].load_some(src + i * params.ldx, valid);
        }
      };
      int stage = 0, turn = 0;
      unsigned phase = 0;
      bool ok = true;
      Unit u;
      for (int step = 0; ok && next_unit(step, u); ++step) {
        for (int kb = u.kb0; kb < u.kb1; ++kb) {
          if (turn == mine) {
            fetch(kb, 0);
            ok = __all_sync(0xffffffffu, mbar_wait(empty_bar(stage), phase ^ 1u));
            if (!ok) break;
            unsigned char* tile = gen_base + stage * C::STAGE_BYTES;
            unsigned char* scales = gen_base + kScales + stage * C::SCALE_BYTES + (kb & 3);
            for (int r0 = 0; r0 < M; r0 += R) {
              block8::Raw4<X> v[R];
#pragma unroll
              for (int i = 0; i < R; ++i) v[i] = next[i];
              if (r0 + R < M) fetch(kb, r0 + R);
              unsigned big = 0u;                               // lane i < R: the pattern of row i's maximum
              auto maxima = [&] {
#pragma unroll
                for (int i = 0; i < R; ++i) {
                  typename block8::Raw4<X>::Max unused;
                  block8::Raw4<X>::clear(unused);
                  const unsigned r = __reduce_max_sync(0xffffffffu, v[i].maxima(unused));
                  if (lane == i) big = r;
                }
              };
              maxima();
              if (__any_sync(0xffffffffu, big >= 0x7f800000u)) {   // an infinity (rare): NaN in its place
#pragma unroll
                for (int i = 0; i < R; ++i) v[i].sanitise();
                maxima();
              }
              const int e = block8::scale_exponent(__uint_as_float(big & block8::Raw4<X>::kMask));
              const float inv_mine = block8::pow2(-e);
#pragma unroll
              for (int i = 0; i < R; ++i) {                    // a row's 16-byte chunks are swizzled by its number mod 8
                const float inv = __shfl_sync(0xffffffffu, inv_mine, i);
                float f[4];
                v[i].get(f);
                *reinterpret_cast<unsigned*>(tile + (r0 + i) * 128 + (((lane >> 2) ^ (i & 7)) << 4) + (lane & 3) * 4) =
                    block8::pack4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
              }
              if (lane < R) {
                const int r = r0 + lane;
                scales[(r & 31) * 16 + (r >> 5) * 4] = (unsigned char)(e + 127);
              }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full_bar(stage));
          }
          if (++turn == C::CONVERT_WARPS) turn = 0;
          if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok && lane == 0) atomicCAS(params.error, 0u, 5u);
    }
  } else {
    // ---------------- epilogue: 32 rows x 64 columns of the tile per warp ----------------
    const int q = warp & 3, part = (warp - 2) >> 2;          // q: the TMEM lane quarter this warp may read
    unsigned char* tile_gen = gen_base + kStore + (warp - 2) * 4096;
    const unsigned tile_u32 = base + kStore + (warp - 2) * 4096;
    int acc = 0;
    unsigned acc_phase = 0;
    bool ok = true;
    Unit u;
    for (int step = 0; next_unit(step, u); ++step) {
      const Problem& p = params.pr[u.which];
      if (p.colsum && u.n0 == 0 && part == 0 && u.split == 0) {
        // the bias gradient of a weight gradient's rows: the partial column sums of the quantiser, added in their order
        // by the warps that have to wait for this tile anyway
        const int row = u.m0 + q * 32 + lane;
        if (row < p.M) {
          float sum = 0.f;
#pragma unroll 8
          for (int i = 0; i < p.colsum_tiles; ++i) sum += __ldg(p.colsum + (long long)i * p.M + row);
          if (p.colsum_f32) static_cast<float*>(p.colsum_out)[row] = sum;
          else static_cast<__nv_bfloat16*>(p.colsum_out)[row] = __float2bfloat16_rn(sum);
        }
      }
      if (p.bias_vec && lane < C::PIECES / C::PARTS && u.n0 + 64 * (part + C::PARTS * lane) + 64 <= p.N) {   // comes closer during the wait
        const long long n0 = u.n0 + 64 * (part + C::PARTS * lane);
        asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const char*>(p.bias) + n0 * (p.out_f32 ? 4 : 2)));
        if (p.out_f32) asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const char*>(p.bias) + n0 * 4 + 128));
      }
      if constexpr (!JOIN) {
        ok = __all_sync(0xffffffffu, mbar_wait(tfull_bar(acc), acc_phase));
        if (!ok) break;
        tc_fence_after();
      }
      const long long out_row0 = (long long)u.split * p.m_pad + u.m0 + q * 32;
      auto drained = [&] {                                   // this warp has read its part of the accumulator
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_cluster_light(map_to_cta(tempty_bar(acc), 0));
          else mbar_arrive(tempty_bar(acc));
        }
      };
      // W columns from n0 on, `width` of them inside the matrix, staged as 128 bytes per row: out in one bulk store, or row by row for any pitch
      auto send = [&](auto f32_tag, int n0, int width) {
        constexpr bool OUT_F32 = decltype(f32_tag)::value;
        constexpr int W = OUT_F32 ? 32 : 64;
        if (p.tma_store) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tma_store_4d(&maps.d[u.which], tile_u32, n0, (int)out_row0, 0, 0);
            bulk_commit_group();
          }
        } else {
          __syncwarp();
          const int rows = min(32, p.M - (u.m0 + q * 32));
          constexpr int ES = OUT_F32 ? 4 : 2;
          using Bits = typename std::conditional<OUT_F32, unsigned, unsigned short>::type;
#pragma unroll
          for (int h = 0; h < W / 32; ++h) {
            const int col = lane + 32 * h, byte = col * ES;
            if (col >= width) continue;
            const unsigned char* src = tile_gen + (byte & 15);
            Bits* dst = static_cast<Bits*>(p.D) + out_row0 * p.ldd + n0 + col;
#pragma unroll 1
            for (int i0 = 0; i0 < rows; i0 += 8) {           // eight rows in flight
              Bits v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const Bits*>(src + (i0 + i) * 128 + (((byte >> 4) ^ i) << 4));
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (i0 + i < rows) dst[i * p.ldd] = v[i];
              dst += 8 * p.ldd;
            }
          }
          __syncwarp();
        }
      };
      auto staging_free = [&] {                              // the previous store has read the staging tile
        if (lane == 0) bulk_wait_read_0();
        __syncwarp();
      };
      const int n0 = u.n0 + 64 * part;                       // a warp's pieces of 64 columns lie 64 * PARTS apart
      auto piece = [&] { return tmem_base + ((unsigned)(q * 32) << 16) + (unsigned)(acc * C::BN + 64 * part); };
      if constexpr (JOIN) {
        float sum[2][32] = {};
        for (int kb = u.kb0; kb < u.kb1; kb += kChunk) {
          ok = __all_sync(0xffffffffu, mbar_wait(tfull_bar(acc), acc_phase));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            unsigned r[32];
            tmem_ld_32x32(piece() + 32u * h, r);
            tmem_ld_wait();
            if (h == 1) drained();
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[h][j] += __uint_as_float(r[j]);
          }
          if (++acc == C::ACCS) { acc = 0; acc_phase ^= 1u; }
        }
        if (!ok) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = n0 + 32 * h, width = min(32, p.N - n);
          if (width <= 0) continue;
          unsigned r[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(sum[h][j]);
          if (p.bias) add_bias(p, n, p.bias_vec && width == 32, r);
          staging_free();
          stage_row(tile_gen + lane * 128, lane & 7, r);
          send(std::true_type{}, n, width);
        }
        continue;
      }
      const unsigned t = piece();
      constexpr int PER = C::PIECES / C::PARTS;
      if (p.out_f32) {
#pragma unroll 1
        for (int i = 0; i < 2 * PER; ++i) {
          const int off = (i >> 1) * 64 * C::PARTS + (i & 1) * 32, n = n0 + off, width = min(32, p.N - n);
          unsigned r[32];
          tmem_ld_32x32(t + (unsigned)off, r);
          tmem_ld_wait();
          if (i == 2 * PER - 1) drained();
          if (width <= 0) continue;
          if (p.bias) add_bias(p, n, p.bias_vec && width == 32, r);
          staging_free();
          stage_row(tile_gen + lane * 128, lane & 7, r);
          send(std::true_type{}, n, width);
        }
      } else {
        unsigned r[64];
        auto load = [&](int off) {
          tmem_ld_32x32(t + (unsigned)off, reinterpret_cast<unsigned(&)[32]>(r[0]));
          tmem_ld_32x32(t + (unsigned)off + 32, reinterpret_cast<unsigned(&)[32]>(r[32]));
          tmem_ld_wait();
        };
        load(0);
        if (PER == 1) drained();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int n = n0 + i * 64 * C::PARTS, width = min(64, p.N - n);
          float v[64];
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = __uint_as_float(r[j]);
          if (p.bias_vec && width == 64) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint4 x = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.bias) + n) + j);
              const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) { v[8 * j + 2 * e] += __uint_as_float(w[e] << 16); v[8 * j + 2 * e + 1] += __uint_as_float(w[e] & 0xffff0000u); }
            }
          } else if (p.bias) {
#pragma unroll
            for (int j = 0; j < 64; ++j)
              if (j < width) v[j] += __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n + j]);
          }
          staging_free();
          unsigned w[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const unsigned*>(&h);
          }
          if (i + 1 < PER) {                                 // the accumulator is let go before anything is stored
            load((i + 1) * 64 * C::PARTS);
            if (i + 2 == PER) drained();
          }
          if (width <= 0) continue;
          stage_row(tile_gen + lane * 128, lane & 7, w);
          send(std::false_type{}, n, width);
        }
      }
      if (++acc == C::ACCS) { acc = 0; acc_phase ^= 1u; }
    }
    if (lane == 0) bulk_wait_all();
    if (!ok) atomicCAS(params.error, 0u, 3u);
  }

  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();      // neither CTA leaves (or frees TMEM) while the other can still signal it
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc2(tmem_base, C::TMEM_COLS);
    else tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// Adds the float32 partial tiles of a split product in their order, then bias and the one rounding.
template <typename T>
__global__ void __launch_bounds__(256) gemm8_join_kernel(const float* __restrict__ ws, int splits, long long M, int N, long long m_pad, int n_pad,
                                                         const T* __restrict__ bias, T* __restrict__ out) {
  const int n4 = n_pad >> 2;
  const bool vec = (N & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < M * n4; e += (long long)gridDim.x * 256) {
    const long long r = e / n4;
    const int c = (int)(e - r * n4) << 2;
    float4 a = *reinterpret_cast<const float4*>(ws + r * n_pad + c);
    for (int s = 1; s < splits; ++s) {
      const float4 v = *reinterpret_cast<const float4*>(ws + (s * m_pad + r) * n_pad + c);
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
    float o[4] = {a.x, a.y, a.z, a.w};
    T* dst = out + r * N + c;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (bias && c + j < N) o[j] += (float)bias[c + j];
    if (vec) {
      if constexpr (sizeof(T) == 2) {
        const __nv_bfloat162 h0 = __floats2bfloat162_rn(o[0], o[1]), h1 = __floats2bfloat162_rn(o[2], o[3]);
        *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const unsigned*>(&h0), *reinterpret_cast<const unsigned*>(&h1));
      } else {
        *reinterpret_cast<float4*>(dst) = make_float4(o[0], o[1], o[2], o[3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < N) dst[j] = (T)o[j];
    }
  }
}

// 4-D map (contiguous index, row, 1, 1) with boxes of box_inner x box_rows.
static int make_map(CUtensorMap* map, const void* ptr, CUtensorMapDataType type, int es, long long inner, long long rows, long long ld,
                    int box_inner, int box_rows, CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promo) {
  gemm::EncodeTiledFn fn = gemm::encode_fn();
  if (!fn) return fail(HAPX_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t dims[4] = {(cuuint64_t)inner, (cuuint64_t)rows, 1, 1};
  cuuint64_t strides[3] = {(cuuint64_t)(ld * es), (cuuint64_t)(ld * es), (cuuint64_t)(ld * es)};
  cuuint32_t box[4] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(map, type, 4, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, promo,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(HAPX_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  return HAPX_OK;
}

// How a product is cut: into tiles of 64 (single kernel), 192 or 256 columns, and into how many ranges of blocks.
struct Plan { int bn, f32, splits, kb_per_split; long long m_pad, tiles; int n_pad, blocks; };

static Plan plan_whole(long long M, long long N, long long K, int f32, int bn) {
  Plan pl;
  pl.bn = bn; pl.f32 = f32;
  const long long bm = bn > 64 ? 2 * BM : BM, m_tiles = (M + bm - 1) / bm;
  pl.tiles = m_tiles * ((N + bn - 1) / bn);
  pl.blocks = (int)((K + BK - 1) / BK);
  pl.splits = 1; pl.kb_per_split = pl.blocks; pl.m_pad = m_tiles * bm; pl.n_pad = (int)((N + 3) / 4 * 4);
  return pl;
}
static bool cut(Plan& pl, int splits) {        // false where a range would be empty or the partial tiles too large
  const int per = (pl.blocks + splits - 1) / splits;
  if (splits > 1 && (splits * 4 > pl.blocks || (splits - 1) * per >= pl.blocks || 4.0 * splits * (double)pl.m_pad * pl.n_pad > 512e6)) return false;
  pl.splits = splits; pl.kb_per_split = per;
  return true;
}
// Microseconds of a tile's unit of so many blocks, fitted to measurements, and of a split: its partial tiles written and
// read back at about 4 TB/s plus a launch.  A block of 256 x 256 is a third more work than one of 256 x 192 for a seventh
// more bytes into shared memory, but its accumulator has no second one, so nothing hides its drain; and 256 columns may
// divide a width better or worse.  (192 against 256: 4096 x 1024 from 8192 36.4 / 27.2 us, 8192^3 396 / 384,
// 16384 x 4096 from 1024 65.5 / 62.7; 8192 x 768 from 2304 15.8 / 18.9, 4096 x 4096 from 1024 19.3 / 20.2.)
// Twice as many bytes of float32 take 0.8 us longer to leave (8192 x 4096 from 1024 with its quantiser: 64.8 us in 256
// columns, 59.1 in 192).  Whole float32 outputs, whose accumulators change hands every kChunk blocks, need two.
static double unit_us(const Plan& pl) {
  const int kb = pl.kb_per_split;
  return pl.bn == 64 ? 0.15 * kb : pl.bn == 192 ? 0.29 * kb + 0.8 : 0.39 * kb + (pl.splits > 1 ? 1.95 : 1.15);
}
static double split_us(const Plan& pl) { return pl.splits > 1 ? 3.0 + pl.splits * 8.0 * (double)pl.m_pad * pl.n_pad / 4e6 : 0.0; }

// A long contraction over few tiles leaves SMs idle, or the last round of tiles nearly empty: cut the blocks into ranges
// whose float32 partial tiles a second kernel adds in a fixed order, where that costs less by a clear margin.
static Plan plan_of(long long M, long long N, long long K, int f32, int sm_count) {
  auto cost = [&](const Plan& q) {
    const int workers = q.bn > 64 ? sm_count / 2 : sm_count;
    return (double)((q.tiles * q.splits + workers - 1) / workers) * unit_us(q) + split_us(q);
  };
  auto best_of = [&](int bn) {
    Plan best = plan_whole(M, N, K, f32, bn), pl = best;
    for (int sp = 2; sp <= 16; ++sp)
      if (cut(pl, sp) && cost(pl) < 0.9 * cost(best)) best = pl;
    return best;
  };
  if (M <= BM) return best_of(64);
  const Plan a = best_of(192);
  if (f32) return a;
  const Plan b = best_of(256);
  return cost(b) < cost(a) ? b : a;
}

// Microseconds until the last worker is done with two products dealt out as the kernel does it, the longer units first;
// and the number of rounds of the second product's units for all workers.
static double makespan(const Plan& a, const Plan& b, int workers, int* rounds) {
  const long long ua = a.tiles * a.splits, ub = b.tiles * b.splits, full = ua / workers, left = ua % workers, all = (ub + workers - 1) / workers;
  const double la = unit_us(a), lb = unit_us(b);
  if (left == 0) {
    *rounds = (int)all;
    return full * la + all * lb;
  }
  const double ideal = (ua * la + ub * lb) / workers;
  const long long guess = (long long)std::max(0.0, (ideal - (full + 1) * la) / lb);
  double best = -1.0;
  for (long long r = guess; r <= guess + 1; ++r) {
    const long long some = std::min(r, all), rest = std::max(0ll, ub - some * workers), more = (rest + workers - left - 1) / (workers - left);
    const double t = std::max((full + 1) * la + some * lb, full * la + (some + more) * lb);
    if (best < 0.0 || t < best) { best = t; *rounds = (int)some; }
  }
  return best;
}

// Two products in one launch of the pair kernel: which goes first, its cut, the other's.
struct PairPlan { Plan pl[2]; int first, rounds; };
static PairPlan plan_two(const Product& x, const Product& y, int sm_count) {
  const int workers = sm_count / 2;
  PairPlan best;
  double best_us = -1.0;
  for (int bn = 192; bn <= (x.out_f32 ? 192 : 256); bn += 64) {
    const Plan whole[2] = {plan_whole(x.m, x.n, x.k, x.out_f32, bn), plan_whole(y.m, y.n, y.k, y.out_f32, bn)};
    for (int cx = 1; cx <= 16; cx = cx < 4 ? cx + 1 : cx * 2) {
      for (int cy = 1; cy <= 16; cy = cy < 4 ? cy + 1 : cy * 2) {
        if (cx > 1 && cy > 1) continue;                       // one of the two at most
        PairPlan t;
        t.pl[0] = whole[0]; t.pl[1] = whole[1];
        if (!cut(t.pl[0], cx) || !cut(t.pl[1], cy)) continue;
        t.first = t.pl[1].kb_per_split > t.pl[0].kb_per_split;
        const double us = makespan(t.pl[t.first], t.pl[!t.first], workers, &t.rounds) + split_us(t.pl[0]) + split_us(t.pl[1]);
        if (best_us < 0.0 || us < 0.95 * best_us) { best = t; best_us = us; }
      }
    }
  }
  return best;
}

static long long partial_bytes(const Plan& pl) { return pl.splits > 1 ? pl.splits * pl.m_pad * pl.n_pad * 4 : 0; }

template <int BN, typename X, bool JOIN>
static int launch(const Maps& maps, const Params& p, int sm_count, cudaStream_t stream) {
  using C = Cfg<BN, !std::is_void<X>::value>;
  constexpr bool PAIR = C::PAIR;
  auto kernel = gemm8_kernel<BN, X, JOIN>;
  static int limit_of[64] = {};             // per device: function attributes and occupancy belong to one
  static std::mutex mutex;
  int device = 0;
  HAPX_CUDA(cudaGetDevice(&device));
  if (device < 0 || device >= 64) return fail(HAPX_ERR_ARGUMENT, "block8_matmul: device index out of range");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR ? 2 : 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int limit = 0;
  {
    std::lock_guard<std::mutex> lock(mutex);
    limit = limit_of[device];
    if (limit == 0) {
      HAPX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM_BYTES));
      limit = sm_count;
      if (PAIR) {
        cfg.gridDim = dim3(sm_count / 2 * 2);
        HAPX_CUDA(cudaOccupancyMaxActiveClusters(&limit, kernel, &cfg));
        if (limit < 1) return fail(HAPX_ERR_CUDA, "block8_matmul: no SM pair can host the two-CTA kernel");
      }
      limit_of[device] = limit;
    }
  }
  const int workers = std::min(p.units[0] + p.units[1], limit);
  cfg.gridDim = dim3((unsigned)(workers * (PAIR ? 2 : 1)));
  HAPX_CUDA(cudaLaunchKernelEx(&cfg, kernel, maps, p));
  count_launch();
  return HAPX_OK;
}

static int launch_plan(const Plan& pl, const Maps& maps, const Params& p, int sm_count, cudaStream_t stream) {
  if (pl.bn == 64) return pl.f32 ? launch<64, void, true>(maps, p, sm_count, stream) : launch<64, void, false>(maps, p, sm_count, stream);
  if (pl.bn == 192) return pl.f32 ? launch<192, void, true>(maps, p, sm_count, stream) : launch<192, void, false>(maps, p, sm_count, stream);
  return launch<256, void, false>(maps, p, sm_count, stream);
}

// The scales as (128 words of an atom, group of 128 rows, four blocks).
static int make_scale_map(CUtensorMap* map, const void* ptr, long long rows, int k_blocks, int box_groups) {
  gemm::EncodeTiledFn fn = gemm::encode_fn();
  if (!fn) return fail(HAPX_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t groups = (cuuint64_t)((rows + 127) / 128);
  cuuint64_t dims[4] = {kAtom / 4, groups, (cuuint64_t)((k_blocks + 3) / 4), 1};
  cuuint64_t strides[3] = {kAtom, kAtom * groups, kAtom * groups};
  cuuint32_t box[4] = {kAtom / 4, (cuuint32_t)box_groups, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(HAPX_ERR_CUDA, "cuTensorMapEncodeTiled (scales) failed with code " + std::to_string((int)r));
  return HAPX_OK;
}

long long workspace_bytes(long long m, long long n, long long k, int sm_count) {      // for either type of the output
  return std::max(partial_bytes(plan_of(m, n, k, 0, sm_count)), partial_bytes(plan_of(m, n, k, 1, sm_count)));
}

// Tiles are walked down the rows, so that the second operand comes from memory once; a first operand too long for half of
// L2 next to what else is there is walked in bands of eight rows of tiles, and then it comes once.  (33280 x 768 from 8192:
// 212 / 164 us without / with bands; 16384 x 4096 from 4096 207 / 190; of 16 MB no difference, but two more divisions.)
constexpr long long kLongOperand = 32ll << 20;
constexpr int kBand = 8;

// One product as entry i of a launch; `partial`: where its partial tiles go.
static int describe(const Product& pr, const Plan& pl, void* partial, int i, Maps* maps, Params* params) {
  const long long M = pr.m, N = pr.n, K = pr.k;
  const int bn = pl.bn, bm = bn > 64 ? 2 * BM : BM;
  Problem& p = params->pr[i];
  p = Problem();
  p.M = (int)M; p.N = (int)N; p.k_blocks = pl.blocks;
  p.splits = pl.splits; p.kb_per_split = pl.kb_per_split; p.m_pad = pl.m_pad;
  p.m_tiles = (p.M + bm - 1) / bm; p.n_tiles = (p.N + bn - 1) / bn;
  p.band = M * K >= kLongOperand && p.m_tiles > kBand ? kBand : 0;
  if (pl.tiles * pl.splits > 0x3fffffff) return fail(HAPX_ERR_EXTENT, "block8_matmul: too many tiles");
  params->units[i] = (int)(pl.tiles * pl.splits);
  long long out_rows = M;
  if (pl.splits > 1) { p.D = partial; p.ldd = pl.n_pad; p.out_f32 = 1; p.bias = nullptr; out_rows = pl.splits * pl.m_pad; }
  else { p.D = pr.d; p.ldd = N; p.out_f32 = pr.out_f32; p.bias = pr.bias; }
  p.bias_vec = p.bias && (reinterpret_cast<uintptr_t>(p.bias) & 15u) == 0;
  p.colsum = pr.colsum; p.colsum_tiles = pr.colsum_tiles; p.colsum_f32 = pr.out_f32; p.colsum_out = pr.colsum_out;
  const int es = p.out_f32 ? 4 : 2;
  if (pr.a)
    if (int e = make_map(&maps->a[i], pr.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, M, pr.lda, BK, BM, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return e;
  if (int e = make_map(&maps->b[i], pr.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, N, pr.ldb, BK, bn > 64 ? bn / 2 : bn, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return e;
  if (pr.a)
    if (int e = make_scale_map(&maps->sa[i], pr.a_scale, M, p.k_blocks, 1)) return e;
  if (int e = make_scale_map(&maps->sb[i], pr.b_scale, N, p.k_blocks, bn > 64 ? 2 : 1)) return e;
  p.tma_store = (reinterpret_cast<uintptr_t>(p.D) & 15u) == 0 && (p.ldd * es) % 16 == 0;
  if (p.tma_store)
    return make_map(&maps->d[i], p.D, p.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, es, pl.splits > 1 ? pl.n_pad : N,
                    out_rows, p.ldd, 128 / es, 32, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE);
  return HAPX_OK;
}

static int join(const Product& pr, const Plan& pl, const void* partial, int sm_count, cudaStream_t stream) {
  if (pl.splits == 1) return HAPX_OK;
  const int grid = (int)std::min<long long>((pr.m * (pl.n_pad / 4) + 255) / 256, (long long)sm_count * 8);
  const float* ws = static_cast<const float*>(partial);
  if (pr.out_f32) gemm8_join_kernel<<<grid, 256, 0, stream>>>(ws, pl.splits, pr.m, (int)pr.n, pl.m_pad, pl.n_pad, static_cast<const float*>(pr.bias),
                                                              static_cast<float*>(pr.d));
  else gemm8_join_kernel<<<grid, 256, 0, stream>>>(ws, pl.splits, pr.m, (int)pr.n, pl.m_pad, pl.n_pad, static_cast<const __nv_bfloat16*>(pr.bias),
                                                   static_cast<__nv_bfloat16*>(pr.d));
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

int run(const Product& pr, int sm_count, cudaStream_t stream) {
  Params params = Params();
  Maps maps;
  std::memset(&maps, 0, sizeof(maps));
  if (int e = gemm::error_word(&params.error, nullptr)) return e;
  const Plan pl = plan_of(pr.m, pr.n, pr.k, pr.out_f32, sm_count);
  if (int e = describe(pr, pl, pr.workspace, 0, &maps, &params)) return e;
  if (int e = launch_plan(pl, maps, params, sm_count, stream)) return e;
  return join(pr, pl, pr.workspace, sm_count, stream);
}

// 64 x 1024 -> 4096 takes 16.4 us this way and 9.0 with the quantiser in front, 16 tokens 8.0 and about 9: the limit lies
// where the launch that is saved (5 us of host time) no longer pays.
bool converts(long long m) { return m <= 32; }

int run_converting(const Product& pr, const void* x, int dtype, long long ldx, int sm_count, cudaStream_t stream) {
  Params params = Params();
  Maps maps;
  std::memset(&maps, 0, sizeof(maps));
  if (int e = gemm::error_word(&params.error, nullptr)) return e;
  const Plan pl = plan_of(pr.m, pr.n, pr.k, pr.out_f32, sm_count);
  if (int e = describe(pr, pl, pr.workspace, 0, &maps, &params)) return e;
  params.x = x; params.ldx = ldx; params.K = (int)pr.k;
  if (int e = dtype == HAPX_BF16 ? launch<64, __nv_bfloat16, false>(maps, params, sm_count, stream) : launch<64, float, true>(maps, params, sm_count, stream))
    return e;
  return join(pr, pl, pr.workspace, sm_count, stream);
}

long long workspace_bytes_two(const Product& x, const Product& y, int sm_count) {
  long long most = 0;
  for (int f32 = 0; f32 < 2; ++f32) {
    Product a = x, b = y;
    a.out_f32 = b.out_f32 = f32;
    const PairPlan t = plan_two(a, b, sm_count);
    most = std::max(most, partial_bytes(t.pl[0]) + partial_bytes(t.pl[1]));
  }
  return most;
}

int run_two(const Product& x, const Product& y, int sm_count, cudaStream_t stream) {
  Params params = Params();
  Maps maps;
  std::memset(&maps, 0, sizeof(maps));
  if (int e = gemm::error_word(&params.error, nullptr)) return e;
  const PairPlan t = plan_two(x, y, sm_count);
  const Product* pr[2] = {&x, &y};
  void* partial[2] = {x.workspace, static_cast<char*>(x.workspace) + partial_bytes(t.pl[0])};
  for (int i = 0; i < 2; ++i)
    if (int e = describe(*pr[i], t.pl[i], partial[i], i == t.first ? 0 : 1, &maps, &params)) return e;
  params.rounds = t.rounds;
  if (int e = launch_plan(t.pl[0], maps, params, sm_count, stream)) return e;
  for (int i = 0; i < 2; ++i)
    if (int e = join(*pr[i], t.pl[i], partial[i], sm_count, stream)) return e;
  return HAPX_OK;
}

}  // namespace gemm8
}  // namespace hapx

using namespace hapx;

extern "C" {

int64_t hapx_block8_matmul_workspace(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0 || m > 0x7fffff00 || n > 0x7fffff00 || k > 0x7fffff00) return 0;
  int n_sm = 0;
  return sm_count(&n_sm) ? 0 : gemm8::workspace_bytes(m, n, k, n_sm);
}

int hapx_block8_matmul(void* d, int out_dtype, const void* a, int64_t lda, const void* a_scale, const void* b, int64_t ldb, const void* b_scale,
                       const void* bias, int64_t m, int64_t n, int64_t k, void* workspace, int64_t workspace_bytes, hapx_stream stream) {
  if (out_dtype != HAPX_F32 && out_dtype != HAPX_BF16) return fail(HAPX_ERR_DTYPE, "block8_matmul: the output is float32 or bfloat16");
  if (m < 0 || n < 0 || k < 1 || m > 0x7fffff00 || n > 0x7fffff00 || k > 0x7fffff00)
    return fail(HAPX_ERR_EXTENT, "block8_matmul: extents must lie below 2^31 - 256, the contraction at 1 or above");
  if (m == 0 || n == 0) return HAPX_OK;
  if (!d || !a || !a_scale || !b || !b_scale) return fail(HAPX_ERR_ARGUMENT, "block8_matmul: null pointer");
  if (lda % 16 != 0 || ldb % 16 != 0 || lda < k || ldb < k || ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15u))
    return fail(HAPX_ERR_EXTENT, "block8_matmul: operands need a 16-byte aligned base and pitch, and a pitch that covers a row");
  if ((reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(b_scale)) & 15u)
    return fail(HAPX_ERR_EXTENT, "block8_matmul: the scales need a 16-byte aligned base");
  int n_sm = 0;
  if (int e = sm_count(&n_sm)) return e;
  const long long need = gemm8::workspace_bytes(m, n, k, n_sm);
  if (workspace_bytes < need || (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u))))
    return fail(HAPX_ERR_ARGUMENT, "block8_matmul: the workspace must be 16-byte aligned and as large as hapx_block8_matmul_workspace says");
  gemm8::Product pr;
  pr.d = d; pr.out_f32 = out_dtype == HAPX_F32; pr.a = a; pr.lda = lda; pr.a_scale = a_scale; pr.b = b; pr.ldb = ldb; pr.b_scale = b_scale;
  pr.bias = bias; pr.m = m; pr.n = n; pr.k = k; pr.workspace = workspace;
  return gemm8::run(pr, n_sm, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
