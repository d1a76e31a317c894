// The block-scaled product on the tensor cores: D[M, N] = sum over blocks kb of 128 along the contraction of
//     a_scale[kb][m] * b_scale[kb][n] * sum_{k in kb} A[m, k] B[n, k]   (+ bias)
// with e4m3 operands, both with the contraction contiguous in memory (hapx_block8.h).
//
// Persistent and warp-specialised like the bfloat16 product (hapx_gemm_sm100.cu), with one difference that shapes it:
// an accumulator lives for ONE block of 128 only.  Its scales differ from the next block's, so tensor memory holds
// block products, and the epilogue warps keep the running float32 sums of the output tile in registers, adding each
// block product with its scales while the tensor cores work on the next one (two accumulators, used alternately).
//   warp 0      : TMA producer (128 x 128 byte tiles, 128-byte swizzle; with 1 x 128 blocks of B also their scales)
//   warp 1      : allocates TMEM; one thread issues tcgen05.mma kind::f8f6f4, four of 32 deep per block
//   warps 4 ... : epilogue; a warp owns 32 rows x CW columns of the tile, a thread one row: CW float32 sums
//
// Pair kernel (M > 128): clusters of two CTAs, 256 x 256 tiles, cta_group::2; each CTA stages its 128 rows of A and half
// of B's rows and sums its 128 x 256 half of the tile with eight epilogue warps (128 sums per thread).  Single kernel
// (M <= 128): 128 x 64 tiles, so that a narrow product still spreads over the SMs.
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

#include "hapx_internal.h"
#include "hapx_tc.h"

namespace hapx {
namespace gemm8 {

using namespace tc;

constexpr int BM = 128;      // rows of the tile per CTA
constexpr int BK = 128;      // one block of the contraction: one 128-byte swizzle row
constexpr int UMMA_K = 32;

struct Params {
  int M, N, k_blocks;
  const float* a_scale; long long lda_scale;
  const float* b_scale; long long ldb_scale;   // square: [k block][block of 128 rows]
  void* D; long long ldd;
  const void* bias;          // N values of D's type, or null
  int out_f32, tma_store;
  int m_tiles, n_tiles;
  int splits, kb_per_split;  // > 1: the blocks are cut into ranges; each writes a float32 partial tile to rows [split * m_pad, ...)
  long long m_pad;
  unsigned* error;
};

__device__ __forceinline__ void umma8(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma8_pair(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Two float32 lanes per instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ f32x2 pair2u(unsigned a, unsigned b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void unpair2(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <bool PAIR, bool SQUARE>
struct Cfg {
  static constexpr int BN = PAIR ? 256 : 64;                 // columns of the tile
  static constexpr int EPI_WARPS = PAIR ? 8 : 4;
  static constexpr int CW = BN / (EPI_WARPS / 4);            // columns per epilogue warp
  static constexpr int THREADS = 128 + 32 * EPI_WARPS;      // warps 2 and 3 only complete the first warpgroup
  static constexpr int STAGES = PAIR ? 5 : 7;
  static constexpr int RING = STAGES + 4;                    // slots of B's scales; see the producer
  static constexpr unsigned A_BYTES = BM * BK;
  static constexpr unsigned B_BYTES = (PAIR ? BN / 2 : BN) * BK;
  static constexpr unsigned STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr unsigned SCALE_BYTES = SQUARE ? 0 : BN * 4;
  static constexpr unsigned STORE_BYTES = EPI_WARPS * 32 * 128;  // one 32-row x 128-byte staging tile per epilogue warp
  static constexpr unsigned TMEM_COLS = 2 * BN;
  static constexpr unsigned SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + STORE_BYTES + RING * SCALE_BYTES + 256;
  // float32 accumulator, e4m3 x e4m3 (format 0), K-major operands, N >> 3, M >> 4
  static constexpr unsigned IDESC = (1u << 4) | ((unsigned)(BN >> 3) << 17) | ((unsigned)((PAIR ? 2 * BM : BM) >> 4) << 24);
};

// One 128-byte row piece per thread, swizzled within the warp's staging tile (chunk ^ row % 8).
template <bool OUT_F32>
__device__ __forceinline__ void stage_row(unsigned char* row, int sw, const float* v) {
  if constexpr (OUT_F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) *reinterpret_cast<float4*>(row + ((j ^ sw) << 4)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      unsigned w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[8 * j + 2 * e], v[8 * j + 2 * e + 1]);
        w[e] = *reinterpret_cast<const unsigned*>(&h);
      }
      *reinterpret_cast<uint4*>(row + ((j ^ sw) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

template <bool PAIR, bool SQUARE>
__global__ void __launch_bounds__(Cfg<PAIR, SQUARE>::THREADS, 1)
gemm8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmS,
             const __grid_constant__ CUtensorMap tmD, const Params p) {
  using C = Cfg<PAIR, SQUARE>;
  extern __shared__ unsigned char smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* gen_base = smem_raw + (base - smem_u32(smem_raw));
  constexpr unsigned kStore = C::STAGES * C::STAGE_BYTES, kScales = kStore + C::STORE_BYTES, kBars = kScales + C::RING * C::SCALE_BYTES;
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
  const int units = p.m_tiles * p.n_tiles * p.splits;
  struct Unit { int m0, n0, split, kb0, kb1; };
  auto decode = [&](int unit) {
    Unit u;
    const int tile = unit / p.splits;
    u.split = unit - tile * p.splits;
    u.m0 = (tile % p.m_tiles) * (PAIR ? 2 * BM : BM) + cta * BM;
    u.n0 = (tile / p.m_tiles) * C::BN;
    u.kb0 = u.split * p.kb_per_split;
    u.kb1 = min(u.kb0 + p.kb_per_split, p.k_blocks);
    return u;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), (PAIR ? 2 : 1) * C::EPI_WARPS); }
    fence_barrier_init();
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
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

  // 384 threads start with 168 registers each; the epilogue's 128 sums and two buffers of 32 need more, the first
  // warpgroup far fewer: 128 x 40 + 256 x 232 = 64,512, the block's all.
  if (warp < 4) {
    if (PAIR) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
    // ---------------- TMA producer (one per CTA) ----------------
    if (lane == 0) {
      int stage = 0, slot = 0;
      unsigned phase = 0;
      bool ok = true;
      for (int unit = worker; unit < units && ok; unit += workers) {
        const Unit u = decode(unit);
        for (int kb = u.kb0; kb < u.kb1; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u)) { ok = false; break; }
          const unsigned sa = base + stage * C::STAGE_BYTES, sb = sa + C::A_BYTES;
          // This stage's block products are done, so the sums of the two blocks before it are too: the accumulator they
          // came from was needed.  A slot of B's scales is therefore free STAGES + 2 blocks after it was filled.
          const unsigned ss = base + kScales + slot * C::SCALE_BYTES;
          if (PAIR) {
            const unsigned bar = map_to_cta(full_bar(stage), 0);
            if (cta == 0) mbar_expect_tx(full_bar(stage), 2 * (C::STAGE_BYTES + C::SCALE_BYTES));     // the bytes of both CTAs
            tma_load_4d_pair(sa, &tmA, kb * BK, u.m0, 0, 0, bar);
            tma_load_4d_pair(sb, &tmB, kb * BK, u.n0 + cta * (C::BN / 2), 0, 0, bar);
            if (!SQUARE) tma_load_4d_pair(ss, &tmS, u.n0, kb, 0, 0, bar);
          } else {
            mbar_expect_tx(full_bar(stage), C::STAGE_BYTES + C::SCALE_BYTES);
            tma_load_4d(sa, &tmA, kb * BK, u.m0, 0, 0, full_bar(stage));
            tma_load_4d(sb, &tmB, kb * BK, u.n0, 0, 0, full_bar(stage));
            if (!SQUARE) tma_load_4d(ss, &tmS, u.n0, kb, 0, 0, full_bar(stage));
          }
          if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
          if (++slot == C::RING) slot = 0;
        }
      }
      if (!ok) atomicCAS(p.error, 0u, 1u);
    }
    } else if (warp == 1) {
    // ---------------- MMA issuer (leader CTA only) ----------------
    if (lane == 0 && cta == 0) {
      int stage = 0, acc = 0;
      unsigned phase = 0, acc_phase = 0;
      bool ok = true;
      for (int unit = worker; unit < units && ok; unit += workers) {
        const Unit u = decode(unit);
        for (int kb = u.kb0; kb < u.kb1; ++kb) {
          if (!mbar_wait(tempty_bar(acc), acc_phase ^ 1u) || !mbar_wait(full_bar(stage), phase)) { ok = false; break; }
          tc_fence_after();
          const unsigned sa = base + stage * C::STAGE_BYTES, sb = sa + C::A_BYTES, d = tmem_base + (unsigned)(acc * C::BN);
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            const unsigned long long da = make_desc(sa + k * 32u, 16u, 1024u), db = make_desc(sb + k * 32u, 16u, 1024u);
            if (PAIR) umma8_pair(d, da, db, C::IDESC, k != 0);
            else umma8(d, da, db, C::IDESC, k != 0);
          }
          if (PAIR) { umma2_commit_both(empty_bar(stage)); umma2_commit_both(tfull_bar(acc)); }
          else { umma_commit(empty_bar(stage)); umma_commit(tfull_bar(acc)); }
          if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
          if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
        }
      }
      if (!ok) atomicCAS(p.error, 0u, 2u);
    }
    }
  } else {
    // ---------------- epilogue: 32 rows x CW columns per warp ----------------
    if (PAIR) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int q = warp & 3, half = (warp - 4) >> 2;          // q: the TMEM lane quarter this warp may read
    const unsigned t_warp = tmem_base + ((unsigned)(q * 32) << 16) + (unsigned)(half * C::CW);
    unsigned char* tile_gen = gen_base + kStore + (warp - 4) * 4096;
    const unsigned tile_u32 = base + kStore + (warp - 4) * 4096;
    int acc = 0, slot = 0;
    unsigned acc_phase = 0;
    bool ok = true;
    for (int unit = worker; unit < units && ok; unit += workers) {
      const Unit u = decode(unit);
      const int row = u.m0 + q * 32 + lane, c0 = u.n0 + half * C::CW;
      f32x2 sum[C::CW / 2];
#pragma unroll
      for (int j = 0; j < C::CW / 2; ++j) sum[j] = 0ull;
      const float* as = p.a_scale + (row < p.M ? row : 0);
      const float* bs = p.b_scale + (SQUARE && c0 < p.N ? c0 >> 7 : 0);
      float sa = as[u.kb0 * p.lda_scale], sb = SQUARE ? bs[u.kb0 * p.ldb_scale] : 1.f;
      for (int kb = u.kb0; kb < u.kb1; ++kb) {
        const f32x2 s2 = SQUARE ? pair2(sa * sb, sa * sb) : pair2(sa, sa);
        const int nx = min(kb + 1, u.kb1 - 1);               // the next block's scales travel during the wait
        sa = as[nx * p.lda_scale];
        if (SQUARE) sb = bs[nx * p.ldb_scale];
        ok = __all_sync(0xffffffffu, mbar_wait(tfull_bar(acc), acc_phase));
        if (!ok) break;
        tc_fence_after();
        const unsigned t = t_warp + (unsigned)(acc * C::BN);
        const float* sb_row = reinterpret_cast<const float*>(gen_base + kScales + slot * C::SCALE_BYTES) + half * C::CW;
        // 32 columns per load, two loads in flight; the accumulator goes back as soon as the last ones have landed
        auto add = [&](const unsigned (&v)[32], int c) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            f32x2 x0 = pair2u(v[4 * j], v[4 * j + 1]), x1 = pair2u(v[4 * j + 2], v[4 * j + 3]);
            if (!SQUARE) {
              const float4 b4 = *reinterpret_cast<const float4*>(sb_row + c + 4 * j);
              x0 = mul2(x0, pair2(b4.x, b4.y));
              x1 = mul2(x1, pair2(b4.z, b4.w));
            }
            sum[c / 2 + 2 * j] = fma2(x0, s2, sum[c / 2 + 2 * j]);
            sum[c / 2 + 2 * j + 1] = fma2(x1, s2, sum[c / 2 + 2 * j + 1]);
          }
        };
        unsigned r0[32], r1[32];
        tmem_ld_32x32(t, r0);
        tmem_ld_32x32(t + 32, r1);
#pragma unroll
        for (int c = 0; c < C::CW; c += 64) {
          tmem_ld_wait();
          if (c + 64 >= C::CW) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (PAIR) mbar_arrive_cluster_light(map_to_cta(tempty_bar(acc), 0));
              else mbar_arrive(tempty_bar(acc));
            }
          }
          add(r0, c);
          if (c + 64 < C::CW) tmem_ld_32x32(t + c + 64, r0);
          add(r1, c + 32);
          if (c + 64 < C::CW) tmem_ld_32x32(t + c + 96, r1);
        }
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
        if (++slot == C::RING) slot = 0;
      }
      if (!ok) break;
      // the finished rows: bias, one rounding, out through the staging tile in pieces of 128 bytes per row
      const long long out_row0 = (long long)u.split * p.m_pad + u.m0 + q * 32;
      auto piece = [&](auto f32_tag, int c) {                // columns c0 + c .. of this warp
        constexpr bool OUT_F32 = decltype(f32_tag)::value;
        constexpr int W = OUT_F32 ? 32 : 64;
        float v[W];
#pragma unroll
        for (int j = 0; j < W / 2; ++j) {
          // `c` is a constant after unrolling
          unpair2(sum[c / 2 + j], v[2 * j], v[2 * j + 1]);
        }
        if (p.bias) {
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const int n = min(c0 + c + j, p.N - 1);
            v[j] += OUT_F32 ? static_cast<const float*>(p.bias)[n] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
          }
        }
        if (lane == 0) bulk_wait_read_0();                   // the previous piece has left the staging tile
        __syncwarp();
        stage_row<OUT_F32>(tile_gen + lane * 128, lane & 7, v);
        if (p.tma_store) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tma_store_4d(&tmD, tile_u32, c0 + c, (int)out_row0, 0, 0);
            bulk_commit_group();
          }
        } else {                                             // any pitch: rows of the tile one after another, coalesced
          __syncwarp();
          for (int r = 0; r < 32; ++r) {
            if (u.m0 + q * 32 + r >= p.M) break;
#pragma unroll
            for (int h = 0; h < W / 32; ++h) {
              const int col = lane + 32 * h, byte = col * (OUT_F32 ? 4 : 2);
              const unsigned char* src = tile_gen + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15);
              if (c0 + c + col < p.N) {
                if (OUT_F32) static_cast<float*>(p.D)[(out_row0 + r) * p.ldd + c0 + c + col] = *reinterpret_cast<const float*>(src);
                else static_cast<__nv_bfloat16*>(p.D)[(out_row0 + r) * p.ldd + c0 + c + col] = *reinterpret_cast<const __nv_bfloat16*>(src);
              }
            }
          }
          __syncwarp();
        }
      };
      if (p.out_f32) {
#pragma unroll
        for (int c = 0; c < C::CW; c += 32)
          if (c0 + c < p.N) piece(std::true_type{}, c);
      } else {
#pragma unroll
        for (int c = 0; c < C::CW; c += 64)
          if (c0 + c < p.N) piece(std::false_type{}, c);
      }
    }
    if (lane == 0) bulk_wait_all();
    if (!ok) atomicCAS(p.error, 0u, 3u);
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

// How a product is cut: the pair kernel or the single one, and into how many ranges of blocks.
struct Plan { bool pair; int splits, kb_per_split; long long m_pad; int n_pad; };

static Plan plan_of(long long M, long long N, long long K, int sm_count) {
  Plan pl;
  pl.pair = M > BM;
  const long long bm = pl.pair ? 2 * BM : BM, bn = pl.pair ? Cfg<true, true>::BN : Cfg<false, true>::BN;
  const long long m_tiles = (M + bm - 1) / bm, tiles = m_tiles * ((N + bn - 1) / bn);
  const int blocks = (int)((K + BK - 1) / BK), workers = pl.pair ? sm_count / 2 : sm_count;
  pl.splits = 1; pl.kb_per_split = blocks; pl.m_pad = m_tiles * bm; pl.n_pad = (int)((N + 3) / 4 * 4);
  // A long contraction over few tiles leaves SMs idle, or the last round of tiles nearly empty: cut the blocks into
  // ranges whose float32 partial tiles a second kernel adds in a fixed order.  In microseconds: rounds x blocks x the
  // time of one block, and for a split the partial tiles written and read back at about 4 TB/s plus a launch.
  const double block_us = pl.pair ? 0.30 : 0.15, partial = 8.0 * (double)pl.m_pad * pl.n_pad / 4e6;
  auto rounds = [&](long long units) { return (double)((units + workers - 1) / workers); };
  double best = rounds(tiles) * blocks * block_us;
  for (int sp = 2; sp <= 16 && sp * 4 <= blocks; ++sp) {
    const int per = (blocks + sp - 1) / sp;
    if ((sp - 1) * per >= blocks) continue;                 // an empty last range
    if (4.0 * sp * (double)pl.m_pad * pl.n_pad > 512e6) break;
    const double cost = rounds(tiles * sp) * per * block_us + 3.0 + sp * partial;
    if (cost < 0.9 * best) { pl.splits = sp; pl.kb_per_split = per; best = cost; }
  }
  return pl;
}

static int sm_count_of(int* out) {
  int device = 0;
  HAPX_CUDA(cudaGetDevice(&device));
  HAPX_CUDA(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, device));
  return HAPX_OK;
}

template <bool PAIR, bool SQUARE>
static int launch(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmS, const CUtensorMap& tmD, const Params& p, int sm_count,
                  cudaStream_t stream) {
  using C = Cfg<PAIR, SQUARE>;
  auto kernel = gemm8_kernel<PAIR, SQUARE>;
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
  const long long units = (long long)p.m_tiles * p.n_tiles * p.splits;
  if (units > 0x7fffffff) return fail(HAPX_ERR_EXTENT, "block8_matmul: too many tiles");
  cfg.gridDim = dim3((unsigned)std::min<long long>(units, limit) * (PAIR ? 2 : 1));
  HAPX_CUDA(cudaLaunchKernelEx(&cfg, kernel, tmA, tmB, tmS, tmD, p));
  count_launch();
  return HAPX_OK;
}

static int run(void* d, int out_f32, const void* a, long long lda, const float* as, long long ldas, const void* b, long long ldb, const float* bs,
               long long ldbs, bool square, const void* bias, long long M, long long N, long long K, void* workspace, cudaStream_t stream) {
  unsigned* error = nullptr;
  int sm_count = 0;
  if (int e = gemm::error_word(&error, &sm_count)) return e;
  const Plan pl = plan_of(M, N, K, sm_count);
  Params p = Params();
  p.M = (int)M; p.N = (int)N; p.k_blocks = (int)((K + BK - 1) / BK);
  p.a_scale = as; p.lda_scale = ldas; p.b_scale = bs; p.ldb_scale = ldbs;
  p.splits = pl.splits; p.kb_per_split = pl.kb_per_split; p.m_pad = pl.m_pad;
  p.error = error;
  const int bm = pl.pair ? 2 * BM : BM, bn = pl.pair ? Cfg<true, true>::BN : Cfg<false, true>::BN;
  p.m_tiles = (p.M + bm - 1) / bm; p.n_tiles = (p.N + bn - 1) / bn;
  long long out_rows = M;
  if (pl.splits > 1) { p.D = workspace; p.ldd = pl.n_pad; p.out_f32 = 1; p.bias = nullptr; out_rows = pl.splits * pl.m_pad; }
  else { p.D = d; p.ldd = N; p.out_f32 = out_f32; p.bias = bias; }
  const int es = p.out_f32 ? 4 : 2;
  CUtensorMap tmA, tmB, tmS, tmD;
  std::memset(&tmS, 0, sizeof(tmS));
  std::memset(&tmD, 0, sizeof(tmD));
  if (int e = make_map(&tmA, a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, M, lda, BK, BM, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return e;
  if (int e = make_map(&tmB, b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, N, ldb, BK, pl.pair ? bn / 2 : bn, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return e;
  if (!square)
    if (int e = make_map(&tmS, bs, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, N, p.k_blocks, ldbs, bn, 1, CU_TENSOR_MAP_SWIZZLE_NONE,
                         CU_TENSOR_MAP_L2_PROMOTION_NONE)) return e;
  p.tma_store = (reinterpret_cast<uintptr_t>(p.D) & 15u) == 0 && (p.ldd * es) % 16 == 0;
  if (p.tma_store)
    if (int e = make_map(&tmD, p.D, p.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, es, pl.splits > 1 ? pl.n_pad : N,
                         out_rows, p.ldd, 128 / es, 32, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE)) return e;
  int e;
  if (pl.pair) e = square ? launch<true, true>(tmA, tmB, tmS, tmD, p, sm_count, stream) : launch<true, false>(tmA, tmB, tmS, tmD, p, sm_count, stream);
  else e = square ? launch<false, true>(tmA, tmB, tmS, tmD, p, sm_count, stream) : launch<false, false>(tmA, tmB, tmS, tmD, p, sm_count, stream);
  if (e) return e;
  if (pl.splits > 1) {
    const int grid = (int)std::min<long long>((M * (pl.n_pad / 4) + 255) / 256, (long long)sm_count * 8);
    const float* ws = static_cast<const float*>(workspace);
    if (out_f32) gemm8_join_kernel<<<grid, 256, 0, stream>>>(ws, pl.splits, M, p.N, pl.m_pad, pl.n_pad, static_cast<const float*>(bias), static_cast<float*>(d));
    else gemm8_join_kernel<<<grid, 256, 0, stream>>>(ws, pl.splits, M, p.N, pl.m_pad, pl.n_pad, static_cast<const __nv_bfloat16*>(bias),
                                                     static_cast<__nv_bfloat16*>(d));
    HAPX_CUDA(cudaGetLastError());
    count_launch();
  }
  return HAPX_OK;
}

}  // namespace gemm8
}  // namespace hapx

using namespace hapx;

extern "C" {

int64_t hapx_block8_matmul_workspace(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0 || m > 0x7fffffff || n > 0x7fffffff || k > 0x7fffffff) return 0;
  int sm_count = 0;
  if (gemm8::sm_count_of(&sm_count)) return 0;
  const gemm8::Plan pl = gemm8::plan_of(m, n, k, sm_count);
  return pl.splits > 1 ? (int64_t)pl.splits * pl.m_pad * pl.n_pad * 4 : 0;
}

int hapx_block8_matmul(void* d, int out_dtype, const void* a, int64_t lda, const float* a_scale, int64_t lda_scale, const void* b, int64_t ldb,
                       const float* b_scale, int64_t ldb_scale, int b_square, const void* bias, int64_t m, int64_t n, int64_t k,
                       void* workspace, int64_t workspace_bytes, hapx_stream stream) {
  if (out_dtype != HAPX_F32 && out_dtype != HAPX_BF16) return fail(HAPX_ERR_DTYPE, "block8_matmul: the output is float32 or bfloat16");
  if (m < 0 || n < 0 || k < 1 || m > 0x7fffffff || n > 0x7fffffff || k > 0x7fffffff)
    return fail(HAPX_ERR_EXTENT, "block8_matmul: extents must lie below 2^31, the contraction at 1 or above");
  if (m == 0 || n == 0) return HAPX_OK;
  if (!d || !a || !a_scale || !b || !b_scale) return fail(HAPX_ERR_ARGUMENT, "block8_matmul: null pointer");
  if (lda % 16 != 0 || ldb % 16 != 0 || lda < k || ldb < k || ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15u))
    return fail(HAPX_ERR_EXTENT, "block8_matmul: operands need a 16-byte aligned base and pitch, and a pitch that covers a row");
  if (lda_scale < m || ldb_scale < (b_square ? (n + 127) / 128 : n))
    return fail(HAPX_ERR_EXTENT, "block8_matmul: a scale pitch does not cover its rows");
  if (!b_square && (ldb_scale % 4 != 0 || (reinterpret_cast<uintptr_t>(b_scale) & 15u)))
    return fail(HAPX_ERR_EXTENT, "block8_matmul: the scales of 1 x 128 blocks of b need a 16-byte aligned base and pitch");
  const int64_t need = hapx_block8_matmul_workspace(m, n, k);
  if (workspace_bytes < need || (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u))))
    return fail(HAPX_ERR_ARGUMENT, "block8_matmul: the workspace must be 16-byte aligned and as large as hapx_block8_matmul_workspace says");
  return gemm8::run(d, out_dtype == HAPX_F32, a, lda, a_scale, lda_scale, b, ldb, b_scale, ldb_scale, b_square != 0, bias, m, n, k, workspace,
                    static_cast<cudaStream_t>(stream));
}

}  // extern "C"
