// Operators that keep their input for the backward pass in 8 bits (hapx_block8.h) instead of in the tensor's own type:
// the FFN's activation (with dropout) and layer_norm.  What is kept is a quarter (float32) or half (bfloat16) of the
// input's bytes, written by the forward kernel that has the values in registers anyway, and the backward kernel reads
// it instead of the input.
//
//   gelu       y = k gelu(x)              dx = dy k gelu'(x~)
//   relu       y = k max(x, 0)            dx = dy / (1 - p) where x > 0 and kept: one bit per element is all there is to keep
//   layer_norm y = (x - mean) rstd w + b  z = (x~ - mean) rstd,  g = dy w,  dx = rstd (g - mean(g) - z mean(g z)) [+ add],
//                                         dw = sum dy z,  db = sum dy      (mean and rstd of x itself, in float32)
//
// x~ is x to half a step of 3 fraction bits; forward results are those of the operators that keep x, to rounding (gelu has a
// distribution function of its own here, layer_norm adds in another order).
#include <algorithm>
#include <mutex>
#include <set>
#include <string>
#include <type_traits>
#include <utility>

#include "hapx_block8.h"
#include "hapx_internal.h"
#include "hapx_rng.h"

namespace hapx {
namespace saved8 {

using namespace block8;

enum Act { ACT_RELU = 1, ACT_GELU = 2 };

// Phi(v) = erfc(-v / sqrt 2) / 2 and e = exp(-v^2 / 2) = 2^(-u^2), u = |v| sqrt(log2(e) / 2).  For v < 0 it is the tail
// e t P(t) with t = 1 / (1 + 0.36 u): P is a least-maximum fit to erfcx(|v| / sqrt 2) / (2 t) over |v| <= 13, so the tail
// keeps most of its relative accuracy, which y = v Phi(v) needs, and shares its exponential with the density.  Degree 7 for
// float32 tensors (the fit is off by 1.0e-7 of itself), degree 5 for bfloat16 ones (4.1e-6, a 950th of their rounding).  The
// rounding of u and u^2 comes on top, which the exponential turns into (2 v^2 + 16) 2^-24 of the tail at most: measured in
// float32 5e-7 on [-1, 0], 2.6e-6 on [-5, -3], 4.8e-6 on [-8, -5], 1.3e-5 at -12.9.
template <bool WIDE>
__device__ __forceinline__ float normal_cdf(float v, float& e) {
  const float u = fabsf(v) * 0.84932180028801907f;
  float t;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.36f, u, 1.f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-u * u));
  float q;
  if (WIDE) {
    q = fmaf(0.03657762301083756f, t, -0.15125760273443148f);
    q = fmaf(q, t, 0.18092026515553128f);
    q = fmaf(q, t, -0.0342253215659978f);
    q = fmaf(q, t, 0.11920223581958944f);
    q = fmaf(q, t, 0.10414048504390966f);
    q = fmaf(q, t, 0.12269694252912236f);
    q = fmaf(q, t, 0.12194542414330234f);
  } else {
    q = fmaf(-0.07647082273966256f, t, 0.19837717655503154f);
    q = fmaf(q, t, -0.0008176733719744526f);
    q = fmaf(q, t, 0.1393556059441193f);
    q = fmaf(q, t, 0.11727338761580286f);
    q = fmaf(q, t, 0.1222832162766118f);
  }
  const float tail = q * t * e;
  return v >= 0.f ? 1.f - tail : tail;
}

// Eight consecutive elements as they are in memory (`vec`: p is aligned to 16 bytes), so that those of the next round can
// wait in registers.
template <typename T> struct Raw8;
template <> struct Raw8<__nv_bfloat16> {
  uint4 w;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, bool vec, int valid) {
    if (vec && valid >= 8) {
      w = *reinterpret_cast<const uint4*>(p);
    } else {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
      unsigned u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = (2 * i < valid ? h[2 * i] : 0u) | (2 * i + 1 < valid ? (unsigned)h[2 * i + 1] << 16 : 0u);
      w = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(u[i] << 16); f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
  }
};
template <> struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p, bool vec, int valid) {
    if (vec && valid >= 8) {
      a = *reinterpret_cast<const float4*>(p);
      b = *reinterpret_cast<const float4*>(p + 4);
    } else {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = j < valid ? p[j] : 0.f;
      a = make_float4(f[0], f[1], f[2], f[3]);
      b = make_float4(f[4], f[5], f[6], f[7]);
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
};
template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, int valid, const float (&f)[8]) {
  if (vec && valid >= 8) {
    if constexpr (sizeof(T) == 2) {
      unsigned u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        u[i] = *reinterpret_cast<const unsigned*>(&h);
      }
      *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
      *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < valid) p[j] = from_f<T>(f[j]);
  }
}

// A thread holds eight consecutive elements (one evaluation of the generator), sixteen lanes a block of 128; a warp takes
// kActUnroll pieces of 256 elements at a time, and fetches those of its next round before it works on the present ones
// (without that, waiting for loads was the largest share: 42 M bfloat16 elements of gelu in 52 us).  HBM-bound: those 42 M
// elements take 38.6 us = 5.4 TB/s each way with gelu, whose instructions come close behind, 28.8 = 6.0 TB/s with relu;
// in float32 62 and 60.
constexpr int kActUnroll = 2;
template <typename T, int ACT, bool DROP>
__global__ void __launch_bounds__(256) act_forward_kernel(const T* __restrict__ x, T* __restrict__ y, unsigned char* __restrict__ saved,
                                                          float* __restrict__ scales, long long n, unsigned threshold, float keep_scale,
                                                          const rng::State* st, unsigned long long call_id) {
  const int lane = threadIdx.x & 31;
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15u) == 0;
  rng::Key key = {0u, 0u, 0u, 0u};
  if (DROP) key = rng::make_key(st, call_id);
  constexpr int kPiece = 256 * kActUnroll;
  const long long pieces = (n + kPiece - 1) / kPiece, stride = (long long)gridDim.x * 8, first = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  Raw8<T> next[kActUnroll];
  auto fetch = [&](long long piece) {
    const long long at = piece * kPiece + 8 * lane;
    const bool inside = vec && (piece + 1) * kPiece <= n;
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      if (inside) next[u].load(x + at + 256 * u, true, 8);
      else next[u].load(x + at + 256 * u, vec, (int)max(0ll, min(8ll, n - (at + 256 * u))));
    }
  };
  auto work = [&](long long piece, auto full_tag) {
    constexpr bool FULL = decltype(full_tag)::value;
    const long long at = piece * kPiece + 8 * lane;
    T* yp = y + at;
    unsigned char* sp = saved + (ACT == ACT_RELU ? at >> 3 : at);
    float* cp = scales + at / kBlock;
    float v[kActUnroll][8];
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) next[u].get(v[u]);
    if (piece + stride < pieces) fetch(piece + stride);
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int valid = FULL ? 8 : (int)max(0ll, min(8ll, n - (at + 256 * u)));
      unsigned keep = 0xffu, bits = 0u;
      if (DROP) keep = rng::keep_bits(rng::philox(key, (unsigned long long)((at + 256 * u) >> 3)), threshold);
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float w = v[u][j];
        if (ACT == ACT_RELU) {
          o[j] = w <= 0.f ? 0.f : w;                // NaN passes
          bits |= (w > 0.f ? 1u : 0u) << j;
        } else {
          float e;
          o[j] = w * normal_cdf<sizeof(T) == 4>(w, e);
        }
        if (DROP) o[j] *= (keep >> j) & 1u ? keep_scale : 0.f;
      }
      store8(yp + 256 * u, FULL || vec, valid, o);
      if (!saved) continue;                         // nothing asks for a gradient
      if (ACT == ACT_RELU) {
        if (FULL || valid > 0) sp[32 * u] = (unsigned char)(bits & keep);
      } else {
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(v[u][j]));          // a NaN loses
        if (__any_sync(0xffffffffu, big == __uint_as_float(0x7f800000u))) {    // rare: infinities become NaN
          big = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) { v[u][j] = finite_or_nan(v[u][j]); big = fmaxf(big, fabsf(v[u][j])); }
        }
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
        const int e = scale_exponent(big);
        const float inv = pow2(-e);
        if ((lane & 15) == 0 && (FULL || valid > 0)) cp[2 * u] = pow2(e);
        if (FULL || valid > 0)        // n rounded up to 8 bytes
          *reinterpret_cast<uint2*>(sp + 256 * u) = make_uint2(pack4(v[u][0] * inv, v[u][1] * inv, v[u][2] * inv, v[u][3] * inv),
                                                               pack4(v[u][4] * inv, v[u][5] * inv, v[u][6] * inv, v[u][7] * inv));
      }
    }
  };
  if (first < pieces) fetch(first);
  const long long whole = vec ? n / kPiece : 0;     // pieces that lie inside the tensor, aligned
  long long piece = first;
  for (; piece < whole; piece += stride) work(piece, std::true_type{});
  for (; piece < pieces; piece += stride) work(piece, std::false_type{});
}

// The same split and the same look-ahead; reads the incoming gradient and the 8-bit input (or the bit).  A scale of 2^120
// (inputs above 2^127) is taken as 2^119: 256 * 2^120 is no float32 number, and the slope is 0 or 1 at either.
template <typename T, int ACT, bool DROP>
__global__ void __launch_bounds__(256) act_backward_kernel(const T* __restrict__ dy, const unsigned char* __restrict__ saved,
                                                           const float* __restrict__ scales, T* __restrict__ dx, long long n,
                                                           unsigned threshold, float keep_scale, const rng::State* st,
                                                           unsigned long long call_id) {
  const int lane = threadIdx.x & 31;
  const bool vec = ((reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(dx)) & 15u) == 0;
  rng::Key key = {0u, 0u, 0u, 0u};
  if (ACT == ACT_GELU && DROP) key = rng::make_key(st, call_id);
  constexpr int kPiece = 256 * kActUnroll;
  const long long pieces = (n + kPiece - 1) / kPiece, stride = (long long)gridDim.x * 8, first = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  Raw8<T> next[kActUnroll];
  uint2 next_w[kActUnroll];
  float next_s[kActUnroll];
  auto fetch = [&](long long piece) {
    const long long at = piece * kPiece + 8 * lane;
    const unsigned char* sp = saved + (ACT == ACT_RELU ? at >> 3 : at);
    const float* cp = scales + at / kBlock;
    const bool inside = vec && (piece + 1) * kPiece <= n;
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int valid = inside ? 8 : (int)max(0ll, min(8ll, n - (at + 256 * u)));
      if (inside) next[u].load(dy + at + 256 * u, true, 8);
      else next[u].load(dy + at + 256 * u, vec, valid);
      next_w[u] = make_uint2(0u, 0u);
      next_s[u] = 0.f;
      if (valid > 0) {
        if (ACT == ACT_RELU) next_w[u].x = sp[32 * u];
        else { next_w[u] = *reinterpret_cast<const uint2*>(sp + 256 * u); next_s[u] = fminf(cp[2 * u], 0x1p119f); }
      }
    }
  };
  auto work = [&](long long piece, auto full_tag) {
    constexpr bool FULL = decltype(full_tag)::value;
    const long long at = piece * kPiece + 8 * lane;
    float d[kActUnroll][8], s[kActUnroll];
    uint2 w[kActUnroll];
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) { next[u].get(d[u]); w[u] = next_w[u]; s[u] = next_s[u]; }
    if (piece + stride < pieces) fetch(piece + stride);
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int valid = FULL ? 8 : (int)max(0ll, min(8ll, n - (at + 256 * u)));
      float o[8];
      if (ACT == ACT_RELU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (w[u].x >> j) & 1u ? d[u][j] * keep_scale : 0.f;
      } else {
        unsigned keep = 0xffu;
        if (DROP) keep = rng::keep_bits(rng::philox(key, (unsigned long long)((at + 256 * u) >> 3)), threshold);
        const unsigned half[4] = {w[u].x & 0xffffu, w[u].x >> 16, w[u].y & 0xffffu, w[u].y >> 16};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 two = unpack2(half[j >> 1]);
          const float h = (j & 1 ? two.y : two.x) * s[u];
          float e;
          const float cdf = normal_cdf<sizeof(T) == 4>(h, e);
          o[j] = d[u][j] * fmaf(h * 0.3989422804014327f, e, cdf);
          if (DROP) o[j] *= (keep >> j) & 1u ? keep_scale : 0.f;
        }
      }
      store8(dx + at + 256 * u, FULL || vec, valid, o);
    }
  };
  if (first < pieces) fetch(first);
  const long long whole = vec ? n / kPiece : 0;     // pieces that lie inside the tensor, aligned
  long long piece = first;
  for (; piece < whole; piece += stride) work(piece, std::true_type{});
  for (; piece < pieces; piece += stride) work(piece, std::false_type{});
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---- layer_norm ---------------------------------------------------------------------------------------
// A row belongs to a team of W warps; warp w of it holds the groups of 256 columns w, w + W, ... (NG of them at most) in
// registers, lane l the columns 8l .. 8l + 7 of each, so that sixteen lanes hold a block of 128.  A thread block has 8 / W
// teams, and a team fetches its next row before it works on the present one.  Rows of up to 8192 columns are read once;
// longer ones take the kernels below these.  VEC: rows and parameters lie on 16 bytes and E is a multiple of 8.
constexpr int kTeamColumns = 8192;

// Sum over a team (`s`: one float per warp of the block, reused after the next call's other buffer).
template <int W>
__device__ __forceinline__ float team_sum(float v, float* s, int warp) {
  v = warp_sum(v);
  if constexpr (W > 1) {
    if ((threadIdx.x & 31) == 0) s[warp] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / W), "n"(32 * W) : "memory");
    const int first = warp / W * W;
    v = s[first];
#pragma unroll
    for (int i = 1; i < W; ++i) v += s[first + i];
  }
  return v;
}

// Columns of a thread's eight that lie inside the row.
template <bool VEC>
__device__ __forceinline__ int valid_of(int E, int c) { return VEC ? (c < E ? 8 : 0) : max(0, min(8, E - c)); }

// A team of W warps holds a row in registers (a lane's eight columns, NG groups of them) and has the next row's loads in
// flight; mean, then the mean of squared distances, then y and the blocks of x from the same registers.  By its bytes
// HBM-bound; measured it is the chain of a row's two sums and sixteen-lane maxima with few warps to hide it (three groups of
// 256 columns take all 128 registers that two blocks per SM leave: 16 warps): bfloat16 8192 x 768 9.4 us = 3.4 TB/s,
// 2048 x 8192 20.5, float32 4000 x 2040 16.1 = 4.6 TB/s.
template <typename T, int W, int NG, bool VEC>
__global__ void __launch_bounds__(256, 2) norm_forward_team_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b,
                                                                   T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                                   unsigned char* __restrict__ q, long long ldq, float* __restrict__ s, long long rows,
                                                                   int E, float eps) {
  __shared__ float s_sum[2][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % W, blocks = (E + kBlock - 1) / kBlock;
  Raw8<T> next[NG];
  const float inv_e = 1.f / (float)E;
  const long long stride = (long long)gridDim.x * (8 / W);
  auto fetch = [&](long long row) {
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int c = (part + k * W) * 256 + 8 * lane;
      next[k].load(x + row * E + c, VEC, valid_of<VEC>(E, c));
    }
  };
  long long row = (long long)blockIdx.x * (8 / W) + warp / W;
  if (row < rows) fetch(row);
  for (; row < rows; row += stride) {
    float v[NG][8], sum = 0.f;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      next[k].get(v[k]);
      sum += ((v[k][0] + v[k][1]) + (v[k][2] + v[k][3])) + ((v[k][4] + v[k][5]) + (v[k][6] + v[k][7]));
    }
    if (row + stride < rows) fetch(row + stride);
    const float mean = team_sum<W>(sum, s_sum[0], warp) * inv_e;
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int valid = valid_of<VEC>(E, (part + k * W) * 256 + 8 * lane);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = j < valid ? v[k][j] - mean : 0.f;
        sq = fmaf(d, d, sq);
      }
    }
    const float rstd = rsqrtf(team_sum<W>(sq, s_sum[1], warp) * inv_e + eps);
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int c = (part + k * W) * 256 + 8 * lane, valid = valid_of<VEC>(E, c);
      float o[8], f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = (v[k][j] - mean) * rstd;
      if (w) {
        Raw8<T> p;
        p.load(w + c, VEC, valid);                 // from the first-level cache, row after row
        p.get(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] *= f[j];
      }
      if (b) {
        Raw8<T> p;
        p.load(b + c, VEC, valid);
        p.get(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += f[j];
      }
      store8(y + row * E + c, VEC, valid, o);
      if (q) {                                     // a gradient is asked for
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(v[k][j]));            // a NaN loses
        if (__any_sync(0xffffffffu, big == __uint_as_float(0x7f800000u))) {      // rare: infinities become NaN
          big = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) { v[k][j] = finite_or_nan(v[k][j]); big = fmaxf(big, fabsf(v[k][j])); }
        }
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
        const int e = scale_exponent(big);
        const float inv = pow2(-e);
        if (valid > 0) {
          if ((lane & 15) == 0) s[row * blocks + c / kBlock] = pow2(e);
          *reinterpret_cast<uint2*>(q + row * ldq + c) = make_uint2(pack4(v[k][0] * inv, v[k][1] * inv, v[k][2] * inv, v[k][3] * inv),
                                                                    pack4(v[k][4] * inv, v[k][5] * inv, v[k][6] * inv, v[k][7] * inv));
        }
      }
    }
    if (q && part == 0 && lane == 0) { mean_out[row] = mean; rstd_out[row] = rstd; }
  }
}

// dx of the rows, and partial[block][0][c] = sum dy z, partial[block][1][c] = sum dy over the rows the thread block took.  The
// running sums of a warp's columns lie in shared memory, owned by the warp: in registers, next to the prefetched row, they
// would leave half of the warps.  Bound by the row's chain, again with 16 warps per SM (bfloat16 rows of 513 to 768 columns and
// of more than 4096 spill a few registers even so), and by adding to those sums (with the join of the partials 8192 x 768
// takes 15.2 us = 2.1 TB/s, with the residual's gradient 16.1; float32 4000 x 2040 25.0 = 2.9 TB/s).
template <typename T, int W, int NG, bool VEC>
__global__ void __launch_bounds__(256, 2) norm_backward_team_kernel(const unsigned char* __restrict__ q, long long ldq, const float* __restrict__ s,
                                                                    const T* __restrict__ dy, const T* __restrict__ w,
                                                                    const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                                    const T* __restrict__ add, T* __restrict__ dx, float* __restrict__ partial,
                                                                    long long rows, int E) {
  extern __shared__ float4 s_acc[];               // [warp][NG][dw: first and second four columns, db: the same][32 lanes]
  __shared__ float s_sum[2][2][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % W, blocks = (E + kBlock - 1) / kBlock;
  constexpr bool KEEP = sizeof(T) == 2;            // the residual gradient of the next row is fetched ahead too
  float4* acc = s_acc + (long long)warp * NG * 128 + lane;
  if (partial) {
#pragma unroll
    for (int k = 0; k < 4 * NG; ++k) acc[32 * k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  Raw8<T> next_g[NG], next_r[KEEP ? NG : 1];
  uint2 next_q[NG];
  float next_s[NG], next_mean = 0.f, next_rstd = 0.f;
  auto fetch = [&](long long row) {
    next_mean = mean_in[row];
    next_rstd = rstd_in[row];
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int c = (part + k * W) * 256 + 8 * lane, valid = valid_of<VEC>(E, c);
      next_g[k].load(dy + row * E + c, VEC, valid);
      if (KEEP && add) next_r[k].load(add + row * E + c, VEC, valid);
      next_q[k] = valid > 0 ? *reinterpret_cast<const uint2*>(q + row * ldq + c) : make_uint2(0u, 0u);
      next_s[k] = valid > 0 ? s[row * blocks + c / kBlock] : 0.f;
    }
  };
  const float inv_e = 1.f / (float)E;
  const long long stride = (long long)gridDim.x * (8 / W);
  int flip = 0;
  long long row = (long long)blockIdx.x * (8 / W) + warp / W;
  if (row < rows) fetch(row);
  for (; row < rows; row += stride, flip ^= 1) {
    const float mean = next_mean, rstd = next_rstd;
    Raw8<T> res[KEEP ? NG : 1];
    float g[NG][8], z[NG][8], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int valid = valid_of<VEC>(E, (part + k * W) * 256 + 8 * lane);
      next_g[k].get(g[k]);
      const unsigned half[4] = {next_q[k].x & 0xffffu, next_q[k].x >> 16, next_q[k].y & 0xffffu, next_q[k].y >> 16};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 two = unpack2(half[i]);
        z[k][2 * i] = 2 * i < valid ? fmaf(two.x, next_s[k], -mean) * rstd : 0.f;       // two.x times its scale is exact
        z[k][2 * i + 1] = 2 * i + 1 < valid ? fmaf(two.y, next_s[k], -mean) * rstd : 0.f;
      }
      if (KEEP && add) res[k] = next_r[k];
    }
    if (row + stride < rows) fetch(row + stride);
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int c = (part + k * W) * 256 + 8 * lane, valid = valid_of<VEC>(E, c);
      if (partial) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float4 a = acc[128 * k + 32 * h], d = acc[128 * k + 64 + 32 * h];
          a.x = fmaf(g[k][4 * h], z[k][4 * h], a.x); a.y = fmaf(g[k][4 * h + 1], z[k][4 * h + 1], a.y);
          a.z = fmaf(g[k][4 * h + 2], z[k][4 * h + 2], a.z); a.w = fmaf(g[k][4 * h + 3], z[k][4 * h + 3], a.w);
          d.x += g[k][4 * h]; d.y += g[k][4 * h + 1]; d.z += g[k][4 * h + 2]; d.w += g[k][4 * h + 3];
          acc[128 * k + 32 * h] = a;
          acc[128 * k + 64 + 32 * h] = d;
        }
      }
      if (w) {
        Raw8<T> p;
        float f[8];
        p.load(w + c, VEC, valid);
        p.get(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[k][j] *= f[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) { s1 += g[k][j]; s2 = fmaf(g[k][j], z[k][j], s2); }
    }
    const float m1 = team_sum<W>(s1, s_sum[flip][0], warp) * inv_e, m2 = team_sum<W>(s2, s_sum[flip][1], warp) * inv_e;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const int c = (part + k * W) * 256 + 8 * lane, valid = valid_of<VEC>(E, c);
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = rstd * (g[k][j] - m1 - z[k][j] * m2);
      if (add) {
        Raw8<T> p;
        float f[8];
        if (KEEP) p = res[k]; else p.load(add + row * E + c, VEC, valid);
        p.get(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += f[j];
      }
      store8(dx + row * E + c, VEC, valid, o);
    }
  }
  if (!partial) return;
  __syncthreads();
  // the block's teams, in their order
  float* out = partial + (long long)blockIdx.x * 2 * E;
  const float* flat = reinterpret_cast<const float*>(s_acc);
  for (int i = threadIdx.x; i < 2 * E; i += 256) {
    const int which = i >= E, c = which ? i - E : i, group = c >> 8, in_lane = c & 7, at = (c >> 3) & 31;
    const int offset = (2 * which + (in_lane >> 2)) * 128 + at * 4 + (in_lane & 3);
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < 8 / W; ++t) sum += flat[((t * W + group % W) * NG + group / W) * 512 + offset];
    out[i] = sum;
  }
}

// Rows of more than kTeamColumns: one warp per row, which is read three times, twice from the caches.
template <typename T>
__global__ void __launch_bounds__(128) norm_forward_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b,
                                                           T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                           unsigned char* __restrict__ q, long long ldq, float* __restrict__ s, long long rows,
                                                           int E, float eps) {
  const int lane = threadIdx.x & 31, blocks = (E + kBlock - 1) / kBlock;
  const bool vec = (E & 3) == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(w) |
                                     reinterpret_cast<uintptr_t>(b)) & (4 * sizeof(T) - 1)) == 0;
  for (long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5); row < rows; row += (long long)gridDim.x * 4) {
    const T* xr = x + row * E;
    float sum = 0.f;
    for (int k = 0; k < blocks; ++k) {
      const int c = k * kBlock + 4 * lane, valid = max(0, min(4, E - c));
      float v[4];
      load4(xr + c, vec, valid, v);
      sum += (v[0] + v[1]) + (v[2] + v[3]);
    }
    const float mean = warp_sum(sum) / (float)E;
    float sq = 0.f;
    for (int k = 0; k < blocks; ++k) {
      const int c = k * kBlock + 4 * lane, valid = max(0, min(4, E - c));
      float v[4];
      load4(xr + c, vec, valid, v);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < valid) sq = fmaf(v[j] - mean, v[j] - mean, sq);
    }
    const float rstd = rsqrtf(warp_sum(sq) / (float)E + eps);
    for (int k = 0; k < blocks; ++k) {
      const int c = k * kBlock + 4 * lane, valid = max(0, min(4, E - c));
      float v[4], g[4] = {1.f, 1.f, 1.f, 1.f}, h[4] = {0.f, 0.f, 0.f, 0.f}, o[4], big = 0.f;
      load4(xr + c, vec, valid, v);
      if (w) load4(w + c, vec, valid, g);
      if (b) load4(b + c, vec, valid, h);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j] = fmaf((v[j] - mean) * rstd, g[j], h[j]);
        v[j] = finite_or_nan(v[j]);
        big = fmaxf(big, fabsf(v[j]));
      }
      store4(y + row * E + c, vec, valid, o);
      if (!q) continue;                             // nothing asks for a gradient
      const int e = scale_exponent(warp_max(big));
      const float inv = pow2(-e);
      if (lane == 0) s[row * blocks + k] = pow2(e);
      if (valid > 0) *reinterpret_cast<unsigned*>(q + row * ldq + c) = pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    }
    if (q && lane == 0) { mean_out[row] = mean; rstd_out[row] = rstd; }
  }
}

// dx of such rows: one warp per row, two passes (the two means, then dx), the second from the caches.
template <typename T>
__global__ void __launch_bounds__(128) norm_backward_kernel(const unsigned char* __restrict__ q, long long ldq, const float* __restrict__ s,
                                                            const T* __restrict__ dy, const T* __restrict__ w, const float* __restrict__ mean_in,
                                                            const float* __restrict__ rstd_in, const T* __restrict__ add, T* __restrict__ dx,
                                                            long long rows, int E) {
  const int lane = threadIdx.x & 31, blocks = (E + kBlock - 1) / kBlock;
  const bool vec = (E & 3) == 0 && ((reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(w) |
                                     reinterpret_cast<uintptr_t>(add)) & (4 * sizeof(T) - 1)) == 0;
  for (long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5); row < rows; row += (long long)gridDim.x * 4) {
    const float mean = mean_in[row], rstd = rstd_in[row];
    auto load = [&](int k, int valid, float (&g)[4], float (&z)[4]) {
      const int c = k * kBlock + 4 * lane;
      float ww[4] = {1.f, 1.f, 1.f, 1.f};
      load4(dy + row * E + c, vec, valid, g);
      if (w) load4(w + c, vec, valid, ww);
      const unsigned v = valid > 0 ? *reinterpret_cast<const unsigned*>(q + row * ldq + c) : 0u;
      const float sc = s[row * blocks + k];
      const float2 lo = unpack2(v & 0xffffu), hi = unpack2(v >> 16);
      const float h[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
      for (int j = 0; j < 4; ++j) { g[j] *= ww[j]; z[j] = j < valid ? (h[j] * sc - mean) * rstd : 0.f; }
    };
    float s1 = 0.f, s2 = 0.f;
    for (int k = 0; k < blocks; ++k) {
      float g[4], z[4];
      load(k, max(0, min(4, E - (k * kBlock + 4 * lane))), g, z);
#pragma unroll
      for (int j = 0; j < 4; ++j) { s1 += g[j]; s2 = fmaf(g[j], z[j], s2); }
    }
    const float m1 = warp_sum(s1) / (float)E, m2 = warp_sum(s2) / (float)E;
    for (int k = 0; k < blocks; ++k) {
      const int c = k * kBlock + 4 * lane, valid = max(0, min(4, E - c));
      float g[4], z[4], o[4], r[4] = {0.f, 0.f, 0.f, 0.f};
      load(k, valid, g, z);
      if (add) load4(add + row * E + c, vec, valid, r);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = rstd * (g[j] - m1 - z[j] * m2) + r[j];
      store4(dx + row * E + c, vec, valid, o);
    }
  }
}

// partial[slice][0][c] = sum dy z, partial[slice][1][c] = sum dy over the slice's rows.
constexpr int kSliceRows = 64;
template <typename T>
__global__ void __launch_bounds__(128) norm_param_partial_kernel(const unsigned char* __restrict__ q, long long ldq, const float* __restrict__ s,
                                                                 const T* __restrict__ dy, const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd, float* __restrict__ partial, long long rows, int E) {
  const int c = blockIdx.x * kBlock + threadIdx.x, blocks = (E + kBlock - 1) / kBlock;
  if (c >= E) return;
  for (long long slice = blockIdx.y; slice * kSliceRows < rows; slice += gridDim.y) {
    float dw = 0.f, db = 0.f;
    for (long long r = slice * kSliceRows; r < min(rows, (slice + 1) * kSliceRows); ++r) {
      const float g = to_f(dy[r * E + c]);
      dw = fmaf(g, (unpack2(q[r * ldq + c]).x * s[r * blocks + blockIdx.x] - mean[r]) * rstd[r], dw);
      db += g;
    }
    partial[slice * 2 * E + c] = dw;
    partial[slice * 2 * E + E + c] = db;
  }
}

// dw[c], db[c]: the partial rows in a fixed order - warp w of 32 takes rows w, w + 32, ..., the 32 sums are added in order.
template <typename T>
__global__ void __launch_bounds__(1024) norm_param_join_kernel(const float* __restrict__ partial, long long slices, int E, T* __restrict__ dw,
                                                               T* __restrict__ db) {
  __shared__ float s_sum[32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (e < 2 * E)
#pragma unroll 4
    for (long long i = warp; i < slices; i += 32) sum += partial[i * 2 * E + e];
  s_sum[warp][lane] = sum;
  __syncthreads();
  if (warp != 0 || e >= 2 * E) return;
#pragma unroll
  for (int w = 1; w < 32; ++w) sum += s_sum[w][lane];
  if (e < E) { if (dw) dw[e] = from_f<T>(sum); }
  else if (db) db[e - E] = from_f<T>(sum);
}

static int grid_for(long long blocks, int per_sm, int* grid) {
  int n_sm = 0;
  if (int e = sm_count(&n_sm)) return e;
  *grid = (int)std::max<long long>(1, std::min<long long>(blocks, (long long)n_sm * per_sm));
  return HAPX_OK;
}

static int check_act(const char* who, int dtype, int64_t n, int act, double p) {
  if (dtype != HAPX_F32 && dtype != HAPX_BF16) return fail(HAPX_ERR_DTYPE, std::string(who) + ": float32 or bfloat16 only");
  if (n < 0) return fail(HAPX_ERR_EXTENT, std::string(who) + ": negative size");
  if (act != ACT_RELU && act != ACT_GELU) return fail(HAPX_ERR_ARGUMENT, std::string(who) + ": act must be 1 (relu) or 2 (gelu)");
  if (!(p >= 0.0 && p < 1.0)) return fail(HAPX_ERR_ARGUMENT, std::string(who) + ": p must be in [0, 1)");
  return HAPX_OK;
}

static int check_norm(const char* who, int dtype, int64_t rows, int64_t E) {
  if (dtype != HAPX_F32 && dtype != HAPX_BF16) return fail(HAPX_ERR_DTYPE, std::string(who) + ": float32 or bfloat16 only");
  if (rows < 0 || E < 1 || E > (1 << 20)) return fail(HAPX_ERR_EXTENT, std::string(who) + ": the normalised dimension must lie in [1, 2^20]");
  return HAPX_OK;
}

// Warps per row, and groups of 256 columns per warp at most, for a row of E <= kTeamColumns.
static int team_warps(long long E) { return E <= 768 ? 1 : E <= 1024 ? 2 : E <= 2048 ? 4 : 8; }
#define HAPX_LN8_SWITCH(E)                  \
  if ((E) <= 256) HAPX_LN8_TEAM(1, 1);      \
  else if ((E) <= 512) HAPX_LN8_TEAM(1, 2); \
  else if ((E) <= 768) HAPX_LN8_TEAM(1, 3); \
  else if ((E) <= 1024) HAPX_LN8_TEAM(2, 2); \
  else if ((E) <= 2048) HAPX_LN8_TEAM(4, 2); \
  else if ((E) <= 4096) HAPX_LN8_TEAM(8, 2); \
  else if ((E) <= kTeamColumns) HAPX_LN8_TEAM(8, 4);

static bool on_16_bytes(const void* a, const void* b, const void* c, const void* d) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(d)) & 15u) == 0;
}

// 64 KiB of dynamic shared memory for a kernel on the current device (asked for once).
static int allow_shared(const void* kernel) {
  static std::mutex mutex;
  static std::set<std::pair<int, const void*>> known;
  int device = 0;
  HAPX_CUDA(cudaGetDevice(&device));
  std::lock_guard<std::mutex> lock(mutex);
  if (known.count({device, kernel})) return HAPX_OK;
  HAPX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024));
  known.insert({device, kernel});
  return HAPX_OK;
}

}  // namespace saved8
}  // namespace hapx

using namespace hapx;
using namespace hapx::saved8;

extern "C" {

int hapx_act_dropout8(void* y, void* saved, float* scales, const void* x, int dtype, int64_t n, int act, double p, uint64_t call_id,
                      hapx_stream stream_) {
  if (int e = check_act("act_dropout8", dtype, n, act, p)) return e;
  if (n == 0) return HAPX_OK;
  if (!y || !x || (act == ACT_GELU && saved && !scales)) return fail(HAPX_ERR_ARGUMENT, "act_dropout8: null pointer");
  if (act == ACT_GELU && (reinterpret_cast<uintptr_t>(saved) & 15u)) return fail(HAPX_ERR_EXTENT, "act_dropout8: `saved` must be 16-byte aligned");
  const unsigned thr = p > 0.0 ? rng::threshold_for(p) : 0u;
  rng::State* st = nullptr;
  if (thr)
    if (int e = rng_state(&st)) return e;
  int grid = 1;
  if (int e = grid_for((n + 2048 * kActUnroll - 1) / (2048 * kActUnroll), 8, &grid)) return e;
  const float ks = thr ? (float)(1.0 / (1.0 - p)) : 1.f;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  unsigned char* sv = static_cast<unsigned char*>(saved);
#define HAPX_ACT8(T, A)                                                                                                                     \
  do {                                                                                                                                      \
    if (thr) act_forward_kernel<T, A, true><<<grid, 256, 0, stream>>>(static_cast<const T*>(x), static_cast<T*>(y), sv, scales, n, thr, ks, st, call_id); \
    else act_forward_kernel<T, A, false><<<grid, 256, 0, stream>>>(static_cast<const T*>(x), static_cast<T*>(y), sv, scales, n, thr, ks, st, call_id);    \
  } while (0)
  if (dtype == HAPX_BF16) { if (act == ACT_RELU) HAPX_ACT8(__nv_bfloat16, ACT_RELU); else HAPX_ACT8(__nv_bfloat16, ACT_GELU); }
  else { if (act == ACT_RELU) HAPX_ACT8(float, ACT_RELU); else HAPX_ACT8(float, ACT_GELU); }
#undef HAPX_ACT8
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

int hapx_act_dropout8_backward(void* dx, const void* dy, const void* saved, const float* scales, int dtype, int64_t n, int act, double p,
                               uint64_t call_id, hapx_stream stream_) {
  if (int e = check_act("act_dropout8_backward", dtype, n, act, p)) return e;
  if (n == 0) return HAPX_OK;
  if (!dx || !dy || !saved || (act == ACT_GELU && !scales)) return fail(HAPX_ERR_ARGUMENT, "act_dropout8_backward: null pointer");
  if (act == ACT_GELU && (reinterpret_cast<uintptr_t>(saved) & 15u))
    return fail(HAPX_ERR_EXTENT, "act_dropout8_backward: `saved` must be 16-byte aligned");
  const unsigned thr = p > 0.0 ? rng::threshold_for(p) : 0u;
  rng::State* st = nullptr;
  if (thr)
    if (int e = rng_state(&st)) return e;
  int grid = 1;
  if (int e = grid_for((n + 2048 * kActUnroll - 1) / (2048 * kActUnroll), 8, &grid)) return e;
  const float ks = thr ? (float)(1.0 / (1.0 - p)) : 1.f;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const unsigned char* sv = static_cast<const unsigned char*>(saved);
#define HAPX_ACT8(T, A)                                                                                                                      \
  do {                                                                                                                                       \
    if (thr) act_backward_kernel<T, A, true><<<grid, 256, 0, stream>>>(static_cast<const T*>(dy), sv, scales, static_cast<T*>(dx), n, thr, ks, st, call_id); \
    else act_backward_kernel<T, A, false><<<grid, 256, 0, stream>>>(static_cast<const T*>(dy), sv, scales, static_cast<T*>(dx), n, thr, ks, st, call_id);    \
  } while (0)
  if (dtype == HAPX_BF16) { if (act == ACT_RELU) HAPX_ACT8(__nv_bfloat16, ACT_RELU); else HAPX_ACT8(__nv_bfloat16, ACT_GELU); }
  else { if (act == ACT_RELU) HAPX_ACT8(float, ACT_RELU); else HAPX_ACT8(float, ACT_GELU); }
#undef HAPX_ACT8
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

int hapx_layer_norm8_forward(const void* x, const void* gamma, const void* beta, void* y, float* mean, float* rstd, void* saved, int64_t ld_saved,
                             float* scales, int dtype, int64_t rows, int64_t E, double eps, hapx_stream stream_) {
  if (int e = check_norm("layer_norm8_forward", dtype, rows, E)) return e;
  if (rows == 0) return HAPX_OK;
  if (!x || !y || (saved && (!mean || !rstd || !scales))) return fail(HAPX_ERR_ARGUMENT, "layer_norm8_forward: null argument");
  if (saved && (ld_saved < E || ld_saved % 16 != 0 || (reinterpret_cast<uintptr_t>(saved) & 15u)))
    return fail(HAPX_ERR_EXTENT, "layer_norm8_forward: `saved` needs a 16-byte aligned base and pitch, and a pitch that covers a row");
  int grid = 1;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  unsigned char* q = static_cast<unsigned char*>(saved);
#define HAPX_LN8(T, KERNEL, THREADS) \
  KERNEL<<<grid, THREADS, 0, stream>>>(static_cast<const T*>(x), static_cast<const T*>(gamma), static_cast<const T*>(beta), static_cast<T*>(y), mean, \
                                       rstd, q, ld_saved, scales, rows, (int)E, (float)eps)
  const bool vec = E % 8 == 0 && on_16_bytes(x, y, gamma, beta);
#define HAPX_LN8_TEAM(W, NG)                                                                                                     \
  do {                                                                                                                           \
    if (int e = grid_for((rows + 8 / W - 1) / (8 / W), 2, &grid)) return e;                                                      \
    if (dtype == HAPX_BF16) { if (vec) HAPX_LN8(__nv_bfloat16, (norm_forward_team_kernel<__nv_bfloat16, W, NG, true>), 256);     \
                              else HAPX_LN8(__nv_bfloat16, (norm_forward_team_kernel<__nv_bfloat16, W, NG, false>), 256); }      \
    else { if (vec) HAPX_LN8(float, (norm_forward_team_kernel<float, W, NG, true>), 256);                                        \
           else HAPX_LN8(float, (norm_forward_team_kernel<float, W, NG, false>), 256); }                                         \
  } while (0)
  HAPX_LN8_SWITCH(E)
  else {
    if (int e = grid_for((rows + 3) / 4, 16, &grid)) return e;
    if (dtype == HAPX_BF16) HAPX_LN8(__nv_bfloat16, norm_forward_kernel<__nv_bfloat16>, 128);
    else HAPX_LN8(float, norm_forward_kernel<float>, 128);
  }
#undef HAPX_LN8_TEAM
#undef HAPX_LN8
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

int64_t hapx_layer_norm8_backward_workspace(int64_t rows, int64_t E) {
  int grid = 1;
  if (E < 1 || rows < 0) return 0;
  int64_t slices = (rows + kSliceRows - 1) / kSliceRows;
  if (E <= kTeamColumns) {
    if (grid_for((rows + 8 / team_warps(E) - 1) / (8 / team_warps(E)), 2, &grid)) return 0;
    slices = grid;
  }
  return std::max<int64_t>(1, slices) * 2 * E * (int64_t)sizeof(float);
}

int hapx_layer_norm8_backward(const void* saved, int64_t ld_saved, const float* scales, const void* dy, const void* gamma, const float* mean,
                              const float* rstd, const void* add, void* dx, void* dgamma, void* dbeta, float* workspace, int dtype, int64_t rows,
                              int64_t E, hapx_stream stream_) {
  if (int e = check_norm("layer_norm8_backward", dtype, rows, E)) return e;
  if (rows > 0 && (!saved || !scales || !dy || !mean || !rstd || !dx)) return fail(HAPX_ERR_ARGUMENT, "layer_norm8_backward: null argument");
  if ((dgamma || dbeta) && !workspace) return fail(HAPX_ERR_ARGUMENT, "layer_norm8_backward: null workspace");
  if (rows > 0 && (ld_saved < E || ld_saved % 16 != 0 || (reinterpret_cast<uintptr_t>(saved) & 15u)))
    return fail(HAPX_ERR_EXTENT, "layer_norm8_backward: `saved` needs a 16-byte aligned base and pitch, and a pitch that covers a row");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const unsigned char* q = static_cast<const unsigned char*>(saved);
  const bool params = dgamma || dbeta;
  float* partial = params ? workspace : nullptr;
  long long slices = 0;
  int grid = 1;
  if (rows > 0) {
    const bool vec = E % 8 == 0 && on_16_bytes(dy, dx, gamma, add);
#define HAPX_LN8_RUN(T, W, NG, VEC)                                                                                                         \
  do {                                                                                                                                      \
    auto kernel = norm_backward_team_kernel<T, W, NG, VEC>;                                                                                 \
    if (int e = allow_shared(reinterpret_cast<const void*>(kernel))) return e;                                                              \
    kernel<<<grid, 256, params ? 8 * NG * 2048 : 0, stream>>>(q, ld_saved, scales, static_cast<const T*>(dy), static_cast<const T*>(gamma), mean, \
                                                              rstd, static_cast<const T*>(add), static_cast<T*>(dx), partial, rows, (int)E); \
  } while (0)
#define HAPX_LN8_TEAM(W, NG)                                                             \
  do {                                                                                   \
    if (int e = grid_for((rows + 8 / W - 1) / (8 / W), 2, &grid)) return e;              \
    slices = grid;                                                                       \
    if (dtype == HAPX_BF16) { if (vec) HAPX_LN8_RUN(__nv_bfloat16, W, NG, true); else HAPX_LN8_RUN(__nv_bfloat16, W, NG, false); } \
    else { if (vec) HAPX_LN8_RUN(float, W, NG, true); else HAPX_LN8_RUN(float, W, NG, false); }                                    \
  } while (0)
    HAPX_LN8_SWITCH(E)
    else {
      slices = (rows + kSliceRows - 1) / kSliceRows;
      if (int e = grid_for((rows + 3) / 4, 16, &grid)) return e;
      const dim3 g2((unsigned)((E + kBlock - 1) / kBlock), (unsigned)std::min<long long>(slices, 65535));
#define HAPX_LN8_LONG(T)                                                                                                                       \
  do {                                                                                                                                         \
    norm_backward_kernel<T><<<grid, 128, 0, stream>>>(q, ld_saved, scales, static_cast<const T*>(dy), static_cast<const T*>(gamma), mean, rstd, \
                                                      static_cast<const T*>(add), static_cast<T*>(dx), rows, (int)E);                          \
    if (params)                                                                                                                                \
      norm_param_partial_kernel<T><<<g2, 128, 0, stream>>>(q, ld_saved, scales, static_cast<const T*>(dy), mean, rstd, workspace, rows, (int)E); \
  } while (0)
      if (dtype == HAPX_BF16) HAPX_LN8_LONG(__nv_bfloat16);
      else HAPX_LN8_LONG(float);
      if (params) count_launch();
#undef HAPX_LN8_LONG
    }
#undef HAPX_LN8_TEAM
#undef HAPX_LN8_RUN
    HAPX_CUDA(cudaGetLastError());
    count_launch();
  }
  if (params) {
    const unsigned joins = (unsigned)((2 * E + 31) / 32);
    if (dtype == HAPX_BF16)
      norm_param_join_kernel<__nv_bfloat16><<<joins, 1024, 0, stream>>>(workspace, slices, (int)E, static_cast<__nv_bfloat16*>(dgamma),
                                                                        static_cast<__nv_bfloat16*>(dbeta));
    else
      norm_param_join_kernel<float><<<joins, 1024, 0, stream>>>(workspace, slices, (int)E, static_cast<float*>(dgamma), static_cast<float*>(dbeta));
    HAPX_CUDA(cudaGetLastError());
    count_launch();
  }
  return HAPX_OK;
}

}  // extern "C"
