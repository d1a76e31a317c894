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
// x~ is x to half a step of 3 fraction bits; forward results are those of the operators that keep x.
#include <algorithm>
#include <string>

#include "hapx_block8.h"
#include "hapx_internal.h"
#include "hapx_rng.h"

namespace hapx {
namespace saved8 {

using namespace block8;

enum Act { ACT_RELU = 1, ACT_GELU = 2 };

// Phi(v) and its density's exponential.
__device__ __forceinline__ float normal_cdf(float v) { return 0.5f * erfcf(-v * 0.70710678118654752f); }
__device__ __forceinline__ float gelu_slope(float v) { return fmaf(v * 0.3989422804014327f, __expf(-0.5f * v * v), normal_cdf(v)); }

// One warp per run of 128 elements; lane l holds elements 4l .. 4l + 3 of it.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) act_forward_kernel(const T* __restrict__ x, T* __restrict__ y, unsigned char* __restrict__ saved,
                                                          float* __restrict__ scales, long long n, unsigned threshold, float keep_scale,
                                                          const rng::State* st, unsigned long long call_id) {
  const int lane = threadIdx.x & 31;
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & (4 * sizeof(T) - 1)) == 0;
  rng::Key key = {0u, 0u, 0u, 0u};
  if (threshold) key = rng::make_key(st, call_id);
  const long long runs = (n + kBlock - 1) / kBlock;
  for (long long run = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); run < runs; run += (long long)gridDim.x * 8) {
    const long long e0 = run * kBlock + 4 * lane;
    const int valid = (int)max(0ll, min(4ll, n - e0));
    float v[4], o[4];
    load4(x + e0, vec, valid, v);
    unsigned keep = 0xfu;
    if (threshold) keep = rng::keep_bits(rng::philox(key, (unsigned long long)(e0 >> 3)), threshold) >> (e0 & 4);
    unsigned bits = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float k = (keep >> j) & 1u ? keep_scale : 0.f;
      if (ACT == ACT_RELU) {
        o[j] = (v[j] <= 0.f ? 0.f : v[j]) * k;      // NaN passes
        bits |= (v[j] > 0.f && k != 0.f && j < valid ? 1u : 0u) << j;
      } else {
        o[j] = v[j] * normal_cdf(v[j]) * k;
      }
    }
    store4(y + e0, vec, valid, o);
    if (!saved) continue;                           // nothing asks for a gradient
    if (ACT == ACT_RELU) {
      bits |= __shfl_down_sync(0xffffffffu, bits, 1) << 4;
      if ((lane & 1) == 0 && valid > 0) saved[e0 >> 3] = (unsigned char)bits;
    } else {
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] = finite_or_nan(v[j]); big = fmaxf(big, fabsf(v[j])); }
      const int e = scale_exponent(warp_max(big));
      const float inv = pow2(-e);
      if (lane == 0) scales[run] = pow2(e);
      if (valid > 0) *reinterpret_cast<unsigned*>(saved + e0) = pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    }
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) act_backward_kernel(const T* __restrict__ dy, const unsigned char* __restrict__ saved,
                                                           const float* __restrict__ scales, T* __restrict__ dx, long long n,
                                                           unsigned threshold, float keep_scale, const rng::State* st,
                                                           unsigned long long call_id) {
  const bool vec = ((reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(dx)) & (4 * sizeof(T) - 1)) == 0;
  rng::Key key = {0u, 0u, 0u, 0u};
  if (ACT == ACT_GELU && threshold) key = rng::make_key(st, call_id);
  const long long groups = (n + 3) / 4;
  for (long long g = (long long)blockIdx.x * 256 + threadIdx.x; g < groups; g += (long long)gridDim.x * 256) {
    const long long e0 = 4 * g;
    const int valid = (int)min(4ll, n - e0);
    float d[4], o[4];
    load4(dy + e0, vec, valid, d);
    if (ACT == ACT_RELU) {
      const unsigned bits = saved[e0 >> 3] >> (e0 & 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = (bits >> j) & 1u ? d[j] * keep_scale : 0.f;
    } else {
      unsigned keep = 0xfu;
      if (threshold) keep = rng::keep_bits(rng::philox(key, (unsigned long long)(e0 >> 3)), threshold) >> (e0 & 4);
      const unsigned w = *reinterpret_cast<const unsigned*>(saved + e0);
      const float s = scales[e0 / kBlock];
      const float2 a = unpack2(w & 0xffffu), b = unpack2(w >> 16);
      const float h[4] = {a.x * s, a.y * s, b.x * s, b.y * s};
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = d[j] * ((keep >> j) & 1u ? keep_scale : 0.f) * gelu_slope(h[j]);
    }
    store4(dx + e0, vec, valid, o);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One warp per row, blocks of 128 columns one after another; the row is read three times, twice from the caches.
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

template <typename T>
__global__ void __launch_bounds__(256) norm_param_join_kernel(const float* __restrict__ partial, long long slices, int E, T* __restrict__ dw,
                                                              T* __restrict__ db) {
  const int e = blockIdx.x * 256 + threadIdx.x;
  if (e >= 2 * E) return;
  float sum = 0.f;
  for (long long i = 0; i < slices; ++i) sum += partial[i * 2 * E + e];
  if (e < E) { if (dw) dw[e] = from_f<T>(sum); }
  else if (db) db[e - E] = from_f<T>(sum);
}

static int grid_for(long long blocks, int per_sm, int* grid) {
  int device = 0, n_sm = 0;
  HAPX_CUDA(cudaGetDevice(&device));
  HAPX_CUDA(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, device));
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
  if (int e = grid_for((n + 8 * kBlock - 1) / (8 * kBlock), 8, &grid)) return e;
  const float ks = (float)(1.0 / (1.0 - p));
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  unsigned char* sv = static_cast<unsigned char*>(saved);
#define HAPX_ACT8(T, A) \
  act_forward_kernel<T, A><<<grid, 256, 0, stream>>>(static_cast<const T*>(x), static_cast<T*>(y), sv, scales, n, thr, ks, st, call_id)
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
  if (int e = grid_for((n + 1023) / 1024, 8, &grid)) return e;
  const float ks = (float)(1.0 / (1.0 - p));
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const unsigned char* sv = static_cast<const unsigned char*>(saved);
#define HAPX_ACT8(T, A) \
  act_backward_kernel<T, A><<<grid, 256, 0, stream>>>(static_cast<const T*>(dy), sv, scales, static_cast<T*>(dx), n, thr, ks, st, call_id)
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
  if (int e = grid_for((rows + 3) / 4, 16, &grid)) return e;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
#define HAPX_LN8(T)                                                                                                                       \
  norm_forward_kernel<T><<<grid, 128, 0, stream>>>(static_cast<const T*>(x), static_cast<const T*>(gamma), static_cast<const T*>(beta),   \
                                                   static_cast<T*>(y), mean, rstd, static_cast<unsigned char*>(saved), ld_saved, scales, \
                                                   rows, (int)E, (float)eps)
  if (dtype == HAPX_BF16) HAPX_LN8(__nv_bfloat16); else HAPX_LN8(float);
#undef HAPX_LN8
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

int64_t hapx_layer_norm8_backward_workspace(int64_t rows, int64_t E) {
  return (std::max<int64_t>(1, (rows + kSliceRows - 1) / kSliceRows)) * 2 * E * (int64_t)sizeof(float);
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
  const long long slices = (rows + kSliceRows - 1) / kSliceRows;
  int grid = 1;
  if (int e = grid_for((rows + 3) / 4, 16, &grid)) return e;
  const unsigned char* q = static_cast<const unsigned char*>(saved);
#define HAPX_LN8(T)                                                                                                                           \
  do {                                                                                                                                        \
    if (rows > 0) {                                                                                                                           \
      norm_backward_kernel<T><<<grid, 128, 0, stream>>>(q, ld_saved, scales, static_cast<const T*>(dy), static_cast<const T*>(gamma), mean,   \
                                                        rstd, static_cast<const T*>(add), static_cast<T*>(dx), rows, (int)E);                 \
      count_launch();                                                                                                                         \
    }                                                                                                                                         \
    if (dgamma || dbeta) {                                                                                                                    \
      if (rows > 0) {                                                                                                                         \
        const dim3 g2((unsigned)((E + kBlock - 1) / kBlock), (unsigned)std::min<long long>(slices, 65535));                                   \
        norm_param_partial_kernel<T><<<g2, 128, 0, stream>>>(q, ld_saved, scales, static_cast<const T*>(dy), mean, rstd, workspace, rows, (int)E); \
        count_launch();                                                                                                                       \
      }                                                                                                                                       \
      norm_param_join_kernel<T><<<(unsigned)((2 * E + 255) / 256), 256, 0, stream>>>(workspace, slices, (int)E, static_cast<T*>(dgamma),      \
                                                                                     static_cast<T*>(dbeta));                                 \
      count_launch();                                                                                                                         \
    }                                                                                                                                         \
  } while (0)
  if (dtype == HAPX_BF16) HAPX_LN8(__nv_bfloat16); else HAPX_LN8(float);
#undef HAPX_LN8
  HAPX_CUDA(cudaGetLastError());
  return HAPX_OK;
}

}  // extern "C"
