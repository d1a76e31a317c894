// The block quantiser: a matrix as e4m3 values with one power-of-two scale per block of 128 (hapx_block8.h), as it
// stands (blocks along the columns), transposed (blocks along the rows), or both from one read; and back.
//
// HBM-bound: the element is read once and written once per form.  A thread block owns a 128 x 128 tile - whole blocks
// in either direction, so no maximum crosses a tile - and keeps it in registers: warp w holds rows 16w .. 16w + 15,
// lane l the columns 4l .. 4l + 3.
#include <algorithm>
#include <string>

#include "hapx_block8.h"
#include "hapx_internal.h"

namespace hapx {
namespace block8 {

struct QuantJobs { QuantJob job[2]; long long tiles0, tiles; };     // tiles of the first matrix, of both

// Four consecutive elements as they are in memory.
template <typename T> struct Raw4;
template <> struct Raw4<__nv_bfloat16> {
  uint2 w;
  __device__ __forceinline__ void zero() { w = make_uint2(0u, 0u); }
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void load_some(const __nv_bfloat16* p, int valid) {
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
    w.x = (valid > 0 ? h[0] : 0u) | (valid > 1 ? (unsigned)h[1] << 16 : 0u);
    w.y = (valid > 2 ? h[2] : 0u) | (valid > 3 ? (unsigned)h[3] << 16 : 0u);
  }
  __device__ __forceinline__ void get(float (&f)[4]) const {
    f[0] = __uint_as_float(w.x << 16); f[1] = __uint_as_float(w.x & 0xffff0000u);
    f[2] = __uint_as_float(w.y << 16); f[3] = __uint_as_float(w.y & 0xffff0000u);
  }
  __device__ __forceinline__ float at(int j) const {
    const unsigned v = j < 2 ? w.x : w.y;
    return __uint_as_float(j & 1 ? v & 0xffff0000u : v << 16);
  }
};
template <> struct Raw4<float> {
  float4 v;
  __device__ __forceinline__ void zero() { v = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void load_some(const float* p, int valid) {
    zero();
    if (valid > 0) v.x = p[0];
    if (valid > 1) v.y = p[1];
    if (valid > 2) v.z = p[2];
    if (valid > 3) v.w = p[3];
  }
  __device__ __forceinline__ void get(float (&f)[4]) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
  __device__ __forceinline__ float at(int j) const { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }
};

// Running maxima of magnitudes of four columns (two per register for bfloat16); a NaN loses against any number.
template <typename T> struct Max4;
template <> struct Max4<__nv_bfloat16> {
  __nv_bfloat162 a, b;
  __device__ __forceinline__ void zero() { a = b = __floats2bfloat162_rn(0.f, 0.f); }
  __device__ __forceinline__ void add(const Raw4<__nv_bfloat16>& r) {
    const unsigned x = r.w.x & 0x7fff7fffu, y = r.w.y & 0x7fff7fffu;
    a = __hmax2(a, *reinterpret_cast<const __nv_bfloat162*>(&x));
    b = __hmax2(b, *reinterpret_cast<const __nv_bfloat162*>(&y));
  }
  __device__ __forceinline__ void get(float (&f)[4]) const {
    f[0] = __low2float(a); f[1] = __high2float(a); f[2] = __low2float(b); f[3] = __high2float(b);
  }
  static __device__ __forceinline__ float of(const Raw4<__nv_bfloat16>& r) {
    const unsigned x = r.w.x & 0x7fff7fffu, y = r.w.y & 0x7fff7fffu;
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
    return fmaxf(fmaxf(__low2float(m), __high2float(m)), 0.f);      // of two NaN: 0
  }
};
template <> struct Max4<float> {
  float m[4];
  __device__ __forceinline__ void zero() { m[0] = m[1] = m[2] = m[3] = 0.f; }
  __device__ __forceinline__ void add(const Raw4<float>& r) {
    m[0] = fmaxf(m[0], fabsf(r.v.x)); m[1] = fmaxf(m[1], fabsf(r.v.y)); m[2] = fmaxf(m[2], fabsf(r.v.z)); m[3] = fmaxf(m[3], fabsf(r.v.w));
  }
  __device__ __forceinline__ void get(float (&f)[4]) const { f[0] = m[0]; f[1] = m[1]; f[2] = m[2]; f[3] = m[3]; }
  static __device__ __forceinline__ float of(const Raw4<float>& r) {
    return fmaxf(fmaxf(fmaxf(fabsf(r.v.x), fabsf(r.v.y)), fmaxf(fabsf(r.v.z), fabsf(r.v.w))), 0.f);
  }
};

// square: one scale per 128 x 128 tile, stored for each of its rows (and columns).
//
// The elements stay in their own type in registers (32 of them for bfloat16), so that three blocks fit an SM; the
// transposed bytes go through shared memory and leave as whole 128-byte rows.
template <typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) quantize_kernel(const __grid_constant__ QuantJobs jobs) {
  __shared__ float s_col[8][kBlock];
  __shared__ uint4 s_t[kBlock * 8];
  __shared__ int s_odd;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (long long both = blockIdx.x; both < jobs.tiles; both += gridDim.x) {
    const QuantJob& p = jobs.job[both >= jobs.tiles0];
    const long long tile = both >= jobs.tiles0 ? both - jobs.tiles0 : both;
    const T* x = static_cast<const T*>(p.x);
    const bool vec = (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0 && (p.ldx & 3) == 0;
    const bool square = p.square != 0;
    const int rt = (int)(tile / p.col_tiles), ct = (int)(tile % p.col_tiles);
    const long long r0 = (long long)rt * kBlock + 16 * warp, c0 = (long long)ct * kBlock + 4 * lane;
    const int valid = (int)max(0ll, min(4ll, p.cols - c0)), live = (int)max(0ll, min(16ll, p.rows - r0));   // columns, rows of this thread
    Raw4<T> v[16];
    {
      const T* src = x + r0 * p.ldx + c0;
      if (vec && valid == 4) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (i < live) v[i].load(src + i * p.ldx);
          else v[i].zero();
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (i < live) v[i].load_some(src + i * p.ldx, valid);
          else v[i].zero();
        }
      }
    }
    if (p.colsum) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float f[4];
        v[i].get(f);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += f[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) s_col[warp][4 * lane + j] = sum[j];
      __syncthreads();
      if (threadIdx.x < kBlock && (long long)ct * kBlock + threadIdx.x < p.cols) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += s_col[w][threadIdx.x];
        p.colsum[(long long)rt * p.cols + (long long)ct * kBlock + threadIdx.x] = t;
      }
      __syncthreads();
    }
    if (threadIdx.x == 0) s_odd = 0;
    Max4<T> cm;
    cm.zero();
#pragma unroll
    for (int i = 0; i < 16; ++i) cm.add(v[i]);
    float colbig[4];
    cm.get(colbig);
    __syncthreads();
    // An infinity anywhere in the tile (rare): NaN in its place, and the maxima once more without it.
    if (fmaxf(fmaxf(colbig[0], colbig[1]), fmaxf(colbig[2], colbig[3])) == __uint_as_float(0x7f800000u)) s_odd = 1;
    __syncthreads();
    if (s_odd) {
      cm.zero();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if constexpr (sizeof(T) == 2) {
          if ((v[i].w.x & 0x7f80u) == 0x7f80u) v[i].w.x |= 0x7fffu;
          if ((v[i].w.x & 0x7f800000u) == 0x7f800000u) v[i].w.x |= 0x7fff0000u;
          if ((v[i].w.y & 0x7f80u) == 0x7f80u) v[i].w.y |= 0x7fffu;
          if ((v[i].w.y & 0x7f800000u) == 0x7f800000u) v[i].w.y |= 0x7fff0000u;
        } else {
          v[i].v = make_float4(finite_or_nan(v[i].v.x), finite_or_nan(v[i].v.y), finite_or_nan(v[i].v.z), finite_or_nan(v[i].v.w));
        }
        cm.add(v[i]);
      }
      cm.get(colbig);
    }
    int ecol[4];
    if (square) {
      const float mine = warp_max(fmaxf(fmaxf(colbig[0], colbig[1]), fmaxf(colbig[2], colbig[3])));
      if (lane == 0) s_col[0][warp] = mine;
      __syncthreads();
      float big = s_col[0][0];
#pragma unroll
      for (int w = 1; w < 8; ++w) big = fmaxf(big, s_col[0][w]);
      ecol[0] = ecol[1] = ecol[2] = ecol[3] = scale_exponent(big);
      const unsigned char byte = (unsigned char)(ecol[0] + 127);
      if (threadIdx.x < kBlock) {
        if (p.q) p.s[scale_at((long long)rt * kBlock + threadIdx.x, ct, p.row_tiles)] = byte;
      } else {
        if (p.qt) p.st[scale_at((long long)ct * kBlock + threadIdx.x - kBlock, rt, p.col_tiles)] = byte;
      }
    } else if (p.qt) {
      *reinterpret_cast<float4*>(&s_col[warp][4 * lane]) = make_float4(colbig[0], colbig[1], colbig[2], colbig[3]);
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const float4 o = *reinterpret_cast<const float4*>(&s_col[w][4 * lane]);
        colbig[0] = fmaxf(colbig[0], o.x); colbig[1] = fmaxf(colbig[1], o.y); colbig[2] = fmaxf(colbig[2], o.z); colbig[3] = fmaxf(colbig[3], o.w);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ecol[j] = scale_exponent(colbig[j]);
        if (warp == j) p.st[scale_at(c0 + j, rt, p.col_tiles)] = (unsigned char)(ecol[j] + 127);
      }
    }
    if (p.q) {
      int mine = 0;
      unsigned char* dst = p.q + r0 * p.ldq + c0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int e = square ? ecol[0] : scale_exponent(warp_max(Max4<T>::of(v[i])));
        if (!square && lane == i) mine = e;
        const float inv = pow2(-e);
        float f[4];
        v[i].get(f);
        if (i < live && valid > 0)     // the pitch is a multiple of 16: a partial group of 4 stays inside it
          *reinterpret_cast<unsigned*>(dst + i * p.ldq) = pack4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
      }
      if (!square && lane < live) p.s[scale_at(r0 + lane, ct, p.row_tiles)] = (unsigned char)(mine + 127);
    }
    if (p.qt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float inv = pow2(-ecol[j]);
        unsigned w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = pack4(v[4 * k].at(j) * inv, v[4 * k + 1].at(j) * inv, v[4 * k + 2].at(j) * inv, v[4 * k + 3].at(j) * inv);
        s_t[(4 * lane + j) * 8 + (warp ^ (lane & 7))] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 4; ++k) {       // a warp writes 4 columns' 128 bytes at a time
        const int col = k * 32 + warp * 4 + (lane >> 3), chunk = lane & 7;
        const long long c = (long long)ct * kBlock + col, r = (long long)rt * kBlock + 16 * chunk;
        if (c < p.cols && r < p.rows) *reinterpret_cast<uint4*>(p.qt + c * p.ldqt + r) = s_t[col * 8 + (chunk ^ ((col >> 2) & 7))];
      }
    }
    __syncthreads();      // the shared arrays are reused by the next tile
  }
}

// out[c] = sum over the row tiles in a fixed order: warp w of 8 takes tiles w, w + 8, ...
template <typename T>
__global__ void __launch_bounds__(256) colsum_join_kernel(const float* __restrict__ partial, int tiles, long long cols, T* __restrict__ out) {
  __shared__ float s_sum[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < cols)
#pragma unroll 4
    for (int t = warp; t < tiles; t += 8) s += partial[(long long)t * cols + c];
  s_sum[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || c >= cols) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) s += s_sum[w][lane];
  out[c] = from_f<T>(s);
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const unsigned char* __restrict__ q, long long ldq, const unsigned char* __restrict__ s,
                                                         T* __restrict__ out, long long rows, long long cols) {
  const long long n = rows * cols, groups = (rows + kBlock - 1) / kBlock;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) {
    const long long r = e / cols, c = e - r * cols;
    out[e] = from_f<T>(unpack2(q[r * ldq + c]).x * pow2((int)s[scale_at(r, c >> 7, groups)] - 127));
  }
}

int quantize(QuantJob* job, int n_jobs, int dtype, cudaStream_t stream) {
  int n_sm = 0;
  if (int e = sm_count(&n_sm)) return e;
  QuantJobs jobs;
  for (int i = 0; i < n_jobs; ++i) {
    job[i].row_tiles = (int)((job[i].rows + kBlock - 1) / kBlock);
    job[i].col_tiles = (int)((job[i].cols + kBlock - 1) / kBlock);
    jobs.job[i] = job[i];
    jobs.tiles = (i ? jobs.tiles0 : 0) + (long long)job[i].row_tiles * job[i].col_tiles;
    if (i == 0) jobs.tiles0 = jobs.tiles;
  }
  const int grid = (int)std::min<long long>(jobs.tiles, (long long)n_sm * 16);
  if (dtype == HAPX_BF16) quantize_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(jobs);
  else quantize_kernel<float><<<grid, 256, 0, stream>>>(jobs);
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

}  // namespace block8
}  // namespace hapx

using namespace hapx;
using namespace hapx::block8;

extern "C" {

int64_t hapx_block8_scale_bytes(int64_t rows, int64_t cols) { return rows > 0 && cols > 0 ? scale_bytes(rows, cols) : 0; }

int hapx_block8_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int square, void* q, int64_t ldq, void* s,
                         void* qt, int64_t ldqt, void* st, float* colsum, hapx_stream stream_) {
  if (dtype != HAPX_F32 && dtype != HAPX_BF16) return fail(HAPX_ERR_DTYPE, "block8_quantize: float32 or bfloat16 only");
  if (rows < 0 || cols < 0 || ldx < cols) return fail(HAPX_ERR_EXTENT, "block8_quantize: bad extent or row pitch");
  if (rows == 0 || cols == 0) return HAPX_OK;
  const int64_t row_tiles = (rows + kBlock - 1) / kBlock, col_tiles = (cols + kBlock - 1) / kBlock;
  if (row_tiles > 0x7fffffff / col_tiles) return fail(HAPX_ERR_EXTENT, "block8_quantize: more than 2^31 blocks");
  if (!x || (!q && !qt) || (q && !s) || (qt && !st)) return fail(HAPX_ERR_ARGUMENT, "block8_quantize: null pointer");
  if (q && (ldq % 16 != 0 || ldq < cols || (reinterpret_cast<uintptr_t>(q) & 15u)))
    return fail(HAPX_ERR_EXTENT, "block8_quantize: values need a 16-byte aligned base and pitch, and a pitch that covers a row");
  if (qt && (ldqt % 16 != 0 || ldqt < rows || (reinterpret_cast<uintptr_t>(qt) & 15u)))
    return fail(HAPX_ERR_EXTENT, "block8_quantize: transposed values need a 16-byte aligned base and pitch, and a pitch that covers a column");
  QuantJob job;
  job.x = x; job.rows = rows; job.cols = cols; job.ldx = ldx; job.square = square;
  job.q = static_cast<unsigned char*>(q); job.ldq = ldq; job.s = static_cast<unsigned char*>(s);
  job.qt = static_cast<unsigned char*>(qt); job.ldqt = ldqt; job.st = static_cast<unsigned char*>(st);
  job.colsum = colsum;
  return quantize(&job, 1, dtype, static_cast<cudaStream_t>(stream_));
}

int hapx_block8_colsum_join(void* out, int dtype, const float* partial, int64_t rows, int64_t cols, hapx_stream stream_) {
  if (dtype != HAPX_F32 && dtype != HAPX_BF16) return fail(HAPX_ERR_DTYPE, "block8_colsum_join: float32 or bfloat16 only");
  if (rows < 0 || cols < 0) return fail(HAPX_ERR_EXTENT, "block8_colsum_join: negative size");
  if (cols == 0) return HAPX_OK;
  if (!out || (rows > 0 && !partial)) return fail(HAPX_ERR_ARGUMENT, "block8_colsum_join: null pointer");
  const int tiles = (int)((rows + kBlock - 1) / kBlock);
  const unsigned grid = (unsigned)((cols + 31) / 32);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (dtype == HAPX_BF16) colsum_join_kernel<<<grid, 256, 0, stream>>>(partial, tiles, cols, static_cast<__nv_bfloat16*>(out));
  else colsum_join_kernel<<<grid, 256, 0, stream>>>(partial, tiles, cols, static_cast<float*>(out));
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

int hapx_block8_dequantize(void* out, int dtype, const void* q, int64_t ldq, const void* s, int64_t rows, int64_t cols, hapx_stream stream_) {
  if (dtype != HAPX_F32 && dtype != HAPX_BF16) return fail(HAPX_ERR_DTYPE, "block8_dequantize: float32 or bfloat16 only");
  if (rows < 0 || cols < 0 || ldq < cols) return fail(HAPX_ERR_EXTENT, "block8_dequantize: bad extent or row pitch");
  if (rows == 0 || cols == 0) return HAPX_OK;
  if (!out || !q || !s) return fail(HAPX_ERR_ARGUMENT, "block8_dequantize: null pointer");
  int n_sm = 0;
  if (int e = sm_count(&n_sm)) return e;
  const int grid = (int)std::min<int64_t>((rows * cols + 255) / 256, (int64_t)n_sm * 16);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const unsigned char *v = static_cast<const unsigned char*>(q), *sc = static_cast<const unsigned char*>(s);
  if (dtype == HAPX_BF16) dequantize_kernel<<<grid, 256, 0, stream>>>(v, ldq, sc, static_cast<__nv_bfloat16*>(out), rows, cols);
  else dequantize_kernel<<<grid, 256, 0, stream>>>(v, ldq, sc, static_cast<float*>(out), rows, cols);
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

}  // extern "C"
