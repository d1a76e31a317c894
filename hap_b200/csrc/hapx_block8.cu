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

struct QuantParams {
  const void* x;
  long long rows, cols, ldx;
  unsigned char* q;  long long ldq;  float* s;  long long lds;       // as it stands: scale of (row, column block) at s[block * lds + row]
  unsigned char* qt; long long ldqt; float* st; long long ldst;      // transposed: scale of (column, row block) at st[block * ldst + column]
  float* colsum;                                                     // [row tile][cols] partial column sums, or null
  int row_tiles, col_tiles;
};

// SQUARE: one scale per 128 x 128 tile (s[column block * lds + row block], st the transposed).
template <typename T, bool SQUARE>
__global__ void __launch_bounds__(256) quantize_kernel(const QuantParams p) {
  __shared__ float s_col[8][kBlock];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(p.x);
  const bool vec = (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0 && (p.ldx & 3) == 0;
  for (long long tile = blockIdx.x; tile < (long long)p.row_tiles * p.col_tiles; tile += gridDim.x) {
    const int rt = (int)(tile / p.col_tiles), ct = (int)(tile % p.col_tiles);
    const long long r0 = (long long)rt * kBlock + 16 * warp, c0 = (long long)ct * kBlock + 4 * lane;
    const int valid = (int)max(0ll, min(4ll, p.cols - c0));
    float v[16][4], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (r0 + i < p.rows && valid > 0) load4(x + (r0 + i) * p.ldx + c0, vec, valid, v[i]);
      else v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
    }
    if (p.colsum) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += v[i][j];
#pragma unroll
      for (int j = 0; j < 4; ++j) s_col[warp][4 * lane + j] = sum[j];
      __syncthreads();
      if (threadIdx.x < kBlock && (long long)ct * kBlock + threadIdx.x < p.cols) {
        float t = 0.f;
        for (int w = 0; w < 8; ++w) t += s_col[w][threadIdx.x];
        p.colsum[(long long)rt * p.cols + (long long)ct * kBlock + threadIdx.x] = t;
      }
      __syncthreads();
    }
    float rowbig[16], colbig[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      rowbig[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[i][j] = finite_or_nan(v[i][j]);
        rowbig[i] = fmaxf(rowbig[i], fabsf(v[i][j]));
        colbig[j] = fmaxf(colbig[j], fabsf(v[i][j]));
      }
    }
    int ecol[4];
    if (SQUARE) {
      const float mine = warp_max(fmaxf(fmaxf(colbig[0], colbig[1]), fmaxf(colbig[2], colbig[3])));
      if (lane == 0) s_col[0][warp] = mine;
      __syncthreads();
      float big = s_col[0][0];
      for (int w = 1; w < 8; ++w) big = fmaxf(big, s_col[0][w]);
      ecol[0] = ecol[1] = ecol[2] = ecol[3] = scale_exponent(big);
      if (threadIdx.x == 0) {
        if (p.q) p.s[(long long)ct * p.lds + rt] = pow2(ecol[0]);
        if (p.qt) p.st[(long long)rt * p.ldst + ct] = pow2(ecol[0]);
      }
    } else if (p.qt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s_col[warp][4 * lane + j] = colbig[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float big = s_col[0][4 * lane + j];
        for (int w = 1; w < 8; ++w) big = fmaxf(big, s_col[w][4 * lane + j]);
        ecol[j] = scale_exponent(big);
        if (warp == 0 && j < valid) p.st[(long long)rt * p.ldst + c0 + j] = pow2(ecol[j]);
      }
    }
    if (p.q) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int e = SQUARE ? ecol[0] : scale_exponent(warp_max(rowbig[i]));
        const float inv = pow2(-e);
        if (r0 + i < p.rows) {
          if (!SQUARE && lane == 0) p.s[(long long)ct * p.lds + r0 + i] = pow2(e);
          if (valid > 0)     // the pitch is a multiple of 16: a partial group of 4 stays inside it
            *reinterpret_cast<unsigned*>(p.q + (r0 + i) * p.ldq + c0) = pack4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
        }
      }
    }
    if (p.qt && r0 < p.rows) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j >= valid) continue;
        const float inv = pow2(-ecol[j]);
        unsigned w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = pack4(v[4 * k][j] * inv, v[4 * k + 1][j] * inv, v[4 * k + 2][j] * inv, v[4 * k + 3][j] * inv);
        *reinterpret_cast<uint4*>(p.qt + (c0 + j) * p.ldqt + r0) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    __syncthreads();      // s_col is reused by the next tile
  }
}

// out[c] = sum over the row tiles, in order.
template <typename T>
__global__ void __launch_bounds__(256) colsum_join_kernel(const float* __restrict__ partial, int tiles, long long cols, T* __restrict__ out) {
  const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
  for (int t = 0; t < tiles; ++t) s += partial[(long long)t * cols + c];
  out[c] = from_f<T>(s);
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const unsigned char* __restrict__ q, long long ldq, const float* __restrict__ s,
                                                         long long lds, int row_shift, T* __restrict__ out, long long rows, long long cols) {
  const long long n = rows * cols;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) {
    const long long r = e / cols, c = e - r * cols;
    out[e] = from_f<T>(unpack2(q[r * ldq + c]).x * s[(c >> 7) * lds + (r >> row_shift)]);
  }
}

static int sms(int* out) {
  int device = 0;
  HAPX_CUDA(cudaGetDevice(&device));
  HAPX_CUDA(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, device));
  return HAPX_OK;
}

}  // namespace block8
}  // namespace hapx

using namespace hapx;
using namespace hapx::block8;

extern "C" {

int hapx_block8_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int square, void* q, int64_t ldq, float* s,
                         int64_t lds, void* qt, int64_t ldqt, float* st, int64_t ldst, float* colsum, hapx_stream stream_) {
  if (dtype != HAPX_F32 && dtype != HAPX_BF16) return fail(HAPX_ERR_DTYPE, "block8_quantize: float32 or bfloat16 only");
  if (rows < 0 || cols < 0 || ldx < cols) return fail(HAPX_ERR_EXTENT, "block8_quantize: bad extent or row pitch");
  if (rows == 0 || cols == 0) return HAPX_OK;
  const int64_t row_tiles = (rows + kBlock - 1) / kBlock, col_tiles = (cols + kBlock - 1) / kBlock;
  if (row_tiles > 0x7fffffff / col_tiles) return fail(HAPX_ERR_EXTENT, "block8_quantize: more than 2^31 blocks");
  if (!x || (!q && !qt) || (q && !s) || (qt && !st)) return fail(HAPX_ERR_ARGUMENT, "block8_quantize: null pointer");
  if (q && (ldq % 16 != 0 || ldq < cols || (reinterpret_cast<uintptr_t>(q) & 15u) || lds < (square ? row_tiles : rows)))
    return fail(HAPX_ERR_EXTENT, "block8_quantize: values need a 16-byte aligned base and pitch, and a pitch that covers a row");
  if (qt && (ldqt % 16 != 0 || ldqt < rows || (reinterpret_cast<uintptr_t>(qt) & 15u) || ldst < (square ? col_tiles : cols)))
    return fail(HAPX_ERR_EXTENT, "block8_quantize: transposed values need a 16-byte aligned base and pitch, and a pitch that covers a column");
  int n_sm = 0;
  if (int e = sms(&n_sm)) return e;
  QuantParams p = {x, rows, cols, ldx, static_cast<unsigned char*>(q), ldq, s, lds, static_cast<unsigned char*>(qt), ldqt, st, ldst, colsum,
                   (int)row_tiles, (int)col_tiles};
  const int grid = (int)std::min<int64_t>(row_tiles * col_tiles, (int64_t)n_sm * 16);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (dtype == HAPX_BF16) {
    if (square) quantize_kernel<__nv_bfloat16, true><<<grid, 256, 0, stream>>>(p);
    else quantize_kernel<__nv_bfloat16, false><<<grid, 256, 0, stream>>>(p);
  } else {
    if (square) quantize_kernel<float, true><<<grid, 256, 0, stream>>>(p);
    else quantize_kernel<float, false><<<grid, 256, 0, stream>>>(p);
  }
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

int hapx_block8_colsum_join(void* out, int dtype, const float* partial, int64_t rows, int64_t cols, hapx_stream stream_) {
  if (dtype != HAPX_F32 && dtype != HAPX_BF16) return fail(HAPX_ERR_DTYPE, "block8_colsum_join: float32 or bfloat16 only");
  if (rows < 0 || cols < 0) return fail(HAPX_ERR_EXTENT, "block8_colsum_join: negative size");
  if (cols == 0) return HAPX_OK;
  if (!out || (rows > 0 && !partial)) return fail(HAPX_ERR_ARGUMENT, "block8_colsum_join: null pointer");
  const int tiles = (int)((rows + kBlock - 1) / kBlock);
  const unsigned grid = (unsigned)((cols + 255) / 256);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (dtype == HAPX_BF16) colsum_join_kernel<<<grid, 256, 0, stream>>>(partial, tiles, cols, static_cast<__nv_bfloat16*>(out));
  else colsum_join_kernel<<<grid, 256, 0, stream>>>(partial, tiles, cols, static_cast<float*>(out));
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

int hapx_block8_dequantize(void* out, int dtype, const void* q, int64_t ldq, const float* s, int64_t lds, int square, int64_t rows,
                           int64_t cols, hapx_stream stream_) {
  if (dtype != HAPX_F32 && dtype != HAPX_BF16) return fail(HAPX_ERR_DTYPE, "block8_dequantize: float32 or bfloat16 only");
  if (rows < 0 || cols < 0 || ldq < cols) return fail(HAPX_ERR_EXTENT, "block8_dequantize: bad extent or row pitch");
  if (rows == 0 || cols == 0) return HAPX_OK;
  if (!out || !q || !s) return fail(HAPX_ERR_ARGUMENT, "block8_dequantize: null pointer");
  int n_sm = 0;
  if (int e = sms(&n_sm)) return e;
  const int grid = (int)std::min<int64_t>((rows * cols + 255) / 256, (int64_t)n_sm * 16);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const unsigned char* v = static_cast<const unsigned char*>(q);
  if (dtype == HAPX_BF16) dequantize_kernel<<<grid, 256, 0, stream>>>(v, ldq, s, lds, square ? 7 : 0, static_cast<__nv_bfloat16*>(out), rows, cols);
  else dequantize_kernel<<<grid, 256, 0, stream>>>(v, ldq, s, lds, square ? 7 : 0, static_cast<float*>(out), rows, cols);
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

}  // extern "C"
