// The block quantiser: a matrix as e4m3 values with one power-of-two scale per block of 128 (hapx_block8.h), as it
// stands (blocks along the columns), transposed (blocks along the rows), or both from one read; and back.
//
// HBM-bound: the element is read once and written once per form.  A thread block owns a 128 x 128 tile - whole blocks
// in either direction, so no maximum crosses a tile - and keeps it in registers: warp w holds rows 16w .. 16w + 15,
// lane l the columns 4l .. 4l + 3.
#include <algorithm>
#include <cstring>
#include <mutex>
#include <string>

#include "hapx_block8.h"
#include "hapx_internal.h"
#include "hapx_tc.h"

namespace hapx {
namespace block8 {

struct QuantJobs {
  QuantJob job[2];
  long long tiles0, tiles;       // tiles of the first matrix, of both
  int bulk[2];                   // the matrix can be fetched by bulk tensor loads (16-byte aligned base and pitch)
  unsigned* error;               // device word: a wait that ran out
};

// square: one scale per 128 x 128 tile, stored for each of its rows (and columns).
//
// Two passes over the tile in registers, where the elements stay in their own type (32 registers for bfloat16, three
// blocks per SM): the maxima of rows and columns, then - once all scales are known - both forms from one unpacking.  The
// transposed bytes go through shared memory and leave as whole 128-byte rows.  What bounds it is the bytes in flight: a
// block fetches its next tile into shared memory by one bulk tensor load while it works on and stores the present one; and,
// close behind, the 18 instructions per element.  bfloat16, 8192 x 33280: 205 us for both forms (5.3 TB/s), 142 for one
// (5.7); 8192 x 768, where the 384 tiles are one round of the SMs: 7.5 us (3.3 TB/s).
template <typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) quantize_kernel(const __grid_constant__ QuantJobs jobs, const __grid_constant__ CUtensorMap map0,
                                                                               const __grid_constant__ CUtensorMap map1) {
  extern __shared__ unsigned char s_dynamic[];   // the next tile, 128 x 128 elements
  unsigned char* s_x = s_dynamic + ((128u - (tc::smem_u32(s_dynamic) & 127u)) & 127u);
  __shared__ unsigned long long s_bar;
  __shared__ uint4 s_col[8][32];                 // column maxima of each warp
  __shared__ float4 s_sum[8][32];                // its column sums
  __shared__ uint4 s_t[kBlock * 8];
  __shared__ int s_odd;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // where this thread's scales lie inside the 512 bytes of a tile (lane i < 16: row 16 warp + i; warp j < 4: column 4 lane + j)
  const int at_row = ((16 * warp + (lane & 15)) & 31) * 16 + (warp >> 1) * 4, at_col = ((4 * lane + (warp & 3)) & 31) * 16 + (lane >> 3) * 4;
  const unsigned bar = tc::smem_u32(&s_bar);
  unsigned phase = 0;
  if (threadIdx.x == 0) {
    tc::mbar_init(bar, 1);
    tc::fence_barrier_init();
  }
  __syncthreads();
  auto fetch = [&](long long both) {             // by one thread: the tile's load, if it is one
    const int which = both >= jobs.tiles0;
    if (both >= jobs.tiles || !jobs.bulk[which]) return;
    const unsigned tile = (unsigned)(which ? both - jobs.tiles0 : both), col_tiles = (unsigned)jobs.job[which].col_tiles, rt = tile / col_tiles;
    tc::mbar_expect_tx(bar, kBlock * kBlock * sizeof(T));
    tc::tma_load_4d(tc::smem_u32(s_x), which ? &map1 : &map0, (int)(tile - rt * col_tiles) * kBlock, (int)rt * kBlock, 0, 0, bar);
  };
  if (threadIdx.x == 0) fetch(blockIdx.x);
  for (long long both = blockIdx.x; both < jobs.tiles; both += gridDim.x) {
    const int which = both >= jobs.tiles0;
    const QuantJob& p = jobs.job[which];
    const unsigned tile = (unsigned)(which ? both - jobs.tiles0 : both);        // fewer than 2^31
    const bool square = p.square != 0, want_q = p.q != nullptr, want_qt = p.qt != nullptr, want_sum = p.colsum != nullptr;
    const int rt = (int)(tile / (unsigned)p.col_tiles), ct = (int)tile - rt * p.col_tiles;
    const long long r0 = (long long)rt * kBlock + 16 * warp, c0 = (long long)ct * kBlock + 4 * lane;
    const int valid = (int)max(0ll, min(4ll, p.cols - c0)), live = (int)max(0ll, min(16ll, p.rows - r0));   // columns, rows of this thread
    Raw4<T> v[16];
    if (jobs.bulk[which]) {                      // outside the matrix the load has put zeros
      const bool ok = __syncthreads_and(tc::mbar_wait(bar, phase));
      phase ^= 1u;
      if (!ok) {                                 // the same in every thread
        if (threadIdx.x == 0) atomicCAS(jobs.error, 0u, 4u);
        return;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i].load_shared(s_x, 16 * warp + i, lane);
      __syncthreads();                           // the tile is in registers: its place is free
    } else {
      const T* src = static_cast<const T*>(p.x) + r0 * p.ldx + c0;
      const bool vec = (reinterpret_cast<uintptr_t>(p.x) & (4 * sizeof(T) - 1)) == 0 && (p.ldx & 3) == 0 && valid == 4;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (i >= live) v[i].zero();
        else if (vec) v[i].load(src + i * p.ldx);
        else v[i].load_some(src + i * p.ldx, valid);
      }
    }
    if (threadIdx.x == 0) fetch(both + gridDim.x);
    if (threadIdx.x == 0) s_odd = 0;
    unsigned rowmax = 0u, col[4];                // lane i < 16: row i's maximum
    typename Raw4<T>::Max cm;
    Raw4<T>::clear(cm);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const unsigned r = __reduce_max_sync(0xffffffffu, v[i].maxima(cm));
      if (lane == i) rowmax = r;
    }
    Raw4<T>::columns(cm, col);
    s_col[warp][lane] = make_uint4(col[0], col[1], col[2], col[3]);
    __syncthreads();
    constexpr unsigned kInf = 0x7f800000u;
    if (max(max(col[0], col[1]), max(col[2], col[3])) >= kInf) s_odd = 1;
    __syncthreads();
    const bool odd = s_odd != 0;
    if (odd) {                                   // an infinity in the tile (rare): NaN in its place, the maxima once more
      float special[4] = {0.f, 0.f, 0.f, 0.f};   // the sums are those of the original values
      Raw4<T>::clear(cm);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float f[4];
        v[i].get(f);
#pragma unroll
        for (int j = 0; j < 4; ++j) special[j] += f[j];
        v[i].sanitise();
        const unsigned r = __reduce_max_sync(0xffffffffu, v[i].maxima(cm));
        if (lane == i) rowmax = r;
      }
      Raw4<T>::columns(cm, col);
      s_col[warp][lane] = make_uint4(col[0], col[1], col[2], col[3]);
      s_sum[warp][lane] = make_float4(special[0], special[1], special[2], special[3]);
      __syncthreads();
    }
    if (want_qt || square) {
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const uint4 o = s_col[w][lane];
        col[0] = max(col[0], o.x); col[1] = max(col[1], o.y); col[2] = max(col[2], o.z); col[3] = max(col[3], o.w);
      }
    }
    if (square) rowmax = col[0] = col[1] = col[2] = col[3] = __reduce_max_sync(0xffffffffu, max(max(col[0], col[1]), max(col[2], col[3])));
    const int erow = scale_exponent(__uint_as_float(rowmax & Raw4<T>::kMask));
    const float inv_row = pow2(-erow);
    if (want_q && lane < live) p.s[((long long)(ct >> 2) * p.row_tiles + rt) * 512 + (ct & 3) + at_row] = (unsigned char)(erow + 127);
    float inv_col[4];
    if (want_qt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = scale_exponent(__uint_as_float(col[j] & Raw4<T>::kMask));
        inv_col[j] = pow2(-e);
        if (warp == j && j < valid) p.st[((long long)(rt >> 2) * p.col_tiles + ct) * 512 + (rt & 3) + at_col] = (unsigned char)(e + 127);
      }
    }
    unsigned char* dst = p.q + r0 * p.ldq + c0;
    const int rows_out = valid > 0 ? live : 0;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    unsigned out_t[4][4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {                // four rows at a time
      float f[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * g + i].get(f[i]);
      if (want_q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float inv = square ? inv_row : __shfl_sync(0xffffffffu, inv_row, 4 * g + i);
          if (4 * g + i < rows_out)              // the pitch is a multiple of 16: a partial group of 4 stays inside it
            *reinterpret_cast<unsigned*>(dst) = pack4(f[i][0] * inv, f[i][1] * inv, f[i][2] * inv, f[i][3] * inv);
          dst += p.ldq;
        }
      }
      if (want_qt) {
#pragma unroll
        for (int j = 0; j < 4; ++j) out_t[j][g] = pack4(f[0][j] * inv_col[j], f[1][j] * inv_col[j], f[2][j] * inv_col[j], f[3][j] * inv_col[j]);
      }
      if (want_sum) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[j] += f[i][j];
      }
    }
    if (want_qt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s_t[(4 * lane + j) * 8 + (warp ^ (lane & 7))] = make_uint4(out_t[j][0], out_t[j][1], out_t[j][2], out_t[j][3]);
    }
    if (want_sum && !odd) s_sum[warp][lane] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    __syncthreads();                             // the maxima have been read, the transposed bytes and sums written
    if (want_qt) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {              // a warp writes 4 columns' 128 bytes at a time
        const int at = k * 32 + warp * 4 + (lane >> 3), chunk = lane & 7;
        const long long c = (long long)ct * kBlock + at, r = (long long)rt * kBlock + 16 * chunk;
        if (c < p.cols && r < p.rows) *reinterpret_cast<uint4*>(p.qt + c * p.ldqt + r) = s_t[at * 8 + (chunk ^ ((at >> 2) & 7))];
      }
    }
    if (want_sum && threadIdx.x < kBlock && (long long)ct * kBlock + threadIdx.x < p.cols) {
      const float* part = reinterpret_cast<const float*>(s_sum);
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += part[w * kBlock + threadIdx.x];
      p.colsum[(long long)rt * p.cols + (long long)ct * kBlock + threadIdx.x] = t;
    }
    // the next tile writes s_t and s_sum behind two barriers of its own
  }
}

// out[c] = sum over the row tiles in a fixed order: warp w of 8 takes tiles w, w + 8, ...  A launch's length (3 us); where a
// weight gradient is computed too, its product does this instead.
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

// x~ = q s, one element per thread at a time: for inspection and tests, on no training path.
template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const unsigned char* __restrict__ q, long long ldq, const unsigned char* __restrict__ s,
                                                         T* __restrict__ out, long long rows, long long cols) {
  const long long n = rows * cols, groups = (rows + kBlock - 1) / kBlock;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) {
    const long long r = e / cols, c = e - r * cols;
    out[e] = from_f<T>(unpack2(q[r * ldq + c]).x * pow2((int)s[scale_at(r, c >> 7, groups)] - 127));
  }
}

// The matrix as (column, row) in boxes of 128 x 128.
static int make_map(CUtensorMap* map, const QuantJob& j, int dtype) {
  gemm::EncodeTiledFn fn = gemm::encode_fn();
  if (!fn) return fail(HAPX_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t pitch = (cuuint64_t)j.ldx * (dtype == HAPX_BF16 ? 2 : 4);
  cuuint64_t dims[4] = {(cuuint64_t)j.cols, (cuuint64_t)j.rows, 1, 1};
  cuuint64_t strides[3] = {pitch, pitch, pitch};
  cuuint32_t box[4] = {kBlock, kBlock, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(map, dtype == HAPX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, const_cast<void*>(j.x), dims, strides,
                  box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(HAPX_ERR_CUDA, "cuTensorMapEncodeTiled (quantise) failed with code " + std::to_string((int)r));
  return HAPX_OK;
}

template <typename T>
static int launch_quantize(const QuantJobs& jobs, const CUtensorMap* maps, int n_sm, cudaStream_t stream) {
  constexpr int kShared = kBlock * kBlock * sizeof(T) + 128;
  {  // function attributes are per device
    static bool set[64] = {};
    static std::mutex mutex;
    int device = 0;
    HAPX_CUDA(cudaGetDevice(&device));
    if (device < 0 || device >= 64) return fail(HAPX_ERR_ARGUMENT, "block8_quantize: device index out of range");
    std::lock_guard<std::mutex> lock(mutex);
    if (!set[device]) {
      HAPX_CUDA(cudaFuncSetAttribute(quantize_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kShared));
      set[device] = true;
    }
  }
  const int grid = (int)std::min<long long>(jobs.tiles, (long long)n_sm * (sizeof(T) == 2 ? 3 : 2));     // one resident wave
  quantize_kernel<T><<<grid, 256, kShared, stream>>>(jobs, maps[0], maps[1]);
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

int quantize(QuantJob* job, int n_jobs, int dtype, cudaStream_t stream) {
  QuantJobs jobs;
  CUtensorMap maps[2];
  std::memset(maps, 0, sizeof(maps));
  int n_sm = 0;
  if (int e = gemm::error_word(&jobs.error, &n_sm)) return e;
  const long long es = dtype == HAPX_BF16 ? 2 : 4;
  for (int i = 0; i < n_jobs; ++i) {
    job[i].row_tiles = (int)((job[i].rows + kBlock - 1) / kBlock);
    job[i].col_tiles = (int)((job[i].cols + kBlock - 1) / kBlock);
    jobs.job[i] = job[i];
    jobs.tiles = (i ? jobs.tiles0 : 0) + (long long)job[i].row_tiles * job[i].col_tiles;
    if (i == 0) jobs.tiles0 = jobs.tiles;
    // the map's extents and its coordinates are 32 bits wide
    jobs.bulk[i] = (reinterpret_cast<uintptr_t>(job[i].x) & 15u) == 0 && job[i].ldx * es % 16 == 0 && job[i].ldx * es < (1ll << 40) &&
                   job[i].rows < 0x7fffff00 && job[i].cols < 0x7fffff00;
    if (jobs.bulk[i])
      if (int e = make_map(&maps[i], job[i], dtype)) return e;
  }
  if (n_jobs == 1) jobs.bulk[1] = 0;
  return dtype == HAPX_BF16 ? launch_quantize<__nv_bfloat16>(jobs, maps, n_sm, stream) : launch_quantize<float>(jobs, maps, n_sm, stream);
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
