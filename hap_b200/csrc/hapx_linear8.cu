// F.linear with its products in 8-bit blocks (hapx_block8.h): one C call per direction.
//
// Forward: x in 1 x 128 blocks (and, for the weight gradient, in 128 x 1 blocks, transposed), w in 128 x 128 tiles (and
// transposed, for the input gradient), both in one launch, then the product.  Backward: g likewise in both forms from one
// read, with the partial sums of the bias gradient, then the two products in one launch, which joins those sums.
//
// 8192 x 768 -> 2304 (bfloat16), forward and both gradients: 80 us (28 + 48 one direction at a time: quantisers 12 + 19,
// products 16 + 28); with bfloat16 products 104.  -> 33280: 765 us (234 + 525) against 1130.
//
// Up to 32 tokens through a weight that is already in 8 bits take one launch: the product's, which converts x by itself.
#include <algorithm>
#include <mutex>
#include <string>

#include "hapx_block8.h"
#include "hapx_internal.h"

namespace hapx {
namespace linear8 {

using namespace block8;

constexpr int kThinTokens = 2;              // 2 x 768 -> 2304 takes 4.1 us here, 2 x 768 -> 33280 14.4; 4 tokens on the tensor cores 5.7 and 12.7
constexpr int kThinElements = 24 * 1024;    // tokens x in_features that fit shared memory as float32 (96 KiB)

// One or two tokens: y[m, n] = sum over blocks of s_x s_w sum of q_x q_w, + bias.  No tensor cores: the time is that of the
// launch and of reading the weight (bytes N K).  Every thread block makes the 8-bit form of x for itself in shared memory, a
// warp multiplies ROWS rows of w, whose loads are in flight together, with all tokens from registers; the values multiplied
// are those of the other path.  One token, 768 -> 2304: 3.0 us, 768 -> 33280: 11.0 us = 2.3 TB/s (of L2), where its blocks are
// too many for one round of the SMs.
// A sum of 16 products of e4m3 numbers is 0 or lies in [2^-18, 2^22): with a weight's scale in [2^-108, 2^105] it stays a
// normal number, and the token's scale then rounds it once at most.
constexpr int kNearLow = 127 - 108, kNearHigh = 127 + 105;
// MT: tokens, rounded up to a power of two.
template <typename T, int MT, int ROWS>
__global__ void __launch_bounds__(256) thin_kernel(const T* __restrict__ x, long long ldx, const unsigned char* __restrict__ w, long long ldw,
                                                   const unsigned char* __restrict__ ws, const T* __restrict__ bias, T* __restrict__ y, int M,
                                                   int N, int K) {
  extern __shared__ float4 s_mem[];
  const int kpad = (K + kBlock - 1) / kBlock * kBlock, blocks = kpad / kBlock;
  float* s_x = reinterpret_cast<float*>(s_mem);          // [token][kpad] e4m3 values, unscaled
  int* s_e = reinterpret_cast<int*>(s_x + (long long)M * kpad);      // [token][block] exponents of the scales
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool vec = (ldx & 3) == 0 && (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0;
  for (int i = warp; i < M * blocks; i += 8) {
    const int m = i / blocks, kb = i - m * blocks, k = kb * kBlock + 4 * lane;
    float v[4];
    load4(x + (long long)m * ldx + k, vec, max(0, min(4, K - k)), v);
    float big = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = finite_or_nan(v[j]); big = fmaxf(big, fabsf(v[j])); }
    const int e = scale_exponent(warp_max(big));
    const float inv = pow2(-e);
    const unsigned q = pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    const float2 lo = unpack2(q & 0xffffu), hi = unpack2(q >> 16);
    *reinterpret_cast<float4*>(s_x + (long long)m * kpad + k) = make_float4(lo.x, lo.y, hi.x, hi.y);
    if (lane == 0) s_e[m * blocks + kb] = e;
  }
  __syncthreads();
  // ROWS rows of w at a time: their loads in flight together, x read from shared memory once for all of them
  const long long groups = ((long long)N + kBlock - 1) / kBlock;
  // (unsigned: N may come within 256 of 2^31, where a row number plus the stride leaves 31 bits)
  for (unsigned first = (blockIdx.x * 8 + warp) * ROWS; first < (unsigned)N; first += gridDim.x * 8 * ROWS) {
    const int n0 = (int)first;
    float acc[ROWS][MT];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[r][m] = 0.f;
    for (int k = 16 * lane; k < K; k += 512) {           // 16 values of one block of 128
      uint4 raw[ROWS];
      int e[ROWS];
      const int kb = k / kBlock;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const int n = min(n0 + r, N - 1);
        raw[r] = __ldg(reinterpret_cast<const uint4*>(w + (long long)n * ldw + k));
        e[r] = ws[scale_at(n, kb, groups)];
      }
      bool far = false;                                  // a scale that may carry a sum of 16 products out of float32 by itself
#pragma unroll
      for (int r = 0; r < ROWS; ++r) far |= (unsigned)(e[r] - kNearLow) > (unsigned)(kNearHigh - kNearLow);
      float part[ROWS][MT];
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int m = 0; m < MT; ++m) part[r][m] = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int left = K - (k + 4 * c);                // bytes behind the row's end are padding
        float4 xv[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) xv[m] = *reinterpret_cast<const float4*>(s_x + (long long)min(m, M - 1) * kpad + k + 4 * c);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const unsigned word = c == 0 ? raw[r].x : c == 1 ? raw[r].y : c == 2 ? raw[r].z : raw[r].w;
          const float2 a = unpack2(word & 0xffffu), b = unpack2(word >> 16);
          const float v[4] = {left > 0 ? a.x : 0.f, left > 1 ? a.y : 0.f, left > 2 ? b.x : 0.f, left > 3 ? b.y : 0.f};
#pragma unroll
          for (int m = 0; m < MT; ++m)
            part[r][m] = fmaf(v[0], xv[m].x, fmaf(v[1], xv[m].y, fmaf(v[2], xv[m].z, fmaf(v[3], xv[m].w, part[r][m]))));
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int ex = s_e[min(m, M - 1) * blocks + kb];
        if (!far) {
#pragma unroll
          for (int r = 0; r < ROWS; ++r) acc[r][m] = fmaf(part[r][m] * pow2(e[r] - 127), pow2(ex), acc[r][m]);
        } else {                                         // rare: both scales as one power of two, in halves that are normal numbers
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            const int both = e[r] - 127 + ex, half = both >> 1;
            acc[r][m] = fmaf(part[r][m] * pow2(half), pow2(both - half), acc[r][m]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[r][m] += __shfl_xor_sync(0xffffffffu, acc[r][m], o);
        if (lane == r * MT + m && m < M && n0 + r < N)
          y[(long long)m * N + n0 + r] = from_f<T>(bias ? acc[r][m] + to_f(bias[n0 + r]) : acc[r][m]);
      }
    }
  }
}

template <typename T, int MT>
static int launch_thin(const void* x, long long ldx, const void* w, long long ldw, const void* ws, const void* bias, void* y, int M, int N, int K,
                       int n_sm, cudaStream_t stream) {
  const int kpad = (K + kBlock - 1) / kBlock * kBlock, smem = M * kpad * 4 + M * (kpad / kBlock) * 4;
  constexpr int ROWS = 4;
  auto kernel = thin_kernel<T, MT, ROWS>;
  {  // function attributes are per device
    static bool set[64] = {};
    static std::mutex mutex;
    int device = 0;
    HAPX_CUDA(cudaGetDevice(&device));
    std::lock_guard<std::mutex> lock(mutex);
    if (device < 0 || device >= 64) return fail(HAPX_ERR_ARGUMENT, "linear8: device index out of range");
    if (!set[device]) {
      HAPX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kThinElements * 4 + kThinElements / kBlock * 4));
      set[device] = true;
    }
  }
  const int grid = std::min((N + 8 * ROWS - 1) / (8 * ROWS), n_sm * (smem <= 48 * 1024 ? 4 : 2));
  kernel<<<grid, 256, smem, stream>>>(static_cast<const T*>(x), ldx, static_cast<const unsigned char*>(w), ldw, static_cast<const unsigned char*>(ws),
                                      static_cast<const T*>(bias), static_cast<T*>(y), M, N, K);
  HAPX_CUDA(cudaGetLastError());
  count_launch();
  return HAPX_OK;
}

static bool thin(long long m, long long k) { return m <= kThinTokens && m * ((k + kBlock - 1) / kBlock * kBlock) <= kThinElements; }

static long long up(long long n, long long to) { return (n + to - 1) / to * to; }

// Pieces of a workspace, 256-byte aligned, in the order they are asked for.
struct Carve {
  char* base;
  long long used = 0;
  explicit Carve(void* p) : base(static_cast<char*>(p)) {}
  unsigned char* take(long long bytes) {
    unsigned char* p = reinterpret_cast<unsigned char*>(base) + used;
    used += up(bytes, 256);
    return p;
  }
};

struct Forward { unsigned char *x8, *x8s, *w8, *w8s, *split; long long bytes; };
// How x reaches the product: kThin, kConvert (both for a weight in 8 bits, when x's form is not kept), kQuantise.
enum Path { kThin, kConvert, kQuantise };
static Path path_of(long long m, long long k, bool prepared, bool keep_x) {
  if (!prepared || keep_x) return kQuantise;
  return thin(m, k) ? kThin : gemm8::converts(m) ? kConvert : kQuantise;
}
static Forward layout_forward(void* base, long long m, long long n, long long k, bool prepared, Path path, int n_sm) {
  Carve c(base);
  Forward f = {};
  if (path != kThin) {
    if (path == kQuantise) {
      f.x8 = c.take(m * up(k, 16));
      f.x8s = c.take(scale_bytes(m, k));
    }
    if (!prepared) { f.w8 = c.take(n * up(k, 16)); f.w8s = c.take(scale_bytes(n, k)); }
    f.split = c.take(gemm8::workspace_bytes(m, n, k, n_sm));
  }
  f.bytes = c.used;
  return f;
}

struct Backward { unsigned char *g8, *g8s, *g8t, *g8ts, *colsum, *split; long long bytes; };
static Backward layout_backward(void* base, long long m, long long n, long long k, bool dx, bool dw, bool db, int n_sm) {
  Carve c(base);
  Backward b = {};
  if (dx || !dw) { b.g8 = c.take(m * up(n, 16)); b.g8s = c.take(scale_bytes(m, n)); }      // the quantiser writes one form at least
  if (dw) { b.g8t = c.take(n * up(m, 16)); b.g8ts = c.take(scale_bytes(n, m)); }
  if (db) b.colsum = c.take((m + kBlock - 1) / kBlock * n * 4);
  long long split = 0;
  if (dx && dw) {
    gemm8::Product x, w;
    x.m = m; x.n = k; x.k = n;
    w.m = n; w.n = k; w.k = m;
    split = gemm8::workspace_bytes_two(x, w, n_sm);
  } else if (dx) {
    split = gemm8::workspace_bytes(m, k, n, n_sm);
  } else if (dw) {
    split = gemm8::workspace_bytes(n, k, m, n_sm);
  }
  b.split = c.take(split);
  b.bytes = c.used;
  return b;
}

static int check(const char* who, int dtype, int64_t m, int64_t n, int64_t k) {
  if (dtype != HAPX_F32 && dtype != HAPX_BF16) return fail(HAPX_ERR_DTYPE, std::string(who) + ": float32 or bfloat16 only");
  if (m < 0 || n < 1 || k < 1 || m > 0x7fffff00 || n > 0x7fffff00 || k > 0x7fffff00)
    return fail(HAPX_ERR_EXTENT, std::string(who) + ": extents must lie below 2^31 - 256, features at 1 or above");
  return HAPX_OK;
}
static bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace linear8
}  // namespace hapx

using namespace hapx;
using namespace hapx::linear8;

extern "C" {

int64_t hapx_linear8_forward_workspace(int64_t m, int64_t n, int64_t k, int prepared, int keep_x) {
  int n_sm = 0;
  if (m < 1 || n < 1 || k < 1 || sm_count(&n_sm)) return 0;
  return layout_forward(nullptr, m, n, k, prepared != 0, path_of(m, k, prepared != 0, keep_x != 0), n_sm).bytes;
}

int hapx_linear8_forward(void* y, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* w8, const void* w8_scale, const void* bias,
                         int dtype, int64_t m, int64_t n, int64_t k, void* x8t, void* x8t_scale, void* w8t, void* w8t_scale, void* workspace,
                         int64_t workspace_bytes, hapx_stream stream_) {
  if (int e = check("linear8_forward", dtype, m, n, k)) return e;
  const bool prepared = w == nullptr;
  if (m == 0 && (prepared || !w8t)) return HAPX_OK;
  if ((m > 0 && (!y || !x)) || (prepared && (!w8 || !w8_scale)) || (x8t && !x8t_scale) || (w8t && !w8t_scale) || (prepared && w8t))
    return fail(HAPX_ERR_ARGUMENT, "linear8_forward: null pointer, or a transposed form asked of a weight that is given in 8 bits");
  if (ldx < k || (!prepared && ldw < k)) return fail(HAPX_ERR_EXTENT, "linear8_forward: a row pitch is smaller than its row");
  if (!aligned(w8) || !aligned(w8_scale) || !aligned(x8t) || !aligned(x8t_scale) || !aligned(w8t) || !aligned(w8t_scale))
    return fail(HAPX_ERR_EXTENT, "linear8_forward: 8-bit operands and their scales need 16-byte aligned bases");
  int n_sm = 0;
  if (int e = sm_count(&n_sm)) return e;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const Path path = path_of(m, k, prepared, x8t != nullptr);
  const Forward f = layout_forward(workspace, m, n, k, prepared, path, n_sm);
  if (workspace_bytes < f.bytes || (f.bytes > 0 && (!workspace || !aligned(workspace))))
    return fail(HAPX_ERR_ARGUMENT, "linear8_forward: the workspace must be 16-byte aligned and as large as hapx_linear8_forward_workspace says");
  if (path == kThin) {
    const int M = (int)m, N = (int)n, K = (int)k;
#define HAPX_THIN(T, MT) return launch_thin<T, MT>(x, ldx, w8, up(k, 16), w8_scale, bias, y, M, N, K, n_sm, stream)
    if (dtype == HAPX_BF16) {
      if (m == 1) HAPX_THIN(__nv_bfloat16, 1);
      HAPX_THIN(__nv_bfloat16, 2);
    }
    if (m == 1) HAPX_THIN(float, 1);
    HAPX_THIN(float, 2);
#undef HAPX_THIN
  }
  gemm8::Product p;
  p.d = y; p.out_f32 = dtype == HAPX_F32; p.lda = up(k, 16);
  p.b = prepared ? w8 : f.w8; p.ldb = up(k, 16); p.b_scale = prepared ? w8_scale : f.w8s;
  p.bias = bias; p.m = m; p.n = n; p.k = k; p.workspace = f.split;
  if (path == kConvert) return gemm8::run_converting(p, x, dtype, ldx, n_sm, stream);
  QuantJob jobs[2];
  int n_jobs = 0;
  if (m > 0) {
    QuantJob& j = jobs[n_jobs++];
    j.x = x; j.rows = m; j.cols = k; j.ldx = ldx; j.q = f.x8; j.ldq = up(k, 16); j.s = f.x8s;
    j.qt = static_cast<unsigned char*>(x8t); j.ldqt = up(m, 16); j.st = static_cast<unsigned char*>(x8t_scale);
  }
  if (!prepared) {
    QuantJob& j = jobs[n_jobs++];
    j.x = w; j.rows = n; j.cols = k; j.ldx = ldw; j.square = 1; j.q = f.w8; j.ldq = up(k, 16); j.s = f.w8s;
    j.qt = static_cast<unsigned char*>(w8t); j.ldqt = up(n, 16); j.st = static_cast<unsigned char*>(w8t_scale);
  }
  if (int e = quantize(jobs, n_jobs, dtype, stream)) return e;
  if (m == 0) return HAPX_OK;
  p.a = f.x8; p.a_scale = f.x8s;
  return gemm8::run(p, n_sm, stream);
}

int64_t hapx_linear8_backward_workspace(int64_t m, int64_t n, int64_t k, int dx, int dw, int db) {
  int n_sm = 0;
  if (m < 1 || n < 1 || k < 1 || sm_count(&n_sm)) return 0;
  return layout_backward(nullptr, m, n, k, dx != 0, dw != 0, db != 0, n_sm).bytes;
}

int hapx_linear8_backward(void* dx, void* dw, void* db, const void* g, int64_t ldg, int dtype, int64_t m, int64_t n, int64_t k, const void* w8t,
                          const void* w8t_scale, const void* x8t, const void* x8t_scale, void* workspace, int64_t workspace_bytes,
                          hapx_stream stream_) {
  if (int e = check("linear8_backward", dtype, m, n, k)) return e;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (m == 0) {                     // no tokens: the parameters' gradients are zero
    const size_t es = dtype == HAPX_F32 ? 4 : 2;
    if (dw) HAPX_CUDA(cudaMemsetAsync(dw, 0, (size_t)n * k * es, stream));
    if (db) HAPX_CUDA(cudaMemsetAsync(db, 0, (size_t)n * es, stream));
    return HAPX_OK;
  }
  if (!dx && !dw && !db) return HAPX_OK;
  if (!g || (dx && (!w8t || !w8t_scale)) || (dw && (!x8t || !x8t_scale))) return fail(HAPX_ERR_ARGUMENT, "linear8_backward: null pointer");
  if (ldg < n) return fail(HAPX_ERR_EXTENT, "linear8_backward: the row pitch is smaller than the row");
  if (!aligned(w8t) || !aligned(w8t_scale) || !aligned(x8t) || !aligned(x8t_scale))
    return fail(HAPX_ERR_EXTENT, "linear8_backward: 8-bit operands and their scales need 16-byte aligned bases");
  int n_sm = 0;
  if (int e = sm_count(&n_sm)) return e;
  const Backward b = layout_backward(workspace, m, n, k, dx, dw, db, n_sm);
  if (workspace_bytes < b.bytes || !workspace || !aligned(workspace))
    return fail(HAPX_ERR_ARGUMENT, "linear8_backward: the workspace must be 16-byte aligned and as large as hapx_linear8_backward_workspace says");
  QuantJob j;
  j.x = g; j.rows = m; j.cols = n; j.ldx = ldg; j.q = b.g8; j.ldq = up(n, 16); j.s = b.g8s; j.qt = b.g8t; j.ldqt = up(m, 16); j.st = b.g8ts;
  j.colsum = reinterpret_cast<float*>(b.colsum);
  if (int e = quantize(&j, 1, dtype, stream)) return e;
  gemm8::Product px, pw;
  if (dx) {
    px.d = dx; px.out_f32 = dtype == HAPX_F32; px.a = b.g8; px.lda = up(n, 16); px.a_scale = b.g8s; px.b = w8t; px.ldb = up(n, 16);
    px.b_scale = w8t_scale; px.m = m; px.n = k; px.k = n; px.workspace = b.split;
  }
  if (dw) {
    pw.d = dw; pw.out_f32 = dtype == HAPX_F32; pw.a = b.g8t; pw.lda = up(m, 16); pw.a_scale = b.g8ts; pw.b = x8t; pw.ldb = up(m, 16);
    pw.b_scale = x8t_scale; pw.m = n; pw.n = k; pw.k = m; pw.workspace = b.split;
    if (db) { pw.colsum = reinterpret_cast<const float*>(b.colsum); pw.colsum_tiles = (int)((m + kBlock - 1) / kBlock); pw.colsum_out = db; }
  }
  if (dx && dw) return gemm8::run_two(px, pw, n_sm, stream);
  if (dw) return gemm8::run(pw, n_sm, stream);
  if (dx)
    if (int e = gemm8::run(px, n_sm, stream)) return e;
  return db ? hapx_block8_colsum_join(db, dtype, reinterpret_cast<const float*>(b.colsum), m, n, stream_) : HAPX_OK;
}

}  // extern "C"
