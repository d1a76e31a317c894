// 8-bit blocks: e4m3 values with one power-of-two scale per block of 128 elements, shared by the quantiser, the
// block-scaled product and the operators that keep their input for the backward pass in 8 bits.
//
// A block's scale is 2^e with the smallest integer e >= -126 for which the block's largest magnitude is at most
// 448 * 2^e (448 = 1.75 * 2^8 is the largest e4m3 number); a block of zeros has e = 0.  Scaling by a power of two is
// exact, so the stored value is the correctly rounded (to nearest, ties to even) e4m3 number of x * 2^-e and the
// only error of a block is that one rounding: half a step of 3 fraction bits, 2^-4 relative, for magnitudes down to
// 2^-14 of the block's largest one.  e4m3 has no infinity: infinities and NaN become NaN and do not enter the maximum.
//
// A matrix's scales are kept as the bytes e + 127 in the order the tensor cores take them: 512 bytes for every 128 rows
// and 4 blocks of columns, in them 16 bytes for each of 32 lanes (row % 32), 4 for each row / 32, one per block.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

namespace hapx {
namespace block8 {

constexpr int kBlock = 128;

// Exponent of the scale of a block whose largest finite magnitude is `big` (>= 0).
__device__ __forceinline__ int scale_exponent(float big) {
  const unsigned b = __float_as_uint(big);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);   // 0x600000: the fraction of 1.75
  return b == 0u ? 0 : max(e, -126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 <= e <= 127

__host__ __device__ __forceinline__ long long scale_bytes(long long rows, long long cols) {
  return ((cols + 511) / 512) * ((rows + 127) / 128) * 512;
}
// Where the scale of row r and column block kb is; `groups` = ceil(rows / 128).
__device__ __forceinline__ long long scale_at(long long r, long long kb, long long groups) {
  return ((kb >> 2) * groups + (r >> 7)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (kb & 3);
}

// Infinities become NaN; fmaxf then leaves both out of a block's maximum.
__device__ __forceinline__ float finite_or_nan(float v) {
  return (__float_as_uint(v) & 0x7fffffffu) >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : v;
}

// Four values, already scaled, as four e4m3 bytes (the first in the low byte); NaN stays NaN.
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d) {
  unsigned r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
__device__ __forceinline__ float2 unpack2(unsigned two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

__device__ __forceinline__ float warp_max(float v) {   // v >= 0 and not NaN: the bit patterns order like the numbers
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Four consecutive elements; `vec` says that p is aligned to all four.
template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vec, int valid, float (&f)[4]) {
  if (vec && valid >= 4) {
    if constexpr (sizeof(T) == 2) {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      f[0] = __uint_as_float(w.x << 16); f[1] = __uint_as_float(w.x & 0xffff0000u);
      f[2] = __uint_as_float(w.y << 16); f[3] = __uint_as_float(w.y & 0xffff0000u);
    } else {
      const float4 v = *reinterpret_cast<const float4*>(p);
      f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = j < valid ? to_f(p[j]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, bool vec, int valid, const float (&f)[4]) {
  if (vec && valid >= 4) {
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
      *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
    } else {
      *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < valid) p[j] = from_f<T>(f[j]);
  }
}

// Four consecutive elements as they are in memory, and what the quantiser asks of them.  A magnitude's pattern is its
// float32 bits (of a bfloat16 the upper half, with anything below); patterns order like the numbers.  A NaN loses
// against any number, an infinity wins.
template <typename T> struct Raw4;
template <> struct Raw4<__nv_bfloat16> {
  uint2 w;
  struct Max { __nv_bfloat162 a, b; };                 // of columns 0, 1 and 2, 3
  static constexpr unsigned kMask = 0xffff0000u;       // a pattern's own bits
  static __device__ __forceinline__ __nv_bfloat162 two(unsigned v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); }
  static __device__ __forceinline__ unsigned bits(__nv_bfloat162 v) { return *reinterpret_cast<const unsigned*>(&v); }
  __device__ __forceinline__ void zero() { w = make_uint2(0u, 0u); }
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void load_shared(const unsigned char* tile, int row, int lane) { w = reinterpret_cast<const uint2*>(tile)[row * 32 + lane]; }
  __device__ __forceinline__ void load_some(const __nv_bfloat16* p, int valid) {
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
    w.x = (valid > 0 ? h[0] : 0u) | (valid > 1 ? (unsigned)h[1] << 16 : 0u);
    w.y = (valid > 2 ? h[2] : 0u) | (valid > 3 ? (unsigned)h[3] << 16 : 0u);
  }
  __device__ __forceinline__ void get(float (&f)[4]) const {
    f[0] = __uint_as_float(w.x << 16); f[1] = __uint_as_float(w.x & 0xffff0000u);
    f[2] = __uint_as_float(w.y << 16); f[3] = __uint_as_float(w.y & 0xffff0000u);
  }
  static __device__ __forceinline__ void clear(Max& m) { m.a = m.b = two(0u); }
  // joins the column maxima, returns the row's pattern
  __device__ __forceinline__ unsigned maxima(Max& m) const {
    const __nv_bfloat162 x = __habs2(two(w.x)), y = __habs2(two(w.y));
    m.a = __hmax2(m.a, x); m.b = __hmax2(m.b, y);
    const __nv_bfloat162 r = __hmax2(__hmax2(x, y), two(0u));                       // of two NaN: 0
    return bits(__hmax2(r, two(__byte_perm(bits(r), 0u, 0x1032))));
  }
  static __device__ __forceinline__ void columns(const Max& m, unsigned (&c)[4]) {
    c[0] = bits(m.a) << 16; c[1] = bits(m.a); c[2] = bits(m.b) << 16; c[3] = bits(m.b);
  }
  // infinities become NaN
  __device__ __forceinline__ void sanitise() {
    if ((w.x & 0x7f80u) == 0x7f80u) w.x |= 0x7fffu;
    if ((w.x & 0x7f800000u) == 0x7f800000u) w.x |= 0x7fff0000u;
    if ((w.y & 0x7f80u) == 0x7f80u) w.y |= 0x7fffu;
    if ((w.y & 0x7f800000u) == 0x7f800000u) w.y |= 0x7fff0000u;
  }
};
template <> struct Raw4<float> {
  float4 v;
  struct Max { float c[4]; };
  static constexpr unsigned kMask = 0xffffffffu;
  __device__ __forceinline__ void zero() { v = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void load_shared(const unsigned char* tile, int row, int lane) { v = reinterpret_cast<const float4*>(tile)[row * 32 + lane]; }
  __device__ __forceinline__ void load_some(const float* p, int valid) {
    zero();
    if (valid > 0) v.x = p[0];
    if (valid > 1) v.y = p[1];
    if (valid > 2) v.z = p[2];
    if (valid > 3) v.w = p[3];
  }
  __device__ __forceinline__ void get(float (&f)[4]) const { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
  static __device__ __forceinline__ void clear(Max& m) { m.c[0] = m.c[1] = m.c[2] = m.c[3] = 0.f; }
  __device__ __forceinline__ unsigned maxima(Max& m) const {
    m.c[0] = fmaxf(m.c[0], fabsf(v.x)); m.c[1] = fmaxf(m.c[1], fabsf(v.y)); m.c[2] = fmaxf(m.c[2], fabsf(v.z)); m.c[3] = fmaxf(m.c[3], fabsf(v.w));
    return __float_as_uint(fmaxf(fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))), 0.f));
  }
  static __device__ __forceinline__ void columns(const Max& m, unsigned (&c)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = __float_as_uint(m.c[j]);
  }
  __device__ __forceinline__ void sanitise() { v = make_float4(finite_or_nan(v.x), finite_or_nan(v.y), finite_or_nan(v.z), finite_or_nan(v.w)); }
};

}  // namespace block8
}  // namespace hapx
