// Activations in 8 bits: of each group of neighbouring values of a row, one fp32 scale, the least power of two with max |v| <= 448 scale,
// and v / scale in e4m3 (rounded to the nearest, ties to even).  A power of two divides exactly, so the only rounding is the format's own.
// Infinities are left out of the maximum and become 448 scale; NaN stays.  A group of zeros has the least scale there is.
// A magnitude just below a power of two rounds up to it, which its type may not have: 256 times the largest scale, 2^120, is no fp32, and 256 times 2^8 no
// fp16.  What is finite stays so: at the scale of 2^120 240 is the most that a byte stands for, and a value in 16 bits is at most the largest there is.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "ttt_elem.cuh"

namespace ttt {

// Largest of eight magnitudes.  NaN is left out by the maximum itself; where an infinity comes of it the finite ones are looked for.
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, fabsf(b)); }
__device__ __forceinline__ float magnitude(const float (&v)[8]) {
  const float a = larger(larger(fabsf(v[0]), v[1]), v[2]), b = larger(larger(fabsf(v[3]), v[4]), v[5]);
  float most = fmaxf(larger(larger(a, v[6]), v[7]), b);
  if (!(most < INFINITY)) {      // (or all of them are NaN)
    most = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = fabsf(v[j]) < INFINITY ? larger(most, v[j]) : most;
  }
  return most;
}
// Exponent field of the scale of a group whose largest magnitude has these bits: 8 less than that of amax / 1.75 rounded up, at least 1.
__device__ __forceinline__ uint32_t scale_exponent(float most) { return max(static_cast<int>((__float_as_uint(most) + 0x1fffffu) >> 23) - 8, 1); }
__device__ __forceinline__ float scale_of(uint32_t e) { return __uint_as_float(e << 23); }
__device__ __forceinline__ float inverse_of(uint32_t e) { return __uint_as_float((254u - e) << 23); }      // (e is at most 255 - 8, of magnitudes above 1.75 2^127: no subnormal)

// Two values to two bytes.
__device__ __forceinline__ uint32_t two_bytes(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 two_values(uint32_t bytes) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(bytes), __NV_E4M3)));
}

constexpr float kLargestScale = 0x1p120f;
// The largest magnitude that unpacking gives.
template <class T> constexpr float kMostOf = std::is_same<T, __half>::value ? 65504.f : 240.f * kLargestScale;

// Eight neighbouring values in memory, in pieces of up to 16 bytes where they start on a boundary.
template <class T> struct Eight {
  alignas(16) T v[8];
  using Piece = typename std::conditional<sizeof(T) == 1, uint2, uint4>::type;
  static constexpr int kPieces = 8 * sizeof(T) / sizeof(Piece);
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) reinterpret_cast<Piece*>(v)[i] = reinterpret_cast<const Piece*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) reinterpret_cast<Piece*>(p)[i] = reinterpret_cast<const Piece*>(v)[i];
  }
  // the first n of them, from and to any boundary
  __device__ __forceinline__ void load(const T* p, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : T();
  }
  __device__ __forceinline__ void store(T* p, int n) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = v[i];
  }
};

}  // namespace ttt
