// Element types, packed fp32 arithmetic and small helpers of the layer-side sequence operators (short convolution,
// state space scan, block end).  Activations are bf16, fp16 or fp32; everything between reading and writing is fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "ttt_internal.h"

namespace ttt {

// First statement of every kernel here: the launch may have come before the one in front of it in the stream is through
// (ttt_launch_overlapped), and nothing global is touched until it is.
__device__ __forceinline__ void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Two fp32 operations in one instruction (sm_100): halves the issue slots of fp32-heavy loops.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// The same names for one value and for two, for code that takes either.
__device__ __forceinline__ float mac(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float2 mac(float2 a, float2 b, float2 c) { return fma2(a, b, c); }
__device__ __forceinline__ float times(float a, float b) { return a * b; }
__device__ __forceinline__ float2 times(float2 a, float2 b) { return mul2(a, b); }
__device__ __forceinline__ float plus(float a, float b) { return a + b; }
__device__ __forceinline__ float2 plus(float2 a, float2 b) { return add2(a, b); }
template <class F> __device__ __forceinline__ F all(float v) {
  if constexpr (sizeof(F) == 8) return both(v);
  else return v;
}
__device__ __forceinline__ float fold(float v) { return v; }
__device__ __forceinline__ float fold(float2 v) { return v.x + v.y; }

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float2 ex2(float2 v) { return make_float2(ex2(v.x), ex2(v.y)); }
__device__ __forceinline__ float2 rcp(float2 v) { return make_float2(rcp(v.x), rcp(v.y)); }
__device__ __forceinline__ float least(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ float2 least(float2 a, float b) { return make_float2(fminf(a.x, b), fminf(a.y, b)); }

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 16, 8 or 4 bytes global -> shared without registers, to a shared address; of a piece of `bytes` the rest becomes zeros and is not read.
__device__ __forceinline__ void cp_async16_at(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_at(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async8_at(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4_at(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {
  cp_async16_at(static_cast<uint32_t>(__cvta_generic_to_shared(dst)), src, bytes);
}
// from a shared address
__device__ __forceinline__ uint4 shared_load16(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
  return r;
}
__device__ __forceinline__ uint2 shared_load8(uint32_t at) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at) : "memory");
  return r;
}
template <class T> __device__ __forceinline__ float shared_load(uint32_t at) {
  if constexpr (sizeof(T) == 4) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
  } else {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
    return to_f32(reinterpret_cast<T&>(v));
  }
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// Sums V values over the L lanes that differ in the bits kStride, 2 kStride, ... of the lane index, by exchanging halves:
// V - V / L exchanges instead of V log2 L.  Value i of the sum ends in the lane whose index bits (lane / kStride) are
// i / (V / L), as its element i % (V / L); with V < L in the L / V lanes whose index bits are i L / V and on.
template <int V, int L, int kStride> __device__ __forceinline__ void spread_sum(float (&v)[V], int lane) {
  int n = V;      // a compile-time value after unrolling
#pragma unroll
  for (int m = L / 2; m >= 1; m /= 2) {
    if (n > 1) {
      n /= 2;
      const bool up = (lane / kStride) & m;
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
        if (i < n) {
          const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, m * kStride);
        }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], m * kStride);
    }
  }
}

// ---- host
inline int fail(const char* msg) { return ttt_set_error(TTT_B200_ERR_BAD_ARGS, msg); }
inline int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}
// what the launch in front has come to
inline int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return TTT_B200_OK;
  static thread_local char buf[160];
  snprintf(buf, sizeof buf, "%s: %s", what, cudaGetErrorString(e));
  return ttt_set_error(TTT_B200_ERR_LAUNCH, buf);
}
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace ttt

// Runs `body` with `Elem` as the activations' type.
#define TTT_WITH_TYPE(dtype, body)                                     \
  switch (dtype) {                                                     \
    case TTT_B200_BF16: { using Elem = __nv_bfloat16; body; break; }   \
    case TTT_B200_FP16: { using Elem = __half; body; break; }          \
    default: { using Elem = float; body; break; }                      \
  }
