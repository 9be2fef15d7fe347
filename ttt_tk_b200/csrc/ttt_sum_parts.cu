// Sums of the parts that the CTAs of a backward pass leave of a gradient that all of them share, in a fixed order, so that the
// same call gives the same bits.  Thread columns run along the values, `ry` thread rows split the parts where there are few
// values; each row adds its parts in order and the rows are added in order.  Bound by the reading of the parts: the scan's 35 MB of 4 x 2048 tokens,
// 1536 channels and 16 states in 11.4 us (3.1 TB/s), the convolution's of 4 x 2048 x 2048 in 3.8 us, a launch for the most part.
#include <algorithm>

#include "ttt_elem.cuh"
#include "ttt_sum_parts.h"

namespace {

using namespace ttt;

struct Jobs {
  ttt_sum_job job[TTT_SUM_JOBS];
  int first[TTT_SUM_JOBS + 1];      // block of a job
  int ry[TTT_SUM_JOBS];
  bool four[TTT_SUM_JOBS];      // four values to a thread
  int count;
};

template <class T> __device__ __forceinline__ void put(void* dst, long i, float v) { static_cast<T*>(dst)[i] = from_f32<T>(v); }

template <class T> __device__ __forceinline__ void put4(void* dst, long i, const float (&v)[4]) {
  alignas(4 * sizeof(T)) T t[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) t[k] = from_f32<T>(v[k]);
  T* to = static_cast<T*>(dst) + i;
  if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(to) = reinterpret_cast<uint4&>(t);
  else *reinterpret_cast<uint2*>(to) = reinterpret_cast<uint2&>(t);
}

// W values to a thread (one or four)
template <int W> __device__ __forceinline__ void add_up(const ttt_sum_job& j, int ry, int block, float4* rows) {
  const int cols = 256 / ry, col = threadIdx.x % cols, r = threadIdx.x / cols;
  const long i = (static_cast<long>(block) * cols + col) * W;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < j.n) {
    const int per = (j.parts + ry - 1) / ry, end = min((r + 1) * per, j.parts);
#pragma unroll 8
    for (int q = r * per; q < end; ++q) {
      if constexpr (W == 4) {
        const float4 v = *reinterpret_cast<const float4*>(j.src + q * j.stride + i);
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      } else {
        s.x += j.src[q * j.stride + i];
      }
    }
  }
  if (ry > 1) {
    rows[threadIdx.x] = s;
    __syncthreads();
    if (r) return;
    for (int q = 1; q < ry; ++q) {
      const float4 v = rows[q * cols + col];
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
  if (i >= j.n) return;
  if constexpr (W == 4) {
    const float v[4] = {s.x, s.y, s.z, s.w};
    if (j.dtype == TTT_B200_BF16) put4<__nv_bfloat16>(j.dst, i, v);
    else if (j.dtype == TTT_B200_FP16) put4<__half>(j.dst, i, v);
    else put4<float>(j.dst, i, v);
  } else {
    const long o = j.turn ? i % j.turn * (j.n / j.turn) + i / j.turn : i;
    if (j.dtype == TTT_B200_BF16) put<__nv_bfloat16>(j.dst, o, s.x);
    else if (j.dtype == TTT_B200_FP16) put<__half>(j.dst, o, s.x);
    else put<float>(j.dst, o, s.x);
  }
}

__global__ void __launch_bounds__(256) sum_parts_kernel(const Jobs jobs) {
  wait_for_predecessor();
  __shared__ float4 rows[256];
  int k = 0;
  while (static_cast<int>(blockIdx.x) >= jobs.first[k + 1]) ++k;
  const int block = blockIdx.x - jobs.first[k];
  if (jobs.four[k]) add_up<4>(jobs.job[k], jobs.ry[k], block, rows);
  else add_up<1>(jobs.job[k], jobs.ry[k], block, rows);
}

}  // namespace

int ttt_sum_parts(const ttt_sum_job* job, int count, cudaStream_t stream) {
  Jobs jobs = {};
  long blocks = 0;
  for (int k = 0; k < count; ++k) {
    if (!job[k].dst || job[k].n == 0) continue;
    const ttt_sum_job& j = job[k];
    const bool four = j.n % 4 == 0 && j.stride % 4 == 0 && !j.turn && aligned16(j.src) && aligned16(j.dst);
    const int width = four ? 4 : 1;
    int ry = 1;      // enough threads to hide the loads' latency, at least four parts to each
    while (j.n / width * ry < 262144 && ry < 16 && ry * 8 <= j.parts) ry *= 2;
    const int c = jobs.count++;
    jobs.job[c] = j;
    jobs.ry[c] = ry;
    jobs.four[c] = four;
    jobs.first[c] = static_cast<int>(blocks);
    const long values = 256 / ry * width;      // of a block
    blocks += (j.n + values - 1) / values;
    if (blocks > 0x7fffffffL) return ttt_set_error(TTT_B200_ERR_BAD_ARGS, "sum of parts: too many values");
    jobs.first[c + 1] = static_cast<int>(blocks);
  }
  if (!jobs.count) return TTT_B200_OK;
  ttt_launch_overlapped(sum_parts_kernel, static_cast<int>(blocks), 256, 0, stream, jobs);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TTT_B200_OK : ttt_set_error(TTT_B200_ERR_LAUNCH, cudaGetErrorString(e));
}
