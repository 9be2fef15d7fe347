// Sums of the parts that the CTAs of a backward pass leave of a gradient that all of them share, in a fixed order, so that the
// same call gives the same bits.  Thread columns run along the values, `ry` thread rows split the parts where there are few
// values; each row adds its parts in order and the rows are added in order.
#include <algorithm>

#include "ttt_elem.cuh"
#include "ttt_sum_parts.h"

namespace {

using namespace ttt;

struct Jobs {
  ttt_sum_job job[TTT_SUM_JOBS];
  int first[TTT_SUM_JOBS + 1];      // block of a job
  int ry[TTT_SUM_JOBS];
  int count;
};

template <class T> __device__ __forceinline__ void put(void* dst, long i, float v) { static_cast<T*>(dst)[i] = from_f32<T>(v); }

__global__ void __launch_bounds__(256) sum_parts_kernel(const Jobs jobs) {
  __shared__ float rows[256];
  int k = 0;
  while (static_cast<int>(blockIdx.x) >= jobs.first[k + 1]) ++k;
  const ttt_sum_job j = jobs.job[k];
  const int ry = jobs.ry[k], cols = 256 / ry, col = threadIdx.x % cols, r = threadIdx.x / cols;
  const long i = static_cast<long>(blockIdx.x - jobs.first[k]) * cols + col;
  float s = 0.f;
  if (i < j.n) {
    const int per = (j.parts + ry - 1) / ry, end = min((r + 1) * per, j.parts);
#pragma unroll 8
    for (int q = r * per; q < end; ++q) s += j.src[q * j.stride + i];
  }
  if (ry > 1) {
    rows[threadIdx.x] = s;
    __syncthreads();
    if (r) return;
    for (int q = 1; q < ry; ++q) s += rows[q * cols + col];
  }
  if (i >= j.n) return;
  const long o = j.turn ? i % j.turn * (j.n / j.turn) + i / j.turn : i;
  if (j.dtype == TTT_B200_BF16) put<__nv_bfloat16>(j.dst, o, s);
  else if (j.dtype == TTT_B200_FP16) put<__half>(j.dst, o, s);
  else put<float>(j.dst, o, s);
}

}  // namespace

int ttt_sum_parts(const ttt_sum_job* job, int count, cudaStream_t stream) {
  Jobs jobs = {};
  long blocks = 0;
  for (int k = 0; k < count; ++k) {
    if (!job[k].dst || job[k].n == 0) continue;
    int ry = 1;
    while (job[k].n < 65536 && ry < 16 && ry * 4 <= job[k].parts) ry *= 2;
    const int c = jobs.count++;
    jobs.job[c] = job[k];
    jobs.ry[c] = ry;
    jobs.first[c] = static_cast<int>(blocks);
    blocks += (job[k].n + 256 / ry - 1) / (256 / ry);
    if (blocks > 0x7fffffffL) return ttt_set_error(TTT_B200_ERR_BAD_ARGS, "sum of parts: too many values");
    jobs.first[c + 1] = static_cast<int>(blocks);
  }
  if (!jobs.count) return TTT_B200_OK;
  sum_parts_kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(jobs);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TTT_B200_OK : ttt_set_error(TTT_B200_ERR_LAUNCH, cudaGetErrorString(e));
}
