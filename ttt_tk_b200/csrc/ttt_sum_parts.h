// Ordered sums of partial gradients (ttt_sum_parts.cu).
#pragma once

#include "ttt_internal.h"

constexpr int TTT_SUM_JOBS = 5;
struct ttt_sum_job {
  const float* src;
  void* dst;       // NULL: nothing to do
  long n;          // values
  long stride;     // part r of value i is src[r * stride + i]
  int parts;
  int dtype;       // of dst
  long turn;       // 0, or the inner length of a matrix that is written transposed
};
int ttt_sum_parts(const ttt_sum_job* jobs, int count, cudaStream_t stream);
