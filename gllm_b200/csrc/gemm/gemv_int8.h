// The 8-bit product of a few rows (gemv_int8.cu): x [M, K] bf16 (rows ldx apart), w [N, K] int8 with w_scale [N] -> c [M, N], gated [M, N / 2].
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

struct GemvInt8 {
  const __nv_bfloat16* x;
  int64_t ldx;
  const uint8_t* w;
  const float* w_scale;
  __nv_bfloat16* c;
  int64_t ldc;
  const __nv_bfloat16* bias;
  int N, K;
};

// whether the rows fit, and whether this is the form to take
bool gemv_int8_fits(int M, int K);
bool gemv_int8_takes(int M, int K);
// 0: launched
int gemv_int8(const GemvInt8& p, int M, bool gated, cudaStream_t st);

}  // namespace b200
