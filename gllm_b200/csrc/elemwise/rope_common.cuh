// What the rotary write kernels share (rope_kv.cu, rope_kv4.cu): their parameters and the choice of a pair's position row.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace b200 {

struct RopeParams {
  __nv_bfloat16* q; int64_t q_ts, q_hs; int Hq;
  __nv_bfloat16* k; int64_t k_ts, k_hs; int Hkv;
  const __nv_bfloat16* v; int64_t v_ts, v_hs;
  const __nv_bfloat16* q_norm_w;
  const __nv_bfloat16* k_norm_w;
  const float* cos_sin;  // [max_pos, rot]: cos | sin
  int D, rot, neox, T;
  const int32_t* positions;  // [T] or [3, T] (mrope)
  const int32_t* slots;      // [T] or null
  float eps;
  __nv_bfloat16* k_cache;
  __nv_bfloat16* v_cache;
  int sec0, sec1, page_size;  // sec0 > 0: chunked M-RoPE [T|H|W]; sec0 < 0: interleaved (H = -sec0, W = sec1)
  int64_t pos_stride;         // row stride of a [3, T] positions tensor
};

// which of the (t, h, w) position rows rotary pair i uses
__device__ __forceinline__ int mrope_axis(int i, int sec0, int sec1) {
  if (sec0 > 0) return i < sec0 ? 0 : (i < sec0 + sec1 ? 1 : 2);
  if (sec0 < 0) {
    const int r = i % 3;
    if (r == 1 && i < -sec0 * 3) return 1;
    if (r == 2 && i < sec1 * 3) return 2;
  }
  return 0;
}

}  // namespace b200
