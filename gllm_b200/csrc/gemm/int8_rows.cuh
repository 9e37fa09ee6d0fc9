// How a row is quantised to 8-bit integers (gemm_int8.cu, gemv_int8.cu): scale a / 127 with its largest magnitude a, 2^-100 at least, values
// to the nearest multiple, ties to even.
#pragma once

#include "../common/ptx.cuh"
#include "../seq/seq_common.cuh"

namespace b200 {

constexpr float kQuantFloor = 7.888609052210118e-31f;    // 2^-100: rows below it are quantised with its step, so that 128 / a and scales are normal numbers

// the larger of two pairs of magnitudes, as bits: NaN is above infinity
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, uint32_t w) { return __vmaxu2(m, w & 0x7fff7fffu); }
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, const uint4& v) {
  return max_abs2(max_abs2(max_abs2(max_abs2(m, v.x), v.y), v.z), v.w);
}
// a from the pair; a NaN stays one
__device__ __forceinline__ float largest(uint32_t m) {
  const float found = __uint_as_float(max(m & 0xffffu, m >> 16) << 16);
  return found < kQuantFloor ? kQuantFloor : found;
}

// Eight bytes from eight bf16. The quotient 127 x / a to the nearest, ties to even, as in exact arithmetic, two at a time: the remainder of the
// first estimate is exact, and adding its share leaves an error far below what lies between a quotient that is no tie and the tie next to it
// (x and a have eight bits each: 1 / 510 of the unit of x's last place against 2^-22 of the quotient), while a tie comes out as one. 4096 rows of
// 4096 take 11.5 us; with one value an instruction and ties told by their remainders 18.1.
struct Quant8 {
  seqk::f2 inv, minus;                                   // 128 / a and -a / 128
  uint32_t keep;                                         // no bits of rows that are not finite: codes of 0, the scale says the rest
  __device__ __forceinline__ explicit Quant8(float a) {
    const float i = __fdiv_rn(128.f, a);
    inv = seqk::pk(i, i);
    minus = seqk::pk(a * -0.0078125f, a * -0.0078125f);
    keep = a <= 3.3895e38f ? 0xffffffffu : 0u;
  }
  __device__ __forceinline__ uint2 operator()(const uint4& raw) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const seqk::f2 t = seqk::mul2(seqk::pk(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u)),
                                    seqk::pk(0.9921875f, 0.9921875f));          // 127 / 128: exact
      const seqk::f2 q = seqk::mul2(t, inv);
      float lo, hi;
      seqk::un(seqk::add2(seqk::fma2(seqk::fma2(q, minus, t), inv, q), seqk::pk(12582912.f, 12582912.f)), lo, hi);
      b[2 * e] = __float_as_uint(lo);                    // 1.5 x 2^23: an integer added to it stands in the low bits
      b[2 * e + 1] = __float_as_uint(hi);
    }
    return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410) & keep,
                      __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410) & keep);
  }
};

}  // namespace b200
