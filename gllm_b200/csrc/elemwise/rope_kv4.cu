// [per-head q / k RMSNorm] -> RoPE -> keys and values coded in 4 bits into their pages, in one pass over the projection's rows;
// and the rows of such a cache read back.
//
// The cache (layout and rounding: ops/kv4.py): uint8 [pages, Hkv, page_size / 16, 9 D], blocks of 16 tokens: 16 rows of D / 2 bytes,
// then 16 x D / 64 pairs (scale, low) of bf16. Each 64 dims y of a token's head:
//   low = min y,  scale = bf16((max y - low) / 15),  code = min(15, rne((y - low) / scale)),  value = code * scale + low.
// y is rounded to bf16 before it is coded (what a bf16 cache would hold), so low needs no rounding of its own. Many quotients
// are ties (both sides are multiples of the same power of two), which a product with the reciprocal alone would send either way. A scale below
// 2^-126 counts as 0 (its reciprocal may be beyond fp32); the steps up to there keep subnormal numbers.
//
// What bounds it: issue slots and the latency of short blocks. 4096 tokens x (32 + 8 + 8) heads of 128 with norms take 22.6 us, 3.9 TB/s of
// what is read and written (floor 13.5 us; 19.3 without norms); with IEEE divisions in every lane it took 80, with one fp32 operation an
// instruction 25.9. So the arithmetic is on pairs of fp32.
//
// Queries are rotated in place; the rotated keys go to the cache only.
#include "../common/host_utils.h"
#include "../common/ptx.cuh"
#include "../seq/seq_common.cuh"
#include "rope_common.cuh"

namespace b200 {

namespace {

using seqk::add2;
using seqk::f2;
using seqk::fma2;
using seqk::mul2;
using seqk::pk;

__device__ __forceinline__ f2 both(float a) { return pk(a, a); }
// a + b of products that are rounded by themselves. The compiler makes one rounding of product and sum where it sees them, and of a factor
// that it knows to be one, so `one` comes with the launch (-one: a - b).
__device__ __forceinline__ f2 plus2(f2 a, f2 b, f2 one) { return fma2(b, one, a); }
__device__ __forceinline__ f2 unpack2(uint32_t w) { return pk(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pack2(f2 v) {
  float a, b;
  seqk::un(v, a, b);
  return pack_bf16(a, b);
}

// where the block of `slot` starts in head 0 of its page, and the row in it; ok: the slot is one of the cache
struct Kv4Place {
  size_t block;
  int row;
  bool ok;
};
__device__ __forceinline__ Kv4Place kv4_place(int slot, int page_size, int64_t pages, int Hkv, int D) {
  const int page = slot / page_size, off = slot - page * page_size;
  return Kv4Place{(static_cast<size_t>(page) * Hkv * (page_size / 16) + off / 16) * (9 * D), off % 16, slot >= 0 && page < pages};
}

__device__ __forceinline__ uint32_t min_nan2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max_nan2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// The ends of a group from those of a lane's values (bf16 pairs): O neighbouring lanes hold the group, all of the warp take part.
template <int O>
__device__ __forceinline__ void kv4_ends(uint32_t& lo, uint32_t& hi) {
  lo = min_nan2(lo, __byte_perm(lo, lo, 0x1032));
  hi = max_nan2(hi, __byte_perm(hi, hi, 0x1032));
#pragma unroll
  for (int o = O / 2; o > 0; o >>= 1) {
    lo = min_nan2(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan2(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
}
__device__ __forceinline__ uint32_t min4(const uint32_t (&w)[4]) { return min_nan2(min_nan2(w[0], w[1]), min_nan2(w[2], w[3])); }
__device__ __forceinline__ uint32_t max4(const uint32_t (&w)[4]) { return max_nan2(max_nan2(w[0], w[1]), max_nan2(w[2], w[3])); }

__device__ __forceinline__ float fma_full(float a, float b, float c) {                // the build flushes subnormal numbers elsewhere
  float d;
  asm("fma.rn.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// A quotient to the nearest from an estimate of the reciprocal: the remainder of the first estimate is exact, and adding its share leaves
// an error far below half a step (Markstein). So a quotient that is a tie between two codes comes out as one.
__device__ __forceinline__ float quotient(float d, float s, float inv) {
  const float q = fma_full(d, inv, 0.f);
  return fma_full(fma_full(q, -s, d), inv, q);          // (-q would be flushed)
}

// A group's pair from its ends, and what its codes are made with. A NaN or an infinity (or a span beyond fp32) makes the scale a
// NaN, and so every value that is read back.
struct Kv4Group {
  float low, scale, inv;
  uint32_t pair;
  __device__ __forceinline__ Kv4Group(uint32_t lo, uint32_t hi) {
    low = __uint_as_float(lo << 16);
    const float high = __uint_as_float(hi << 16);
    uint32_t bits = __bfloat16_as_ushort(__float2bfloat16_rn(quotient(fma_full(-1.f, low, high), 15.f, 1.f / 15.f)));
    bits = bits < 0x0080u ? 0u : bits < 0x7f80u ? bits : 0x7fffu;          // below 2^-126: 0; infinities and NaN
    scale = __uint_as_float(bits << 16);
    const bool fine = bits < 0x7f80u;
    pair = (lo & 0xffff0000u) | bits;
    inv = fine && scale > 0.f ? __fdividef(1.f, scale) : 0.f;       // no scale: codes of 0
  }
  // Eight codes. The scale is at least (1 - 2^-8) / 15 of the span, so none is over 15.
  __device__ __forceinline__ uint32_t codes(const uint32_t (&w)[4]) const {
    constexpr float kMagic = 12582912.f;                 // 1.5 x 2^23: an integer added to it stands in the low bits
    uint32_t v = 0;
#pragma unroll
    for (int e = 3; e >= 0; --e) {
      const f2 d = add2(unpack2(w[e]), both(-low)), q = mul2(d, both(inv));
      float a, b;
      seqk::un(add2(fma2(fma2(q, both(-scale), d), both(inv), q), both(kMagic)), a, b);           // `quotient`, two at a time
      v = (v * 16u + __float_as_uint(b)) * 16u + __float_as_uint(a);
    }
    // sum of 16^e (kMagic's bits) mod 2^32: 0x4b400000 (1 + 16 + 256), the rest is shifted out
    return inv > 0.f ? v - (0x4b400000u + 0xb4000000u + 0x40000000u) : 0u;
  }
};

__device__ __forceinline__ float squares(const f2 (&x)[4]) {
  f2 v = mul2(x[0], x[0]);
#pragma unroll
  for (int e = 1; e < 4; ++e) v = fma2(x[e], x[e], v);
  float a, b;
  seqk::un(v, a, b);
  return a + b;
}
// x inv w, rounded to bf16 as on a bf16 cache
__device__ __forceinline__ void normed(f2 (&x)[4], float inv, const __nv_bfloat16* w) {
  const uint4 v = *reinterpret_cast<const uint4*>(w);
  const uint32_t ww[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = unpack2(pack2(mul2(mul2(x[e], both(inv)), unpack2(ww[e]))));
}

__device__ __forceinline__ uint8_t* kc_of(const RopeParams& p) { return reinterpret_cast<uint8_t*>(p.k_cache); }
__device__ __forceinline__ uint8_t* vc_of(const RopeParams& p) { return reinterpret_cast<uint8_t*>(p.v_cache); }

// A lane holds eight dims of a head, L = D / 8 lanes a head, NB heads a lane group, all loaded before the first is worked on.
template <int L, int NB>
__global__ void __launch_bounds__(128) rope_kv4_kernel(const RopeParams p, const int64_t pages, const int wide, const float one) {
  griddep_launch();
  griddep_wait();
  constexpr int D = 8 * L, G = D / 64, kHeadsPerWarp = 32 / L, kStep = 4 * kHeadsPerWarp;
  const int t = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = lane % L, e0 = gl * 8;
  const int half = p.rot >> 1;
  const int n_qk = p.Hq + p.Hkv, n_heads = n_qk + p.Hkv;
  const int first = blockIdx.y * (kStep * NB) + warp * kHeadsPerWarp + lane / L;

  uint4 raw[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int hh = first + n * kStep;
    raw[n] = make_uint4(0u, 0u, 0u, 0u);
    if (hh < n_heads) {
      const __nv_bfloat16* src = hh < p.Hq ? p.q + t * p.q_ts + hh * p.q_hs
                                 : hh < n_qk ? p.k + t * p.k_ts + (hh - p.Hq) * p.k_hs
                                             : p.v + t * p.v_ts + (hh - n_qk) * p.v_hs;
      raw[n] = *reinterpret_cast<const uint4*>(src + e0);
    }
  }
  // this lane's rotation row: the pair of element e is (e0 + e) % half (NeoX) or (e0 + e) / 2 (neighbours)
  const f2 plus = both(one), minus = both(-one);
  f2 c[4], s[4];
  const bool in_rot = e0 < p.rot, lo = e0 < half;
  if (in_rot && p.sec0 == 0 && wide) {
    const float* row = p.cos_sin + static_cast<size_t>(p.positions[t]) * p.rot;
    if (p.neox) {
      const int i = e0 - (lo ? 0 : half);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float4 cv = *reinterpret_cast<const float4*>(row + i + 4 * g), sv = *reinterpret_cast<const float4*>(row + half + i + 4 * g);
        c[2 * g] = pk(cv.x, cv.y); c[2 * g + 1] = pk(cv.z, cv.w);
        s[2 * g] = pk(sv.x, sv.y); s[2 * g + 1] = pk(sv.z, sv.w);
      }
    } else {
      const float4 cv = *reinterpret_cast<const float4*>(row + e0 / 2), sv = *reinterpret_cast<const float4*>(row + half + e0 / 2);
      c[0] = both(cv.x); c[1] = both(cv.y); c[2] = both(cv.z); c[3] = both(cv.w);
      s[0] = both(sv.x); s[1] = both(sv.y); s[2] = both(sv.z); s[3] = both(sv.w);
    }
  } else if (in_rot) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float cs[2][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = p.neox ? e0 + 2 * e + j - (lo ? 0 : half) : (e0 + 2 * e) >> 1;
        const int pos = p.sec0 != 0 ? p.positions[mrope_axis(i, p.sec0, p.sec1) * p.pos_stride + t] : p.positions[t];
        const float* row = p.cos_sin + static_cast<size_t>(pos) * p.rot;
        cs[0][j] = row[i];
        cs[1][j] = row[half + i];
      }
      c[e] = pk(cs[0][0], cs[0][1]);
      s[e] = pk(cs[1][0], cs[1][1]);
    }
  }
  const int dl = half / 8;
  const int partner = (lane & ~(L - 1)) | ((lo ? gl + dl : gl - dl) & (L - 1));
  const Kv4Place at = kv4_place(p.slots[t], p.page_size, pages, p.Hkv, D);
  const size_t head_stride = static_cast<size_t>(p.page_size / 16) * (9 * D);
  const int group = e0 / 64, unit = (e0 % 64) / 8 * G + group;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int hh = first + n * kStep;
    if (hh - lane / L >= n_heads) break;                 // none for the whole warp
    const bool is_q = hh < p.Hq, is_qk = hh < n_qk;
    uint32_t w[4] = {raw[n].x, raw[n].y, raw[n].z, raw[n].w};
    f2 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = unpack2(w[e]);
    const __nv_bfloat16* nw = is_q ? p.q_norm_w : p.k_norm_w;
    if (p.q_norm_w != nullptr || p.k_norm_w != nullptr) {
      float ss = squares(x);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (is_qk && nw != nullptr) normed(x, rsqrtf(ss * (1.f / D) + p.eps), nw + e0);
    }
    if (p.rot > 0) {
      // products and sum rounded one by one: a contraction would turn the last bit of some keys, and with it their codes
      if (p.neox) {
        f2 y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = __shfl_sync(0xffffffffu, x[e], partner);
        if (in_rot && is_qk) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f2 a = mul2(x[e], c[e]), b = mul2(y[e], s[e]);
            x[e] = plus2(a, b, lo ? minus : plus);
          }
        }
      } else if (in_rot && is_qk) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {                    // (a c - b s, b c + a s): the halves of c and of s are equal
          float a, b, si, same;
          seqk::un(x[e], a, b);
          seqk::un(s[e], si, same);
          x[e] = plus2(mul2(x[e], c[e]), mul2(pk(b, a), pk(-si, si)), plus);
        }
      }
    }
    if (is_qk) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = pack2(x[e]);
    }
    if (is_q) *reinterpret_cast<uint4*>(p.q + t * p.q_ts + hh * p.q_hs + e0) = make_uint4(w[0], w[1], w[2], w[3]);
    if (__all_sync(0xffffffffu, is_q)) continue;
    uint32_t low = min4(w), high = max4(w);
    kv4_ends<8>(low, high);
    const Kv4Group made(low, high);
    if (!is_q && hh < n_heads && at.ok) {
      uint8_t* block = (is_qk ? kc_of(p) + (hh - p.Hq) * head_stride : vc_of(p) + (hh - n_qk) * head_stride) + at.block;
      *reinterpret_cast<uint32_t*>(block + at.row * (D / 2) + unit * 4) = made.codes(w);
      if (e0 % 64 == 0) *reinterpret_cast<uint32_t*>(block + 8 * D + (at.row * G + group) * 4) = made.pair;
    }
  }
}

// NeoX rotation of whole heads (rot = D), the common form: a lane holds eight dims of the lower half and their partners of the upper
// one, L = D / 16 lanes a head, so that nothing is exchanged for the rotation; heads of 128: its two words are neighbours in the cache.
template <int L, int NB>
__global__ void __launch_bounds__(128) rope_kv4_pair_kernel(const RopeParams p, const int64_t pages, const float one) {
  griddep_launch();
  griddep_wait();
  constexpr int D = 16 * L, H = D / 2, G = D / 64, kHeadsPerWarp = 32 / L, kStep = 4 * kHeadsPerWarp;
  const int t = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gl = lane % L, e0 = gl * 8;
  const int n_qk = p.Hq + p.Hkv, n_heads = n_qk + p.Hkv;
  const int first = blockIdx.y * (kStep * NB) + warp * kHeadsPerWarp + lane / L;

  uint4 raw[NB][2];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int hh = first + n * kStep;
    raw[n][0] = raw[n][1] = make_uint4(0u, 0u, 0u, 0u);
    if (hh < n_heads) {
      const __nv_bfloat16* src = hh < p.Hq ? p.q + t * p.q_ts + hh * p.q_hs
                                 : hh < n_qk ? p.k + t * p.k_ts + (hh - p.Hq) * p.k_hs
                                             : p.v + t * p.v_ts + (hh - n_qk) * p.v_hs;
      raw[n][0] = *reinterpret_cast<const uint4*>(src + e0);
      raw[n][1] = *reinterpret_cast<const uint4*>(src + H + e0);
    }
  }
  const f2 plus = both(one), minus = both(-one);
  f2 c[4], s[4];
  const float* row = p.cos_sin + static_cast<size_t>(p.positions[t]) * D + e0;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float4 cv = *reinterpret_cast<const float4*>(row + 4 * g), sv = *reinterpret_cast<const float4*>(row + H + 4 * g);
    c[2 * g] = pk(cv.x, cv.y); c[2 * g + 1] = pk(cv.z, cv.w);
    s[2 * g] = pk(sv.x, sv.y); s[2 * g + 1] = pk(sv.z, sv.w);
  }
  const Kv4Place at = kv4_place(p.slots[t], p.page_size, pages, p.Hkv, D);
  const size_t head_stride = static_cast<size_t>(p.page_size / 16) * (9 * D);
  const bool norm = p.q_norm_w != nullptr || p.k_norm_w != nullptr;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int hh = first + n * kStep;
    if (hh - lane / L >= n_heads) break;                 // none for the whole warp
    const bool is_q = hh < p.Hq, is_qk = hh < n_qk;
    uint32_t w[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i][0] = raw[n][i].x; w[i][1] = raw[n][i].y; w[i][2] = raw[n][i].z; w[i][3] = raw[n][i].w;
    }
    if (__any_sync(0xffffffffu, is_qk)) {
      f2 x[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = unpack2(w[i][e]);
      }
      if (norm) {
        float ss = squares(x[0]) + squares(x[1]);        // the order of the sums is the other kernel's, and so are the bits
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const __nv_bfloat16* nw = is_q ? p.q_norm_w : p.k_norm_w;
        if (is_qk && nw != nullptr) {
          const float inv = rsqrtf(ss * (1.f / D) + p.eps);
          normed(x[0], inv, nw + e0);
          normed(x[1], inv, nw + H + e0);
        }
      }
      if (is_qk) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {                    // rounded one by one, as above
          w[0][e] = pack2(plus2(mul2(x[0][e], c[e]), mul2(x[1][e], s[e]), minus));
          w[1][e] = pack2(plus2(mul2(x[1][e], c[e]), mul2(x[0][e], s[e]), plus));
        }
      }
    }
    if (is_q) {
      __nv_bfloat16* dst = p.q + t * p.q_ts + hh * p.q_hs + e0;
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
      *reinterpret_cast<uint4*>(dst + H) = make_uint4(w[1][0], w[1][1], w[1][2], w[1][3]);
    }
    if (__all_sync(0xffffffffu, is_q)) continue;
    const bool stored = !is_q && hh < n_heads && at.ok;
    uint8_t* block = is_q || !at.ok ? nullptr : (is_qk ? kc_of(p) + (hh - p.Hq) * head_stride : vc_of(p) + (hh - n_qk) * head_stride) + at.block;
    if constexpr (G == 2) {                              // the halves are the groups
      uint32_t lo[2] = {min4(w[0]), min4(w[1])}, hi[2] = {max4(w[0]), max4(w[1])};
      kv4_ends<L>(lo[0], hi[0]);
      kv4_ends<L>(lo[1], hi[1]);
      const Kv4Group a(lo[0], hi[0]), b(lo[1], hi[1]);
      if (stored) {
        *reinterpret_cast<uint2*>(block + at.row * (D / 2) + gl * 8) = make_uint2(a.codes(w[0]), b.codes(w[1]));
        if (gl == 0) *reinterpret_cast<uint2*>(block + 8 * D + at.row * 8) = make_uint2(a.pair, b.pair);
      }
    } else {
      uint32_t lo = min_nan2(min4(w[0]), min4(w[1])), hi = max_nan2(max4(w[0]), max4(w[1]));
      kv4_ends<L>(lo, hi);
      const Kv4Group a(lo, hi);
      if (stored) {
        *reinterpret_cast<uint32_t*>(block + at.row * (D / 2) + gl * 4) = a.codes(w[0]);
        *reinterpret_cast<uint32_t*>(block + at.row * (D / 2) + (gl + L) * 4) = a.codes(w[1]);
        if (gl == 0) *reinterpret_cast<uint32_t*>(block + 8 * D + at.row * 4) = a.pair;
      }
    }
  }
}

// Rows of a 4-bit cache as bf16 (code * scale + low, rounded once): a lane makes the eight dims of a unit of the keys and of the values, of two
// heads where there are as many, all loaded before the first is worked on. 4096 tokens of 8 heads of 128: 7.3 us under the profiler for 3.3 of
// bytes; issue slots and ALU at 60 % of a launch that short.
template <int L, int NB>
__global__ void __launch_bounds__(128)
kv4_rows_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const int32_t* __restrict__ slots,
                __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int T, int Hkv, int page_size, int64_t pages) {
  griddep_launch();
  griddep_wait();
  constexpr int D = 8 * L, G = D / 64;
  const int groups = (Hkv + NB - 1) / NB;                // of heads
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x, row = i / L;
  if (row >= static_cast<int64_t>(T) * groups) return;
  const int unit = static_cast<int>(i % L), group = unit % G, e0 = 64 * group + unit / G * 8;
  const int t = static_cast<int>(row / groups), h0 = static_cast<int>(row % groups) * NB;
  const Kv4Place at = kv4_place(slots[t], page_size, pages, Hkv, D);
  const size_t head_stride = static_cast<size_t>(page_size / 16) * (9 * D);
  uint32_t codes[NB][2], pair[NB][2];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      codes[n][kv] = pair[n][kv] = 0u;                   // stands for zeros
      if (at.ok && h0 + n < Hkv) {
        const uint8_t* block = (kv ? v_cache : k_cache) + at.block + (h0 + n) * head_stride;
        codes[n][kv] = *reinterpret_cast<const uint32_t*>(block + at.row * (D / 2) + unit * 4);
        pair[n][kv] = *reinterpret_cast<const uint32_t*>(block + 8 * D + (at.row * G + group) * 4);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    if (h0 + n >= Hkv) break;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const float2 p = unpack_bf16(pair[n][kv]);
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = fma_full(static_cast<float>((codes[n][kv] >> (4 * e)) & 15u), p.x, p.y);
      *reinterpret_cast<uint4*>((kv ? v_out : k_out) + (static_cast<int64_t>(t) * Hkv + h0 + n) * D + e0) =
          make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
    }
  }
}

template <int L>
cudaError_t launch_rope_kv4(const RopeParams& p, int64_t pages, cudaStream_t st) {
  constexpr int kStep = 4 * (32 / L);
  const int n_heads = p.Hq + 2 * p.Hkv;
  const int wide = (reinterpret_cast<uintptr_t>(p.cos_sin) & 15) == 0 && p.rot % 8 == 0;       // rotation rows in pieces of 16 bytes
  // many tokens: several heads a lane, fewer and longer blocks; a decode batch: one, so that it still fills the machine
  // (2000 tokens x 64 heads of 128, half of them rotated: 24.3 us with one, 21.6 with two, 19.3 with four, 20.5 with five)
  if (static_cast<int64_t>(p.T) * n_heads >= static_cast<int64_t>(num_sms()) * 16 * kStep * 2)
    return launch_pdl(rope_kv4_kernel<L, 4>, dim3(p.T, (n_heads + 4 * kStep - 1) / (4 * kStep)), dim3(128), 0, st, p, pages, wide, 1.f);
  return launch_pdl(rope_kv4_kernel<L, 1>, dim3(p.T, (n_heads + kStep - 1) / kStep), dim3(128), 0, st, p, pages, wide, 1.f);
}

template <int L>
cudaError_t launch_rope_kv4_pair(const RopeParams& p, int64_t pages, cudaStream_t st) {
  constexpr int kStep = 4 * (32 / L);
  const int n_heads = p.Hq + 2 * p.Hkv;
  // as above, with two: 4096 tokens x 80 heads 32.4 us with one, 30.2 with two, 30.9 with three, 31.8 with four
  if (static_cast<int64_t>(p.T) * n_heads >= static_cast<int64_t>(num_sms()) * 16 * kStep * 2)
    return launch_pdl(rope_kv4_pair_kernel<L, 2>, dim3(p.T, (n_heads + 2 * kStep - 1) / (2 * kStep)), dim3(128), 0, st, p, pages, 1.f);
  return launch_pdl(rope_kv4_pair_kernel<L, 1>, dim3(p.T, (n_heads + kStep - 1) / kStep), dim3(128), 0, st, p, pages, 1.f);
}

}  // namespace

}  // namespace b200

using namespace b200;

// As gllm_rope_kv_write, on 4-bit caches of `pages` pages; k is left as it is. Slots outside of the cache are left out. Rows, norm
// weights and caches on 16-byte boundaries, D 64 or 128, pages of a multiple of 16 tokens up to 512, rot a multiple of 16 (of 8 for
// neighbouring pairs).
GLLM_EXPORT int gllm_rope_kv4_write(void* q, int64_t q_ts, int64_t q_hs, int Hq, const void* k, int64_t k_ts, int64_t k_hs, int Hkv,
                                    const void* v, int64_t v_ts, int64_t v_hs, const void* q_norm_w, const void* k_norm_w,
                                    const void* cos_sin, int D, int rot, int neox, int T, const void* positions,
                                    const void* slots, float eps, void* k_cache, void* v_cache, int64_t pages, int sec0,
                                    int sec1, int page_size, int64_t pos_stride, void* stream) {
  if (T <= 0) return 0;
  auto al16 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  if ((D != 64 && D != 128) || page_size < 16 || page_size > 512 || page_size % 16 != 0 || rot < 0 || rot > D || rot % (neox ? 16 : 8) != 0 ||
      ((q_ts | q_hs | k_ts | k_hs | v_ts | v_hs) & 7) != 0 || !al16(q) || !al16(k) || !al16(v) || !al16(q_norm_w) ||
      !al16(k_norm_w) || !al16(k_cache) || !al16(v_cache)) {
    fprintf(stderr, "[gllm_b200] rope_kv4_write: unsupported D=%d rot=%d page_size=%d, or rows off 16-byte boundaries\n", D, rot,
            page_size);
    return 1;
  }
  RopeParams p;
  p.q = reinterpret_cast<__nv_bfloat16*>(q); p.q_ts = q_ts; p.q_hs = q_hs; p.Hq = Hq;
  p.k = const_cast<__nv_bfloat16*>(reinterpret_cast<const __nv_bfloat16*>(k)); p.k_ts = k_ts; p.k_hs = k_hs; p.Hkv = Hkv;
  p.v = reinterpret_cast<const __nv_bfloat16*>(v); p.v_ts = v_ts; p.v_hs = v_hs;
  p.q_norm_w = reinterpret_cast<const __nv_bfloat16*>(q_norm_w);
  p.k_norm_w = reinterpret_cast<const __nv_bfloat16*>(k_norm_w);
  p.cos_sin = reinterpret_cast<const float*>(cos_sin);
  p.D = D; p.rot = rot; p.neox = neox; p.T = T;
  p.positions = reinterpret_cast<const int32_t*>(positions);
  p.slots = reinterpret_cast<const int32_t*>(slots);
  p.eps = eps;
  p.k_cache = reinterpret_cast<__nv_bfloat16*>(k_cache);
  p.v_cache = reinterpret_cast<__nv_bfloat16*>(v_cache);
  p.sec0 = sec0; p.sec1 = sec1; p.page_size = page_size; p.pos_stride = pos_stride;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (neox && rot == D && sec0 == 0 && al16(cos_sin))
    CUDA_CHECK_RET(D == 64 ? launch_rope_kv4_pair<4>(p, pages, st) : launch_rope_kv4_pair<8>(p, pages, st));
  else
    CUDA_CHECK_RET(D == 64 ? launch_rope_kv4<8>(p, pages, st) : launch_rope_kv4<16>(p, pages, st));
  return 0;
}

// k_out, v_out [T, Hkv, D] bf16: what the caches hold at `slots`; zeros for slots outside of the cache
GLLM_EXPORT int gllm_kv4_rows(const void* k_cache, const void* v_cache, const void* slots, void* k_out, void* v_out, int T, int Hkv,
                              int D, int page_size, int64_t pages, void* stream) {
  if (T <= 0) return 0;
  if ((D != 64 && D != 128) || page_size < 16 || page_size > 512 || page_size % 16 != 0) {
    fprintf(stderr, "[gllm_b200] kv4_rows: unsupported D=%d page_size=%d\n", D, page_size);
    return 1;
  }
  const int nb = static_cast<int64_t>(T) * Hkv >= 4096 ? 2 : 1;             // one head a lane where that does not fill the machine
  const int64_t blocks = (static_cast<int64_t>(T) * ((Hkv + nb - 1) / nb) * (D / 8) + 127) / 128;
  if (blocks > 0x7fffffff) {
    fprintf(stderr, "[gllm_b200] kv4_rows: %lld blocks\n", static_cast<long long>(blocks));
    return 1;
  }
  auto kern = D == 64 ? (nb == 2 ? kv4_rows_kernel<8, 2> : kv4_rows_kernel<8, 1>) : (nb == 2 ? kv4_rows_kernel<16, 2> : kv4_rows_kernel<16, 1>);
  CUDA_CHECK_RET(launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(128), 0, reinterpret_cast<cudaStream_t>(stream),
                            reinterpret_cast<const uint8_t*>(k_cache), reinterpret_cast<const uint8_t*>(v_cache),
                            reinterpret_cast<const int32_t*>(slots), reinterpret_cast<__nv_bfloat16*>(k_out),
                            reinterpret_cast<__nv_bfloat16*>(v_out), T, Hkv, page_size, pages));
  return 0;
}
