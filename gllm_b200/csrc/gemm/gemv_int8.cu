// 8-bit products of a few rows (the decode step of a sequence or two), the rows quantised on the way:
//
//   a_m = max(max_k |x_mk|, 2^-100),  X_mk = rne(127 x_mk / a_m),  y_mn = (a_m / 127) s_n sum_k X_mk W_nk (+ b_n);  gated: W = [gate rows ; up rows]
//
// Bound by the weight bytes and, for the matrices of a layer, by latency: launch, one trip to HBM, the sum. As in gemv_bf16.cu a warp owns
// one or two weight rows with the whole of K and has its first 4 KB of weights in flight before the previous kernel ends. Meanwhile
// every block, one an SM, quantises the rows for itself (8 KB of reads at K = 4096; four blocks an SM: 0.8 us more), so that there is one
// launch and no scratch. Four products to an instruction; sums are int32 and exact, so the results are the bits of the other forms.
// One row, here and in the other forms with their quantiser, us, cold: 6144 x 4096 6.1 / 8.9 (4.1 TB/s; its bytes alone take 3.8), 4096 x 12,288 10.8 / 13.6,
// 10,240 x 8192 15.9 / 18.3, 57,344 x 8192 gated 69.6 / 80.7, 8192 x 28,672 40.3 / 43.2, 2048 x 2048 2.6 / 5.7. Two: 6.9 / 9.0, 12.0 / 13.8,
// 16.9 / 18.3, 70.5 / 80.0, 42.4 / 43.1, 3.1 / 5.7. Three and four read the rows from shared memory too often where K is long (four of 10,240 x 8192: 21.3 / 18.3),
// but not up to 4096 (6144 x 4096 7.9 and 9.0 / 9.0, 24,576 x 4096 gated 19.4 and 20.4 / 21.5, 2048 x 2048 3.7 and 4.4 / 5.8).
#include "../common/host_utils.h"
#include "../common/ptx.cuh"
#include "gemv_int8.h"
#include "int8_rows.cuh"

namespace b200 {

namespace {

constexpr int kV8Warps = 16, kV8Threads = kV8Warps * 32;               // one block an SM: it quantises the rows once
constexpr int kV8Rows = 4, kV8Smem = 160 * 1024;                        // rows of x and their bytes, at most

__device__ __forceinline__ uint4 ldg_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// MT: rows of x; R weight rows per warp, U 16-byte loads per lane and row at a time. Gated: R = 2, a gate and its up.
template <int MT, int R, int U, bool GATED>
__global__ void __launch_bounds__(kV8Threads, 1) gemv_int8_kernel(const GemvInt8 p, const int units) {
  extern __shared__ __align__(16) uint8_t gemv8_smem[];                 // [MT][K]
  __shared__ uint32_t part[MT][kV8Warps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wid = warp * gridDim.x + blockIdx.x, nw = gridDim.x * kV8Warps;      // a last round spreads over the SMs
  const int chunks = (p.K + 512 * U - 1) / (512 * U);
  griddep_launch();
  auto row_of = [&](int u, int r) { return GATED ? u + r * (p.N / 2) : u * R + r; };
  auto load = [&](int u, int c, uint4 (&v)[R][U]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int n = row_of(u, r);
      const uint8_t* src = p.w + static_cast<size_t>(n) * p.K;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int k = (c * U + i) * 512 + lane * 16;
        v[r][i] = n < p.N && k < p.K ? ldg_stream(src + k) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  uint4 cur[R][U], nxt[R][U];
  int u = wid, c = 0;
  if (u < units) load(u, 0, cur);
  griddep_wait();
  // the rows: this thread's pieces, the first two of a row kept
  constexpr int kKept = 2;
  uint4 raw[MT][kKept];
  uint32_t most[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      const int k = (threadIdx.x + i * kV8Threads) * 8;
      raw[m][i] = k < p.K ? __ldcg(reinterpret_cast<const uint4*>(p.x + m * p.ldx + k)) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    most[m] = 0;
#pragma unroll
    for (int i = 0; i < kKept; ++i) most[m] = max_abs2(most[m], raw[m][i]);
    for (int k = (threadIdx.x + kKept * kV8Threads) * 8; k < p.K; k += kV8Threads * 8)
      most[m] = max_abs2(most[m], __ldcg(reinterpret_cast<const uint4*>(p.x + m * p.ldx + k)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most[m] = __vmaxu2(most[m], __shfl_xor_sync(0xffffffffu, most[m], o));
    if (lane == 0) part[m][warp] = most[m];
  }
  __syncthreads();
  float scale = 0.f;                                     // of row `lane`
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    uint32_t all = part[m][lane % kV8Warps];
#pragma unroll
    for (int o = kV8Warps / 2; o > 0; o >>= 1) all = __vmaxu2(all, __shfl_xor_sync(0xffffffffu, all, o));
    const float a = largest(all);
    const Quant8 quant(a);
    if (lane == m) scale = __fdiv_rn(a, 127.f);
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      const int k = (threadIdx.x + i * kV8Threads) * 8;
      if (k < p.K) *reinterpret_cast<uint2*>(gemv8_smem + m * p.K + k) = quant(raw[m][i]);
    }
    for (int k = (threadIdx.x + kKept * kV8Threads) * 8; k < p.K; k += kV8Threads * 8)
      *reinterpret_cast<uint2*>(gemv8_smem + m * p.K + k) = quant(__ldcg(reinterpret_cast<const uint4*>(p.x + m * p.ldx + k)));
  }
  __syncthreads();
  int acc[R][MT];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[r][m] = 0;
  while (u < units) {
    int nu = u, nc = c + 1;
    if (nc == chunks) { nc = 0; nu += nw; }
    if (nu < units) load(nu, nc, nxt);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = (c * U + i) * 512 + lane * 16;
      if (k < p.K) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 x = *reinterpret_cast<const uint4*>(gemv8_smem + m * p.K + k);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            acc[r][m] = __dp4a(static_cast<int>(cur[r][i].x), static_cast<int>(x.x), acc[r][m]);
            acc[r][m] = __dp4a(static_cast<int>(cur[r][i].y), static_cast<int>(x.y), acc[r][m]);
            acc[r][m] = __dp4a(static_cast<int>(cur[r][i].z), static_cast<int>(x.z), acc[r][m]);
            acc[r][m] = __dp4a(static_cast<int>(cur[r][i].w), static_cast<int>(x.w), acc[r][m]);
          }
        }
      }
    }
    if (nc == 0) {                                       // the rows are done: lane m has those of row m
      float sum[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        sum[r] = 0.f;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int s = __reduce_add_sync(0xffffffffu, acc[r][m]);
          if (lane == m) sum[r] = static_cast<float>(s);
          acc[r][m] = 0;
        }
      }
      if (lane < MT) {
        if constexpr (GATED) {
          const float g = sum[0] * (scale * p.w_scale[u]), up = sum[R - 1] * (scale * p.w_scale[u + p.N / 2]);
          p.c[lane * p.ldc + u] = __float2bfloat16(g / (1.0f + __expf(-g)) * up);
        } else {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const int n = row_of(u, r);
            if (n < p.N) {
              const float y = sum[r] * (scale * p.w_scale[n]);
              p.c[lane * p.ldc + n] = __float2bfloat16(p.bias != nullptr ? y + __bfloat162float(p.bias[n]) : y);
            }
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < U; ++i) cur[r][i] = nxt[r][i];
    u = nu;
    c = nc;
  }
}

template <int MT, int R, int U, bool GATED>
int launch(const GemvInt8& p, cudaStream_t st) {
  static PerDeviceOnce configured;
  if (configured.need()) {
    CUDA_CHECK_RET(cudaFuncSetAttribute(gemv_int8_kernel<MT, R, U, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kV8Smem));
    configured.done();
  }
  const int units = GATED ? p.N / 2 : (p.N + R - 1) / R, sms = num_sms();
  CUDA_CHECK_RET(launch_pdl(gemv_int8_kernel<MT, R, U, GATED>, dim3(units < sms ? units : sms), dim3(kV8Threads), MT * p.K, st, p, units));
  return 0;
}

template <int MT>
int launch_rows(const GemvInt8& p, bool gated, cudaStream_t st) {
  if (gated) return launch<MT, 2, 4, true>(p, st);
  if (p.K <= 2048) return launch<MT, 2, 4, false>(p, st);       // two short rows at a time share the reads of x; longer ones leave a worse last round
  return launch<MT, 1, 8, false>(p, st);
}

}  // namespace

bool gemv_int8_fits(int M, int K) { return M >= 1 && M <= kV8Rows && K <= 131072 && M * K <= kV8Smem; }
bool gemv_int8_takes(int M, int K) { return gemv_int8_fits(M, K) && (M <= 2 || K <= 4096); }

int gemv_int8(const GemvInt8& p, int M, bool gated, cudaStream_t st) {
  switch (M) {
    case 1: return launch_rows<1>(p, gated, st);
    case 2: return launch_rows<2>(p, gated, st);
    case 3: return launch_rows<3>(p, gated, st);
    default: return launch_rows<4>(p, gated, st);
  }
}

}  // namespace b200
