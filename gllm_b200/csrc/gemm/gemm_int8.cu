// Products in 8-bit integers with a scale per token and per output channel:
//
//   a_t = max(max_k |x_tk|, 2^-100),  X_tk = rne(127 x_tk / a_t),  y_tn = (a_t / 127) s_n sum_k X_tk W_nk (+ b_n)  -> bf16
//
// x bf16, W int8 with fp32 scales s; gated: W = [gate rows ; up rows] and y = silu(gate) * up. The sums are int32, exact for K up to
// 131,072 (127 x 128 x K < 2^31); scales, bias and gate are fp32, and y is rounded once.
//
// A row or two (up to four where K is short) are multiplied while they are read (gemv_int8.cu). Otherwise two launches: the rows are
// quantised (here), then multiplied on the tensor cores (tcgen05.mma kind::i8) by one of two kernels:
// prompts on pairs of SMs (gemm_bf16_pair.cu), decode batches with K cut over a cluster (gemm_bf16_cluster.cu), which copies its first
// weights while the rows are quantised. `gllm_linear_int8` chooses by what their time is made of. (Rows quantised in every CTA of the
// cluster kernel, to save the launch: 10.0 us for one row of 6144 x 4096 instead of 9.1, 12.8 for four, 16 for eight.)
#include "../common/host_utils.h"
#include "../common/ptx.cuh"
#include "gemm_cluster.h"
#include "gemm_pair.h"
#include "gemv_int8.h"
#include "int8_rows.cuh"

namespace b200 {

namespace {

// A row is T threads' (a warp's or a block's), eight values a piece, NV pieces a thread kept in registers; NV = 0: any length, read
// twice.
template <int T, int NV>
__global__ void __launch_bounds__(256)
int8_quant_rows_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, float* __restrict__ scales, int M, int K) {
  griddep_launch();
  griddep_wait();
  constexpr int kRows = 256 / T;
  const int row = blockIdx.x * kRows + threadIdx.x / T, at = threadIdx.x % T, pieces = K / 8;
  const bool in = row < M;
  const __nv_bfloat16* src = x + static_cast<int64_t>(in ? row : 0) * ldx;
  uint4 raw[NV > 0 ? NV : 1];
  uint32_t most = 0;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (in && at + i * T < pieces) raw[i] = *reinterpret_cast<const uint4*>(src + (at + i * T) * 8);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) most = max_abs2(most, raw[i]);
  } else {
    for (int i = at; i < pieces; i += T) most = max_abs2(most, *reinterpret_cast<const uint4*>(src + i * 8));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, o));
  if constexpr (T > 32) {
    __shared__ uint32_t part[T / 32];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 32; ++i) most = __vmaxu2(most, part[i]);
  }
  if (!in) return;
  const float a = largest(most);
  const Quant8 quant(a);
  if (at == 0) scales[row] = __fdiv_rn(a, 127.f);
  uint8_t* dst = q + static_cast<int64_t>(row) * K;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (at + i * T < pieces) *reinterpret_cast<uint2*>(dst + (at + i * T) * 8) = quant(raw[i]);
  } else {
    for (int i = at; i < pieces; i += T) *reinterpret_cast<uint2*>(dst + i * 8) = quant(*reinterpret_cast<const uint4*>(src + i * 8));
  }
}

// Does nothing, launched in stream order: what comes before it is complete when it starts, whenever that let its dependents go ahead.
__global__ void int8_rows_complete_kernel() {}

int quant_rows(const __nv_bfloat16* x, int64_t ldx, uint8_t* q, float* scales, int M, int K, cudaStream_t st) {
  auto go = [&](auto kern, int rows) {
    return launch_pdl(kern, dim3((M + rows - 1) / rows), dim3(256), 0, st, x, ldx, q, scales, M, K);
  };
  if (K <= 512) CUDA_CHECK_RET(go(int8_quant_rows_kernel<32, 2>, 8));
  else if (K <= 1024) CUDA_CHECK_RET(go(int8_quant_rows_kernel<32, 4>, 8));
  else if (K <= 4096) CUDA_CHECK_RET(go(int8_quant_rows_kernel<256, 2>, 1));
  else if (K <= 8192) CUDA_CHECK_RET(go(int8_quant_rows_kernel<256, 4>, 1));
  else if (K <= 16384) CUDA_CHECK_RET(go(int8_quant_rows_kernel<256, 8>, 1));
  else CUDA_CHECK_RET(go(int8_quant_rows_kernel<256, 0>, 1));
  return 0;
}

// The faster form of a product of this size: true with a plan for the cluster kernel, false for the pairs. Fitted to 933 products (1 to 700
// rows, weights of 512 to 57,344 rows and 640 to 28,672 columns, a third gated; every plan timed with cold weights, the rows'
// quantiser included). A plan costs what is more of its copies (an SM takes 100 KB per us) and its weights (6.36 TB/s, less where few
// SMs draw), and a fixed sum a round, which counts as 14 us here, more than the 0.8 us that it takes: a second round is rarely worth it.
// The choice takes 1.5 % longer than the best plan on average (27 of 933 over 10 %, 1.42 at worst). Against the pairs both are estimated in
// us; the choice between them loses 0.4 % (19 over 10 %, 1.28 at worst); the pairs win 91 of the 933, all but a few over 256 rows. Some, pairs and
// chosen, us: 64 rows 24,576 x 4096 gated 33.9 and 24.8, 64 of 4096 x 12,288 37.5 and 18.4, 256 of 6144 x
// 4096 19.7 and 19.1, 777 of 10,240 x 8192 71.7 and 80.1.
bool plan_int8(int M, int N, int K, bool gated, ClusterPlan* plan) {
  if (M > 1024) return false;
  const int sms = num_sms(), num_kb = (K + 127) / 128, tiles_n = (N + 127) / 128;
  const double bytes = static_cast<double>(N) * K / 6.36e6;
  double best = 1e30, takes = 1e30;
  for (int tm = 1; tm <= 8; ++tm) {
    const int bt = ((M + tm - 1) / tm + 15) / 16 * 16;
    if (bt > 256) continue;
    if (tm > 1 && bt < 32) break;
    for (const int parts : {1, 2, 3, 4, 6, 8}) {
      if (parts > 1 && parts * 2 > num_kb) break;
      const int side = cluster_slots(1, parts) - (parts == 3 ? 2 : 0);      // of three, fewer run at once than the query says
      if (side <= 0) continue;
      for (int per_sm = 1; per_sm <= 2; ++per_sm) {
        const ClusterPlan one{bt, parts, per_sm == 1 ? 220 * 1024 : 108 * 1024};
        const int stages = (one.smem - 2048) / ((128 + bt) * 128);
        if (stages < per_sm + 1 || cluster_smem(one, gated) == 0) continue;
        const int tiles = tiles_n * ((M + bt - 1) / bt), rounds = (tiles + side * per_sm - 1) / (side * per_sm);
        const double ctas = static_cast<double>(tiles < side * per_sm ? tiles : side * per_sm) * parts;
        const double copies = static_cast<double>(rounds) * per_sm * ((num_kb + parts - 1) / parts) * ((128 + bt) * 128) * 1e-5;
        auto drawn = [&](double share, double less) {                       // ... by so many SMs
          const double n = per_sm == 1 ? ctas : share * ctas;
          return bytes * (1.0 + less * (sms / (n < sms ? n : sms) - 1.0));
        };
        auto most = [](double a, double b) { return a > b ? a : b; };
        const double memory = drawn(0.92, 0.3);
        const double t = most(copies, memory) + 0.018 * (copies < memory ? copies : memory) + rounds * (14.3 + 0.0054 * bt) +
                         (per_sm == 2 ? 0.0014 * bt : 0.0);
        if (t < best) {
          best = t;
          takes = most(0.924 * copies, drawn(0.38, 0.1)) + rounds * (0.76 + 0.0434 * bt) + 4.1;
          *plan = one;
        }
      }
    }
  }
  if (best == 1e30) return false;
  const int tiles = ((M + 255) / 256) * ((N + 255) / 256), rounds = (tiles + sms / 2 - 1) / (sms / 2);
  const double products = rounds * (0.297 * num_kb + 0.08), memory = 1.95 * bytes;
  return takes < 1.1 * ((products > memory ? products : memory) + 8.5);
}

}  // namespace

}  // namespace b200

using namespace b200;

// x [M, K] bf16 (rows ldx apart) -> q [M, K] int8, scales [M] (largest magnitude, 2^-100 at least, / 127). These may be the weights of a
// product that is launched next. Products fetch their first weights before they wait for the kernels ahead of them, and the quantiser lets its
// dependents start at once, so an empty kernel without an early start stands between the two (1 us: 6144 x 4096 14.9 us for 13.7; the product's
// own rows go without).
GLLM_EXPORT int gllm_int8_quant_rows(const void* x, int64_t ldx, void* q, void* scales, int M, int K, void* stream) {
  if (M <= 0 || K <= 0) return 0;
  if (K % 16 != 0 || ldx % 8 != 0 || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(q)) & 15) != 0) {
    fprintf(stderr, "[gllm_b200] int8_quant_rows: K %% 16 and rows on 16-byte boundaries required\n");
    return 1;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (const int rc = quant_rows(reinterpret_cast<const __nv_bfloat16*>(x), ldx, reinterpret_cast<uint8_t*>(q), reinterpret_cast<float*>(scales),
                                M, K, st))
    return rc;
  int8_rows_complete_kernel<<<1, 1, 0, st>>>();
  CUDA_CHECK_RET(cudaGetLastError());
  return 0;
}

// Whether the form that is taken for M rows needs no scratch.
GLLM_EXPORT int gllm_int8_rows_inside(int M, int K) { return gemv_int8_takes(M, K) ? 1 : 0; }

// y [M, N] (gated: [M, N / 2]) of x [M, K] and W8 [N, K] int8 (contiguous) with w_scale [N]; xq [M, K] and x_scale [M] are scratch (null
// where gllm_int8_rows_inside says so).
// form: 0 = by size, 1 = pairs of SMs, 2 = clusters with bt rows of x a tile and K in `parts`, 3 = a few rows (tests, tuning).
GLLM_EXPORT int gllm_linear_int8(const void* x, int64_t ldx, void* xq, void* x_scale, const void* W8, const void* w_scale, void* C,
                                 int64_t ldc, int M, int N, int K, const void* bias, int gated, int form, int bt, int parts, int smem,
                                 void* stream) {
  if (M <= 0 || N <= 0) return 0;
  const int out_N = gated ? N / 2 : N;
  if (K <= 0 || K % 16 != 0 || K > 131072 || N % 8 != 0 || out_N % 8 != 0 || (gated && (N % 2 != 0 || bias != nullptr)) || ldx % 8 != 0 ||
      ldc % 8 != 0 || form < 0 || form > 3 || (form == 3 && !gemv_int8_fits(M, K)) ||
      ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(xq) | reinterpret_cast<uintptr_t>(W8) | reinterpret_cast<uintptr_t>(w_scale) |
        reinterpret_cast<uintptr_t>(C) | reinterpret_cast<uintptr_t>(bias)) & 15) != 0 ||
      (form == 2 && (bt % 16 != 0 || bt < 16 || bt > 256 || parts < 1 || parts > 8 || parts > (K + 127) / 128))) {
    fprintf(stderr, "[gllm_b200] linear_int8: M=%d N=%d K=%d (K %% 16, K <= 131072, N %% 8, gated N %% 16; 16-byte boundaries)\n", M, N, K);
    return 1;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (form == 0 && gemv_int8_takes(M, K)) form = 3;
  if (form == 3)
    return gemv_int8(GemvInt8{reinterpret_cast<const __nv_bfloat16*>(x), ldx, reinterpret_cast<const uint8_t*>(W8),
                              reinterpret_cast<const float*>(w_scale), reinterpret_cast<__nv_bfloat16*>(C), ldc,
                              reinterpret_cast<const __nv_bfloat16*>(bias), N, K}, M, gated != 0, st);
  if (xq == nullptr || x_scale == nullptr) {
    fprintf(stderr, "[gllm_b200] linear_int8: no room for the quantised rows\n");
    return 1;
  }
  if (const int rc = quant_rows(reinterpret_cast<const __nv_bfloat16*>(x), ldx, reinterpret_cast<uint8_t*>(xq),
                                reinterpret_cast<float*>(x_scale), M, K, st))
    return rc;
  const float *as = reinterpret_cast<const float*>(x_scale), *ws = reinterpret_cast<const float*>(w_scale);
  __nv_bfloat16* c = reinterpret_cast<__nv_bfloat16*>(C);
  const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(bias);
  ClusterPlan plan{bt, parts, smem};
  if (form == 0) form = plan_int8(M, N, K, gated != 0, &plan) ? 2 : 1;
  if (form == 2)
    return gemm_int8_cluster(ClusterGemmInt8{ClusterGemm{xq, W8, K, K, c, ldc, M, N, K, b, gated != 0, 0}, as, ws}, plan, st);
  return gemm_int8_pair(PairGemmInt8{PairGemm{xq, W8, K, K, c, ldc, M, N, K, b, gated, 0.f, 0.f, 0}, as, ws}, st);
}
