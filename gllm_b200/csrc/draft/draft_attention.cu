// Attention of drafted nodes over a paged bf16 cache. Definition: ops/draft.py.
#include "../common/host_utils.h"
#include "../common/ptx.cuh"

namespace b200 {

static constexpr int kNodes = 64;
static constexpr int kWarps = 4;

struct DraftAttnParams {
  const __nv_bfloat16* q;
  int64_t q_ts;
  __nv_bfloat16* out;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t pages;
  const int32_t* table;
  int64_t table_ld;
  const int32_t* seq_lens;
  const int32_t* q_start;
  const int64_t* seen;
  int table_width, num_seqs, rows, Hq, Hkv, page_size;
  float scale_log2;
};

// One CTA per (node, query head), its warps take every fourth key; a lane has D / 32 neighbouring dims. Grid: (heads, 64 nodes, sequences).
template <int D>
__global__ void __launch_bounds__(kWarps * 32) draft_attention_plain_kernel(const DraftAttnParams p) {
  constexpr int E = D / 32;
  griddep_wait();
  const int seq = blockIdx.z, node = blockIdx.y, head = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = p.q_start[seq], n = min(p.q_start[seq + 1], p.rows) - first;
  if (first < 0 || node >= n) return;
  const int ctx = max(p.seq_lens[seq] - n, 0), len = ctx + min(n, kNodes), kvh = head / (p.Hq / p.Hkv);
  const unsigned long long seen = static_cast<unsigned long long>(p.seen[first + node]);
  const int64_t row = first + node;
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(p.q[row * p.q_ts + static_cast<int64_t>(head) * D + lane * E + e]) * p.scale_log2;
    o[e] = 0.f;
  }
  for (int key = warp; key < len; key += kWarps) {
    if (key >= ctx && !((seen >> (key - ctx)) & 1)) continue;
    const int block = key / p.page_size;
    const int64_t page = block < p.table_width ? p.table[seq * p.table_ld + block] : -1;
    if (page < 0 || page >= p.pages) continue;
    const int64_t at = (((page * p.Hkv + kvh) * (D / 64) + lane * E / 64) * p.page_size + key % p.page_size) * 64 + lane * E % 64;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += q[e] * __bfloat162float(p.k[at + e]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float top = s > m ? s : m, alpha = m == -INFINITY ? 0.f : exp2f(m - top), w = exp2f(s - top);
    m = top;
    l = l * alpha + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * alpha + w * __bfloat162float(p.v[at + e]);
  }
  __shared__ float so[kWarps][D], sm[kWarps], sl[kWarps];
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w]);
  for (int w = 0; w < kWarps; ++w) sum += sm[w] == -INFINITY ? 0.f : sl[w] * exp2f(sm[w] - top);
  for (int d = threadIdx.x; d < D; d += kWarps * 32) {
    float x = 0.f;
    for (int w = 0; w < kWarps; ++w) x += sm[w] == -INFINITY ? 0.f : so[w][d] * exp2f(sm[w] - top);
    p.out[(row * p.Hq + head) * D + d] = __float2bfloat16(sum == 0.f ? 0.f : x / sum);
  }
}

}  // namespace b200

using namespace b200;

GLLM_EXPORT int gllm_draft_attention(const void* q, int64_t q_ts, void* out, const void* k_cache, const void* v_cache, int64_t pages,
                                     const void* table, int64_t table_ld, int table_width, const void* seq_lens, const void* q_start,
                                     const void* seen, int num_seqs, int rows, int max_nodes, int Hq, int Hkv, int D, int page_size,
                                     float scale, void* stream) {
  if (num_seqs <= 0 || rows <= 0 || max_nodes <= 0) return 0;
  if ((D != 64 && D != 128) || Hkv <= 0 || Hq % Hkv || num_seqs > 65535) return 1;
  DraftAttnParams p;
  p.q = reinterpret_cast<const __nv_bfloat16*>(q); p.q_ts = q_ts;
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  p.k = reinterpret_cast<const __nv_bfloat16*>(k_cache);
  p.v = reinterpret_cast<const __nv_bfloat16*>(v_cache);
  p.pages = pages;
  p.table = reinterpret_cast<const int32_t*>(table); p.table_ld = table_ld; p.table_width = table_width;
  p.seq_lens = reinterpret_cast<const int32_t*>(seq_lens);
  p.q_start = reinterpret_cast<const int32_t*>(q_start);
  p.seen = reinterpret_cast<const int64_t*>(seen);
  p.num_seqs = num_seqs; p.rows = rows; p.Hq = Hq; p.Hkv = Hkv; p.page_size = page_size;
  p.scale_log2 = scale * 1.4426950408889634f;
  const dim3 grid(Hq, max_nodes < kNodes ? max_nodes : kNodes, num_seqs);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (D == 128) CUDA_CHECK_RET(launch_pdl(draft_attention_plain_kernel<128>, grid, dim3(kWarps * 32), 0, st, p));
  else CUDA_CHECK_RET(launch_pdl(draft_attention_plain_kernel<64>, grid, dim3(kWarps * 32), 0, st, p));
  return 0;
}
