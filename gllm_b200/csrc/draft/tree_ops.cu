// Drafted trees: their layout behind the paged cache (plan), and keys and values of the nodes that were taken moved up (keep).
// Definitions: ops/draft.py.
#include "../common/host_utils.h"
#include "../common/ptx.cuh"

namespace b200 {

static constexpr int kMostNodes = 64;

// ---------------------------------------------------------------------------------------------------------------------
// plan: a warp per sequence, two nodes a lane. With up_i the parent and seen_i = {i}, six rounds of
//   seen_i |= seen[up_i],  up_i = up[up_i]
// reach ancestors 64 levels above. Latency bounds it: lengths, parents, then the table's entries, one trip to memory each (1 sequence of
// 8 nodes 4.1 us, 256 of 5 and 256 of up to 64 4.2).
// ---------------------------------------------------------------------------------------------------------------------
static constexpr int kPlanWarps = 4;

__global__ void __launch_bounds__(kPlanWarps * 32)
draft_plan_kernel(const int32_t* __restrict__ parents, const int32_t* __restrict__ q_start, const int32_t* __restrict__ seq_lens,
                  const int32_t* __restrict__ table, int64_t table_ld, int table_width, int num_seqs, int rows, int page_size,
                  int64_t* __restrict__ seen, int32_t* __restrict__ positions, int32_t* __restrict__ slots) {
  griddep_wait();
  const int lane = threadIdx.x & 31, seq = blockIdx.x * kPlanWarps + (threadIdx.x >> 5);
  if (seq > num_seqs) return;
  if (seq == num_seqs) {                       // rows behind the last sequence
    for (int i = max(q_start[num_seqs], 0) + lane; i < rows; i += 32) {
      seen[i] = 0;
      positions[i] = 0;
      slots[i] = -1;
    }
    return;
  }
  const int first = q_start[seq], n_all = min(q_start[seq + 1], rows) - first;
  if (first < 0 || n_all <= 0) return;
  const int n = min(n_all, kMostNodes), ctx = max(seq_lens[seq] - n_all, 0);
  int up[2];
  unsigned long long mask[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = lane + 32 * h, p = i < n ? parents[first + i] : -1;
    up[h] = p >= 0 && p < i ? p : -1;
    mask[h] = 1ull << i;
  }
#pragma unroll
  for (int round = 0; round < 6; ++round) {
    unsigned long long more[2];
    int next[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int from = up[h] & 31;
      const unsigned long long m0 = __shfl_sync(0xffffffffu, mask[0], from), m1 = __shfl_sync(0xffffffffu, mask[1], from);
      const int u0 = __shfl_sync(0xffffffffu, up[0], from), u1 = __shfl_sync(0xffffffffu, up[1], from);
      more[h] = up[h] < 0 ? 0 : up[h] < 32 ? m0 : m1;
      next[h] = up[h] < 0 ? -1 : up[h] < 32 ? u0 : u1;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mask[h] |= more[h];
      up[h] = next[h];
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = lane + 32 * h;
    if (i >= n) break;
    const int place = ctx + i, page = place / page_size;
    seen[first + i] = static_cast<int64_t>(mask[h]);
    positions[first + i] = ctx + __popcll(mask[h]) - 1;
    slots[first + i] = page < table_width ? table[seq * table_ld + page] * page_size + (place - page * page_size) : -1;
  }
  for (int i = n + lane; i < n_all; i += 32) {  // more than a sequence may have
    seen[first + i] = 0;
    positions[first + i] = 0;
    slots[first + i] = -1;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// keep: rows of 16-byte words; a thread has one word of a token's row in one cache and walks the sequence's path. Node indexes
// ascend along a path (path_j >= j), so a row is written only behind the one that it is read from and what is loaded later
// is never overwritten before: all words of a batch of rows are on their way at once, no buffer between. A CTA has a sequence in one cache, all
// layers' caches are in one launch. Bytes bound it where many rows move: 64 sequences, 36 layers
// of 8 heads of 128: 29 us back to back, of which 22 the kernel, for 18 of bytes; one sequence 4.2. An eager call of 72 caches is the host's, 41.
// ---------------------------------------------------------------------------------------------------------------------
static constexpr int kMostCaches = 256;
struct CachePtrs { uint4* at[kMostCaches]; };

struct KeepParams {
  const int32_t* path;
  const int32_t* count;
  const int32_t* q_start;
  const int32_t* seq_lens;
  const int32_t* table;
  int64_t table_ld, pages;
  int table_width, rows, page_size, slabs, words;   // slabs: heads x slabs of a page; words: 16-byte words of a slab's row
};

static constexpr int kKeepThreads = 128, kKeepBatch = 4;

__global__ void __launch_bounds__(kKeepThreads)
draft_keep_kernel(const __grid_constant__ CachePtrs caches, const KeepParams p) {
  __shared__ int64_t from[kMostNodes], to[kMostNodes];   // rows, counted in slab rows of a page: (page * slabs * page_size + row)
  __shared__ int moves;
  griddep_wait();
  const int seq = blockIdx.x;
  const int first = p.q_start[seq], n_all = min(p.q_start[seq + 1], p.rows) - first;
  if (first < 0 || n_all <= 0) return;
  const int n = min(n_all, kMostNodes), ctx = max(p.seq_lens[seq] - n_all, 0), taken = min(p.count[seq], n);
  if (taken < 2) return;
  if (threadIdx.x < 32) {                        // rows that move, in order
    int have = 0;
    for (int j0 = 0; j0 < taken; j0 += 32) {
      const int j = j0 + threadIdx.x;
      const int way = j < taken ? p.path[first + j] : -1;
      bool moves_up = j > 0 && way > j && way < n;
      int64_t a = 0, b = 0;
      if (moves_up) {
        const int oldp = ctx + way, newp = ctx + j;
        if (oldp / p.page_size < p.table_width) {
          const int64_t pa = p.table[seq * p.table_ld + oldp / p.page_size], pb = p.table[seq * p.table_ld + newp / p.page_size];
          a = pa * p.slabs * p.page_size + oldp % p.page_size;
          b = pb * p.slabs * p.page_size + newp % p.page_size;
          moves_up = pa >= 0 && pa < p.pages && pb >= 0 && pb < p.pages;
        } else {
          moves_up = false;
        }
      }
      const unsigned all = __ballot_sync(0xffffffffu, moves_up);
      if (moves_up) {
        const int at = have + __popc(all & ((1u << threadIdx.x) - 1));
        from[at] = a;
        to[at] = b;
      }
      have += __popc(all);
    }
    if (threadIdx.x == 0) moves = have;
  }
  __syncthreads();
  const int total = moves, columns = p.slabs * p.words;
  uint4* cache = caches.at[blockIdx.y];
  for (int c = threadIdx.x; c < columns; c += kKeepThreads) {
    const int slab = c / p.words, w = c - slab * p.words;
    uint4* base = cache + static_cast<int64_t>(slab) * p.page_size * p.words + w;
    for (int j = 0; j < total; j += kKeepBatch) {
      uint4 v[kKeepBatch];
#pragma unroll
      for (int e = 0; e < kKeepBatch; ++e)
        if (j + e < total) v[e] = base[from[j + e] * p.words];
#pragma unroll
      for (int e = 0; e < kKeepBatch; ++e)
        if (j + e < total) base[to[j + e] * p.words] = v[e];
    }
  }
}

}  // namespace b200

using namespace b200;

GLLM_EXPORT int gllm_draft_plan(const void* parents, const void* q_start, const void* seq_lens, const void* table, int64_t table_ld,
                                int table_width, int num_seqs, int rows, int page_size, void* seen, void* positions, void* slots,
                                void* stream) {
  if (rows <= 0) return 0;
  if (num_seqs < 0 || page_size < 1) return 1;
  const int blocks = num_seqs / kPlanWarps + 1;          // one warp more than sequences: the rows behind them
  CUDA_CHECK_RET(launch_pdl(draft_plan_kernel, dim3(blocks), dim3(kPlanWarps * 32), 0, reinterpret_cast<cudaStream_t>(stream),
                            reinterpret_cast<const int32_t*>(parents), reinterpret_cast<const int32_t*>(q_start),
                            reinterpret_cast<const int32_t*>(seq_lens), reinterpret_cast<const int32_t*>(table), table_ld, table_width,
                            num_seqs, rows, page_size, reinterpret_cast<int64_t*>(seen), reinterpret_cast<int32_t*>(positions),
                            reinterpret_cast<int32_t*>(slots)));
  return 0;
}

// caches: n device pointers (on the host) to tensors of one shape: pages of `slabs` slabs of page_size rows of `words` 16-byte words
GLLM_EXPORT int gllm_draft_keep(const void* const* caches, int n, int64_t pages, int slabs, int page_size, int words, const void* path,
                                const void* count, const void* q_start, const void* seq_lens, const void* table, int64_t table_ld,
                                int table_width, int num_seqs, int rows, void* stream) {
  if (n <= 0 || num_seqs <= 0 || rows <= 0 || slabs <= 0 || words <= 0) return 0;
  if (n > kMostCaches || page_size < 1) return 1;
  CachePtrs ptrs;
  for (int i = 0; i < n; ++i) ptrs.at[i] = reinterpret_cast<uint4*>(const_cast<void*>(caches[i]));
  KeepParams p;
  p.path = reinterpret_cast<const int32_t*>(path);
  p.count = reinterpret_cast<const int32_t*>(count);
  p.q_start = reinterpret_cast<const int32_t*>(q_start);
  p.seq_lens = reinterpret_cast<const int32_t*>(seq_lens);
  p.table = reinterpret_cast<const int32_t*>(table);
  p.table_ld = table_ld; p.pages = pages;
  p.table_width = table_width; p.rows = rows; p.page_size = page_size; p.slabs = slabs; p.words = words;
  CUDA_CHECK_RET(launch_pdl(draft_keep_kernel, dim3(num_seqs, n), dim3(kKeepThreads), 0, reinterpret_cast<cudaStream_t>(stream), ptrs, p));
  return 0;
}
