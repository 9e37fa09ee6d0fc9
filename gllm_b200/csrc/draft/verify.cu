// Verification of drafted trees: which nodes the target takes, one path from node 0 on, and the token behind the last. Definitions:
// ops/draft.py.
//
// The walk needs single probabilities (gathered for all nodes at once); the rows of the vocabulary are read only where a node's child is
// not taken, sum max(p - S q, 0), and for the token behind the path, whose sums say where to look. Probabilities are fp32 and
// what is made of them fp64: a running sum over 150,000 fp32 steps would move a border by more than many tokens' share. A CTA, or a
// cluster of them, has a sequence; each CTA has an equal range of the row, each warp an equal range of that, so that a warp's sum is
// that of consecutive tokens. All CTAs of a cluster walk alike: they exchange their sums of a row and add them in one order.
#include "../common/host_utils.h"
#include "../common/ptx.cuh"

namespace b200 {

static constexpr int kNodes = 64;
static constexpr int kVerifyThreads = 1024, kVerifyWarps = kVerifyThreads / 32;
static constexpr int kVerifyParts = 8;                 // CTAs of a cluster at most

enum VerifyForm : int { kMatch = 0, kGiven = 1, kDraws = 2 };

struct VerifyParams {
  const int32_t* tokens;
  const int32_t* parents;
  const int32_t* q_start;
  const int32_t* chosen;     // kMatch: the target's token at every node
  const float* target;
  const float* draft;        // kDraws
  const float* uniform;
  int64_t ld_target, ld_draft;
  int vocab, num_seqs, rows, parts;
  int32_t* said;
  int32_t* path;
  int32_t* count;
};

struct VerifyShared {
  int up[kNodes], word[kNodes];
  unsigned long long children[kNodes];
  double p[kNodes], q[kNodes], u[kNodes];       // of a node's own token, at its parent
  int taken[kNodes], chosen[kNodes];
  double warp_sum[kVerifyWarps];
  double part_sum[2][kVerifyParts];             // of the cluster's CTAs
  int after;
};

// Four tokens at once where both rows allow it: the row's first 16-byte boundary is `lead` tokens before its first token, group g has
// the tokens 4 g - lead and on.
struct Rows {
  const float* p;
  const float* q;            // null: none
  int vocab, lead, groups;
  bool together;
  double past;
  const int* word;           // tokens of the nodes
  unsigned long long gone;   // kGiven: nodes whose tokens are out of the row (those in this warp's range: `near`)

  __device__ __forceinline__ Rows(const float* p_, const float* q_, int v) : p(p_), q(q_), vocab(v), past(0.0), word(nullptr), gone(0) {
    lead = static_cast<int>((reinterpret_cast<uintptr_t>(p) >> 2) & 3);
    groups = (lead + v + 3) / 4;
    together = q == nullptr || ((reinterpret_cast<uintptr_t>(q) ^ reinterpret_cast<uintptr_t>(p)) & 15) == 0;
  }
  __device__ __forceinline__ void raw(int g, float (&a)[4], float (&b)[4]) const {
    const int i = 4 * g - lead;
    if (i >= 0 && i + 4 <= vocab) {
      const float4 x = *reinterpret_cast<const float4*>(p + i);
      a[0] = x.x; a[1] = x.y; a[2] = x.z; a[3] = x.w;
      if (q != nullptr) {
        if (together) {
          const float4 y = *reinterpret_cast<const float4*>(q + i);
          b[0] = y.x; b[1] = y.y; b[2] = y.z; b[3] = y.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) b[e] = q[i + e];
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = i + e >= 0 && i + e < vocab;
        a[e] = in ? p[i + e] : 0.f;
        if (q != nullptr) b[e] = in ? q[i + e] : 0.f;
      }
    }
  }
  // of the nodes in `gone`, those whose tokens lie in groups [g0, g1): none for most warps
  __device__ __forceinline__ unsigned long long near(int g0, int g1) const {
    unsigned long long m = 0;
    for (unsigned long long e = gone; e != 0ull; e &= e - 1) {
      const int i = __ffsll(static_cast<long long>(e)) - 1, at = word[i] + lead;
      if (word[i] >= 0 && word[i] < vocab && at >= 4 * g0 && at < 4 * g1) m |= 1ull << i;
    }
    return m;
  }
  __device__ __forceinline__ void mass(int g, unsigned long long out, const float (&a)[4], const float (&b)[4], double (&r)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      double x = static_cast<double>(a[e]);
      if (q != nullptr) x = __dadd_rn(x, -__dmul_rn(past, static_cast<double>(b[e])));
      r[e] = x > 0.0 ? x : 0.0;
    }
    for (; out != 0ull; out &= out - 1) {
      const int at = word[__ffsll(static_cast<long long>(out)) - 1] + lead - 4 * g;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e == at) r[e] = 0.0;
    }
  }
};

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// groups of this warp: [first, end)
__device__ __forceinline__ void share(int groups, int part, int parts, int warp, int& first, int& end) {
  const int64_t all = static_cast<int64_t>(parts) * kVerifyWarps, w = static_cast<int64_t>(part) * kVerifyWarps + warp;
  first = static_cast<int>(groups * w / all);
  end = static_cast<int>(groups * (w + 1) / all);
}

// sum of the row's mass, the same in every thread of the cluster
__device__ __forceinline__ double row_sum(const Rows& r, VerifyShared& s, int part, int parts, int pass) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int g0, g1;
  share(r.groups, part, parts, warp, g0, g1);
  double sum = 0.0;
  const unsigned long long out = r.near(g0, g1);
  for (int g = g0 + lane; g < g1; g += 32) {
    float a[4], b[4];
    double m[4];
    r.raw(g, a, b);
    r.mass(g, out, a, b, m);
    sum += (m[0] + m[1]) + (m[2] + m[3]);
  }
  sum = warp_sum(sum);
  __syncthreads();                                       // the sums of the pass before have been read
  if (lane == 0) s.warp_sum[warp] = sum;
  __syncthreads();
  double mine = 0.0;
  for (int w = 0; w < kVerifyWarps; ++w) mine += s.warp_sum[w];
  if (parts == 1) return mine;
  if (threadIdx.x < parts) {
    const uint32_t at = cluster_addr(&s.part_sum[pass & 1][part], threadIdx.x);
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(mine) : "memory");
  }
  __syncwarp();
  cluster_sync();
  double all = 0.0;
  for (int i = 0; i < parts; ++i) all += s.part_sum[pass & 1][i];
  return all;
}

__global__ void __launch_bounds__(kVerifyThreads)
draft_verify_kernel(const VerifyParams v) {
  __shared__ VerifyShared s;
  if (v.parts > 1) cluster_sync();                       // every CTA's shared memory is there
  griddep_wait();
  const int parts = v.parts, seq = blockIdx.x / parts, part = blockIdx.x % parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int form = v.target == nullptr ? kMatch : v.draft == nullptr ? kGiven : kDraws;
  if (seq == v.num_seqs) {                               // rows behind the last sequence
    if (part == 0)
      for (int i = max(v.q_start[v.num_seqs], 0) + threadIdx.x; i < v.rows; i += kVerifyThreads) v.said[i] = v.path[i] = -1;
    return;
  }
  const int first = v.q_start[seq], n_all = first < 0 ? 0 : min(v.q_start[seq + 1], v.rows) - first;
  if (n_all <= 0) {
    if (part == 0 && threadIdx.x == 0) v.count[seq] = 0;
    return;
  }
  const int n = min(n_all, kNodes);
  if (threadIdx.x < kNodes) s.children[threadIdx.x] = 0ull;
  if (threadIdx.x < n) {
    const int i = threadIdx.x, up = v.parents[first + i], word = v.tokens[first + i];
    s.up[i] = up >= 0 && up < i ? up : -1;
    s.word[i] = word;
    if (form == kMatch) {
      s.chosen[i] = v.chosen[first + i];
    } else {
      const int64_t row = first + max(s.up[i], 0);
      const bool in = word >= 0 && word < v.vocab;
      const float p = in ? v.target[row * v.ld_target + word] : 0.f;
      s.p[i] = static_cast<double>(p);
      s.q[i] = form == kGiven || !in ? 1.0 : static_cast<double>(v.draft[row * v.ld_draft + word]);
      s.u[i] = static_cast<double>(v.uniform[first + i]);
    }
  }
  __syncthreads();
  if (threadIdx.x < n && s.up[threadIdx.x] >= 0) atomicOr(&s.children[s.up[threadIdx.x]], 1ull << threadIdx.x);
  if (threadIdx.x == 0) s.taken[0] = 0;
  __syncthreads();

  int node = 0, depth = 1, pass = 0;
  double past = 0.0, total = 0.0;
  bool summed = false;                                   // total is that of the row left at `node`
  for (;;) {
    // children of `node`, in every thread alike
    unsigned long long left = s.children[node];
    int step = -1;
    double mass = 1.0;
    past = 0.0;
    summed = false;
    while (left != 0ull) {
      const int i = __ffsll(static_cast<long long>(left)) - 1;
      left &= left - 1;
      if (form == kMatch) {
        if (s.word[i] == s.chosen[node]) step = i;
      } else if (form == kGiven) {
        double have = s.p[i] > 0.0 ? s.p[i] : 0.0;
        for (unsigned long long e = s.children[node] & ((1ull << i) - 1); e != 0ull; e &= e - 1)
          if (s.word[__ffsll(static_cast<long long>(e)) - 1] == s.word[i]) have = 0.0;
        if (s.u[i] * mass < have) step = i;
        else mass = fmax(mass - have, 0.0);
      } else {
        const double r = __dadd_rn(s.p[i], -__dmul_rn(past, s.q[i]));
        const bool in = s.word[i] >= 0 && s.word[i] < v.vocab;
        if (in && s.u[i] * mass * s.q[i] < (r > 0.0 ? r : 0.0)) {
          step = i;
        } else {
          past += mass;
          Rows rows(v.target + (first + node) * v.ld_target, v.draft + (first + node) * v.ld_draft, v.vocab);
          rows.past = past;
          mass = total = row_sum(rows, s, part, parts, pass++);
          summed = true;
        }
      }
      if (step >= 0) break;
    }
    if (step < 0) break;
    node = step;
    if (threadIdx.x == 0) s.taken[depth] = step;
    ++depth;
  }

  int after;
  if (form == kMatch) {
    after = s.chosen[node];
  } else {
    __syncthreads();                                     // s.taken
    Rows rows(v.target + (first + node) * v.ld_target, form == kDraws ? v.draft + (first + node) * v.ld_draft : nullptr, v.vocab);
    rows.past = past;
    rows.word = s.word;
    rows.gone = form == kGiven ? s.children[node] : 0ull;
    if (!summed) total = row_sum(rows, s, part, parts, pass++);
    if (!(total > 0.0)) {                                // nothing is left of p: p itself
      rows.gone = 0ull;
      rows.past = 0.0;
      total = row_sum(rows, s, part, parts, pass++);
    }
    // the warp that the border lies in: its range's running sum is the first over u x total, or the last with mass
    const double border = s.u[0] * total;
    double before = 0.0;
    int owner = -1;
    if (parts > 1) {
      double run = 0.0;
      for (int i = 0; i < parts; ++i) {
        const double m = s.part_sum[(pass - 1) & 1][i];
        if (m > 0.0) {
          owner = i;
          before = run;
        }
        run += m;
        if (m > 0.0 && run > border) break;
      }
      if (owner < 0 ? part != 0 : part != owner) return;
    } else if (total > 0.0) {
      owner = 0;
    }
    int mine = -1;
    double start = 0.0;
    if (owner >= 0) {
      double run = before;
      for (int w = 0; w < kVerifyWarps; ++w) {
        const double m = s.warp_sum[w];
        if (m > 0.0) {
          mine = w;
          start = run;
        }
        run += m;
        if (m > 0.0 && run > border) break;
      }
    }
    if (warp == max(mine, 0)) {
      int found = -1, last = 0;
      if (mine >= 0) {
        int g0, g1;
        share(rows.groups, part, parts, warp, g0, g1);
        double run = start;
        const unsigned long long out = rows.near(g0, g1);
        for (int g = g0; g < g1 && found < 0; g += 32) {
          float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
          double m[4] = {0.0, 0.0, 0.0, 0.0};
          if (g + lane < g1) {
            rows.raw(g + lane, a, b);
            rows.mass(g + lane, out, a, b, m);
          }
          const double own = (m[0] + m[1]) + (m[2] + m[3]);
          double upto = own;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
          }
          const unsigned with = __ballot_sync(0xffffffffu, own > 0.0), over = __ballot_sync(0xffffffffu, own > 0.0 && run + upto > border);
          const int lane_hit = over != 0u ? __ffs(over) - 1 : -1, lane_last = with != 0u ? 31 - __clz(with) : -1;
          double at = run + (upto - own);
          int hit = -1, end = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            at += m[e];
            if (m[e] > 0.0) {
              end = 4 * (g + lane) - rows.lead + e;
              if (hit < 0 && at > border) hit = end;
            }
          }
          if (hit < 0) hit = end;                        // the group's sum is over the border, rounding left no token of it there
          if (lane_last >= 0) last = __shfl_sync(0xffffffffu, end, lane_last);
          if (lane_hit >= 0) found = __shfl_sync(0xffffffffu, hit, lane_hit);
          run += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (found < 0) found = last;
      }
      if (lane == 0) s.after = max(found, 0);
    }
    __syncthreads();
    after = s.after;
  }
  if (part != 0 && form == kMatch) return;
  if (form == kMatch) __syncthreads();                   // s.taken
  for (int j = threadIdx.x; j < n_all; j += kVerifyThreads) {
    v.path[first + j] = j < depth ? s.taken[j] : -1;
    v.said[first + j] = j + 1 < depth ? s.word[s.taken[j + 1]] : j + 1 == depth ? after : -1;
  }
  if (threadIdx.x == 0) v.count[seq] = depth;
}

}  // namespace b200

using namespace b200;

// chosen: the target's tokens (comparison), or target (and draft, or null) probabilities with uniform
GLLM_EXPORT int gllm_draft_verify(const void* tokens, const void* parents, const void* q_start, const void* chosen, const void* target,
                                  int64_t ld_target, const void* draft, int64_t ld_draft, const void* uniform, int vocab, int num_seqs,
                                  int rows, void* said, void* path, void* count, int parts, void* stream) {
  if (num_seqs < 0 || (chosen == nullptr) == (target == nullptr) || parts < 1 || parts > kVerifyParts) return 1;
  if (num_seqs == 0 && rows <= 0) return 0;
  VerifyParams v;
  v.tokens = reinterpret_cast<const int32_t*>(tokens);
  v.parents = reinterpret_cast<const int32_t*>(parents);
  v.q_start = reinterpret_cast<const int32_t*>(q_start);
  v.chosen = reinterpret_cast<const int32_t*>(chosen);
  v.target = reinterpret_cast<const float*>(target);
  v.draft = reinterpret_cast<const float*>(draft);
  v.uniform = reinterpret_cast<const float*>(uniform);
  v.ld_target = ld_target; v.ld_draft = ld_draft;
  v.vocab = vocab; v.num_seqs = num_seqs; v.rows = rows; v.parts = parts;
  v.said = reinterpret_cast<int32_t*>(said);
  v.path = reinterpret_cast<int32_t*>(path);
  v.count = reinterpret_cast<int32_t*>(count);
  const dim3 grid(static_cast<unsigned>(num_seqs + 1) * parts);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (parts > 1) CUDA_CHECK_RET(launch_pdl_cluster(draft_verify_kernel, grid, parts, dim3(kVerifyThreads), 0, st, v));
  else CUDA_CHECK_RET(launch_pdl(draft_verify_kernel, grid, dim3(kVerifyThreads), 0, st, v));
  return 0;
}
