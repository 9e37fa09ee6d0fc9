// Verification of drafted trees: which nodes the target takes, one path from node 0 on, and the token behind the last. Definitions:
// ops/draft.py.
//
// The walk needs single probabilities (gathered for all nodes at once); the rows of the vocabulary are read only where a node's child is
// not taken, sum max(p - S q, 0), and for the token behind the path, whose sums say where to look. Probabilities are fp32 and
// what is made of them fp64: a running sum over 150,000 fp32 steps would move a border by more than many tokens' share. A CTA, or a
// cluster of them, has a sequence; each CTA has an equal range of the row, each warp an equal range of that, so that a warp's sum is
// that of consecutive tokens. All CTAs of a cluster walk alike: they exchange their sums of a row and add them in one order.
//
// What bounds it: latency. A row is read behind the decisions that lead to it (lengths, tokens, their probabilities: three trips to memory, then the
// cluster's barrier), and its warp's range once more for the border: one chain of 151,936 tokens 9.0 us, 64 chains of 128,257 18.0 for 10 of bytes
// (66 MB, all sequences in the same phase at the same time), 256 of 151,936 60 for 47. The draft's row is read where a child was refused: where all
// are taken these are 8.5, 15.2 and 43.
#include "../common/host_utils.h"
#include "../common/ptx.cuh"

namespace b200 {

static constexpr int kNodes = 64;
static constexpr int kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32;
static constexpr int kVerifyParts = 16;                // CTAs of a cluster at most

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
  int after, first_over, last_with;
};

// Four tokens at once: the row's first 16-byte boundary is `lead` tokens before its first token, group g has the tokens 4 g - lead and on
struct Rows {
  const float* p;
  const float* q;            // null: none, the mass is p's
  int vocab, lead, groups;
  bool together;             // both rows have their boundaries at the same tokens
  double past;
  const int* word;           // tokens of the nodes
  unsigned long long gone;   // kGiven: nodes whose tokens are out of the row

  __device__ __forceinline__ Rows(const float* p_, const float* q_, int v) : p(p_), q(q_), vocab(v), past(0.0), word(nullptr), gone(0) {
    lead = static_cast<int>((reinterpret_cast<uintptr_t>(p) >> 2) & 3);
    groups = (lead + v + 3) / 4;
    together = q == nullptr || ((reinterpret_cast<uintptr_t>(q) ^ reinterpret_cast<uintptr_t>(p)) & 15) == 0;
  }
  // any group
  __device__ __forceinline__ void raw(int g, float4& a, float4& b) const {
    const int i = 4 * g - lead;
    float x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = i + e >= 0 && i + e < vocab;
      x[e] = in ? p[i + e] : 0.f;
      y[e] = in && q != nullptr ? q[i + e] : 0.f;
    }
    a = make_float4(x[0], x[1], x[2], x[3]);
    b = make_float4(y[0], y[1], y[2], y[3]);
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
  __device__ __forceinline__ double left_of(float a, float b) const {
    const double x = __dadd_rn(static_cast<double>(a), -__dmul_rn(past, static_cast<double>(b)));
    return x > 0.0 ? x : 0.0;
  }
  __device__ __forceinline__ void mass(int g, unsigned long long out, const float4& a, const float4& b, double (&r)[4]) const {
    if (q != nullptr) {
      r[0] = left_of(a.x, b.x); r[1] = left_of(a.y, b.y); r[2] = left_of(a.z, b.z); r[3] = left_of(a.w, b.w);
    } else {
      r[0] = fmaxf(a.x, 0.f); r[1] = fmaxf(a.y, 0.f); r[2] = fmaxf(a.z, 0.f); r[3] = fmaxf(a.w, 0.f);   // not a number: 0
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

// groups of a warp: [first, end)
__device__ __forceinline__ void share(int groups, int part, int parts, int warp, int& first, int& end) {
  const int64_t all = static_cast<int64_t>(parts) * kVerifyWarps, w = static_cast<int64_t>(part) * kVerifyWarps + warp;
  first = static_cast<int>(groups * w / all);
  end = static_cast<int>(groups * (w + 1) / all);
}

// This lane's part of the mass of groups [g0, g1). Whole groups have their loads two at a time ahead of their arithmetic: one at a time the
// latency of each is waited for; four at a time need more than 64 registers (64 chains of 128,257 tokens, both rows read for each: 20.9 us, four
// 21.6, six 27).
__device__ __forceinline__ double range_mass(const Rows& r, int g0, int g1, int lane) {
  constexpr int kAhead = 2;
  const unsigned long long out = r.near(g0, g1);
  const int w0 = max(g0, r.lead != 0 ? 1 : 0), w1 = min(g1, (r.lead + r.vocab) / 4);
  double sum = 0.0, m[4];
  float4 a[kAhead], b[kAhead];
  for (int g = w0 + lane; g < w1; g += 32 * kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = g + 32 * u;
      a[u] = b[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (h < w1) {
        a[u] = *reinterpret_cast<const float4*>(r.p + 4 * h - r.lead);
        if (r.q != nullptr) {
          const float* at = r.q + 4 * h - r.lead;
          b[u] = r.together ? *reinterpret_cast<const float4*>(at) : make_float4(at[0], at[1], at[2], at[3]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      r.mass(g + 32 * u, out, a[u], b[u], m);
      sum += (m[0] + m[1]) + (m[2] + m[3]);
    }
  }
  // the groups at the row's ends
  const int edge = lane == 0 && g0 < min(w0, g1) ? g0 : lane == 1 && w1 < g1 && w1 >= w0 ? w1 : -1;
  if (edge >= 0) {
    r.raw(edge, a[0], b[0]);
    r.mass(edge, out, a[0], b[0], m);
    sum += (m[0] + m[1]) + (m[2] + m[3]);
  }
  return sum;
}

// sum of the row's mass, the same in every thread of the cluster
__device__ __forceinline__ double row_sum(const Rows& r, VerifyShared& s, int part, int parts, int pass) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int g0, g1;
  share(r.groups, part, parts, warp, g0, g1);
  const double sum = warp_sum(range_mass(r, g0, g1, lane));
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

__global__ void __launch_bounds__(kVerifyThreads, 2)
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
    // The draft's row counts where a child was refused only (past is 1 or more then): others may hold anything, NaN among it
    Rows rows(v.target + (first + node) * v.ld_target, form == kDraws && past > 0.0 ? v.draft + (first + node) * v.ld_draft : nullptr, v.vocab);
    rows.past = past;
    rows.word = s.word;
    rows.gone = form == kGiven ? s.children[node] : 0ull;
    if (!summed) total = row_sum(rows, s, part, parts, pass++);
    if (!(total > 0.0)) {                                // nothing is left of p: p itself
      rows.gone = 0ull;
      rows.q = nullptr;
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
    // Its range, by the whole CTA: consecutive groups a thread, their running sums, the first thread whose sum is over the border (or the last
    // with mass) looks at its tokens
    int g0 = 0, g1 = 0;
    if (mine >= 0) share(rows.groups, part, parts, mine, g0, g1);
    const unsigned long long out = rows.near(g0, g1);
    const int each = (g1 - g0 + kVerifyThreads - 1) / kVerifyThreads;
    const int h0 = min(g0 + static_cast<int>(threadIdx.x) * each, g1), h1 = min(h0 + each, g1);
    float4 a, b;
    double m[4], own = 0.0;
    for (int g = h0; g < h1; ++g) {
      rows.raw(g, a, b);
      rows.mass(g, out, a, b, m);
      own += (m[0] + m[1]) + (m[2] + m[3]);
    }
    double upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    __syncthreads();                                     // s.warp_sum has been read
    if (lane == 31) s.warp_sum[warp] = upto;
    if (threadIdx.x == 0) {
      s.first_over = kVerifyThreads;
      s.last_with = -1;
      s.after = 0;
    }
    __syncthreads();
    double before_me = start;
    for (int w = 0; w < warp; ++w) before_me += s.warp_sum[w];
    before_me += upto - own;
    if (own > 0.0) {
      atomicMax(&s.last_with, static_cast<int>(threadIdx.x));
      if (before_me + own > border) atomicMin(&s.first_over, static_cast<int>(threadIdx.x));
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) == (s.first_over < kVerifyThreads ? s.first_over : s.last_with)) {
      int hit = -1, last = 0;
      double at = before_me;
      for (int g = h0; g < h1; ++g) {
        rows.raw(g, a, b);
        rows.mass(g, out, a, b, m);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          at += m[e];
          if (m[e] > 0.0) {
            last = 4 * g - rows.lead + e;
            if (hit < 0 && at > border) hit = last;
          }
        }
      }
      s.after = hit >= 0 ? hit : last;                   // rounding left no token of it over the border: the last one
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
  if (parts > 8) {                                       // more than every device has to take
    static PerDeviceOnce configured;
    if (configured.need()) {
      CUDA_CHECK_RET(cudaFuncSetAttribute(draft_verify_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
      configured.done();
    }
  }
  if (parts > 1) CUDA_CHECK_RET(launch_pdl_cluster(draft_verify_kernel, grid, parts, dim3(kVerifyThreads), 0, st, v));
  else CUDA_CHECK_RET(launch_pdl(draft_verify_kernel, grid, dim3(kVerifyThreads), 0, st, v));
  return 0;
}
