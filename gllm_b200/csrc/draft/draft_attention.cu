// Attention of drafted nodes over a paged bf16 cache. Definition: ops/draft.py.
//
// Work: a unit is a sequence, a kv head and a block of its rows (node x query head), as long as the sequence's 128-key tiles. A block's scores
// S = Q K^T and results O += P V are tcgen05 products of M = 128, whatever the rows: 1024 cycles of tensor core per 128 keys (heads of 128),
// where their 64 KB take some 2700 of an SM's share of the memory. All units lie in one row that is cut into equal shares for the CTAs, one an
// SM, on the device, so that lengths may differ from those at the time a graph was captured and long contexts beside short ones leave no SM
// idle. A share's units are whole but for the first and the last; those parts (O in fp32, maximum, sum) are joined by a second launch in a
// fixed order, which costs 5 to 9 us. Or no unit is cut, where none has more than 16 tiles and that costs less (ops/sm100_draft.py): the SM with the
// longest ends last then.
//
// Rows, by what a sequence may have (host):  up to 32, 64, 128  one block; with few rows 4 or 2 TMEM lanes share a row, each has a part of
// every tile's keys, so that all four schedulers form exponentials (a lane's 128 take a warp 1700 cycles and more, 32 take 650).
// More: blocks of two halves of 128, so that keys and values are read once for 256 rows. Where a row has one lane two warps share it, with 64
// keys of a tile each (16 of 8000 tokens, 64 nodes, 32 / 8 heads: 123.5 us with one warp, 121 with two; 128 x 600, 24 nodes: 67.2 and 65.5, or
// 66.6 to 67.1 since blocks of up to 128 rows meet once more a tile).
//
//   softmax            two groups of four warps, or of eight (two a row); a row a lane (tcgen05.ld 32x32b). The groups have the CTA's items
//                      in turn: one's results, some 3000 cycles of which most is instruction fetch, are written while the other has the
//                      next one. (Tiles in turn, with one reference of the exponents handed on: the case above 79 us, items 69.) The
//                      reference follows the maximum in steps of 2^8; P goes over S, as the A operand of the product with V
//   two warps          copies of K and V: page boxes [page][64] -> one ring of tiles [D / 64][128][64] (SW128), K a tile ahead of V. (One
//                      warp for both issues 32 boxes of 2 KB in 3300 cycles, more than their bytes take)
//   one thread         products: S of the tile to come before P V of this one (S and P in two buffers of TMEM, O in two). It is found by
//                      elect.sync: eight products are issued in 300 to 420 cycles then, behind `lane == 0` in some 600
//   one thread         queries, a box a block, of the items to come (two buffers)
//
// Masks: only tiles that reach behind the context are masked, with the bits of the row's word shifted to the tile. A value that is not seen must
// not reach the sum even as 0 x NaN: rows behind the last key are zeroed, and so are values of nodes that are no numbers; rows that see
// those have them added at the end.
//
// What bounds it: HBM where histories are long (two of 60,000, 64 / 8 heads, 16 nodes: 82 us for 61 of bytes, the copies alone 69; 64 of 2500, 8
// nodes 89 for 74; some 10 us are the first data and the last results). Blocks of 256 rows: the chain softmax -> P V -> S of a half, 3960 cycles
// per 128 keys for 2048 of tensor core and of the 2^x unit each (4 of 30,000, 64 nodes, 64 / 8 heads: 165 us, 775 TFLOP/s): maximum 600,
// exponentials 1300 to 1600, the two hand-overs 530, the products 1250. The prefill kernel has the same chain at 1221 TFLOP/s, with a row of scores
// in the registers of one thread (setmaxnreg) instead of two readings of TMEM by two; that form was not tried here. A product with the first half
// of P while the other half is formed gains 1 % (the issuing thread's waits take the rest), exponentials by polynomial lose 6 %, a thread for
// either half's products loses 20 % (one thread's order keeps one half at its exponentials while the other is at its products); steps of 64 keys
// with two buffers of S a half were slower (278 for 173): twice the products and commits of that thread.
#include "../attn/attn_common.cuh"
#include "../common/bounded.cuh"

namespace b200 {

static constexpr int kNodes = 64;
static constexpr int kRows = 128, kKeys = 128;           // of a unit's block, of a tile
constexpr int softmax_warps(int rep) { return rep <= 1 ? 16 : 8; }
constexpr int cta_threads(int rep) { return (softmax_warps(rep) + 4) * 32; }
static constexpr float kLazy = 8.f;                      // P stays below 2^8 between two rescales of O

struct DraftAttnParams {
  const __nv_bfloat16* q;
  int64_t q_ts;
  __nv_bfloat16* out;
  const __nv_bfloat16* v;                                // for nodes whose values are no numbers
  int64_t pages;
  const int32_t* table;
  int64_t table_ld;
  const int32_t* seq_lens;
  const int32_t* q_start;
  const int64_t* seen;
  int table_width, num_seqs, rows, Hq, Hkv, G, page_shift;   // a page has 2^page_shift tokens
  int whole;                                             // no unit is cut: nothing to join
  int block_rows, half_rows, part_rows;                  // of a block, of a box of queries; rows that parts have room for
  float scale_log2;
  float4* part_o;                                        // [2 CTA][D / 4][128 rows]
  float2* part_ml;                                       // [2 CTA][128 rows]: reference of the exponents, sum
  int4* cut;                                             // [CTA][2]: what the join of a unit that the CTA begins needs
  WaitConfig waits;
};

inline int part_rows_of(int max_rows) { return max_rows > kRows ? 2 * kRows : kRows; }

template <int D>
struct DraftSmem {
  static constexpr int kQBytes = kRows * D * 2, kTileBytes = kKeys * D * 2;
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr int kRingOff = 2 * kQBytes, kBarOff = kRingOff + kStages * kTileBytes;
  // barriers and words (see the kernel), and up to 1 KB before the first 1024-byte boundary
  static constexpr int kBarBytes = (2 * kStages + 17) * 8 + 8 + 4 * 8 + 5 * 8 + 20 * 8 + 2 * kRows * 4 + kStages * 4;
  static constexpr int kBytes = kBarOff + (kBarBytes + 15) / 16 * 16 + 1024;
  static_assert(kBytes <= 232448, "shared memory of a CTA");
  static constexpr int kTmemO = 2 * kKeys, kTmemCols = 512;
};

__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// P of 16 keys, the kk-th of a tile: in the first columns of its 32 keys' scores
__device__ __forceinline__ uint32_t p_column(uint32_t kk) { return (kk >> 1) * 32 + (kk & 1) * 8; }
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// V as it lies in the cache, keys along the rows: MN-major, 64 dims (128 bytes) then the next slab LBO bytes on, 8 keys SBO
__device__ __forceinline__ uint64_t mn_major_desc(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFF) | static_cast<uint64_t>((kKeys * 128) >> 4) << 16 |
         static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
// an order of fp32 that integers have too (and back: the same)
__device__ __forceinline__ int ordered(int bits) { return bits ^ ((bits >> 31) & 0x7fffffff); }
static constexpr int kNoScore = static_cast<int>(0x807fffffu);       // -infinity
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// What a sequence is to the units: rows [first, first + n) of the batch, ctx tokens before its nodes
struct Seq {
  int first, n, ctx, len, tiles, blocks;
  __device__ __forceinline__ void set(const DraftAttnParams& p, int start, int end, int seq_len) {
    first = start;
    const int n_all = first < 0 ? 0 : min(end, p.rows) - first;
    n = max(min(n_all, kNodes), 0);
    ctx = min(max(seq_len - max(n_all, 0), 0), p.table_width << p.page_shift);
    len = min(ctx + n, p.table_width << p.page_shift);   // what the table holds
    blocks = (n * p.G + p.block_rows - 1) / p.block_rows;
    tiles = n > 0 ? (len + kKeys - 1) / kKeys : 0;
  }
  __device__ __forceinline__ int work(const DraftAttnParams& p) const { return tiles * blocks * p.Hkv; }
};

// The CTA's items: its share of one unit each, tiles [t0, t1). What the next sequence is to be made of is on its way while this one's items run.
struct Items : Seq {
  const DraftAttnParams& p;
  int s;
  int off, left;                                         // in the sequence's work; tiles to come
  int kvh, blk, t0, t1;
  int end, next_end, next_len;                           // q_start[s + 1], q_start[s + 2], seq_lens[s + 1]
  __device__ __forceinline__ Items(const DraftAttnParams& p_, int s_, int off_, int left_) : p(p_), s(s_), off(off_), left(left_) {
    end = p.q_start[s + 1];
    set(p, p.q_start[s], end, p.seq_lens[s]);
    ahead();
  }
  __device__ __forceinline__ void ahead() {
    const int t = min(s + 1, p.num_seqs - 1);
    next_end = p.q_start[t + 1];
    next_len = p.seq_lens[t];
  }
  __device__ __forceinline__ bool next() {
    if (left <= 0) return false;
    while (off >= work(p)) {                             // the sequence that `off` lies in: there is one, as tiles are left
      off = 0;
      if (++s >= p.num_seqs) {
        left = 0;
        return false;
      }
      set(p, end, next_end, next_len);
      end = next_end;
      ahead();
    }
    const int unit = off / tiles;
    t0 = off - unit * tiles;
    t1 = min(tiles, t0 + left);
    kvh = unit / blocks;
    blk = unit - kvh * blocks;
    off += t1 - t0;
    left -= t1 - t0;
    return true;
  }
  __device__ __forceinline__ int block_rows() const { return min(p.block_rows, n * p.G - blk * p.block_rows); }
  // keys of tile t that there are
  __device__ __forceinline__ int keys(int t) const { return min(len - t * kKeys, kKeys); }
};

template <int D, int REP>
__global__ void __launch_bounds__(cta_threads(REP), 1)
draft_attention_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_q,
                       const DraftAttnParams p) {
  using SM = DraftSmem<D>;
  constexpr int NS = SM::kStages;
  // A block's rows are whole nodes. REP 1, 2, 4: at most BR = 128 / REP rows, TMEM lane = part of the keys x BR + row, the warpgroups
  // take the items in turn. REP 0 (WIDE): two halves of at most 128 rows, each warpgroup has one of them of every item.
  // PAIR: two threads have a TMEM lane, 64 keys of a tile each.
  constexpr bool WIDE = REP == 0, PAIR = REP <= 1;
  constexpr int kLanes = WIDE ? 1 : REP, kParts = PAIR ? 2 : REP;    // TMEM lanes, threads of a row
  constexpr int BR = kRows / kLanes;
  constexpr int kChunks = kKeys / 32 / kParts;           // of 32 keys that a thread has of a tile
  constexpr int kThreads = cta_threads(REP), W0 = softmax_warps(REP), kGroup = W0 * 16;   // a warpgroup's (a half's) threads
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + SM::kBarOff);   // [NS] copies -> products (and softmax: V)
  uint64_t* empty = full + NS;                           // [NS] products -> copies
  uint64_t* s_full = empty + NS;                         // [2 warpgroups][2] S of the warpgroup's k-th tile: barrier k % 2 (WIDE: the first)
  uint64_t* p_full = s_full + 4;                         // [2] P of the CTA's tile g written (4 warps): barrier g % 2 (WIDE: of a half)
  uint64_t* pv_full = p_full + 2;                        // [2 warpgroups][2] P V of its k-th tile is in O: barrier k % 2 (WIDE: the first)
  uint64_t* o_free = pv_full + 4;                        // [2 warpgroups] O of its item has been read (4 warps)
  uint64_t* q_full = o_free + 2;                         // [2] queries of item i: barrier i % 2 (WIDE: the first)
  uint64_t* q_free = q_full + 2;                         // [2]
  uint64_t* mma_end = q_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_end + 1);
  const WaitGuard guard{tmem_slot + 1, p.waits};
  unsigned long long* bad_nodes = reinterpret_cast<unsigned long long*>(tmem_slot + 2);   // [item % 4]
  int64_t* begin = reinterpret_cast<int64_t*>(bad_nodes + 4);         // share: first sequence, offset in it, end; all tiles; begin
  int64_t* warp_work = begin + 5;                        // [20]
  volatile uint32_t* filled = reinterpret_cast<uint32_t*>(warp_work + 20);   // [NS] copies into a stage
  int* row_max = reinterpret_cast<int*>(warp_work + 20) + NS;        // PAIR: [2 warpgroups][128] maximum of a row's scores, as an integer of the same order

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); filled[i] = 0; }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[2 * i], 1); mbar_init(&s_full[2 * i + 1], 1); mbar_init(&p_full[i], W0 / 2);
      mbar_init(&pv_full[2 * i], 1); mbar_init(&pv_full[2 * i + 1], 1); mbar_init(&o_free[i], W0 / 2); mbar_init(&q_full[i], 1); mbar_init(&q_free[i], REP > 1 ? 2 : 1);
      bad_nodes[2 * i] = bad_nodes[2 * i + 1] = 0ull;
    }
    mbar_init(mma_end, 1);
    *guard.dead = 0;
    begin[0] = begin[1] = begin[2] = begin[4] = 0;
    fence_mbar_init();
  }
  if (warp == W0 + 1) tmem_alloc<1>(tmem_slot, SM::kTmemCols);
  if (PAIR && threadIdx.x < 2 * kRows) row_max[threadIdx.x] = kNoScore;
  if (warp == W0 && lane < 3) tma_prefetch_desc(lane == 0 ? &tmap_k : lane == 1 ? &tmap_v : &tmap_q);
  griddep_launch();
  griddep_wait();

  // ---- the share: prefix sums of the sequences' work, a run of sequences a thread
  {
    const int per = (p.num_seqs + kThreads - 1) / kThreads, s0 = threadIdx.x * per, s1 = min(s0 + per, p.num_seqs);
    int64_t mine = 0;
    Seq q;
    for (int s = s0; s < s1; ++s) {
      q.set(p, p.q_start[s], p.q_start[s + 1], p.seq_lens[s]);
      mine += q.work(p);
    }
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) warp_work[warp] = upto;
    __syncthreads();
    int64_t before = upto - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += warp_work[w];
      all += warp_work[w];
    }
    // no more CTAs than tiles take part, so that no share between two others is empty
    const int64_t ctas = min(static_cast<int64_t>(gridDim.x), all);
    if (blockIdx.x < ctas) {
      const int64_t x[2] = {all * blockIdx.x / ctas, all * (blockIdx.x + 1) / ctas};
#pragma unroll
      for (int i = 0; i < 2; ++i) {                        // where the share begins and ends; WHOLE: at the next unit's first tile
        if (x[i] < before || x[i] >= before + mine) continue;
        int64_t at = before;
        int s = s0;
        for (;; ++s) {
          q.set(p, p.q_start[s], p.q_start[s + 1], p.seq_lens[s]);
          const int w = q.work(p);
          if (x[i] < at + w || s + 1 >= s1) break;
          at += w;
        }
        int off = static_cast<int>(x[i] - at);
        if (p.whole) off = (off + q.tiles - 1) / q.tiles * q.tiles;
        if (i == 0) {
          begin[0] = s;
          begin[1] = off;
          begin[4] = at + off;
        } else {
          begin[2] = at + off;
        }
      }
      if (threadIdx.x == 0 && x[1] == all) begin[2] = all;
    }
    if (threadIdx.x == 0) begin[3] = all;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Items it(p, static_cast<int>(begin[0]), static_cast<int>(begin[1]), static_cast<int>(begin[2] - begin[4]));
  const bool idle = begin[2] <= begin[4];

  if (warp >= W0) {
    if ((warp == W0 || warp == W0 + 2) && !idle) {
      // ------------------------------------------------------------------ copies: K, V
      const bool is_v = warp == W0 + 2;
      const CUtensorMap* map = is_v ? &tmap_v : &tmap_k;
      const int box = 1 << min(p.page_shift, 6), boxes = kKeys / box, j = lane % boxes, sl = lane / boxes;
      const int in_page = (1 << p.page_shift) - 1;
      uint32_t g = 0;
      bool ok = true;
      while (ok && it.next()) {
        const int32_t* bt = p.table + it.s * p.table_ld;
        const int last_page = min((it.len - 1) >> p.page_shift, p.table_width - 1);
        auto page_of = [&](int tile) { return bt[min((tile * kKeys + j * box) >> p.page_shift, last_page)]; };
        int page = page_of(it.t0);
        for (int t = it.t0; t < it.t1; ++t, ++g) {
          const int next = t + 1 < it.t1 ? page_of(t + 1) : 0;
          const int n = (((it.keys(t) + 15) & ~15) + box - 1) / box;   // boxes with a key that there is, in steps of the product with V
          // places in the ring: K0, K1, V0, K2, V1, ..., V of the last
          const uint32_t pos = is_v ? (t + 1 < it.t1 || it.left > 0 ? 2 * g + 2 : 2 * g + 1) : g == 0 ? 0 : 2 * g - 1;
          const uint32_t st = pos % NS;
          ok = __all_sync(0xffffffffu, pos < NS || guard.wait<true>(&empty[st], ((pos / NS) & 1) ^ 1));
          if (!ok) break;
          if (lane == 0) {
            filled[st] = pos / NS + 1;
            mbar_expect_tx(&full[st], n * box * D * 2);
          }
          __syncwarp();
          if (sl < D / 64 && j < n)
            tma_load_3d(smem + SM::kRingOff + st * SM::kTileBytes + sl * (kKeys * 128) + j * box * 128, map, &full[st], 0,
                        (t * kKeys + j * box) & in_page, (page * p.Hkv + it.kvh) * (D / 64) + sl);
          page = next;
        }
      }
    } else if (warp == W0 + 1 && !idle && elect_one()) {
      // ------------------------------------------------------------------ products
      constexpr uint32_t idesc_s = make_idesc_bf16(kRows, kKeys);
      constexpr uint32_t idesc_pv = make_idesc_bf16(kRows, D) | (1u << 16);
      uint32_t pos = 0, g = 0;                             // place in the ring, tile
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { return guard.wait<true>(bar, parity); };
      // S in buffer s_buf from the queries in buffer q_buf and the tile in stage st
      uint32_t own0 = 0, own1 = 0, own_pv0 = 0, own_pv1 = 0;   // tiles of either warpgroup whose S, whose P V has been issued
      auto issue_s = [&](uint32_t s_buf, uint32_t q_buf, uint32_t st) {
        const uint32_t q_addr = smem_u32(smem + q_buf * SM::kQBytes), k_addr = smem_u32(smem + SM::kRingOff + st * SM::kTileBytes);
        const uint32_t d_tmem = tmem + s_buf * kKeys;
#pragma unroll
        for (int kd = 0; kd < D / 64; ++kd) {
          const uint64_t da = make_sw128_kmajor_desc(q_addr + kd * (kRows * 128)), db = make_sw128_kmajor_desc(k_addr + kd * (kKeys * 128));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_bf16<1>(d_tmem, da + kk * 2, db + kk * 2, idesc_s, (kd | kk) != 0);
        }
        uint32_t& own = q_buf == 0 ? own0 : own1;          // the queries' buffer goes with the warpgroup
        umma_commit(&s_full[2 * q_buf + (WIDE ? 0 : own & 1)]);
        ++own;
      };
      // P in buffer s_buf times the tile in stage st, added to O in o_buf: the steps of 16 keys that there are
      auto issue_pv = [&](uint32_t s_buf, uint32_t o_buf, uint32_t st, int keys, uint32_t acc) {
        const uint64_t dv = mn_major_desc(smem_u32(smem + SM::kRingOff + st * SM::kTileBytes));
        const uint32_t o_tmem = tmem + SM::kTmemO + o_buf * D, p_tmem = tmem + s_buf * kKeys;
        if (keys == kKeys) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk) umma_ts(o_tmem, p_tmem + p_column(kk), dv + static_cast<uint64_t>(kk) * (2048 >> 4), idesc_pv, kk != 0 ? 1u : acc);
        } else {
#pragma unroll 1
          for (int kk = 0; kk < (keys + 15) / 16; ++kk)
            umma_ts(o_tmem, p_tmem + p_column(kk), dv + static_cast<uint64_t>(kk) * (2048 >> 4), idesc_pv, kk != 0 ? 1u : acc);
        }
        uint32_t& own = o_buf == 0 ? own_pv0 : own_pv1;
        umma_commit(&pv_full[2 * o_buf + (WIDE ? 0 : own & 1)]);
        ++own;
      };
      if constexpr (WIDE) {
        uint32_t seen0 = 0, seen1 = 0, items1 = 0;           // tiles of each half so far; items that had a second half
        for (uint32_t item = 0; ok && it.next(); ++item) {
          const int halves = it.block_rows() > p.half_rows ? 2 : 1;
          if (item == 0) ok = guard.first(&q_full[0]);
          ok = ok && wait(&q_full[0], item & 1);
          uint32_t k_pos = g == 0 ? 0 : 2 * g - 1;
          ok = ok && wait(&full[k_pos % NS], (k_pos / NS) & 1);
          if (!ok) break;
          tc_fence_after();
          for (int h = 0; h < halves; ++h) issue_s(h, h, k_pos % NS);
          umma_commit(&empty[k_pos % NS]);
          if (it.t0 + 1 == it.t1) umma_commit(&q_free[0]);
          for (int t = it.t0; ok && t < it.t1; ++t, ++g) {
            const bool more = t + 1 < it.t1;
            const uint32_t v_pos = more || it.left > 0 ? 2 * g + 2 : 2 * g + 1;
            k_pos = 2 * g + 1;
            if (more) ok = wait(&full[k_pos % NS], (k_pos / NS) & 1);
            ok = ok && wait(&full[v_pos % NS], (v_pos / NS) & 1);
            for (int h = 0; h < halves && ok; ++h) {
              uint32_t& seen = h == 0 ? seen0 : seen1;
              // O of this half's item before has been read
              if (t == it.t0) ok = h == 0 ? item == 0 || wait(&o_free[0], (item & 1) ^ 1) : items1 == 0 || wait(&o_free[1], (items1 & 1) ^ 1);
              ok = ok && wait(&p_full[h], seen & 1);
              if (!ok) break;
              tc_fence_after();
              issue_pv(h, h, v_pos % NS, it.keys(t), t == it.t0 ? 0u : 1u);
              if (more) issue_s(h, h, k_pos % NS);
              ++seen;
            }
            if (!ok) break;
            umma_commit(&empty[v_pos % NS]);
            if (more) umma_commit(&empty[k_pos % NS]);
            if (t + 2 == it.t1) umma_commit(&q_free[0]);
          }
          items1 += halves == 2;
        }
      } else {
      // S of tile `tile_no`, from the queries in buffer `buf`
      auto scores = [&](uint32_t tile_no, uint32_t buf, bool last) {
        const uint32_t st = pos % NS;
        ok = wait(&full[st], (pos / NS) & 1);
        if (!ok) return;
        tc_fence_after();
        issue_s(tile_no & 1, buf, st);
        umma_commit(&empty[st]);
        if (last) umma_commit(&q_free[buf]);
        ++pos;
      };
      bool have = it.next();                               // the tile whose P V is to come: of item `now`, with `keys` keys
      ok = have && guard.first(&q_full[0]) && guard.wait<true>(&q_full[0], 0);
      int t = it.t0;
      if (ok) scores(0, 0, t + 1 == it.t1);
      uint32_t now = 0;
      while (ok) {
        const int keys = it.keys(t);
        const bool first_tile = t == it.t0, last_tile = t + 1 == it.t1;
        // scores of the next tile
        bool more = true;
        uint32_t next = now;
        if (!last_tile) {
          ++t;
        } else {
          more = it.next();
          if (more) {
            t = it.t0;
            next = now + 1;
            ok = guard.wait<true>(&q_full[next & 1], (next >> 1) & 1);
            if (!ok) break;
          }
        }
        if (more) scores(g + 1, next & 1, t + 1 == it.t1);
        if (!ok) break;
        // P V of this one
        const uint32_t buf = now & 1, st = pos % NS;
        ok = guard.wait<true>(&full[st], (pos / NS) & 1) && guard.wait<true>(&p_full[g & 1], (g >> 1) & 1) &&
             (!first_tile || now < 2 || guard.wait<true>(&o_free[buf], ((now >> 1) & 1) ^ 1));
        if (!ok) break;
        tc_fence_after();
        issue_pv(g & 1, buf, st, keys, first_tile ? 0u : 1u);
        umma_commit(&empty[st]);
        ++pos;
        ++g;
        if (!more) break;
        now = next;
      }
      }
      umma_commit(mma_end);                                // nothing is in flight when the columns are given back
      guard.land(mma_end, 0);
    } else if (warp == W0 + 3 && lane == 0 && !idle) {
      // ------------------------------------------------------------------ queries: a box is a block's (a half's) nodes x heads, 64 columns
      uint32_t item = 0;
      for (; it.next(); ++item) {
        const uint32_t buf = WIDE ? 0 : item & 1;
        if (WIDE) {                                        // both buffers have this item's rows
          if (item >= 1 && !guard.wait<true>(&q_free[0], (item & 1) ^ 1)) break;
        } else if (item >= 2 && !guard.wait<true>(&q_free[buf], ((item >> 1) & 1) ^ 1)) {
          break;
        }
        const int copies = WIDE ? (it.block_rows() > p.half_rows ? 2 : 1) : REP, nodes = p.half_rows / p.G;
        const int node = it.first + it.blk * (p.block_rows / p.G);
        mbar_expect_tx(&q_full[buf], copies * p.half_rows * D * 2);
        for (int i = 0; i < copies; ++i)
          for (int sl = 0; sl < D / 64; ++sl)
            tma_load_3d(smem + (WIDE ? i : buf) * SM::kQBytes + sl * (kRows * 128) + (WIDE ? 0 : i * BR * 128), &tmap_q, &q_full[buf], sl * 64,
                        it.kvh * p.G, node + (WIDE ? i * nodes : 0));
      }
      // the last copies land, whichever role gave up (after a wait that did not, they have)
      for (uint32_t i = WIDE ? (item >= 1 ? item - 1 : 0) : (item >= 2 ? item - 2 : 0); i < item; ++i)
        guard.land(&q_full[WIDE ? 0 : i & 1], (WIDE ? i : i >> 1) & 1);
    }
  } else {
    // ------------------------------------------------------------------ softmax
    const int wg = threadIdx.x / kGroup, tl = threadIdx.x & 127;   // TMEM lane
    const int row = WIDE ? wg * p.half_rows + tl : tl % BR, part = PAIR ? (warp >> 2) & 1 : kLanes == 1 ? 0 : (warp & 3) / (4 / kLanes);
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t g = 0, mine = 0;                              // tile of the CTA, of this warpgroup
    bool cut_tail = false;
    // A wait that gives up leaves the warps in step: they go on with what is there, and every later wait ends at once
    auto await = [&](uint64_t* bar, uint32_t parity) {
      guard.wait<true>(bar, parity);
      __syncwarp();
      tc_fence_after();
    };
    // P V of the warpgroup's tile k. A wait tells a phase from the next one only: tile k + 2 needs this warpgroup's P, and S of tile k + 1, or of
    // tile k itself, which it has, was formed behind P V of tile k - 2 (WIDE: k - 1), the phase before.
    auto await_pv = [&](uint32_t k) {
      if (WIDE) await(&pv_full[2 * wg], k & 1);
      else await(&pv_full[2 * wg + (k & 1)], (k >> 1) & 1);
    };
    auto sync_group = [&] {
      if (wg == 0) asm volatile("bar.sync 1, %0;" ::"n"(kGroup) : "memory");
      else asm volatile("bar.sync 2, %0;" ::"n"(kGroup) : "memory");
    };
    // WIDE, the first half: the second one has done with the items before this one. Its barrier is in the phase of the last of them that it had a
    // part in, or in the next: for more it needs this half's P.
    uint32_t halves2 = 0;                                  // items before this one that have a second half
    auto wait_second = [&] {
      if (halves2 > 0) guard.wait<true>(&o_free[1], (halves2 & 1) ^ 1);
    };
    // PAIR: the two warps that have a row between them
    auto sync_pair = [&] { asm volatile("bar.sync %0, 64;" ::"r"(3 + wg * 4 + (warp & 3)) : "memory"); };
    for (uint32_t item = 0; it.next(); ++item) {
      const bool cut = it.t0 > 0 || it.t1 < it.tiles;
      if (it.t0 == 0 && it.t1 < it.tiles) cut_tail = true; // the last item, if any
      const int rows = it.block_rows();
      const bool row_ok = row < rows && (!WIDE || tl < p.half_rows), warp_ok = row - lane < rows && (!WIDE || tl - lane < p.half_rows);
      const int at = it.blk * p.block_rows + row, node = at / p.G, head = it.kvh * p.G + at - node * p.G;
      const int64_t tok = it.first + (row_ok ? node : 0);
      const unsigned long long word_all = row_ok ? static_cast<unsigned long long>(p.seen[tok]) : 0ull;   // first used where nodes are
      const int placed = it.len - it.ctx;                  // nodes behind the table's end have no place: nobody sees them
      const unsigned long long nodes = placed < kNodes ? (1ull << placed) - 1 : ~0ull;
      unsigned long long* bad_here = bad_nodes + (item & 3);
      const uint32_t t_o = tmem + SM::kTmemO + wg * D + lane_base;
      if (WIDE ? wg * p.half_rows >= rows : (item & 1) != static_cast<uint32_t>(wg)) {   // no second half; the other's
        g += it.t1 - it.t0;
        continue;
      }
      float m_run = -INFINITY, l_run = 0.f;                // reference of the exponents, their sum
      for (int t = it.t0; t < it.t1; ++t, ++g) {
        const int key0 = t * kKeys;
        const uint32_t s_buf = WIDE ? wg : g & 1, t_s = tmem + s_buf * kKeys + lane_base;
        if (WIDE) await(&s_full[2 * wg], mine & 1);
        else await(&s_full[2 * wg + (mine & 1)], (mine >> 1) & 1);
        const bool behind = key0 + kKeys > it.ctx;         // the tile has nodes, or ends behind the last key
        float mx = -INFINITY;
        // 32 scores at a time in loops that are not unrolled: the warps are at different places of the code, and what is not in the instruction
        // caches costs some five cycles an instruction (and a row of 128 in registers spills)
        float f[32];
        auto load = [&](int c) {
          tmem_ld_32x32(t_s + (part * kChunks + c) * 32, reinterpret_cast<uint32_t(&)[32]>(f));
          tmem_ld_wait();
        };
        if (warp_ok) {
#pragma unroll 1
          for (int c = 0; c < kChunks; ++c) {
            load(c);
            if (behind) {
              // bits of these keys: all of the context, then the row's word from its first node on
              const unsigned long long word = word_all & nodes;
              const int j0 = key0 + (part * kChunks + c) * 32 - it.ctx;   // node of the first of 32 keys
              const uint32_t bits = j0 >= 64 ? 0u
                                    : j0 >= 0 ? static_cast<uint32_t>(word >> j0)
                                    : j0 <= -32 ? 0xffffffffu : (static_cast<uint32_t>(word << -j0) | ((1u << -j0) - 1u));
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((bits >> e) & 1u)) f[e] = -INFINITY;
              if (c + 1 < kChunks) {                       // read once more below
                tmem_store16(t_s + (part * kChunks + c) * 32, *reinterpret_cast<uint32_t(*)[16]>(f));
                tmem_store16(t_s + (part * kChunks + c) * 32 + 16, *reinterpret_cast<uint32_t(*)[16]>(f + 16));
              }
            }
            float m4[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
#pragma unroll
              for (int i = 0; i < 4; ++i) m4[i] = fmaxf(m4[i], fmaxf(f[e + i], f[e + 4 + i]));
            }
            mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          }
          if (kChunks > 1 && behind) tmem_store_wait();
          if constexpr (PAIR) {
            // The item's maximum so far, of both warps. Neither may add the next tile's before the other has read it. WIDE: S of the next tile is
            // formed behind both's P. Else it may be there already, and they meet once more.
            if (!WIDE && t > it.t0) sync_pair();
            atomicMax(&row_max[wg * kRows + tl], ordered(__float_as_int(mx)));
            sync_pair();
            mx = __int_as_float(ordered(*static_cast<volatile int*>(&row_max[wg * kRows + tl])));
          }
          mx *= p.scale_log2;
          float alpha = 1.f;
          if (mx > m_run + kLazy) {
            alpha = ex2(m_run - mx);
            m_run = mx;
            l_run *= alpha;
          }
          if (t > it.t0 && __any_sync(0xffffffffu, alpha != 1.f)) {
            // O is free when the product of the warpgroup's tile before has ended (WIDE: S of this tile was formed behind it)
            if (!WIDE) await_pv(mine - 1);
#pragma unroll 1
            for (int c = PAIR ? part * (D / 2) : 0; c < (PAIR ? (part + 1) * (D / 2) : D); c += 16) {
              uint32_t v[16];
              tmem_ld_32x16(t_o + c, v);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha);
              tmem_store16(t_o + c, v);
            }
          }
          const float m_use = m_run == -INFINITY ? 0.f : m_run;
          const uint64_t sc2 = pair(p.scale_log2, p.scale_log2), nm2 = pair(-m_use, -m_use);
          uint64_t sum2[2] = {0, 0};
#pragma unroll 1
          for (int c = kChunks - 1; c >= 0; --c) {         // 32 keys: 16 columns of P over their scores; the last ones are still there
            if (c + 1 < kChunks) load(c);
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 x = unpair(fma_pair(pair(f[2 * e], f[2 * e + 1]), sc2, nm2));
              const float2 y = make_float2(ex2(x.x), ex2(x.y));
              sum2[e & 1] = add_pair(sum2[e & 1], pair(y.x, y.y));
              pk[e] = pack_bf16(y.x, y.y);                 // probabilities enter the product in bf16, the sum in fp32
            }
            tmem_store16(t_s + (part * kChunks + c) * 32, pk);
          }
          if (kLanes > 1) {                                // the keys that other lanes have of this row
            uint32_t none[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) none[e] = 0u;
#pragma unroll
            for (int c = 0; c < kKeys / 32; ++c)
              if (c / kChunks != part) tmem_store16(t_s + c * 32, none);
          }
          const float2 sa = unpair(add_pair(sum2[0], sum2[1]));
          l_run += sa.x + sa.y;
          tmem_store_wait();
        }
        if (WIDE && threadIdx.x == 0 && t == it.t0 && *static_cast<volatile unsigned long long*>(bad_nodes + ((item + 1) & 3)) != 0ull) {
          wait_second();                                   // the next item's word was that of the item three before
          bad_nodes[(item + 1) & 3] = 0ull;
        }
        if (behind && (!WIDE || wg == 0)) {                // (WIDE: the first half's product comes first)
          // Values that nobody sees, or not every row, are finite before the product reads them
          const uint32_t vp = (t + 1 < it.t1 || it.left > 0) ? 2 * g + 2 : 2 * g + 1, st = vp % NS;    // where V of tile g is in the ring
          await(&full[st], (vp / NS) & 1);
          uint8_t* tile = smem + SM::kRingOff + st * SM::kTileBytes;
          const int lo = max(it.ctx - key0, 0), hi = it.keys(t), end = min((hi + 15) & ~15, kKeys);
          for (int e = lo * (D / 8) + (threadIdx.x & (kGroup - 1)); e < end * (D / 8); e += kGroup) {
            const int r = e / (D / 8), c = e % (D / 8);
            uint4* w = reinterpret_cast<uint4*>(tile + (c >> 3) * (kKeys * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
            if (r >= hi) {
              *w = make_uint4(0, 0, 0, 0);
              continue;
            }
            uint4 x = *w;
            uint32_t* u = reinterpret_cast<uint32_t*>(&x);
            bool bad = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t b = ((u[i] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((u[i] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
              if (b != 0u) { u[i] &= ~b; bad = true; }
            }
            if (bad) {
              *w = x;
              if (WIDE) wait_second();                     // the word was that of the item four before
              atomicOr(bad_here, 1ull << (key0 + r - it.ctx));
            }
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();                                 // P and the rescaled O are in TMEM, S has been read
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[s_buf]);
        ++mine;
      }
      // ---- results; the other warpgroup has the next item meanwhile
      await_pv(mine - 1);
      // The word of the item after the next is free: it was that of the group's item before, whose results all of it has
      if (!WIDE && tl == 0 && (!PAIR || part == 0)) bad_nodes[(item + 2) & 3] = 0ull;
      // Lanes that have a row's keys between them: maximum and sum of all, this lane's weight
      float2* lanes = reinterpret_cast<float2*>(smem + (item & 1) * SM::kQBytes);    // the item's queries have been read
      if (kLanes > 1) lanes[tl] = make_float2(m_run, l_run);
      sync_group();                                        // and bad_here of all four warps
      if constexpr (PAIR) {                                // the row's sum, by way of its maximum's place
        volatile float* place = reinterpret_cast<volatile float*>(&row_max[wg * kRows + tl]);
        if (part == 0) *place = l_run;
        sync_pair();
        if (part == 1) *place = l_run += *place;
        sync_pair();
        if (part == 0) {
          l_run = *place;
          *reinterpret_cast<volatile int*>(place) = kNoScore;
        }
        sync_pair();
      }
      float weight = 1.f;
      if (kLanes > 1) {
        float2 o[kLanes];
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
          o[i] = lanes[i * BR + row];
          top = fmaxf(top, o[i].x);
        }
        if (top != -INFINITY) {
#pragma unroll
          for (int i = 0; i < kLanes; ++i) sum += o[i].y * ex2(o[i].x - top);
          weight = ex2(m_run - top);
        }
        m_run = top;
        l_run = sum;
      }
      const unsigned long long bad = *static_cast<volatile unsigned long long*>(bad_here) & word_all & nodes;
      {
        const float inv = weight * (cut ? 1.f : l_run > 0.f ? __frcp_rn(l_run) : 0.f);
        const int slot = 2 * blockIdx.x + (it.t0 == 0 ? 1 : 0);
        __nv_bfloat16* op = p.out + (tok * p.Hq + head) * D;
        constexpr int kPartRows = WIDE ? 2 * kRows : kRows;
        float4* po = p.part_o + static_cast<size_t>(slot) * (D / 4) * kPartRows + row;
        // F finished columns from column c on
        auto put = [&](int c, auto& x) {
          constexpr int F = sizeof(x) / sizeof(float);
          for (unsigned long long b = bad; b != 0ull; b &= b - 1) {   // seen values that are no numbers
            const int place = it.ctx + __ffsll(static_cast<long long>(b)) - 1;
            const int64_t page = p.table[it.s * p.table_ld + min(place >> p.page_shift, p.table_width - 1)];
            if (page < 0 || page >= p.pages) continue;
            const __nv_bfloat16* vr =
                p.v + ((((page * p.Hkv + it.kvh) * (D / 64) + c / 64) << p.page_shift) + (place & ((1 << p.page_shift) - 1))) * 64 + c % 64;
#pragma unroll
            for (int e = 0; e < F; ++e) {
              const float y = __bfloat162float(vr[e]);
              if (!(fabsf(y) < INFINITY)) x[e] += y;
            }
          }
          if (!row_ok) return;
          if (cut) {
#pragma unroll
            for (int e = 0; e < F / 4; ++e) po[(c / 4 + e) * kPartRows] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
          } else {
#pragma unroll
            for (int e = 0; e < F / 8; ++e) {
              uint4 w;
              w.x = pack_bf16(x[8 * e], x[8 * e + 1]);
              w.y = pack_bf16(x[8 * e + 2], x[8 * e + 3]);
              w.z = pack_bf16(x[8 * e + 4], x[8 * e + 5]);
              w.w = pack_bf16(x[8 * e + 6], x[8 * e + 7]);
              *reinterpret_cast<uint4*>(op + c + e * 8) = w;
            }
          }
        };
        if constexpr (kLanes == 1) {
          if (warp_ok) {
#pragma unroll 1
            for (int c = part * (D / 2); c < (part + 1) * (D / 2); c += 32) {
              float x[32];
              tmem_ld_32x32(t_o + c, reinterpret_cast<uint32_t(&)[32]>(x));
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] *= inv;
              put(c, x);
              __syncwarp();
            }
          }
        } else {
          // A row's lanes hand each other, by way of the item's query buffer, what they have of the columns that the other one finishes: F columns
          // a lane, half of all columns at a time
          constexpr int F = D / 2 / REP;
          float4* stage = reinterpret_cast<float4*>(smem + (item & 1) * SM::kQBytes + kRows * 8);   // [part][its sources][F / 4][row]
          static_assert(REP * (REP - 1) * F * 4 * BR + kRows * 8 <= SM::kQBytes, "lanes' results fit in a query buffer");
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += D / 2) {
            float own[F];
            if (warp_ok) {
              uint32_t v[D / 64][32];
#pragma unroll
              for (int c = 0; c < D / 64; ++c) tmem_ld_32x32(t_o + c0 + c * 32, v[c]);
              tmem_ld_wait();
#pragma unroll
              for (int to = 0; to < REP; ++to) {
                float x[F];
#pragma unroll
                for (int e = 0; e < F; ++e) x[e] = __uint_as_float(v[(to * F + e) / 32][(to * F + e) % 32]) * inv;
                if (to == part) {
#pragma unroll
                  for (int e = 0; e < F; ++e) own[e] = x[e];
                } else {
                  float4* at = stage + (to * (REP - 1) + (part < to ? part : part - 1)) * (F / 4) * BR + row;
#pragma unroll
                  for (int e = 0; e < F / 4; ++e) at[e * BR] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
                }
              }
            }
            fence_proxy_async_smem();                      // the next queries are copied into this buffer
            sync_group();
            if (warp_ok) {
#pragma unroll
              for (int i = 0; i < REP - 1; ++i) {
                const float4* at = stage + (part * (REP - 1) + i) * (F / 4) * BR + row;
#pragma unroll
                for (int e = 0; e < F / 4; ++e) {
                  const float4 y = at[e * BR];
                  own[4 * e] += y.x; own[4 * e + 1] += y.y; own[4 * e + 2] += y.z; own[4 * e + 3] += y.w;
                }
              }
              put(c0 + part * F, own);
              __syncwarp();
            }
            sync_group();
          }
        }
        tc_fence_before();                                 // O has been read
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[wg]);
        if (kLanes > 1 && tl == 0) mbar_arrive(&q_free[item & 1]);
      }
      if (WIDE) halves2 += rows > p.half_rows;
      if (warp_ok && part == 0) {
        const int slot = 2 * blockIdx.x + (it.t0 == 0 ? 1 : 0);
        if (cut && row_ok) p.part_ml[static_cast<size_t>(slot) * (WIDE ? 2 * kRows : kRows) + row] = make_float2(m_run, l_run);
        if (cut && it.t0 == 0 && row == 0) {
          // CTAs before the one whose share ends at the unit's end or behind it
          const int64_t all = begin[3], ctas = min(static_cast<int64_t>(gridDim.x), all);
          const int64_t end = all * (blockIdx.x + 1) / ctas + (it.tiles - it.t1);
          const int last = static_cast<int>((end * ctas + all - 1) / all) - 1;
          p.cut[2 * blockIdx.x] = make_int4(last, it.first, it.kvh, it.blk);
          p.cut[2 * blockIdx.x + 1] = make_int4(rows, 0, 0, 0);
        }
      }
    }
    if (threadIdx.x == 0 && !cut_tail && !p.whole) p.cut[2 * blockIdx.x] = make_int4(-1, 0, 0, 0);   // no unit begins here that ends elsewhere
  }
  tc_fence_before();
  __syncthreads();
  // copies that nobody waited for, because a wait gave up, land before the CTA ends
  if (threadIdx.x < NS && guard.gave_up() && filled[threadIdx.x] != 0) guard.land(&full[threadIdx.x], (filled[threadIdx.x] - 1) & 1);
  if (warp == W0 + 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc<1>(tmem, SM::kTmemCols);
  }
}

// Joins the parts of the unit that CTA blockIdx.x begins and CTA `last` ends: 32 rows a block, a lane each. A warp has 32 columns and every
// second part (fourth, with heads of 64), two of them on their way at a time, in order; the warps' results are joined in order. Latency bounds
// it: few parts and many units (256 rows, two parts) want few blocks, many parts (16 units of ten) few waits one after the other.
static constexpr int kJoinWarps = 8;
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) draft_join_kernel(const DraftAttnParams p) {
  constexpr int kColumns = D / 32, kSub = kJoinWarps / kColumns;      // warps beside and behind one another
  __shared__ float sm[kSub][kColumns][32], sl[kSub][kColumns][32];
  __shared__ float4 so[kSub - 1][kColumns][8][32];
  griddep_wait();
  const int cta = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.y * 32 + lane;
  const int column = warp % kColumns, sub = warp / kColumns;
  const int4 c0 = p.cut[2 * cta], c1 = p.cut[2 * cta + 1];
  const int last = c0.x, rows = c1.x;
  if (last <= cta || last >= static_cast<int>(gridDim.x) || static_cast<int>(blockIdx.y) * 32 >= rows) return;
  const bool ok = row < rows;
  float m = -INFINITY, l = 0.f;
  float4 o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto slot = [&](int c) { return static_cast<size_t>(2 * c + (c == cta ? 1 : 0)); };
  auto load = [&](int c, float2& ml, float4 (&x)[8]) {
    ml = p.part_ml[slot(c) * p.part_rows + row];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p.part_o[(slot(c) * (D / 4) + column * 8 + i) * p.part_rows + row];
  };
  auto add = [&](const float2& ml, const float4 (&x)[8]) {
    const float top = fmaxf(m, ml.x), use = top == -INFINITY ? 0.f : top, a = ex2(m - use), w = ex2(ml.x - use);
    m = top;
    l = l * a + ml.y * w;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i].x = o[i].x * a + x[i].x * w; o[i].y = o[i].y * a + x[i].y * w;
      o[i].z = o[i].z * a + x[i].z * w; o[i].w = o[i].w * a + x[i].w * w;
    }
  };
  for (int c = cta + sub; c <= last && ok; c += 2 * kSub) {
    float2 ml[2];
    float4 x[2][8];
    const bool more = c + kSub <= last;
    load(c, ml[0], x[0]);
    if (more) load(c + kSub, ml[1], x[1]);
    add(ml[0], x[0]);
    if (more) add(ml[1], x[1]);
  }
  if (sub > 0) {
    sm[sub][column][lane] = m;
    sl[sub][column][lane] = l;
#pragma unroll
    for (int i = 0; i < 8; ++i) so[sub - 1][column][i][lane] = o[i];
  }
  __syncthreads();
  if (!ok || sub > 0) return;
  for (int w = 1; w < kSub && cta + w <= last; ++w) {
    float4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = so[w - 1][column][i][lane];
    add(make_float2(sm[w][column][lane], sl[w][column][lane]), x);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int at = c0.w * p.block_rows + row, node = at / p.G, head = c0.z * p.G + at - node * p.G;
  __nv_bfloat16* op = p.out + (static_cast<int64_t>(c0.y + node) * p.Hq + head) * D + column * 32;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 w;
    w.x = pack_bf16(o[2 * i].x * inv, o[2 * i].y * inv);
    w.y = pack_bf16(o[2 * i].z * inv, o[2 * i].w * inv);
    w.z = pack_bf16(o[2 * i + 1].x * inv, o[2 * i + 1].y * inv);
    w.w = pack_bf16(o[2 * i + 1].z * inv, o[2 * i + 1].w * inv);
    *reinterpret_cast<uint4*>(op + i * 8) = w;
  }
}

// boxes of one 64-wide slab of a page ([page][64], at most 64 rows)
static int page_tmap(const void* base, int64_t pages, int Hkv, int D, int page_size, CUtensorMap* out) {
  const cuuint64_t dims[3] = {64, static_cast<cuuint64_t>(page_size), static_cast<cuuint64_t>(pages * Hkv * (D / 64))};
  const cuuint64_t strides[2] = {128, static_cast<cuuint64_t>(page_size) * 128};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(page_size < 64 ? page_size : 64), 1}, estr[3] = {1, 1, 1};
  const CUresult r = get_encode_fn()(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    fprintf(stderr, "[gllm_b200] cache tensor-map encode failed (%d)\n", static_cast<int>(r));
    return 1;
  }
  return 0;
}

template <int D, int REP>
static int launch_draft_attention(const CUtensorMap& tk, const CUtensorMap& tv, DraftAttnParams p, int ctas, int max_rows, cudaStream_t st) {
  using SM = DraftSmem<D>;
  static PerDeviceOnce configured;
  if (configured.need()) {
    CUDA_CHECK_RET(cudaFuncSetAttribute(draft_attention_kernel<D, REP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::kBytes));
    configured.done();
  }
  constexpr int most = kRows / (REP == 0 ? 1 : REP);
  const int nodes = most / p.G;                            // of a box
  p.half_rows = nodes * p.G;
  p.block_rows = REP == 0 ? 2 * p.half_rows : p.half_rows;
  p.part_rows = part_rows_of(max_rows);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + static_cast<size_t>(2) * ctas * (D / 4) * p.part_rows);
  p.cut = reinterpret_cast<int4*>(p.part_ml + static_cast<size_t>(2) * ctas * p.part_rows);
  CUtensorMap tq;                                          // queries [row][head][D]
  const cuuint64_t dims[3] = {D, static_cast<cuuint64_t>(p.Hq), static_cast<cuuint64_t>(p.rows)};
  const cuuint64_t strides[2] = {D * 2, static_cast<cuuint64_t>(p.q_ts) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.G), static_cast<cuuint32_t>(nodes)}, estr[3] = {1, 1, 1};
  const CUresult r = get_encode_fn()(&tq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(p.q), dims, strides, box, estr,
                                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    fprintf(stderr, "[gllm_b200] query tensor-map encode failed (%d)\n", static_cast<int>(r));
    return 1;
  }
  CUDA_CHECK_RET(launch_pdl(draft_attention_kernel<D, REP>, dim3(ctas), dim3(cta_threads(REP)), SM::kBytes, st, tk, tv, tq, p));
  if (p.whole) return 0;
  CUDA_CHECK_RET(launch_pdl(draft_join_kernel<D>, dim3(ctas, (p.block_rows + 31) / 32), dim3(kJoinWarps * 32), 0, st, p));
  return 0;
}

}  // namespace b200

using namespace b200;

// bytes of scratch for a launch of `ctas` CTAs over sequences of at most max_rows rows (nodes x query heads a kv head)
GLLM_EXPORT int64_t gllm_draft_attention_scratch(int D, int max_rows, int ctas) {
  return static_cast<int64_t>(ctas) * (2 * part_rows_of(max_rows) * (D * 4 + 8) + 32);
}

GLLM_EXPORT int gllm_draft_attention(const void* q, int64_t q_ts, void* out, const void* k_cache, const void* v_cache, int64_t pages,
                                     const void* table, int64_t table_ld, int table_width, const void* seq_lens, const void* q_start,
                                     const void* seen, int num_seqs, int rows, int max_nodes, int whole, int Hq, int Hkv, int D,
                                     int page_size, float scale, int ctas, void* scratch, int64_t scratch_bytes, void* stream) {
  if (num_seqs <= 0 || rows <= 0 || max_nodes <= 0) return 0;
  if ((D != 64 && D != 128) || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > kRows || page_size < 8 || kKeys % page_size || (page_size & (page_size - 1)) || pages <= 0 || table_width <= 0 || ctas <= 0 ||
      q_ts % 8 || (reinterpret_cast<uintptr_t>(q) & 15))
    return 1;
  if (!whole && ((reinterpret_cast<uintptr_t>(scratch) & 15) || scratch_bytes < gllm_draft_attention_scratch(D, (max_nodes < kNodes ? max_nodes : kNodes) * (Hq / Hkv), ctas)))
    return 1;
  CUtensorMap tk, tv;
  if (page_tmap(k_cache, pages, Hkv, D, page_size, &tk) || page_tmap(v_cache, pages, Hkv, D, page_size, &tv)) return 1;
  DraftAttnParams p;
  p.q = reinterpret_cast<const __nv_bfloat16*>(q); p.q_ts = q_ts;
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  p.v = reinterpret_cast<const __nv_bfloat16*>(v_cache);
  p.pages = pages;
  p.table = reinterpret_cast<const int32_t*>(table); p.table_ld = table_ld; p.table_width = table_width;
  p.seq_lens = reinterpret_cast<const int32_t*>(seq_lens);
  p.q_start = reinterpret_cast<const int32_t*>(q_start);
  p.seen = reinterpret_cast<const int64_t*>(seen);
  p.num_seqs = num_seqs; p.rows = rows; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv;
  p.page_shift = 31 - __builtin_clz(static_cast<unsigned>(page_size));
  p.scale_log2 = scale * 1.4426950408889634f;
  p.whole = whole;
  p.part_o = reinterpret_cast<float4*>(scratch);
  p.part_ml = nullptr;
  p.cut = nullptr;
  p.waits = g_wait_config;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // Rows that a sequence may have decide how many lanes share a row (a sequence with more has more blocks)
  const int max_rows = (max_nodes < kNodes ? max_nodes : kNodes) * p.G;
#define GLLM_DRAFT(REP) \
  (D == 128 ? launch_draft_attention<128, REP>(tk, tv, p, ctas, max_rows, st) : launch_draft_attention<64, REP>(tk, tv, p, ctas, max_rows, st))
  return max_rows <= 32 ? GLLM_DRAFT(4) : max_rows <= 64 ? GLLM_DRAFT(2) : max_rows <= kRows ? GLLM_DRAFT(1) : GLLM_DRAFT(0);
#undef GLLM_DRAFT
}
