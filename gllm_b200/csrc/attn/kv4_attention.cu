// Attention of decoding sequences over a paged cache held in 4 bits, and such a cache expanded to bf16 tiles for prompts.
//
// The cache (ops/kv4.py): per page and kv head blocks of 16 tokens, 16 rows of D / 2 bytes and 16 x D / 64 pairs (scale, low); a
// code c of a group stands for c scale + low. With the groups g of a head's dims, key j and query row r
//   score  = sum_g scale_jg (q_rg . c_jg) + low_jg sum(q_rg)
//   output = sum_j p_j (c'_jg scale'_jg + low'_jg) = sum_j (p_j scale'_jg) c'_jg + sum_j p_j low'_jg
// so the codes go into the matrix instructions as they are and scales and low ends stay outside: four fused operations a score, two a
// probability, instead of one or two for each of the D values of a key.
//
// Codes as 16-bit operands: the lower half of a byte of two codes is the fp16 subnormal c0 2^-24, the upper one 16 c1 2^-24, both exact, and
// the matrix instructions take subnormals: four ANDs and a byte move for eight codes. A query's factor of c1 is divided by 16 (exact), sums of
// values by 16 at their end. Queries are scaled by a power of two to the upper end of fp16, so that their eight bits are exact down to 2^-28 of a
// head's largest. (The whole byte as c0's operand saves an instruction, but q0 c0 + q1 c1 = q0 (c0 + 16 c1) + (q1 / 16 - q0) 16 c1 rounds the
// second factor, which costs odd dims 2^-7 of their even neighbour's query.) Probabilities times scales are rounded to
// fp16 (2^-11 of each): the exponentials' reference is the head's maximum plus the logarithm of the largest scale met so far, so that
// they stay below 2^14, and what vanishes below 2^-25 is 2^-32 of the largest that can stand beside it.
//
// Keys are the rows of the products (m16n8k16: 16 keys x 8 query heads, then 16 dims x 8 heads), so eight query heads of
// one kv head fill an instruction. A lane (g, t) = (lane / 4, lane % 4) holds
//   codes of keys g, g + 8: 16 bytes (D = 128), the t-th quarter of the row: eight dims at a time of each group
//   codes of values: tokens 2t, 2t + 1, 2t + 8, 2t + 9, eight bytes each: eight dims of each group, chunk g
//   scores: keys g, g + 8 of heads 2t, 2t + 1; movmatrix turns the probabilities into the second product's operand
//
// A warp walks tiles of 32 keys by itself: it copies them (cp.async.bulk, one contiguous block of 9 D bytes for 16 tokens' keys or
// values) into its own ring, two tiles deep. The tiles of all sequences and heads lie in one row, which is cut into equal shares on the
// device, for CTAs and then for their warps: ragged batches, many short sequences and few long ones fill the machine alike. A head that
// lies in one warp's share is finished there; the warps of a CTA add their parts of others up at its end, once; what goes on in another
// CTA goes to scratch, and a second kernel joins it.
//
// The reference follows only when a score passes the head's maximum by 2^8 or a scale the largest one (one vote instead of shuffles).
//
// What bounds it: bytes beside the ALU. Four sequences of up to 60,000 tokens, 64 / 8 heads of 128: 191 MB in 47.2 us, join included (copies
// without arithmetic 38.7, of which some 9 are the start, uneven ends and the join). 616 warp instructions a tile of 32 keys, all counted: ALU 57 %,
// issue slots 57 %, tensor pipe 24 %. 64 sequences of up to 2500 (32 / 8): 40.4 us (copies 32.8); one of 700: 8.2 (6.9), latency. More than eight
// query heads of a kv head (two column tiles, 244 registers, eight warps an SM), 32 / 2 heads: 64 of up to 2500 26.0 us for 5.5 of bytes
// (bf16 cache 35.8), 8 of up to 32,000 30.6 for 8.2 (40.2), one of 700 11.7. Pages of 16 to 64: the same times. With operands that took one
// instruction less: two CTAs of eight warps an SM 47.8 for 45.5; without gain the base folded into the scores, 12 warps with 168 registers, larger
// shares for some CTAs; a join by the CTA that finds all parts there (flags behind fences) instead of a second launch 49.2, one of 700 9.9.
#include "../common/bounded.cuh"
#include "attn_common.cuh"

namespace b200 {

namespace {

constexpr int kV4Keys = 32, kV4Stages = 2, kV4Least = 8;      // tiles of a CTA's share, at least
constexpr int kV4Snap = 1;                               // tiles by which a cut moves to a head group's start or end (two: 256 x 75 16.5 for 18.5 us, all others longer, by up to 5 %)
constexpr uint32_t kEven = 0x000f000fu, kOdd = 0x00f000f0u;      // the two codes of bytes 0 and 2
constexpr float kV4Lazy = 8.f;                           // scores pass the maximum that the reference is taken from by no more than this
constexpr float kV4Room = 6.f;                           // and exponentials times scales stay below 2^(kV4Lazy + kV4Room)

struct Kv4Params {
  const __nv_bfloat16* q;
  int64_t q_ts;
  __nv_bfloat16* out;                                    // [B, Hq, D]
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  uint32_t last_page;
  const int32_t* block_table;
  const int32_t* seq_lens;
  int64_t pitch;                                         // between the rows of the block table, which has max_blocks columns
  int B, max_blocks, Hq, Hkv, G, GP;                     // GP query heads (at most 8 NT) of the G of a kv head at a time
  int page_blocks;                                       // blocks of 16 tokens in a page
  uint32_t page_magic;                                   // floor(b / page_blocks) = umulhi(b, page_magic), exact while b x page_blocks < 2^32 (0: one block)
  float scale_log2;
  float* part_o;                                         // [2 CTAs, 8 NT, D]
  float* part_ml;                                        // [2 CTAs, 8 NT, 2]
  int4* meta;                                            // [CTAs] (sequence, head group, last CTA, slot) of what starts here and goes on; sequence -1: nothing
  WaitConfig waits;
};

template <int D, int NT>
struct Kv4Smem {
  // As many warps as registers allow, in one CTA: of two CTAs on an SM the first had the better of the second (its warps were done after 32 us, the
  // other's after 37), where all of one get on alike.
  static constexpr int kV4Warps = NT == 1 ? 16 : 8, kV4Threads = kV4Warps * 32;
  static constexpr int kV4Lens = kV4Threads;             // lengths that a CTA keeps in shared memory, from its first sequence on
  static constexpr int kBlock = 9 * D;                   // 16 tokens' keys or values
  static constexpr int kStage = 4 * kBlock;
  static constexpr int kRing = kV4Warps * kV4Stages * kStage;
  static constexpr int kSums = kV4Warps * 32 * (D / 16 * 4 * NT) * 4;
  static_assert(kSums / kV4Warps <= kV4Stages * kStage, "a warp's last part takes its ring's place");
  static constexpr int kMl = 2 * kV4Warps * 8 * NT * 2 * 4;
  static constexpr int kBytes = kRing + kSums + kMl + kV4Lens * 4 + kV4Warps * (kV4Stages * 8 + 32) + 64;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void lds64(uint32_t addr, uint32_t& a, uint32_t& b) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr));
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t a;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(a) : "r"(addr));
  return a;
}
// d += a b, 16 x 8 x 16
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  return d;
}
__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// tiles of a sequence; one at least, so that a sequence of no keys gets its zeros
__device__ __forceinline__ int kv4_tiles(int len) { return max(1, (len + kV4Keys - 1) / kV4Keys); }

template <int D, int NT>
__global__ void __launch_bounds__(Kv4Smem<D, NT>::kV4Threads, 1) kv4_decode_kernel(const Kv4Params p) {
  using SM = Kv4Smem<D, NT>;
  constexpr int kV4Warps = SM::kV4Warps, kV4Threads = SM::kV4Threads, kV4Lens = SM::kV4Lens;
  constexpr int GR = D / 64;                             // groups of a head
  constexpr int KS = D / 16;                             // 16-dim steps of the first product, and dim tiles of the second
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kPieces = NT * GR * 4;                   // of a part: four sums a lane
  float4* firsts = reinterpret_cast<float4*>(smem + SM::kRing);                    // [warp][piece][lane]: parts that an earlier warp starts
  float* ml = reinterpret_cast<float*>(smem + SM::kRing + SM::kSums);              // [first or last][warp][head][base, l]
  int* lens = reinterpret_cast<int*>(smem + SM::kRing + SM::kSums + SM::kMl);
  uint64_t* bars = reinterpret_cast<uint64_t*>(lens + kV4Lens);
  int4* info = reinterpret_cast<int4*>(bars + kV4Warps * kV4Stages);               // [first or last][warp] (sequence or -1, head group, ends, last CTA)
  uint32_t* words = reinterpret_cast<uint32_t*>(info + 2 * kV4Warps);              // gave up, first sequence, its first tile
  const WaitGuard guard{words, p.waits};
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

  if (tid == 0) *guard.dead = 0;
  if (tid < kV4Warps * kV4Stages) mbar_init(&bars[tid], 1);
  fence_mbar_init();
  __syncthreads();
  griddep_launch();
  griddep_wait();

  // ---- this CTA's share [begin, end) of all tiles: sequence by sequence, head group by head group
  const int H = p.Hkv * (p.G / p.GP);
  __shared__ int scan[kV4Warps + 1];
  auto block_scan = [&](int v, int& total) {             // inclusive
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kV4Warps; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    return x + before;
  };
  int all = 0, mine_len = 0, mine_upto = 0, seq0, tiles0;      // all tiles of a head group, this CTA's first sequence and the tiles before it
  int64_t share, begin, end;
  auto cut = [&] {
    const int64_t work = static_cast<int64_t>(all) * H;
    share = max((work + gridDim.x - 1) / gridDim.x, static_cast<int64_t>(kV4Least));
    begin = share * blockIdx.x;
    end = min(begin + share, work);
  };
  if (tid == 0) p.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (p.B <= 64) {
    // few sequences: every warp for itself, without barriers (a lone sequence of 700: 8.6 -> 8.3 us)
    int len[2], n[2], upto[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      len[i] = lane + 32 * i < p.B ? p.seq_lens[lane + 32 * i] : 0;
      n[i] = lane + 32 * i < p.B ? kv4_tiles(len[i]) : 0;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      upto[i] = n[i];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto[i], o);
        if (lane >= o) upto[i] += y;
      }
      upto[i] += all;
      all = __shfl_sync(0xffffffffu, upto[i], 31);
    }
    cut();
    if (begin >= end) return;
    seq0 = tiles0 = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t here = __ballot_sync(0xffffffffu, begin >= static_cast<int64_t>(upto[i] - n[i]) * H && begin < static_cast<int64_t>(upto[i]) * H);
      if (here != 0) {
        const int from = __ffs(here) - 1;
        seq0 = 32 * i + from;
        tiles0 = __shfl_sync(0xffffffffu, upto[i] - n[i], from);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (lane + 32 * i >= seq0) lens[lane + 32 * i - seq0] = len[i];        // every warp the same
    __syncwarp();
  } else {
    // up to one sequence a thread, one pass has it all; beyond that the first counts, the second finds this CTA's
    for (int s0 = 0; s0 < p.B; s0 += kV4Threads) {
      int total;
      mine_len = s0 + tid < p.B ? p.seq_lens[s0 + tid] : 0;
      mine_upto = block_scan(s0 + tid < p.B ? kv4_tiles(mine_len) : 0, total);
      all += total;
    }
    cut();
    if (begin >= end) return;
    int base = 0;                                        // tiles of one head group before these sequences
    for (int s0 = 0; s0 < p.B; s0 += kV4Threads) {
      int total = 0;
      if (p.B > kV4Threads) mine_len = s0 + tid < p.B ? p.seq_lens[s0 + tid] : 0;
      const int n = s0 + tid < p.B ? kv4_tiles(mine_len) : 0;
      const int upto = (p.B > kV4Threads ? block_scan(n, total) : mine_upto) + base;
      if (begin >= static_cast<int64_t>(upto - n) * H && begin < static_cast<int64_t>(upto) * H) {
        words[1] = s0 + tid;
        words[2] = upto - n;
      }
      base += total;
    }
    __syncthreads();
    seq0 = words[1];
    tiles0 = words[2];
    if (p.B > kV4Threads) {
      for (int i = tid; i < kV4Lens; i += kV4Threads) lens[i] = seq0 + i < p.B ? p.seq_lens[seq0 + i] : 0;
    } else if (tid >= seq0) {
      lens[tid - seq0] = mine_len;                       // kV4Lens == kV4Threads
    }
    __syncthreads();
  }
  auto len_of = [&](int s) { return s - seq0 < kV4Lens ? lens[s - seq0] : p.seq_lens[s]; };

  const int first_in = static_cast<int>(begin - static_cast<int64_t>(tiles0) * H), tiles = static_cast<int>(end - begin);
  const int hg = p.G / p.GP;
  struct Place {                                         // a head group of a sequence
    int seq, head, len, n;
  } at;
  at.seq = seq0;
  at.len = len_of(seq0);
  at.n = kv4_tiles(at.len);
  at.head = first_in / at.n;
  int at_tile = first_in - at.head * at.n;               // the first tile of the segment that is worked on
  auto next_head = [&](Place& x) {                       // behind the last one: never used
    if (++x.head < H) return;
    x.head = 0;
    if (++x.seq >= p.B) return;
    x.len = len_of(x.seq);
    x.n = kv4_tiles(x.len);
  };

  auto settle = [&](Place& x, int& tile) {               // tile counted from x's first: into the head group that it lies in
    while (tile >= x.n && x.seq < p.B) {
      tile -= x.n;
      next_head(x);
    }
  };
  // This warp's part [my_begin, my_end) of the share.
  const int each = tiles / kV4Warps, over = tiles % kV4Warps;        // the first ones have one more: a warp without tiles has none behind it
  int my_begin = warp * each + min(warp, over), my_end = my_begin + each + (warp < over ? 1 : 0);
  at_tile += my_begin;
  settle(at, at_tile);
  // A cut that lies next to a head group's start or end moves there, where warps have two tiles and more: a part less (256 sequences of some 75:
  // 22.3 -> 18.6 us).
  const bool snap = share >= 2 * kV4Warps;
  auto moves = [&](int n, int tile) {
    return !snap ? 0 : tile <= kV4Snap && 2 * tile <= n ? -tile : n - tile <= kV4Snap ? n - tile : 0;
  };
  if (snap) {
    Place stop = at;
    int stop_tile = at_tile + (my_end - my_begin);
    settle(stop, stop_tile);
    if (stop.seq < p.B) my_end += moves(stop.n, stop_tile);
    if (at.seq < p.B) {
      const int by = moves(at.n, at_tile);
      my_begin += by;
      at_tile += by;
      settle(at, at_tile);
    }
  }
  const uint32_t my_tiles = static_cast<uint32_t>(my_end - my_begin);
  auto last_cta = [&](int64_t stop, int n) {             // the CTA that ends a head group of n tiles up to `stop`
    const int64_t cta = (stop - 1) / share;
    const int tile = n - static_cast<int>(stop - cta * share);         // where its share begins, from the group's start
    return static_cast<int>(tile > 0 && moves(n, tile) > 0 ? cta - 1 : cta);
  };
  if (lane < 2) info[lane * kV4Warps + warp] = make_int4(-1, 0, 0, 0);
  __syncwarp();

  // ---- copies. Eight of the warp's tiles are prepared at a time, a block a lane: tile lane / 4, keys or values, 16 tokens. A table entry
  // that is no page reads another one.
  const uint32_t ring = smem_u32(smem) + warp * (kV4Stages * SM::kStage);
  uint64_t* bar = bars + warp * kV4Stages;
  Place fetch = at;                                      // of this lane's next block
  int fetch_x = my_begin + (lane >> 2), fetch_tile = at_tile + (lane >> 2);
  const uint8_t* src = nullptr;
  int blocks = 0;                                        // of this lane's tile (none: an empty sequence)
  auto prepare = [&] {
    settle(fetch, fetch_tile);
    blocks = 0;
    if (fetch_x < my_end) {
      const int blk = 2 * fetch_tile + (lane & 1);
      blocks = min(2, (fetch.len - fetch_tile * kV4Keys + 15) / 16);
      if ((lane & 1) < blocks) {
        const int i = p.page_magic != 0 ? static_cast<int>(__umulhi(static_cast<uint32_t>(blk), p.page_magic)) : blk;
        const uint32_t page = min(static_cast<uint32_t>(p.block_table[fetch.seq * p.pitch + min(i, p.max_blocks - 1)]),
                                  p.last_page);
        src = (lane & 2 ? p.v_cache : p.k_cache) +
              ((static_cast<uint64_t>(page) * p.Hkv + fetch.head / hg) * p.page_blocks + (blk - i * p.page_blocks)) * SM::kBlock;
      }
    }
    fetch_x += 8;
    fetch_tile += 8;
  };
  uint32_t issued = 0, used = 0;
  auto issue = [&](int stage) {
    if ((issued & 7u) == 0) prepare();
    if (static_cast<uint32_t>(lane >> 2) == (issued & 7u)) {
      if ((lane & 3) == 0) {
        if (blocks > 0) mbar_expect_tx(&bar[stage], blocks * 2 * SM::kBlock);
        else mbar_arrive(&bar[stage]);
      }
      if ((lane & 1) < blocks) bulk_load(ring + stage * SM::kStage + (lane & 3) * SM::kBlock, src, SM::kBlock, &bar[stage]);
    }
    ++issued;
  };
#pragma unroll
  for (int s = 0; s < kV4Stages; ++s)
    if (issued < my_tiles) issue(s);

  // ---- segment by segment (the tiles of one head group of one sequence)
  bool ok = true;
  if (guard.cfg.limit_ns == 0) ok = __all_sync(0xffffffffu, my_tiles == 0 || guard.first(&bar[0]));
  int seg = my_begin;
  while (seg < my_end) {
    const int seg_end = min(my_end, seg + (at.n - at_tile));
    const int len = at.len;
    const int head0 = at.head / hg * p.G + at.head % hg * p.GP;
    const __nv_bfloat16* q = p.q + at.seq * p.q_ts + static_cast<int64_t>(head0) * D;

    // queries of heads 8 nt + g as operands; sums and factors of heads 8 nt + 2t, + 2t + 1
    uint32_t qf[NT][KS][2];
    float unscale[NT][2], qsum[NT][2][GR];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = 8 * nt + g;
      uint32_t raw[GR][2][4];                            // chunk 2t, 2t + 1 of each group, eight dims each
      float most = 0.f, sum[GR];
#pragma unroll
      for (int gr = 0; gr < GR; ++gr) {
        sum[gr] = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (h < p.GP) v = *reinterpret_cast<const uint4*>(q + h * D + gr * 64 + (2 * t + c) * 8);
          raw[gr][c][0] = v.x; raw[gr][c][1] = v.y; raw[gr][c][2] = v.z; raw[gr][c][3] = v.w;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack_bf16(raw[gr][c][e]);
            most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
            sum[gr] += f.x + f.y;
          }
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], o);
      }
      // 2^k with the largest |q| in [2^14, 2^15); rows below 2^-112 (zeros, say) are taken as that, rows beyond 2^117 become
      // infinities
      const int ex = max(static_cast<int>(__float_as_uint(most) >> 23), 15);
      const float up = ex > 244 ? 1.f : __uint_as_float(static_cast<uint32_t>(268 - ex) << 23);
      const float back = ex > 244 ? 16777216.f : __uint_as_float(static_cast<uint32_t>(ex + 10) << 23);      // 2^24 / up
#pragma unroll
      for (int gr = 0; gr < GR; ++gr) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 v = unpack_bf16(raw[gr][c][e]);
            f[2 * e] = v.x * up;
            f[2 * e + 1] = v.y * up;
          }
          // step 2c: bytes 0 and 2 (codes 0, 1 and 4, 5); step 2c + 1: bytes 1 and 3. The second code of a byte comes as 16 c1.
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            qf[nt][gr * 4 + 2 * c + i][0] = pack_f16(f[2 * i], f[2 * i + 4]);
            qf[nt][gr * 4 + 2 * c + i][1] = pack_f16(f[2 * i + 1] * 0.0625f, f[2 * i + 5] * 0.0625f);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {                      // lane 4 (2t + c) has head 2t + c
        unscale[nt][c] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + c)) * p.scale_log2;
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) qsum[nt][c][gr] = __shfl_sync(0xffffffffu, sum[gr], 4 * (2 * t + c)) * p.scale_log2;
      }
    }

    // o: sums of codes of even dims and of 16 times those of odd dims, in units of 2^-24; o, l and lows relative to
    // 2^base, base = maximum (m) + log2 of the largest scale (top_scale) - kV4Room
    float o[NT][KS][4], lows[NT][GR][2], m[NT][2], l[NT][2], base[NT][2], top_scale = 8.6736174e-19f;      // 2^-60: scales below it count as that
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[nt][c] = -INFINITY;
        l[nt][c] = base[nt][c] = 0.f;
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) lows[nt][gr][c] = 0.f;
      }
    }

    for (int tile = at_tile; tile < at_tile + seg_end - seg && ok; ++tile) {
      const int stage = used % kV4Stages;
      const int key0 = tile * kV4Keys;
      ok = __all_sync(0xffffffffu, guard.wait(&bar[stage], (used / kV4Stages) & 1));
      if (!ok) break;
      const uint32_t kb = ring + stage * SM::kStage, vb = kb + 2 * SM::kBlock;
      const bool tail = key0 + kV4Keys > len;

      // scores of keys 16 sub + g, + 8
      float s[NT][2][4];
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const uint32_t b = kb + sub * SM::kBlock;
        float acc[NT][GR][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int gr = 0; gr < GR; ++gr)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][gr][e] = 0.f;
        uint32_t w[2][2 * GR];                           // keys g, g + 8: chunks 2t, 2t + 1 of each group
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if constexpr (D == 128) lds128(b + (g + 8 * r) * 64 + t * 16, w[r]);
          else lds64(b + (g + 8 * r) * 32 + t * 8, w[r][0], w[r][1]);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) {
            const uint32_t x = w[0][c * GR + gr], y = w[1][c * GR + gr], x1 = x >> 8, y1 = y >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(acc[nt][gr], x & kEven, y & kEven, x & kOdd, y & kOdd, qf[nt][gr * 4 + 2 * c][0], qf[nt][gr * 4 + 2 * c][1]);
              mma_f16(acc[nt][gr], x1 & kEven, y1 & kEven, x1 & kOdd, y1 & kOdd, qf[nt][gr * 4 + 2 * c + 1][0], qf[nt][gr * 4 + 2 * c + 1][1]);
            }
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t pr[2];
          if constexpr (GR == 2) lds64(b + 8 * D + (g + 8 * r) * 8, pr[0], pr[1]);
          else pr[0] = lds32(b + 8 * D + (g + 8 * r) * 4);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float dot = low_half(pr[0]) * acc[nt][0][2 * r + c], add = high_half(pr[0]) * qsum[nt][c][0];
              if constexpr (GR == 2) {
                dot = fmaf(low_half(pr[1]), acc[nt][1][2 * r + c], dot);
                add = fmaf(high_half(pr[1]), qsum[nt][c][1], add);
              }
              s[nt][sub][2 * r + c] = fmaf(unscale[nt][c], dot, add);
            }
          }
        }
      }
      // the values' scales and low ends; what lies behind the last token may be anything
      uint32_t vp[2][2][GR];
      float scale_max = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t (&pr)[GR] = vp[i / 2][i % 2];
        const uint32_t at_pair = vb + i / 2 * SM::kBlock + 8 * D + (g + 8 * (i % 2)) * (4 * GR);
        if constexpr (GR == 2) lds64(at_pair, pr[0], pr[1]);
        else pr[0] = lds32(at_pair);
      }
      if (tail) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (key0 + 8 * i + g >= len) {
            vp[i / 2][i % 2][0] = vp[i / 2][i % 2][GR - 1] = 0u;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][i / 2][i % 2 * 2] = s[nt][i / 2][i % 2 * 2 + 1] = -INFINITY;
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) scale_max = fmaxf(scale_max, low_half(vp[i / 2][i % 2][gr]));
      // the reference of the exponentials
      float mx[NT][2];
      bool follow = scale_max > top_scale;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          mx[nt][c] = fmaxf(fmaxf(s[nt][0][c], s[nt][0][2 + c]), fmaxf(s[nt][1][c], s[nt][1][2 + c]));
          follow = follow || mx[nt][c] > m[nt][c] + kV4Lazy;
        }
      }
      if (__any_sync(0xffffffffu, follow)) {
        // the next power of two: the reference moves by whole steps
        const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(scale_max, top_scale)));
        top_scale = __uint_as_float(min((bits + 0x7fffffu) & 0x7f800000u, 0x7f000000u));
        const float room = static_cast<float>(static_cast<int>(__float_as_uint(top_scale) >> 23) - 127) - kV4Room;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int of = 4; of < 32; of <<= 1) mx[nt][c] = fmaxf(mx[nt][c], __shfl_xor_sync(0xffffffffu, mx[nt][c], of));
            const float m_new = fmaxf(m[nt][c], mx[nt][c]);
            const float to = m_new == -INFINITY ? 0.f : m_new + room;
            const float alpha = m[nt][c] == -INFINITY ? 0.f : exp2f(base[nt][c] - to);       // nothing is there yet where m is -inf
            m[nt][c] = m_new;
            base[nt][c] = to;
            l[nt][c] *= alpha;
#pragma unroll
            for (int gr = 0; gr < GR; ++gr) lows[nt][gr][c] *= alpha;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              o[nt][i][c] *= alpha;
              o[nt][i][2 + c] *= alpha;
            }
          }
        }
      }
      // probabilities, times the values' scales: operands of the second product
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const uint32_t b = vb + sub * SM::kBlock;
        uint32_t pf[NT][GR][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t (&pr)[GR] = vp[sub][r];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float e[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              e[c] = exp2f(s[nt][sub][2 * r + c] - base[nt][c]);
              l[nt][c] += e[c];
#pragma unroll
              for (int gr = 0; gr < GR; ++gr) lows[nt][gr][c] = fmaf(e[c], high_half(pr[gr]), lows[nt][gr][c]);
            }
#pragma unroll
            for (int gr = 0; gr < GR; ++gr) pf[nt][gr][r] = movmatrix(pack_f16(e[0] * low_half(pr[gr]), e[1] * low_half(pr[gr])));
          }
        }
        uint32_t w[4][2];                                // tokens 2t, 2t + 1, 2t + 8, 2t + 9: chunk g of each group
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a = b + (2 * t + (i & 1) + (i >> 1) * 8) * (D / 2) + g * (4 * GR);
          if constexpr (GR == 2) lds64(a, w[i][0], w[i][1]);
          else w[i][0] = lds32(a);
        }
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {                  // bytes 2i, 2i + 1 of the chunk: dims 4i .. 4i + 3
            const uint32_t x = __byte_perm(w[0][gr], w[1][gr], i == 0 ? 0x5410 : 0x7632), y = __byte_perm(w[2][gr], w[3][gr], i == 0 ? 0x5410 : 0x7632);
            const uint32_t x1 = x >> 8, y1 = y >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(o[nt][gr * 4 + 2 * i], x & kEven, x & kOdd, y & kEven, y & kOdd, pf[nt][gr][0], pf[nt][gr][1]);
              mma_f16(o[nt][gr * 4 + 2 * i + 1], x1 & kEven, x1 & kOdd, y1 & kEven, y1 & kOdd, pf[nt][gr][0], pf[nt][gr][1]);
            }
          }
        }
      }
      ++used;
      __syncwarp();                                      // every lane has read the stage
      if (issued < my_tiles) issue(stage);
    }

    // ---- the head group's end, or this warp's: l and lows are of this lane's keys so far
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int of = 4; of < 32; of <<= 1) {
          l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], of);
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) lows[nt][gr][c] += __shfl_xor_sync(0xffffffffu, lows[nt][gr][c], of);
        }
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          o[nt][i][c] = fmaf(o[nt][i][c], 16777216.f, lows[nt][i / 4][c]);
          o[nt][i][2 + c] = fmaf(o[nt][i][2 + c], 1048576.f, lows[nt][i / 4][c]);
        }
        if (m[nt][c] == -INFINITY) base[nt][c] = -INFINITY;          // no keys: no part in a sum
      }
    }
    const bool starts = at_tile == 0, ends = at_tile + seg_end - seg == at.n;
    if (starts && ends) {                                // all of it: eight dims of a group of heads 2t, 2t + 1 a lane
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int h = 8 * nt + 2 * t + c;
          const float inv = l[nt][c] > 0.f || l[nt][c] != l[nt][c] ? 1.f / l[nt][c] : 0.f;       // no keys: zeros
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_bf16(o[nt][gr * 4 + i][c] * inv, o[nt][gr * 4 + i][2 + c] * inv);
            if (h < p.GP)
              *reinterpret_cast<uint4*>(p.out + (static_cast<int64_t>(at.seq) * p.Hq + head0 + h) * D + gr * 64 + 8 * g) =
                  make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    } else {
      // a part: what does not start here goes to `firsts` (a warp's first part), what does is the warp's last and takes its ring's place
      float4* to = starts ? reinterpret_cast<float4*>(smem + warp * (kV4Stages * SM::kStage)) : firsts + warp * kPieces * 32;
      float* to_ml = ml + ((starts ? kV4Warps : 0) + warp) * 16 * NT;
      if (lane == 0)
        info[(starts ? kV4Warps : 0) + warp] = make_int4(at.seq, at.head, ends ? 1 : 0, starts ? last_cta(begin + seg + at.n, at.n) : 0);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (g == 0) *reinterpret_cast<float2*>(to_ml + (nt * 8 + 2 * t + c) * 2) = make_float2(base[nt][c], l[nt][c]);
#pragma unroll
          for (int gr = 0; gr < GR; ++gr)
#pragma unroll
            for (int half = 0; half < 2; ++half)
              to[((nt * GR + gr) * 4 + c * 2 + half) * 32 + lane] =
                  make_float4(o[nt][gr * 4 + 2 * half][c], o[nt][gr * 4 + 2 * half][2 + c], o[nt][gr * 4 + 2 * half + 1][c],
                              o[nt][gr * 4 + 2 * half + 1][2 + c]);
        }
      }
    }
    at_tile = 0;                                         // only a warp's last head group ends after it does
    next_head(at);
    seg = seg_end;
  }
  __syncthreads();
  // ---- the parts of this CTA's warps: a row starts with a warp's last part, or with what the CTA before began, and goes on through
  // the first parts of the warps behind. Four dims of a head a thread.
  constexpr uint32_t kAll = (1u << kV4Warps) - 1;
  static_assert(2 * kV4Warps <= 32);
  const int4 mine = lane < 2 * kV4Warps ? info[lane] : make_int4(-1, 0, 0, 0);
  const uint32_t parts = __ballot_sync(0xffffffffu, mine.x >= 0), ending = __ballot_sync(0xffffffffu, mine.x >= 0 && mine.z != 0) & kAll;
  constexpr int kTeam = kPieces < kV4Warps ? kPieces : kV4Warps, kTeams = kV4Warps / kTeam;       // as many warps as a row has pieces
  int turn = 0;
  for (uint32_t rows = (parts >> kV4Warps) << 1 | (parts & 1u); rows != 0; rows &= rows - 1) {        // bit 0: what the CTA before began
    const int row = __ffs(rows) - 2;
    if (turn++ % kTeams != warp / kTeam) continue;
    const uint32_t behind = (parts & kAll) >> (row + 1), stops = ending >> (row + 1);
    const int run = __ffs(~behind) - 1, stop = __ffs(stops);                 // first parts in a row, place of the one that ends (from 1 on)
    const bool done = stop != 0 && stop <= run;
    const int last = row + (done ? stop : run), at_info = row < 0 ? 0 : kV4Warps + row;          // the last warp with a part
    const int4 what = make_int4(__shfl_sync(0xffffffffu, mine.x, at_info), __shfl_sync(0xffffffffu, mine.y, at_info), 0,
                                __shfl_sync(0xffffffffu, mine.w, at_info));
    const int head0 = what.y / hg * p.G + what.y % hg * p.GP, slot = 2 * static_cast<int>(blockIdx.x) + (row < 0 ? 0 : 1);
    for (int x = warp % kTeam; x < kPieces; x += kTeam) {
      const int nt = x / (GR * 4), gr = x / 4 % GR, c = x / 2 % 2, half = x % 2;
      const int h = 8 * nt + 2 * t + c, dim = gr * 64 + 8 * g + 4 * half;
      float top = -INFINITY, sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = max(row, 0); w <= last; ++w)
        top = fmaxf(top, ml[((w == row ? kV4Warps : 0) + w) * 16 * NT + h * 2]);
      for (int w = max(row, 0); w <= last; ++w) {
        const float2 y = *reinterpret_cast<const float2*>(ml + ((w == row ? kV4Warps : 0) + w) * 16 * NT + h * 2);
        const float4* from = w == row ? reinterpret_cast<const float4*>(smem + w * (kV4Stages * SM::kStage)) : firsts + w * kPieces * 32;
        const float4 z = from[x * 32 + lane];
        const float f = y.x == -INFINITY ? 0.f : exp2f(y.x - top);
        sum = fmaf(y.y, f, sum);
        v.x = fmaf(z.x, f, v.x); v.y = fmaf(z.y, f, v.y); v.z = fmaf(z.z, f, v.z); v.w = fmaf(z.w, f, v.w);
      }
      if (h < p.GP) {
        if (row >= 0 && done) {
          const float inv = 1.f / sum;
          *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(what.x) * p.Hq + head0 + h) * D + dim) =
              make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
        } else {
          *reinterpret_cast<float4*>(p.part_o + (static_cast<int64_t>(slot) * 8 * NT + h) * D + dim) = v;
          if (g == 0 && gr == 0 && half == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * 8 * NT + h) * 2) = make_float2(top, sum);
        }
      }
    }
    if (row >= 0 && !done && warp % kTeam == 0 && lane == 0) p.meta[blockIdx.x] = make_int4(what.x, what.y, what.w, slot);     // goes on in the next share
  }
  // copies in flight land before the CTA ends, where the waits were given up
  for (; used < issued; ++used) guard.land(&bar[used % kV4Stages], (used / kV4Stages) & 1);
}

// Joins the parts of a head group that several CTAs share: one CTA for each that starts one and does not end it. A thread has four dims of a
// head and every WAYS-th part; three parts' sums are on their way at a time. Four ways where few head groups have many parts (one sequence
// of 80 thousand, 64 / 8 heads: 45 -> 38 us in all), one where many have two (64 of some 500: 21 us, 23 in four).
template <int D, int NT, int WAYS>
__global__ void __launch_bounds__(256 * WAYS) kv4_join_kernel(const Kv4Params p) {
  __shared__ float4 sums[WAYS][256];
  __shared__ float2 tops[WAYS][256];
  griddep_launch();
  griddep_wait();
  const int4 meta = p.meta[blockIdx.x];                  // sequence, head group, last CTA, slot of the first part
  if (meta.x < 0) return;
  const int hg = p.G / p.GP, parts = meta.z - static_cast<int>(blockIdx.x) + 1;
  const int head0 = meta.y / hg * p.G + meta.y % hg * p.GP, way = WAYS == 1 ? 0 : threadIdx.x / 256, at = threadIdx.x % 256;
  for (int i0 = 0; i0 < p.GP * (D / 4); i0 += 256) {
    const int i = i0 + at, h = i / (D / 4), d = i % (D / 4) * 4;
    const bool in = h < p.GP;
    float m = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int n0 = way; in && n0 < parts; n0 += 3 * WAYS) {
      float2 ml[3];
      float4 o[3];
#pragma unroll
      for (int n = 0; n < 3; ++n) {                      // behind the last part: that one again, with no weight
        const int part = min(n0 + n * WAYS, parts - 1), slot = part == 0 ? meta.w : 2 * (static_cast<int>(blockIdx.x) + part);
        ml[n] = *reinterpret_cast<const float2*>(p.part_ml + (slot * 8 * NT + h) * 2);
        o[n] = *reinterpret_cast<const float4*>(p.part_o + (static_cast<int64_t>(slot) * 8 * NT + h) * D + d);
      }
      const float m_new = fmaxf(fmaxf(m, ml[0].x), fmaxf(ml[1].x, ml[2].x)), old = m == -INFINITY ? 0.f : exp2f(m - m_new);
      m = m_new;
      sum *= old; v.x *= old; v.y *= old; v.z *= old; v.w *= old;
#pragma unroll
      for (int n = 0; n < 3; ++n) {
        if (n0 + n * WAYS >= parts) break;
        const float f = ml[n].x == -INFINITY ? 0.f : exp2f(ml[n].x - m);
        sum = fmaf(ml[n].y, f, sum);
        v.x = fmaf(o[n].x, f, v.x); v.y = fmaf(o[n].y, f, v.y);
        v.z = fmaf(o[n].z, f, v.z); v.w = fmaf(o[n].w, f, v.w);
      }
    }
    if constexpr (WAYS > 1) {
      __syncthreads();
      sums[way][at] = v;
      tops[way][at] = make_float2(m, sum);
      __syncthreads();
    }
    if (way == 0 && in) {
      float top = m;
#pragma unroll
      for (int w = 1; w < WAYS; ++w) top = fmaxf(top, tops[w][at].x);
      const float mine = m == -INFINITY ? 0.f : exp2f(m - top);
      sum *= mine; v.x *= mine; v.y *= mine; v.z *= mine; v.w *= mine;
#pragma unroll
      for (int w = 1; w < WAYS; ++w) {
        const float2 y = tops[w][at];
        const float4 z = sums[w][at];
        const float f = y.x == -INFINITY ? 0.f : exp2f(y.x - top);
        sum = fmaf(y.y, f, sum);
        v.x = fmaf(z.x, f, v.x); v.y = fmaf(z.y, f, v.y); v.z = fmaf(z.z, f, v.z); v.w = fmaf(z.w, f, v.w);
      }
      const float inv = 1.f / sum;
      *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(meta.x) * p.Hq + head0 + h) * D + d) =
          make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
    }
  }
}

template <int D, int NT>
int launch_kv4_decode(const Kv4Params& p, int ctas, cudaStream_t st) {
  using SM = Kv4Smem<D, NT>;
  static PerDeviceOnce configured;
  if (configured.need()) {
    CUDA_CHECK_RET(cudaFuncSetAttribute(kv4_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::kBytes));
    configured.done();
  }
  CUDA_CHECK_RET(launch_pdl(kv4_decode_kernel<D, NT>, dim3(ctas), dim3(SM::kV4Threads), SM::kBytes, st, p));
  if (static_cast<int64_t>(p.B) * (p.Hq / p.GP) * 3 < ctas) CUDA_CHECK_RET(launch_pdl(kv4_join_kernel<D, NT, 4>, dim3(ctas), dim3(1024), 0, st, p));
  else CUDA_CHECK_RET(launch_pdl(kv4_join_kernel<D, NT, 1>, dim3(ctas), dim3(256), 0, st, p));
  return 0;
}

// Pages of the sequences of a launch expanded to bf16 tiles [tile][Hkv][D / 64][64 tokens][64], as the prefill kernels read a cache with
// pages of 64, and the tiles' table. Sequence s has ceil(len / 64) tiles, from the sum of those before it on. A CTA makes a tile of a
// head's keys or values, zeros behind the last token; a thread has several units of eight dims on their way. Memory-bound: 9 D / 16 bytes in,
// 2 D out a token; three prompts with up to 1700 tokens of 8 heads of 64: 4 us of the step's 71.
constexpr int kV4ExpandThreads = 256;
template <int D>
__global__ void __launch_bounds__(kV4ExpandThreads)
kv4_expand_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const int32_t* __restrict__ block_table,
                  int64_t pitch, int max_blocks, const int32_t* __restrict__ seq_lens, int Hkv, int page_size, int64_t pages, int64_t tiles,
                  __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int32_t* __restrict__ table, int max_tiles) {
  griddep_launch();
  griddep_wait();
  constexpr int G = D / 64, kBlock = 9 * D, kUnits = D / 8, kN = 64 * kUnits / kV4ExpandThreads;
  const int seq = blockIdx.y, in_seq = blockIdx.x;       // tile of the sequence
  const int len = seq_lens[seq];
  if (in_seq * 64 >= len) return;
  __shared__ int part[kV4ExpandThreads / 32];
  int before = 0;
  for (int s = threadIdx.x; s < seq; s += kV4ExpandThreads) before += (seq_lens[s] + 63) / 64;
  before = __reduce_add_sync(0xffffffffu, before);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = before;
  __syncthreads();
  int64_t tile = in_seq;
#pragma unroll
  for (int w = 0; w < kV4ExpandThreads / 32; ++w) tile += part[w];
  if (tile >= tiles) return;                             // more tokens than the caller has made room for
  if (threadIdx.x == 0 && blockIdx.z == 0) table[static_cast<size_t>(seq) * max_tiles + in_seq] = static_cast<int>(tile);
  const bool is_v = static_cast<int>(blockIdx.z) >= Hkv;
  const int h = is_v ? blockIdx.z - Hkv : blockIdx.z;
  const uint8_t* cache = is_v ? v_cache : k_cache;
  __nv_bfloat16* out = (is_v ? v_out : k_out) + (tile * Hkv + h) * G * 64 * 64;
  const int32_t* row = block_table + seq * pitch;
  uint32_t codes[kN], pair[kN];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    const int i = threadIdx.x + n * kV4ExpandThreads, r = i / kUnits, unit = i % kUnits, tok = in_seq * 64 + r;
    codes[n] = pair[n] = 0u;                             // stands for zeros
    if (tok < len) {
      const int at = tok / page_size, off = tok - at * page_size;
      const int64_t page = min(static_cast<int64_t>(static_cast<uint32_t>(row[min(at, max_blocks - 1)])), pages - 1);
      const uint8_t* block = cache + ((page * Hkv + h) * (page_size / 16) + off / 16) * kBlock;
      codes[n] = *reinterpret_cast<const uint32_t*>(block + off % 16 * (D / 2) + unit * 4);
      pair[n] = *reinterpret_cast<const uint32_t*>(block + 8 * D + (off % 16 * G + unit % G) * 4);
    }
  }
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    const int i = threadIdx.x + n * kV4ExpandThreads, r = i / kUnits, unit = i % kUnits;
    const float2 p = unpack_bf16(pair[n]);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fmaf(static_cast<float>((codes[n] >> (4 * e)) & 15u), p.x, p.y);
    *reinterpret_cast<uint4*>(out + (unit % G * 64 + r) * 64 + unit / G * 8) =
        make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
}

}  // namespace

}  // namespace b200

using namespace b200;

// Bytes of scratch that gllm_kv4_decode needs on `ctas` CTAs.
GLLM_EXPORT int64_t gllm_kv4_decode_scratch(int D, int ctas) {
  return static_cast<int64_t>(ctas) * (2 * 16 * (D + 2) * 4 + 16);
}

// Attention of B sequences with one new token each over 4-bit caches of `pages` pages: q [B, Hq * D] (token stride q_ts), out [B, Hq, D]
// contiguous; keys [0, seq_lens[s]) of each, zeros where there are none.
GLLM_EXPORT int gllm_kv4_decode(const void* q, int64_t q_ts, void* out, const void* k_cache, const void* v_cache, int64_t pages,
                                const void* block_table, int64_t pitch, int max_blocks, const void* seq_lens, int B, int Hq, int Hkv,
                                int D, int page_size, float scale, int ctas, void* scratch, int64_t scratch_bytes, void* stream) {
  if (B <= 0) return 0;
  auto al16 = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  if ((D != 64 && D != 128) || page_size < 16 || page_size > 512 || page_size % 16 != 0 || Hkv <= 0 || Hq % Hkv != 0 || q_ts % 8 != 0 || !al16(q) ||
      !al16(out) || !al16(k_cache) || !al16(v_cache) || !al16(scratch) || pages <= 0 || max_blocks <= 0 || ctas <= 0 ||
      scratch_bytes < gllm_kv4_decode_scratch(D, ctas)) {
    fprintf(stderr, "[gllm_b200] kv4_decode: unsupported D=%d page_size=%d Hq=%d Hkv=%d (%lld pages, %d a sequence), or rows off 16-byte boundaries\n",
            D, page_size, Hq, Hkv, static_cast<long long>(pages), max_blocks);
    return 1;
  }
  Kv4Params p;
  p.q = reinterpret_cast<const __nv_bfloat16*>(q);
  p.q_ts = q_ts;
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  p.k_cache = reinterpret_cast<const uint8_t*>(k_cache);
  p.v_cache = reinterpret_cast<const uint8_t*>(v_cache);
  p.last_page = static_cast<uint32_t>(pages < 0x80000000ll ? pages - 1 : 0x7fffffffll);
  p.block_table = reinterpret_cast<const int32_t*>(block_table);
  p.seq_lens = reinterpret_cast<const int32_t*>(seq_lens);
  p.pitch = pitch; p.B = B; p.max_blocks = max_blocks; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv;
  p.page_blocks = page_size / 16;
  p.page_magic = p.page_blocks == 1 ? 0u : static_cast<uint32_t>((0x100000000ull + p.page_blocks - 1) / p.page_blocks);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part_o = reinterpret_cast<float*>(scratch);
  p.part_ml = p.part_o + static_cast<int64_t>(ctas) * 2 * 16 * D;
  p.meta = reinterpret_cast<int4*>(p.part_ml + static_cast<int64_t>(ctas) * 2 * 16 * 2);
  p.waits = g_wait_config;
  // The largest divisor of a kv head's query heads up to 16 of them at a time: a kv head's codes are read G / GP times, once up to 16. (G = 17 has
  // none and takes one at a time: 64 sequences of up to 1000, 34 / 2 heads, 57 us; the bf16 cache 91.)
  p.GP = 1;
  for (int d = 2; d <= 16 && d <= p.G; ++d)
    if (p.G % d == 0) p.GP = d;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p.GP <= 8) return D == 64 ? launch_kv4_decode<64, 1>(p, ctas, st) : launch_kv4_decode<128, 1>(p, ctas, st);
  return D == 64 ? launch_kv4_decode<64, 2>(p, ctas, st) : launch_kv4_decode<128, 2>(p, ctas, st);
}

// Keys and values of B sequences from 4-bit caches to bf16 tiles k_out, v_out [tiles, Hkv, D / 64, 64, 64], sequence after sequence, each
// rounded up to 64 tokens; table [B, max_tiles]: their tiles. max_len: the longest.
GLLM_EXPORT int gllm_kv4_expand(const void* k_cache, const void* v_cache, const void* block_table, int64_t pitch, int max_blocks,
                                const void* seq_lens, int B, int Hkv, int D, int page_size, int64_t pages, int64_t tiles, void* k_out, void* v_out,
                                void* table, int max_tiles, int max_len, void* stream) {
  if (B <= 0 || max_len <= 0) return 0;
  if ((D != 64 && D != 128) || page_size < 16 || page_size > 512 || page_size % 16 != 0 || pages <= 0 || max_blocks <= 0 || B > 65535 || Hkv > 32767 ||
      static_cast<int64_t>(max_tiles) * 64 < max_len) {
    fprintf(stderr, "[gllm_b200] kv4_expand: unsupported D=%d page_size=%d, %d sequences\n", D, page_size, B);
    return 1;
  }
  const dim3 grid((max_len + 63) / 64, B, 2 * Hkv);
  CUDA_CHECK_RET(launch_pdl(D == 64 ? kv4_expand_kernel<64> : kv4_expand_kernel<128>, grid, dim3(kV4ExpandThreads), 0,
                            reinterpret_cast<cudaStream_t>(stream), reinterpret_cast<const uint8_t*>(k_cache),
                            reinterpret_cast<const uint8_t*>(v_cache), reinterpret_cast<const int32_t*>(block_table), pitch, max_blocks,
                            reinterpret_cast<const int32_t*>(seq_lens), Hkv, page_size, pages, tiles,
                            reinterpret_cast<__nv_bfloat16*>(k_out), reinterpret_cast<__nv_bfloat16*>(v_out),
                            reinterpret_cast<int32_t*>(table), max_tiles));
  return 0;
}
