// w4_kv8_prompt.cu - attention over the paged 8-bit KV cache for many query
// rows a sequence (prompts, chunks of prompts), on the 5th-generation tensor
// cores.
//
// The maths, the split and the join are those of w4_kv8_attn.cu; there a step's
// few rows make the cache's bytes the bound, here 4 D operations a (row, token)
// pair do. An item is 128 query rows of one cache head (G query heads times the
// new tokens), worked through in tiles of 128 tokens by one CTA an SM, the tiles
// in turn by two streams that meet at the item's end:
//   copy warp      : the pages' runs of 16 tokens by bulk copies into three buffers
//                    of a K or a V tile, and the scales;
//   4 widen warps  : e4m3 to fp16 (exact), K and V alike token by token in the 128B-swizzled
//                    layout (K is the K-major operand of Q K^T; of P V the same
//                    rows are the MN-major operand V, so nothing is transposed);
//   item warp      : walks the CTA's share and leaves the items in a ring, so that
//                    no other warp carries the walk in its registers and code;
//   MMA warp       : one thread issues S = Q K^T of one stream (M = N = 128),
//                    then O += P V of the other, so that the tensor cores work
//                    for one while the other's softmax does;
//   2 x 4 softmax warps: a thread a row of its stream. S from tensor memory, the
//                    exponent's argument with the page's scales folded in (as in
//                    the other kernel), P' in fp16 back into tensor memory over
//                    the S that it came from. O stays in tensor memory, one a
//                    stream with a maximum of its own, and is rescaled only when
//                    a row's running maximum has grown by more than 2^kGrowth since
//                    the last time (P' may then reach 2^15, inside fp16's range).
// Two O, two S (with P over them) fill the tensor memory: 4 x 128 columns. A tile's
// products at their best rate and its 128 x 128 exponentials at 16 a clock are 1024
// clocks each, its traffic on shared memory 1750. A tile takes 2600: a stream's
// S, softmax (2400), P V and next S follow one another, and two streams are all that
// the tensor memory holds. 2 x 256 tokens of 32 heads on 8 over 4096: 71 us, 480
// TFLOP/s of the causal products (16 us of it before the first S, after the last P V
// and in the empty join's launch); 8192 tokens from nothing 876 us, 630 TFLOP/s.
#include "w4_kv8_attn.cuh"
#include "w4_tcgen05.cuh"

#include <algorithm>

namespace w4 {

namespace {

constexpr int kSoftWarps = 4, kWidenWarps = 4;  // softmax warps of a stream
constexpr int kWidenWarp = 2 * kSoftWarps;
constexpr int kMmaWarp = kWidenWarp + kWidenWarps;
constexpr int kItemWarp = kMmaWarp + 1, kCopyWarp = kMmaWarp + 2;
constexpr int kPromptThreads = 32 * (kMmaWarp + 4);  // four warpgroups; one warp idles
// Registers a thread: 128 at launch, then by warpgroup (their sum is four times
// that, which is what the block has). 8192 tokens, when chosen: softmax 176 922 us, 184
// 885, 192 905.
constexpr int kSoftRegs = 184, kWidenRegs = 80, kMmaRegs = 64;
static_assert(2 * kSoftRegs + kWidenRegs + kMmaRegs <= 4 * 128, "registers of the block");
constexpr int kPromptTile = 128;   // tokens of a tile, and rows of an item
// P' of the maximum that O is scaled by is 2^kPromptShift, and the running maximum may
// exceed it by kGrowth (and by 2^-3, the roundings of scores below 2^20): P' stays below
// fp16's 2^16. What is more than 2^28 below the maximum falls under fp16's normal range,
// off by 2^-25 at most: 2^-39 of the maximum's, as in the other kernel. (A shift of 8 and a
// growth of 6 spare rescales, 2 x 256 over 4096 70.4 and 71.3 us, but weights of 2^-30 are
// then off by a seventh.)
constexpr float kPromptShift = 14.0f;
constexpr float kGrowth = 1.75f;
constexpr int kErrPromptWait = 9;
// Factors of S are at least this, so that a masked -inf stays -inf under a scale of
// zero; below it a score is none of the argument's 24 bits.
constexpr float kLeast = 1e-37f;

// Items in units of tokens: a row tile is as long as its own last row sees, near
// enough (a step of 128 rows is ceil(128 / G) tokens), so that the triangle of a
// long prompt is shared out evenly.
struct Rows128 {
  static constexpr int kRows = kPromptTile;
  static constexpr int kTile = kPromptTile;
  static constexpr int kUnit = kPromptTile;
  static constexpr int kOver = 3 * kPromptTile;  // queries, first tile's latency, output
  static constexpr int kMinShare = 4 * kPromptTile;
  static __device__ __forceinline__ int tiles(const AttnP&, const Seq&, int limit) {
    return (limit + kTile - 1) / kTile;
  }
  static __device__ __forceinline__ int row_tiles(const AttnP& p, const Seq& s) {
    return (s.n * p.group + kRows - 1) / kRows;
  }
  static __device__ __forceinline__ int step(const AttnP& p) {
    return (kRows + p.group - 1) / p.group;
  }
  // Items are not cut if the longest CTA ends at most this much later than with equal
  // shares: a cut costs two first tiles, the parts and their join. 2 sequences of
  // up to 256 tokens, 32 heads on 8, cut and not, when chosen: over 1000 45.2 and 31.3 us, 4096 81.7
  // and 68.0, 12000 (13 tiles later) 165.7 and 165.6; 512 tokens of 16 heads over 3000 (17) 44.3 and 54.7.
  static constexpr int kCut = 12 * kPromptTile;
  static constexpr int kMore = 3 * kPromptTile;  // what first() and length() have beside past
  // Length of the first row tile, then of row tile rt: above kOver + kUnit * tiles
  // for every limit.
  static __device__ __forceinline__ int64_t first(const AttnP& p, const Seq& s) {
    return (int64_t)kOver + s.past + step(p) + kUnit;
  }
  static __device__ __forceinline__ int64_t length(const AttnP& p, const Seq& s, int64_t rt) {
    return first(p, s) + step(p) * rt;
  }
  // Length of row tiles 0 .. rt - 1 together.
  static __device__ __forceinline__ int64_t upto(const AttnP& p, const Seq& s, int64_t rt) {
    return rt * first(p, s) + step(p) * (rt * (rt - 1) / 2);
  }
  static __device__ __forceinline__ int64_t seq_work(const AttnP& p, const Seq& s) {
    return s.n > 0 ? p.kv_heads * upto(p, s, row_tiles(p, s)) : 0;
  }
  static __device__ __forceinline__ void locate(const AttnP& p, const Seq& s, int64_t off, int* h,
                                                int* rt, int64_t* at, int64_t* len) {
    const int nrt = row_tiles(p, s);
    const int64_t head = upto(p, s, nrt);
    *h = (int)divide(off, head);
    off -= *h * head;
    // the largest r with upto(r) <= off: the root in fp32, then to the integer
    const float a = 0.5f * step(p), b = (float)first(p, s) - a;
    int64_t r = (int64_t)((sqrtf(b * b + 4.f * a * (float)off) - b) / (2.f * a));
    r = min(max(r, (int64_t)0), (int64_t)nrt - 1);
    while (r > 0 && upto(p, s, r) > off) --r;
    while (r + 1 < nrt && upto(p, s, r + 1) <= off) ++r;
    *rt = (int)r;
    *at = off - upto(p, s, r);
    *len = length(p, s, r);
  }
};

// An item as the item warp leaves it; t0 == t1: there are no more.
struct Item {
  int t0, t1;        // its tiles
  int limit;         // tokens that its last row sees
  int past;          // tokens before the sequence's rows
  int b, h;          // sequence, cache head
  int first;         // the sequence's first row
  int r0, n_rows;    // first query row, all query rows of the head
  int whole, slot;   // all tiles of the item are here, or where the part goes
  int pad;
};
constexpr int kItems = 4;  // ring
constexpr int kRaws = 3;   // buffers of codes, K and V tiles in turn
constexpr int kScales = 8;  // tiles whose scales are kept

template <int D>
struct PromptShape {
  static constexpr int kHalf = kPromptTile * 128;         // 128 rows of 64 fp16
  static constexpr int kOperand = kHalf * (D / 64);       // Q, or a K or V tile
  static constexpr int kPitch = D + 4;
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kOffQ + kOperand;          // two buffers
  static constexpr int kOffV = kOffK + 2 * kOperand;      // two buffers
  static constexpr int kRaw = kPromptTile * D;            // a K or V tile's codes
  static constexpr int kOffRaw = kOffV + 2 * kOperand;    // kRaws buffers
  // tiles of 8 x (K scale, log2 and inverse of the V scale, the tile's blocks whose V scale
  // is far below another's: 8 bits), their blocks with a page
  static constexpr int kOffScale = kOffRaw + kRaws * kRaw;
  static constexpr int kOffPages = kOffScale + kScales * 8 * 16;
  // two items in turn: a factor a row, maxima and sums of the stream that meets the other
  static constexpr int kOffMul = kOffPages + kScales * 4;
  static constexpr int kOffSums = kOffMul + 2 * kPromptTile * 4;
  static constexpr int kOffMarks = kOffSums + 2 * kPromptTile * 8;
  static constexpr int kMarks = kPromptTile * D / 8;      // of an item; four items
  static constexpr int kOffItems = kOffMarks + 4 * kMarks;
  static constexpr int kOffBar = kOffItems + kItems * (int)sizeof(Item);
  static constexpr int kBars = 9 * 2 + 3 + 2 * kItems + 2 * kRaws;
  static constexpr int kOffTmem = kOffBar + kBars * 8;
  static constexpr int kSmem = 1024 + kOffTmem + 16;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// Byte offset of 16-byte chunk c (8 fp16) of row r in an operand half.
__device__ __forceinline__ uint32_t operand_at(int r, int c) {
  return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ void sts128(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

// A run of bytes into shared memory; they count at the barrier as they land.
__device__ __forceinline__ void bulk_load(uint32_t to, const void* from, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(to),
      "l"(from), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// mbar_wait with the clock for its limit, about a second: little code, for a
// dozen waits in each role.
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity) {
  const long long began = clock64();
  while (!mbar_try_wait(bar, parity))
    if (clock64() - began > 2000000000ll) return false;
  return true;
}

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kPromptThreads, 1) kv8_prompt_kernel(const AttnP p) {
  using S = PromptShape<D>;
  using G = Rows128;
  constexpr int kRows = kPromptTile;
  extern __shared__ uint8_t smem_prompt[];
  uint8_t* base = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_prompt) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sm = smem_u32(base);
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + S::kOffBar);
  // two of each, by stream (the parity of the tile)
  uint64_t* k_full = bars;        // widened K tile there (widen warps)
  uint64_t* k_empty = bars + 2;   // its product is done (commit)
  uint64_t* v_full = bars + 4;
  uint64_t* v_empty = bars + 6;
  uint64_t* s_full = bars + 8;    // S is in tensor memory (commit)
  uint64_t* p_full = bars + 10;   // all of P' is in its place (softmax warps)
  uint64_t* pv_done = bars + 12;  // P V is done (commit)
  // Two, by item: a stream that writes an item out may be at its queries when the
  // other one prepares those of the item after. (Never two after: that takes a
  // second S of the first stream, which has read its factors by then.)
  uint64_t* q_full = bars + 14;   // an item's queries are in shared memory, factors in mul_s
  uint64_t* b_done = bars + 16;   // the stream without the item's last tile is through with it
  uint64_t* o_empty = bars + 17;  // an item's outputs are read (the other one)
  uint64_t* item_full = bars + 18;             // an item is in the ring
  uint64_t* item_empty = item_full + kItems;   // MMA, copy, widen and softmax warps are through with it
  uint64_t* raw_full = item_empty + kItems;    // a tile's codes have landed (bytes), its scales are there
  uint64_t* raw_empty = raw_full + kRaws;      // widened
  uint64_t* p_half = raw_empty + kRaws;        // O is rescaled, P' of 64 tokens is in its place
  uint64_t* mma_done = p_half + 2;             // all products are done (commit)
  Item* items = reinterpret_cast<Item*>(base + S::kOffItems);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base + S::kOffTmem);
  // Marks of four items in turn: the widen warps may be two tiles ahead, that is
  // two short items, of the item whose output is read, but no more than that:
  // they have seen a product of the item before theirs but one, whose first waits
  // for the output of the one before it.
  const float4* scale_s = reinterpret_cast<const float4*>(base + S::kOffScale);
  uint32_t* marks = reinterpret_cast<uint32_t*>(base + S::kOffMarks);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], kWidenWarps);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], kWidenWarps);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kSoftWarps);
      mbar_init(&p_half[i], kSoftWarps);
      mbar_init(&pv_done[i], 1);
      mbar_init(&q_full[i], kSoftWarps);
    }
    mbar_init(b_done, kSoftWarps);
    mbar_init(o_empty, kSoftWarps);
    mbar_init(mma_done, 1);
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 2 + kWidenWarps + 2 * kSoftWarps);
    }
    for (int i = 0; i < kRaws; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], kWidenWarps);
    }
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {  // all of it: two S, two O
    tc_alloc(tmem_slot, 512);
    tc_fence_before();
  }
  for (int i = tid; i < S::kMarks; i += kPromptThreads) marks[i] = 0u;
  grid_dependency_wait();
  grid_launch_dependents();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_o = tmem + 2 * kPromptTile;  // O of stream u: + 128 u
  // A wait that gives up ends its role; the others give up in turn. A warp gives up as a
  // whole, since what follows needs all its lanes. (The MMA role is one lane: wait_on.)
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return (bool)__all_sync(0xffffffffu, wait_on(bar, parity));
  };
  int n = 0;     // tiles that this CTA has begun, over all items
  int item = 0;  // items
  bool ok = true;
  Item it;
  // Item `item` of the ring; false when there is none.
  auto next_by = [&](auto& wait) {
    if (!(ok = wait(&item_full[item % kItems], (item / kItems) & 1))) return false;
    it = items[item % kItems];
    return it.t0 < it.t1;
  };
  auto next_item = [&]() { return next_by(wait); };
  auto done_item = [&]() {  // by a whole warp
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[item % kItems]);
    ++item;
  };

  if (warp >= kMmaWarp) {
    // ------------------------------------------------------------ MMA
    fewer_registers<kMmaRegs>();
    if (warp == kItemWarp) {
      const Share share = find_share<G>(p);
      if (lane == 0) p.join[blockIdx.x].count = 0;
      Walk<G> walk;
      walk.start(share);
      for (;; ++item) {
        const bool more = share.x < share.end && walk.next(p);
        const int at = item % kItems;
        if (item >= kItems && !(ok = wait(&item_empty[at], ((item / kItems) & 1) ^ 1u))) break;
        if (lane == 0) {
          it.t0 = it.t1 = 0;
          if (more) {
            it.t0 = walk.t0, it.t1 = walk.t1, it.limit = walk.limit, it.past = walk.s.past;
            it.b = walk.b, it.h = walk.h, it.first = walk.s.first;
            it.r0 = walk.rt * kRows, it.n_rows = walk.s.n * p.group;
            it.whole = walk.whole, it.slot = walk.slot(share);
            if (!walk.whole) walk.describe(p, share);
          }
          items[at] = it;
          mbar_arrive(&item_full[at]);
        }
        __syncwarp();
        if (!more) break;
      }
    } else if (warp == kCopyWarp) {
      // Lane 8 j + b has block b (16 tokens) of tile t + j: its page and scales are
      // read for four tiles at once, its codes are one run of 16 D bytes in K and V.
      const int j = lane >> 3, b = lane & 7;
      constexpr uint32_t kRun = 16 * D;
      float4* scales = reinterpret_cast<float4*>(base + S::kOffScale);
      uint32_t* pages = reinterpret_cast<uint32_t*>(base + S::kOffPages);
      uint32_t stage = 0, turn = 0;
      while (ok && next_item()) {
        int most_lv = -100;  // largest log2 of the item's V scales so far (of kLeastScale: -80)
        for (int t = it.t0; t < it.t1 && ok; t += 4) {
          const int tok = (t + j) * kPromptTile + 16 * b;
          int id = -1;
          if (t + j < it.t1 && tok < it.limit) {
            const int pi = tok >> p.page_shift;
            if (pi < p.max_pages) id = p.page_table[it.b * p.table_stride + pi];
            if ((uint32_t)id >= (uint32_t)p.pages) {
              id = -1;
              atomicCAS(p.err, 0, kErrKvRange);
            }
          }
          const int64_t blk = (int64_t)max(id, 0) * p.kv_heads + it.h;
          const int64_t at = ((blk << p.page_shift) + (tok & (p.page - 1))) * D;
          float sc_k = 0.f, sc_v = 0.f, lv = -INFINITY;
          if (id >= 0) {
            sc_k = p.k_scale[blk];
            sc_v = fmaxf(p.v_scale[blk], kLeastScale);
            lv = lg2(sc_v);
          }
          const int whole_lv = __float2int_rd(fmaxf(lv, -100.0f));
          most_lv = max(most_lv, __reduce_max_sync(0xffffffffu, whole_lv));
          const uint32_t there = __ballot_sync(0xffffffffu, id >= 0);
          const uint32_t far = __ballot_sync(0xffffffffu, id >= 0 && whole_lv < most_lv - (int)kFar);
          for (int jj = 0; jj < min(4, it.t1 - t) && ok; ++jj, ++n) {
            const uint32_t blocks = there >> (8 * jj) & 0xffu;
#pragma unroll 1
            for (int kv = 0; kv < 2; ++kv) {
              if (!(ok = wait(&raw_empty[stage], turn ^ 1u))) break;
              if (kv == 0) {
                // K scale, log2 and inverse of the V scale, the tile's far blocks; no page: -inf
                if (j == jj) {
                  const float w = __uint_as_float(far >> (8 * jj) & 0xffu);
                  scales[(n % kScales) * 8 + b] = id >= 0 ? make_float4(sc_k, lv, 1.0f / sc_v, w)
                                                          : make_float4(0.f, -INFINITY, 0.f, w);
                }
                if (lane == 0) pages[n % kScales] = blocks;
              }
              __syncwarp();
              if (lane == 0) mbar_arrive_expect_tx(&raw_full[stage], __popc(blocks) * kRun);
              __syncwarp();
              if (j == jj && id >= 0)
                bulk_load(sm + S::kOffRaw + stage * S::kRaw + b * kRun, (kv ? p.v : p.k) + at, kRun,
                          &raw_full[stage]);
              if (++stage == kRaws) stage = 0, turn ^= 1u;
            }
          }
        }
        done_item();
      }
      // No copy stays in flight where the others no longer wait for it: each buffer's last,
      // of this turn or of the one before.
      for (int i = 0; i < kRaws && !ok; ++i)
        wait(&raw_full[i], (uint32_t)i < stage ? turn : turn ^ 1u);
    } else if (warp == kMmaWarp && lane == 0) {
      constexpr uint32_t idesc_s = tc_idesc(0, 0, kPromptTile), idesc_o = tc_idesc(0, 1, D);
      const uint64_t q_desc = tc_operand(sm + S::kOffQ, 16, 1024);
      // O += P V of tile m of item `of`, its first of the stream or not
      auto output = [&](int m, bool first, int of) {
        const int u = m & 1;
        if (!wait_on(&p_half[u], (m >> 1) & 1) || !wait_on(&v_full[u], (m >> 1) & 1) ||
            (first && of > 0 && !wait_on(o_empty, (of - 1) & 1)))
          return false;
        tc_fence_after();
        const uint64_t v_desc = tc_operand(sm + S::kOffV + u * S::kOperand, S::kHalf, 1024);
#pragma unroll
        for (int k = 0; k < kPromptTile / 16; ++k) {  // 16 tokens: 8 columns of P, 16 rows of V
          if (k == kPromptTile / 32) {
            if (!wait_on(&p_full[u], (m >> 1) & 1)) return false;
            tc_fence_after();
          }
          tc_mma_ts(tmem_o + u * kPromptTile, tmem + u * kPromptTile + 8 * k,
                     v_desc + ((k * 16 * 128) >> 4), idesc_o, first && k == 0 ? 0u : 1u);
        }
        __threadfence_block();  // the widen warps' marks, for those who wait for pv_done
        tc_commit(&v_empty[u]);
        tc_commit(&pv_done[u]);
        return true;
      };
      // A tile's P V comes after the next tile's S, the next item's first too, so that
      // there is a softmax to do while the item's last one is done.
      bool first = false;
      int of = 0;
      while (ok && next_by(wait_on)) {
        if (!(ok = wait_on(&q_full[item & 1], (item >> 1) & 1))) break;
        const int n0 = n;
        for (int t = it.t0; t < it.t1 && ok; ++t, ++n) {
          const int u = n & 1;
          // the stream's last P lies where this S goes
          ok = wait_on(&k_full[u], (n >> 1) & 1) &&
               (n < 2 || wait_on(&pv_done[u], ((n >> 1) & 1) ^ 1u));
          if (!ok) break;
          tc_fence_after();
          const uint64_t k_desc = tc_operand(sm + S::kOffK + u * S::kOperand, 16, 1024);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {  // 16 dims: 32 bytes along the swizzled rows
            const uint32_t at = ((k >> 2) * S::kHalf + (k & 3) * 32) >> 4;
            tc_mma(tmem + u * kPromptTile, q_desc + at, k_desc + at, idesc_s, k > 0);
          }
          __threadfence_block();  // the widen warps' scales, for those who wait for s_full
          tc_commit(&k_empty[u]);
          tc_commit(&s_full[u]);
          if (n > 0) ok = output(n - 1, first, of);
          first = n - n0 < 2;
          of = item;
        }
        mbar_arrive(&item_empty[item++ % kItems]);
      }
      if (ok && n > 0) ok = output(n - 1, first, of);
      // every product is done before the tensor memory is freed, also where a role gave up
      tc_commit(mma_done);
      ok = wait_on(mma_done, 0) && ok;
    }
  } else if (warp >= kWidenWarp) {
    // ------------------------------------------------------------ widen
    fewer_registers<kWidenRegs>();
    constexpr int CPR = D / 16, RPP = 128 / CPR, NP = kPromptTile / RPP;  // chunks a row, rows a pass
    // A quarter warp takes one chunk of each of eight rows, by an exclusive or that
    // gives its 16-byte reads of the plain codes and its stores of both halves of
    // the chunk into the swizzled rows all banks alike. A pass is RPP rows.
    const int w = warp - kWidenWarp, j = lane & 7, q = lane >> 3;
    const int c = CPR == 8 ? j ^ (q + 4 * (w & 1)) : ((j & 2) | (((j >> 2) ^ (j >> 1)) & 1)) ^ q;
    const int rr = j + 8 * (CPR == 8 ? w >> 1 : w);
    const uint32_t raw0 = sm + S::kOffRaw + rr * D + 16 * c;  // + 2048 a pass
    // where the halves go: rows a pass apart have the same swizzle
    const uint32_t to_a = (c >> 2) * S::kHalf + operand_at(rr, 2 * (c & 3)), to_b = to_a ^ 16u;
    uint32_t stage = 0, turn = 0;
    // A tile's codes, 16 a chunk, to two chunks of fp16 in an operand row each; the
    // reads of four passes go out together. Zeros for tokens of no page and behind
    // the limit (bit i of keep: pass i).
    auto widen = [&](uint32_t to, uint32_t from, uint32_t keep) {
#pragma unroll
      for (int i0 = 0; i0 < NP; i0 += 4) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = make_uint4(0u, 0u, 0u, 0u);
          if (keep >> (i0 + i) & 1u) v[i] = lds128(from + 2048 * (i0 + i));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t row = to + (i0 + i) * RPP * 128;
          sts128(row + to_a, make_uint4(e4m3_lo(v[i].x), e4m3_hi(v[i].x), e4m3_lo(v[i].y),
                                        e4m3_hi(v[i].y)));
          sts128(row + to_b, make_uint4(e4m3_lo(v[i].z), e4m3_hi(v[i].z), e4m3_lo(v[i].w),
                                        e4m3_hi(v[i].w)));
        }
      }
    };
    auto widened = [&](uint64_t* full) {
      fence_async_shared();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(full);
        mbar_arrive(&raw_empty[stage]);
      }
      if (++stage == kRaws) stage = 0, turn ^= 1u;
    };
    while (ok && next_item()) {
      uint32_t* mine = marks + (item & 3) * (S::kMarks / 4);
      const int low = min(it.past + by_group(p, it.r0) + 1, p.capacity);  // what the first row sees
      for (int t = it.t0; t < it.t1 && ok; ++t, ++n) {
        const int u = n & 1;
        if (!(ok = wait(&raw_full[stage], turn))) break;
        const uint32_t blocks = *reinterpret_cast<const volatile uint32_t*>(base + S::kOffPages +
                                                                            4 * (n % kScales));
        const int limit_in = it.limit - t * kPromptTile;
        uint32_t keep = (1u << NP) - 1u;
        if (blocks != 0xffu || limit_in < kPromptTile) {
          keep = 0u;
#pragma unroll
          for (int i = 0; i < NP; ++i)
            if ((blocks >> ((i * RPP + rr) >> 4) & 1u) && i * RPP + rr < limit_in) keep |= 1u << i;
        }
        if (n >= 2 && !(ok = wait(&k_empty[u], ((n >> 1) & 1) ^ 1u))) break;
        widen(sm + S::kOffK + u * S::kOperand, raw0 + stage * S::kRaw, keep);
        widened(&k_full[u]);
        if (!(ok = wait(&raw_full[stage], turn)) ||
            (n >= 2 && !(ok = wait(&v_empty[u], ((n >> 1) & 1) ^ 1u))))
          break;
        if ((t + 1) * kPromptTile > low && low < it.limit) {
          // Rows of the item end at different tokens here, and a NaN that one row
          // sees must not reach a row that does not (0 * NaN): NaN codes leave V,
          // and the outputs that they belong to are marked.
#pragma unroll 4
          for (int i = 0; i < NP; ++i) {
            if (!(keep >> i & 1u)) continue;
            if (!any_nan(lds128(raw0 + stage * S::kRaw + 2048 * i))) continue;
            const int tok = t * kPromptTile + i * RPP + rr;
#pragma unroll 1
            for (int k = 0; k < 4; ++k) {
              const uint32_t at = raw0 + stage * S::kRaw + 2048 * i + 4 * k;
              const uint32_t v = lds32(at);
              const uint32_t nan = nan_codes(v);
              if (nan == 0u) continue;
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(v & ~nan) : "memory");
              const uint32_t bits = ((nan & 1u) | (nan >> 7 & 2u) | (nan >> 14 & 4u) |
                                     (nan >> 21 & 8u)) << (16 * (c & 1) + 4 * k);
#pragma unroll 1
              for (int r = it.r0; r < min(it.n_rows, it.r0 + kRows); ++r)
                if (tok < min(it.past + by_group(p, r) + 1, p.capacity))
                  atomicOr(mine + (r - it.r0) * (D / 32) + (c >> 1), bits);
            }
          }
        }
        // (fence_async_shared in widened also stands between these stores and the next copy)
        widen(sm + S::kOffV + u * S::kOperand, raw0 + stage * S::kRaw, keep);
        widened(&v_full[u]);
      }
      done_item();
    }
  } else {
    // ------------------------------------------------------------ softmax
    more_registers<kSoftRegs>();
    const int stream = warp / kSoftWarps, r = tid % kPromptTile;  // row of the item
    const uint32_t lanes = (uint32_t)(32 * (warp % kSoftWarps)) << 16;  // its lanes of tensor memory
    const uint32_t tmem_s = tmem + lanes + stream * kPromptTile;
    float* mul_s = reinterpret_cast<float*>(base + S::kOffMul);
    float2* sums_s = reinterpret_cast<float2*>(base + S::kOffSums);
    bool prepares = stream == 1;  // the queries of the next item
    while (ok && next_item()) {
      const int row = it.r0 + r;
      const bool in = row < it.n_rows;
      const int qi = by_group(p, row);
      const int lim = in ? min(it.past + qi + 1, p.capacity) : 0;
      float q_mul;
      if (prepares) {
        // ---- this row's query, scaled to 2^14, as the A operand
        const uint16_t* src = p.q + (int64_t)(it.first + qi) * p.q_row +
                              (int64_t)(it.h * p.group + row - qi * p.group) * p.q_head;
        uint4 raw[D / 8];
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < D / 8; ++k)
          raw[k] = in ? reinterpret_cast<const uint4*>(src)[k] : make_uint4(0u, 0u, 0u, 0u);
        auto two = [&](uint32_t w) {
          if constexpr (BF16)
            return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
          else
            return __half22float2(*reinterpret_cast<const __half2*>(&w));
        };
#pragma unroll
        for (int k = 0; k < D / 8; ++k)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float2 f = two(reinterpret_cast<const uint32_t*>(&raw[k])[w]);
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 126);
        // (an infinite query has no softmax: NaN, as in the other kernel)
        const float up = amax <= 3.4028234e38f
                             ? copysignf(__uint_as_float((uint32_t)(14 - e + 127) << 23), p.scale_log2)
                             : __int_as_float(0x7fffffff);
        q_mul = fabsf(p.scale_log2) * __uint_as_float((uint32_t)(e - 14 + 127) << 23);
        mul_s[(item & 1) * kPromptTile + r] = q_mul;
        // the last item's last S, which the other stream's tile was
        if (n > 0 && !(ok = wait(&s_full[(n - 1) & 1], ((n - 1) >> 1) & 1))) break;
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          uint32_t o[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float2 f = two(reinterpret_cast<const uint32_t*>(&raw[k])[w]);
            o[w] = half2_bits(f.x * up, f.y * up);
          }
          sts128(sm + S::kOffQ + (k >> 3) * S::kHalf + operand_at(r, k & 7),
                 make_uint4(o[0], o[1], o[2], o[3]));
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[item & 1]);
      } else {
        if (!(ok = wait(&q_full[item & 1], (item >> 1) & 1))) break;
        q_mul = mul_s[(item & 1) * kPromptTile + r];
      }
      float m = -INFINITY;  // the running maximum that the stream's O and l are scaled by
      float l = 0.f;
      bool coarse = false;  // m's steps in fp32 are no small part of one, in some row
      int last = -1;        // the stream's last tile
      for (int t = it.t0; t < it.t1 && ok; ++t, ++n) {
        if ((n & 1) != stream) continue;
        if (!(ok = wait(&s_full[stream], (n >> 1) & 1))) break;
        tc_fence_after();
        const float4* sc = scale_s + (n % kScales) * 8;
        const int left = lim - t * kPromptTile;  // tokens of the tile that the row sees
        const bool cut = __any_sync(0xffffffffu, left < kPromptTile);
        // A row of S stays in registers from its maximum to its P'.
        float x[kPromptTile];
        tc_ld64(tmem_s, x);
        tc_ld64(tmem_s + 64, x + 64);
        if (cut) {
#pragma unroll
          for (int k = 0; k < kPromptTile; ++k)
            if (k >= left) x[k] = -INFINITY;
        }
        float top = -INFINITY;
        const uint32_t far = __float_as_uint(sc[0].w);
#pragma unroll
        for (int b = 0; b < 8; ++b) {  // the largest of a block, then its score: no factor is negative
          float t[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            t[k] = max3(max3(x[16 * b + k], x[16 * b + k + 4], x[16 * b + k + 8]),
                        x[16 * b + k + 12], -INFINITY);
          const float4 f = sc[b];
          top = fmaxf(top, fmaf(max3(max3(t[0], t[1], t[2]), t[3], -INFINITY),
                                fmaxf(f.x * q_mul, kLeast), f.y));
        }
        // ---- a row's maximum much larger: all rows' O and l move to theirs (the
        // stream's last product is done: S came after it)
        if (__any_sync(0xffffffffu, top > __fadd_rd(m, kGrowth))) {
          const float most = fmaxf(m, top);
          // (l's in two steps: between far scales it is below fp32, the product is not)
          const float root = m == -INFINITY ? 0.f : ex2(0.5f * (m - most)), al = root * root;
          m = most;
          coarse = __any_sync(0xffffffffu, fabsf(m) > 0x1p20f && m != -INFINITY);
          l *= root;
          l *= root;
          if (last >= 0) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              const uint32_t at = tmem_o + lanes + stream * kPromptTile + 32 * c;
              float o[32];
              tc_ld32(at, o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] *= al;
              tc_st32(at, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        const float sub = m == -INFINITY ? 0.f : __fadd_ru(m, -kPromptShift);
        // 64 columns of P' are in their place.
        auto stored = [&](int c) {
          if (c & 1) {
            tc_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(c == 1 ? &p_half[stream] : &p_full[stream]);
          }
        };
        last = n;
        if (coarse || far != 0u) {
          // Seldom. Scores whose steps in fp32 are no small part of one: the argument in one
          // rounding, with the maximum's two in `less`, could be off by several, so they get
          // the maximum's own rounding first. And scales so far apart that P' may vanish and
          // P' / sv not: the sum is made without it. S is read again: P' lies over what is read.
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float y[32];
            uint32_t w[16];
            tc_ld32(tmem_s + 32 * c, y);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const float4 f = sc[2 * c + b];
              const float ks = fmaxf(f.x * q_mul, kLeast);
              const bool apart = far >> (2 * c + b) & 1u;
              const float over = apart ? f.y : 0.f;
              float sum = 0.f;
#pragma unroll
              for (int k = 16 * b; k < 16 * b + 16; ++k) {
                const float a = 32 * c + k < left ? fmaf(y[k], ks, f.y) - sub : -INFINITY;
                y[k] = ex2(a);
                sum += ex2(a - over);
              }
#pragma unroll
              for (int k = 0; k < 8; ++k) w[8 * b + k] = half2_bits(y[16 * b + 2 * k], y[16 * b + 2 * k + 1]);
              l = fmaf(sum, apart ? 1.f : f.z, l);
            }
            tc_st16(tmem_s + 16 * c, w);
            stored(c);
          }
          continue;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const float4 f = sc[2 * c + b];
            const float ks = fmaxf(f.x * q_mul, kLeast), less = f.y - sub;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float a = ex2(fmaf(x[32 * c + 16 * b + 2 * k], ks, less)),
                          e = ex2(fmaf(x[32 * c + 16 * b + 2 * k + 1], ks, less));
              sum[k & 3] += a + e;
              w[8 * b + k] = half2_bits(a, e);
            }
            l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), f.z, l);
          }
          tc_st16(tmem_s + 16 * c, w);
          stored(c);
        }
      }
      if (!ok || (last >= 0 && !(ok = wait(&pv_done[stream], (last >> 1) & 1)))) break;
      // ---- the streams meet. The one without the item's last tile leaves maximum and
      // sum and prepares the next item's queries; the other one writes the item out.
      prepares = ((n - 1) & 1) != stream;
      if (prepares) {
        sums_s[(item & 1) * kPromptTile + r] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(b_done);
        done_item();
        continue;
      }
      if (!(ok = wait(b_done, item & 1))) break;
      tc_fence_after();
      const float2 other = sums_s[(item & 1) * kPromptTile + r];
      const float most = fmaxf(m, other.x);
      const float ra = m == -INFINITY ? 0.f : ex2(0.5f * (m - most)), fa = ra * ra;
      const float rb = other.x == -INFINITY ? 0.f : ex2(0.5f * (other.x - most)), fb = rb * rb;
      l = l * ra * ra + other.y * rb * rb;
      const bool has_b = it.t1 - it.t0 > 1;
      uint32_t* mine = marks + (item & 3) * (S::kMarks / 4) + r * (D / 32);  // this thread's alone
      const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
      uint16_t* dst = p.out + (int64_t)(it.first + qi) * p.out_row +
                      (int64_t)(it.h * p.group + row - qi * p.group) * p.out_head;
      float* part = p.parts + (((size_t)blockIdx.x * 2 + it.slot) * kRows + r) * S::kPitch;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32], o2[32];
        tc_ld32(tmem_o + lanes + stream * kPromptTile + 32 * c, o);
        if (has_b) tc_ld32(tmem_o + lanes + (stream ^ 1) * kPromptTile + 32 * c, o2);
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = o[k] * fa + (has_b ? o2[k] * fb : 0.f);
        const uint32_t mark = mine[c];
        if (mark) {
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (mark >> k & 1u) o[k] = __int_as_float(0x7fffffff);
          mine[c] = 0u;
        }
        if (!in) continue;
        if (it.whole) {
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float a = o[k + 2 * j] * inv, d = o[k + 2 * j + 1] * inv;
              if constexpr (BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(a, d);
                w[j] = *reinterpret_cast<const uint32_t*>(&h);
              } else {
                w[j] = half2_bits(a, d);
              }
            }
            *reinterpret_cast<uint4*>(dst + 32 * c + k) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            *reinterpret_cast<float4*>(part + 32 * c + k) =
                make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
        }
      }
      if (!it.whole && in) *reinterpret_cast<float2*>(part + D) = make_float2(most, l);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_empty);
      done_item();
    }
  }
  if (!ok && p.err) atomicCAS(p.err, 0, kErrPromptWait);
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tc_dealloc(tmem, 512);
  }
}

template <int D>
int launch_prompt(AttnP p, const DeviceInfo& di, cudaStream_t stream) {
  using S = PromptShape<D>;
  p.join = reinterpret_cast<Join*>(p.parts + (size_t)(kMaxCtas / 2) * 2 * kPromptTile * S::kPitch);
  // (16 tokens of 16 heads on 4 over 100: 12.9 us, with all CTAs 15.8; the other
  // kernel's CTAs are smaller, and fewer of them gain nothing)
  const int ctas = useful_ctas<Rows128>(p, std::min(kMaxCtas / 2, di.sm_count));
  cudaError_t e =
      launch_overlapped(p.bf16 ? kv8_prompt_kernel<D, true> : kv8_prompt_kernel<D, false>,
                        dim3((unsigned)ctas), kPromptThreads, S::kSmem, stream, p);
  if (e != cudaSuccess) return cuda_fail(e, "w4_kv8_attention prompt launch");
  e = launch_overlapped(kv8_join_kernel<D, kPromptTile>, dim3((unsigned)ctas, kPromptTile / kJoinWarps),
                        kJoinThreads, 0, stream, p);
  return e == cudaSuccess ? W4_OK : cuda_fail(e, "w4_kv8_attention join launch");
}

template <int D>
int init_prompt(const DeviceInfo& di) {
  constexpr int smem = PromptShape<D>::kSmem;
  if (smem > di.max_smem_optin)
    return fail(W4_ERR_UNSUPPORTED, "w4_kv8_attention needs %d B of shared memory", smem);
  cudaError_t e = cudaFuncSetAttribute(kv8_prompt_kernel<D, true>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kv8_prompt_kernel<D, false>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  return e == cudaSuccess ? W4_OK : cuda_fail(e, "cudaFuncSetAttribute(kv8 prompt)");
}

}  // namespace

size_t kv8_prompt_workspace_bytes(int head_dim) {
  return (size_t)(kMaxCtas / 2) * (2 * kPromptTile * (head_dim + 4) * 4 + sizeof(Join));
}

int kv8_prompt_init_device(const DeviceInfo& di) {
  const int st = init_prompt<64>(di);
  return st == W4_OK ? init_prompt<128>(di) : st;
}

int launch_kv8_prompt(AttnP p, int head_dim, const DeviceInfo& di, cudaStream_t stream) {
  return head_dim == 128 ? launch_prompt<128>(p, di, stream) : launch_prompt<64>(p, di, stream);
}

}  // namespace w4
