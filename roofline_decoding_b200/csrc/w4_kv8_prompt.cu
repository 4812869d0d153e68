// w4_kv8_prompt.cu - attention over the paged 8-bit KV cache for many query
// rows a sequence (prompts, chunks of prompts), on the 5th-generation tensor
// cores.
//
// The maths, the split and the join are those of w4_kv8_attn.cu; there a step's
// few rows make the cache's bytes the bound, here 4 D operations a (row, token)
// pair do. An item is 128 query rows of one cache head (G query heads times the
// new tokens), worked through in tiles of 128 tokens by one CTA an SM:
//   4 widen warps  : the tile's pages from global memory into registers, a tile
//                    ahead; e4m3 to fp16 (exact) and into shared memory as MMA
//                    operands, K and V alike token by token in the 128B-swizzled
//                    layout (K is the K-major operand of Q K^T; of P V the same
//                    rows are the MN-major operand V, so nothing is transposed);
//   MMA warp       : one thread issues S = Q K^T (M = N = 128) of tile i + 1
//                    before O += P V of tile i, so that the tensor cores work
//                    while the softmax does;
//   4 softmax warps: a thread a row. S from tensor memory, the exponent's
//                    argument with the page's scales folded in (as in the other
//                    kernel), P' in fp16 into shared memory. O stays in tensor
//                    memory; it is rescaled only when the running maximum has
//                    grown by more than 2^3 since the last time (P' may then
//                    reach 2^14, inside fp16's range).
// S and the widened tiles are double-buffered. The exponentials are the floor of
// this split: 128 x 128 of them a tile at 16 a clock are 1024 clocks, as long as
// the tile's two products together at their best rate.
#include "w4_kv8_attn.cuh"

#include <algorithm>

namespace w4 {

namespace {

constexpr int kSoftWarps = 4, kWidenWarps = 4;
constexpr int kMmaWarp = kSoftWarps + kWidenWarps;
constexpr int kPromptThreads = 32 * (kMmaWarp + 1);
constexpr int kPromptTile = 128;   // tokens of a tile, and rows of an item
constexpr float kPromptShift = 11.0f;  // P' of the maximum that O is scaled by is 2^kPromptShift
constexpr float kGrowth = 3.0f;        // the running maximum may exceed it by this much
constexpr int kErrPromptWait = 9;

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
  // Length of row tile rt: above kOver + kUnit * tiles for every limit.
  static __device__ __forceinline__ int64_t first(const AttnP& p, const Seq& s) {
    return (int64_t)kOver + s.past + step(p) + kUnit;
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
    *len = first(p, s) + step(p) * r;
  }
};

template <int D>
struct PromptShape {
  static constexpr int kHalf = kPromptTile * 128;         // 128 rows of 64 fp16
  static constexpr int kOperand = kHalf * (D / 64);       // Q, or a K or V tile
  static constexpr int kP = kPromptTile * kPromptTile * 2;
  static constexpr int kPitch = D + 4;
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kOffQ + kOperand;          // two buffers
  static constexpr int kOffV = kOffK + 2 * kOperand;      // two buffers
  static constexpr int kOffP = kOffV + 2 * kOperand;
  static constexpr int kOffScale = kOffP + kP;            // four tiles of 8 x (K, log2 V, 1 / V, 0)
  static constexpr int kOffMarks = kOffScale + 4 * 8 * 16;
  static constexpr int kMarks = kPromptTile * D / 8;      // of an item; four items
  static constexpr int kOffBar = kOffMarks + 4 * kMarks;
  static constexpr int kBars = 2 + 2 + 2 + 2 + 2 + 2 + 1 + 1 + 1 + 1;
  static constexpr int kOffTmem = kOffBar + kBars * 8;
  static constexpr int kSmem = 1024 + kOffTmem + 16;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// ------------------------------------------------------------ tcgen05

__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  // 128B swizzle, version 1; offsets in bytes
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 |
         (uint64_t)((sbo >> 4) & 0x3FFFu) << 32 | (uint64_t)1u << 46 | (uint64_t)2u << 61;
}
// kind::f16, fp16 operands, fp32 sums, M = 128; b_mn: B is MN-major.
__host__ __device__ constexpr uint32_t prompt_idesc(int n, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :
      : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_to(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void before_sync() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void after_sync() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void to_async_proxy() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// 32 columns of this warp's 32 lanes; several loads may be in flight until ld_wait.
__device__ __forceinline__ void ld32(uint32_t addr, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
        "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
        "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]),
        "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]),
        "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr));
}
__device__ __forceinline__ void ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void st32(uint32_t addr, const float* r) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(r);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(
          u[0]),
      "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]),
      "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]),
      "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]),
      "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]),
      "r"(u[30]), "r"(u[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Byte offset of 16-byte chunk c (8 fp16) of row r in an operand half.
__device__ __forceinline__ uint32_t operand_at(int r, int c) {
  return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
}
__device__ __forceinline__ void sts128(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

template <int D>
__global__ void __launch_bounds__(kPromptThreads, 1) kv8_prompt_kernel(const AttnP p) {
  using S = PromptShape<D>;
  using G = Rows128;
  constexpr int kRows = kPromptTile;
  extern __shared__ uint8_t smem_prompt[];
  uint8_t* base = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_prompt) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sm = smem_u32(base);
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + S::kOffBar);
  uint64_t* k_full = bars;          // [2] widened K tile there (widen warps)
  uint64_t* k_empty = bars + 2;     // [2] its product is done (commit)
  uint64_t* v_full = bars + 4;      // [2]
  uint64_t* v_empty = bars + 6;     // [2]
  uint64_t* s_full = bars + 8;      // [2] S of a tile is in tensor memory (commit)
  uint64_t* s_empty = bars + 10;    // [2] the softmax threads have read it, and the tile's scales
  uint64_t* p_full = bars + 12;     // P' is in shared memory, O is rescaled
  uint64_t* pv_done = bars + 13;    // P V of a tile is done (commit)
  uint64_t* q_full = bars + 14;     // an item's queries are in shared memory
  uint64_t* o_empty = bars + 15;    // an item's output is read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base + S::kOffTmem);
  int* abort_flag = reinterpret_cast<int*>(base + S::kOffTmem + 4);
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
      mbar_init(&s_empty[i], kSoftWarps);
    }
    mbar_init(p_full, kSoftWarps);
    mbar_init(pv_done, 1);
    mbar_init(q_full, kSoftWarps);
    mbar_init(o_empty, kSoftWarps);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {  // S twice 128 columns, O: 512 is the next size that there is
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    before_sync();
  }
  for (int i = tid; i < S::kMarks; i += kPromptThreads) marks[i] = 0u;
  grid_dependency_wait();
  grid_launch_dependents();
  const Share share = find_share<G>(p);
  if (tid == 0) p.join[blockIdx.x].count = 0;
  __syncthreads();
  after_sync();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_o = tmem + 256;
  // A wait that gives up ends its role; the others give up in turn.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_wait(bar, parity)) return true;
    if (p.err) atomicCAS(p.err, 0, kErrPromptWait);
    *reinterpret_cast<volatile int*>(abort_flag) = 1;
    return false;
  };

  Walk<G> walk;
  walk.start(share);
  int n = 0;     // tiles that this CTA has begun, over all items
  int item = 0;  // items
  bool ok = true;

  if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA
    if (lane == 0) {
      constexpr uint32_t idesc_s = prompt_idesc(kPromptTile, 0), idesc_o = prompt_idesc(D, 1);
      const uint64_t q_desc = operand_desc(sm + S::kOffQ, 16, 1024);
      const uint64_t p_desc = operand_desc(sm + S::kOffP, 16, 1024);
      // O += P V of tile m, the first of its item or not
      auto output = [&](int m, bool first) {
        const int u = m & 1;
        if (!wait(p_full, m & 1) || !wait(&v_full[u], (m >> 1) & 1) ||
            (first && item > 0 && !wait(o_empty, (item - 1) & 1)))
          return false;
        after_sync();
        const uint64_t v_desc = operand_desc(sm + S::kOffV + u * S::kOperand, S::kHalf, 1024);
#pragma unroll
        for (int k = 0; k < kPromptTile / 16; ++k)  // 16 tokens: 32 bytes of P, 16 rows of V
          mma_f16(tmem_o, p_desc + (((k >> 2) * S::kHalf + (k & 3) * 32) >> 4),
                  v_desc + ((k * 16 * 128) >> 4), idesc_o, first && k == 0 ? 0u : 1u);
        __threadfence_block();  // the widen warps' marks, for those who wait for pv_done
        commit_to(&v_empty[u]);
        commit_to(pv_done);
        return true;
      };
      while (ok && walk.next(p)) {
        if (!(ok = wait(q_full, item & 1))) break;
        const int tiles = walk.t1 - walk.t0;
        for (int i = 0; i < tiles && ok; ++i, ++n) {
          const int u = n & 1;
          ok = wait(&k_full[u], (n >> 1) & 1) &&
               (n < 2 || wait(&s_empty[u], ((n >> 1) & 1) ^ 1u));
          if (!ok) break;
          after_sync();
          const uint64_t k_desc = operand_desc(sm + S::kOffK + u * S::kOperand, 16, 1024);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {  // 16 dims: 32 bytes along the swizzled rows
            const uint32_t at = ((k >> 2) * S::kHalf + (k & 3) * 32) >> 4;
            mma_f16(tmem + u * kPromptTile, q_desc + at, k_desc + at, idesc_s, k > 0);
          }
          __threadfence_block();  // the widen warps' scales, for those who wait for s_full
          commit_to(&k_empty[u]);
          commit_to(&s_full[u]);
          if (i > 0) ok = output(n - 1, i == 1);
        }
        if (ok) ok = output(n - 1, tiles == 1);
        ++item;
      }
    }
  } else if (warp >= kSoftWarps) {
    // ------------------------------------------------------------ widen
    constexpr int CPR = D / 16, RPP = 128 / CPR, NP = kPromptTile / RPP;  // chunks a row, rows a pass
    const int wt = tid - kSoftWarps * 32;
    const int c = wt % CPR, rr = wt / CPR;
    uint4 kr[NP], vr[NP];
    int ids = -1;       // lane 8 j + b: block b of tile t + j, j < 4
    Walk<G> next = walk;  // the item of the tile that is loaded
    bool more = next.next(p);
    int lt = more ? next.t0 : 0, id_at = 4;
    // Loads the next tile's bytes, and writes its scales to slot m & 3.
    auto load = [&](int m) {
      if (!more) return;
      if (id_at == 4) {
        const int tok = (lt + (lane >> 3)) * kPromptTile + 16 * (lane & 7);
        ids = -1;
        if (lt + (lane >> 3) < next.t1 && tok < next.limit) {
          const int pi = tok >> p.page_shift;
          if (pi < p.max_pages) ids = p.page_table[next.b * p.table_stride + pi];
          if ((uint32_t)ids >= (uint32_t)p.pages) {
            ids = -1;
            atomicCAS(p.err, 0, kErrKvRange);
          }
        }
        id_at = 0;
      }
      const int id_b = __shfl_sync(0xffffffffu, ids, 8 * id_at + (lane & 7));
      if (wt < 8) {  // a block's scales; no page: a score of minus infinity
        const int id = id_b;
        float4 sc = make_float4(0.f, -INFINITY, 0.f, 0.f);
        if (id >= 0) {
          const size_t blk = (size_t)id * p.kv_heads + next.h;
          const float vs = p.v_scale[blk];
          sc = vs > 0.f ? make_float4(p.k_scale[blk], lg2(vs), 1.0f / vs, 0.f) : sc;
        }
        reinterpret_cast<float4*>(base + S::kOffScale)[(m & 3) * 8 + wt] = sc;
      }
      const int tok0 = lt * kPromptTile;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int row = i * RPP + rr, tok = tok0 + row;
        const int id = __shfl_sync(0xffffffffu, ids, 8 * id_at + (row >> 4));
        const bool real = id >= 0 && tok < next.limit;
        const size_t at = ((((size_t)max(id, 0) * p.kv_heads + next.h) << p.page_shift) +
                           (tok & (p.page - 1))) * D + 16 * c;
        kr[i] = vr[i] = make_uint4(0u, 0u, 0u, 0u);
        if (real) {
          kr[i] = __ldg(reinterpret_cast<const uint4*>(p.k + at));
          vr[i] = __ldg(reinterpret_cast<const uint4*>(p.v + at));
        }
      }
      ++id_at;
      if (++lt >= next.t1) {
        more = next.next(p);
        lt = next.t0;
        id_at = 4;
      }
    };
    // 16 codes to two chunks of an operand row
    auto widen = [&](uint32_t to, int row, const uint4& v) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
      const uint4 a = make_uint4(e4m3_lo(w[0]), e4m3_hi(w[0]), e4m3_lo(w[1]), e4m3_hi(w[1]));
      const uint4 b = make_uint4(e4m3_lo(w[2]), e4m3_hi(w[2]), e4m3_lo(w[3]), e4m3_hi(w[3]));
      const uint32_t half = to + (c >> 2) * S::kHalf;
      const int j = 2 * (c & 3), first = c >> 2;  // the halves' lanes write in other orders:
      sts128(half + operand_at(row, j + first), first ? b : a);  // no bank twice
      sts128(half + operand_at(row, j + 1 - first), first ? a : b);
    };
    load(0);
    while (ok && walk.next(p)) {
      const int n_rows = walk.s.n * p.group;
      const int cur_r0 = walk.rt * kRows;
      uint32_t* mine = marks + (item & 3) * (S::kMarks / 4);
      const int low = seen(p, walk.s, cur_r0);  // tokens that the first row sees
      for (int t = walk.t0; t < walk.t1 && ok; ++t, ++n) {
        const int u = n & 1;
        if (n >= 2 && !(ok = wait(&k_empty[u], ((n >> 1) & 1) ^ 1u))) break;
#pragma unroll
        for (int i = 0; i < NP; ++i) widen(sm + S::kOffK + u * S::kOperand, i * RPP + rr, kr[i]);
        to_async_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_full[u]);
        if (n >= 2 && !(ok = wait(&v_empty[u], ((n >> 1) & 1) ^ 1u))) break;
        const bool mixed = (t + 1) * kPromptTile > low && low < walk.limit;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          uint4 v = vr[i];
          if (mixed) {
            // A NaN that one row of the item sees must not reach a row that does
            // not (0 * NaN): NaN codes leave V, and the outputs that they belong
            // to are marked.
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t nan = __vcmpeq4(w[k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              if (nan == 0u) continue;
              w[k] &= ~nan;
              const uint32_t bits = ((nan & 1u) | (nan >> 7 & 2u) | (nan >> 14 & 4u) |
                                     (nan >> 21 & 8u)) << (16 * (c & 1) + 4 * k);
              const int tok = t * kPromptTile + i * RPP + rr;
#pragma unroll 1
              for (int r = cur_r0; r < min(n_rows, cur_r0 + kRows); ++r)
                if (tok < seen(p, walk.s, r))
                  atomicOr(mine + (r - cur_r0) * (D / 32) + (c >> 1), bits);
            }
          }
          widen(sm + S::kOffV + u * S::kOperand, i * RPP + rr, v);
        }
        to_async_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[u]);
        load(n + 1);
      }
      ++item;
    }
  } else {
    // ------------------------------------------------------------ softmax
    const uint32_t lanes = (uint32_t)(32 * warp) << 16;  // this warp's lanes of tensor memory
    while (ok && walk.next(p)) {
      const int n_rows = walk.s.n * p.group;
      const int row = walk.rt * kRows + tid;
      const bool in = row < n_rows;
      const int qi = by_group(p, row);
      const int lim = in ? seen(p, walk.s, row) : 0;
      // ---- this row's query, scaled to 2^14, as the A operand. The last item's
      // products are done: its last S has been read.
      float q_mul;
      {
        const uint16_t* src = p.q + (int64_t)(walk.s.first + qi) * p.q_row +
                              (int64_t)(walk.h * p.group + row - qi * p.group) * p.q_head;
        uint4 raw[D / 8];
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < D / 8; ++k)
          raw[k] = in ? __ldg(reinterpret_cast<const uint4*>(src) + k) : make_uint4(0u, 0u, 0u, 0u);
        auto two = [&](uint32_t w) {
          return p.bf16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u))
                        : __half22float2(*reinterpret_cast<const __half2*>(&w));
        };
#pragma unroll
        for (int k = 0; k < D / 8; ++k)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float2 f = two(reinterpret_cast<const uint32_t*>(&raw[k])[w]);
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 126);
        const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
        q_mul = p.scale_log2 * __uint_as_float((uint32_t)(e - 14 + 127) << 23);
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          uint32_t o[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float2 f = two(reinterpret_cast<const uint32_t*>(&raw[k])[w]);
            o[w] = half2_bits(f.x * up, f.y * up);
          }
          sts128(sm + S::kOffQ + (k >> 3) * S::kHalf + operand_at(tid, k & 7),
                 make_uint4(o[0], o[1], o[2], o[3]));
        }
        to_async_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }
      float m = -INFINITY;  // the running maximum that O and l are scaled by
      float l = 0.f;
      const int n0 = n;
      for (int t = walk.t0; t < walk.t1 && ok; ++t, ++n) {
        const int u = n & 1;
        if (!(ok = wait(&s_full[u], (n >> 1) & 1))) break;
        after_sync();
        float x[kPromptTile];
#pragma unroll
        for (int c = 0; c < 4; ++c) ld32(tmem + lanes + u * kPromptTile + 32 * c, x + 32 * c);
        ld_wait();
        const float4* sc = scale_s + (n & 3) * 8;
        const int left = lim - t * kPromptTile;  // tokens of the tile that the row sees
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          const float4 f = sc[b];
          const float ks = f.x * q_mul;
#pragma unroll
          for (int k = 0; k < 16; ++k) x[16 * b + k] = fmaf(x[16 * b + k], ks, f.y);
        }
        if (__any_sync(0xffffffffu, left < kPromptTile)) {
#pragma unroll
          for (int k = 0; k < kPromptTile; ++k)
            if (k >= left) x[k] = -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < kPromptTile; ++k) top = fmaxf(top, x[k]);
        // ---- a much larger maximum: O and l move to it
        const bool grow = top > m + kGrowth;  // also from minus infinity
        const bool any_grow = __any_sync(0xffffffffu, grow);
        // P V of the tile before: P' may be overwritten, O is at rest
        if (n > n0 && !(ok = wait(pv_done, (n - 1) & 1))) break;
        after_sync();
        if (any_grow) {
          const float al = grow ? (m == -INFINITY ? 0.f : ex2(m - top)) : 1.f;
          if (grow) m = top;
          l *= al;
          if (n > n0) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              ld32(tmem_o + lanes + 32 * c, o);
              ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] *= al;
              st32(tmem_o + lanes + 32 * c, o);
            }
            st_wait();
          }
        }
        const float sub = m == -INFINITY ? 0.f : m - kPromptShift;
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          float sum = 0.f;
          uint32_t w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float a = ex2(x[16 * b + 2 * k] - sub), d = ex2(x[16 * b + 2 * k + 1] - sub);
            sum += a + d;
            w[k] = half2_bits(a, d);
          }
          l = fmaf(sum, sc[b].z, l);
          const uint32_t to = sm + S::kOffP + (b >> 2) * S::kHalf;
          sts128(to + operand_at(tid, 2 * (b & 3)), make_uint4(w[0], w[1], w[2], w[3]));
          sts128(to + operand_at(tid, 2 * (b & 3) + 1), make_uint4(w[4], w[5], w[6], w[7]));
        }
        to_async_proxy();
        before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s_empty[u]);
          mbar_arrive(p_full);
        }
      }
      if (!ok) break;
      // ---- the item's output, or the part of it
      if (!(ok = wait(pv_done, (n - 1) & 1))) break;
      after_sync();
      uint32_t* mine = marks + (item & 3) * (S::kMarks / 4) + tid * (D / 32);  // this thread's alone
      const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
      uint16_t* dst = p.out + (int64_t)(walk.s.first + qi) * p.out_row +
                      (int64_t)(walk.h * p.group + row - qi * p.group) * p.out_head;
      float* part = p.parts + (((size_t)blockIdx.x * 2 + walk.slot(share)) * kRows + tid) * S::kPitch;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        ld32(tmem_o + lanes + 32 * c, o);
        ld_wait();
        const uint32_t mark = mine[c];
        if (mark) {
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (mark >> k & 1u) o[k] = __int_as_float(0x7fffffff);
          mine[c] = 0u;
        }
        if (!in) continue;
        if (walk.whole) {
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float a = o[k + 2 * j] * inv, d = o[k + 2 * j + 1] * inv;
              if (p.bf16) {
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
      if (!walk.whole) {
        // in the other kernel's terms the maximum is m, with P' scaled by 2^14:
        // only the ratio of outputs and sum counts
        if (in) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
        if (tid == 0) walk.describe(p, share);
      }
      before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_empty);
      ++item;
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
  }
}

template <int D>
int launch_prompt(AttnP p, const DeviceInfo& di, cudaStream_t stream) {
  using S = PromptShape<D>;
  p.join = reinterpret_cast<Join*>(p.parts + (size_t)(kMaxCtas / 2) * 2 * kPromptTile * S::kPitch);
  const int ctas = std::min(kMaxCtas / 2, di.sm_count);
  cudaError_t e = launch_overlapped(kv8_prompt_kernel<D>, dim3((unsigned)ctas), kPromptThreads,
                                    S::kSmem, stream, p);
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
  const cudaError_t e = cudaFuncSetAttribute(kv8_prompt_kernel<D>,
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
