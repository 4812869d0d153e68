// w4_kv8_prompt.cu - attention over the paged 8-bit KV cache for many query
// rows a sequence (prompts, chunks of prompts), on the 5th-generation tensor
// cores.
//
// The maths, the split and the join are those of w4_kv8_attn.cu; there a step's
// few rows make the cache's bytes the bound, here 4 D operations a (row, token)
// pair do. An item is 128 query rows of one cache head (G query heads times the
// new tokens), worked through in tiles of 128 tokens by one CTA an SM, the tiles
// in turn by two streams that meet at the item's end:
//   4 widen warps  : the tile's pages by cp.async into shared memory, a tile ahead
//                    (a thread copies, waits for and reads its own chunks: no
//                    barrier); e4m3 to fp16 (exact) and back as MMA operands, K and V alike token by token in the 128B-swizzled
//                    layout (K is the K-major operand of Q K^T; of P V the same
//                    rows are the MN-major operand V, so nothing is transposed);
//   MMA warp       : one thread issues S = Q K^T of one stream (M = N = 128),
//                    then O += P V of the other, so that the tensor cores work
//                    for one while the other's softmax does;
//   2 x 4 softmax warps: a thread a row of its stream. S from tensor memory, the
//                    exponent's argument with the page's scales folded in (as in
//                    the other kernel), P' in fp16 back into tensor memory over
//                    the S that it came from. O stays in tensor memory, one a
//                    stream with a maximum of its own, and is rescaled only when
//                    a row's running maximum has grown by more than 2^3 since the
//                    last time (P' may then reach 2^14, inside fp16's range).
// Two O, two S (with P over them) fill the tensor memory: 4 x 128 columns. The
// exponentials are the floor of this split: 128 x 128 of them a tile at 16 a clock
// are 1024 clocks, as long as the tile's two products together at their best rate.
#include "w4_kv8_attn.cuh"

#include <algorithm>

namespace w4 {

namespace {

constexpr int kSoftWarps = 4, kWidenWarps = 4;  // softmax warps of a stream
constexpr int kWidenWarp = 2 * kSoftWarps;
constexpr int kMmaWarp = kWidenWarp + kWidenWarps;
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
  static constexpr int kPitch = D + 4;
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kOffQ + kOperand;          // two buffers
  static constexpr int kOffV = kOffK + 2 * kOperand;      // two buffers
  static constexpr int kRaw = kPromptTile * D;            // a K or V tile's codes
  static constexpr int kOffRaw = kOffV + 2 * kOperand;    // K, then V
  static constexpr int kOffScale = kOffRaw + 2 * kRaw;  // four tiles of 8 x (K, log2 V, 1 / V, 0)
  static constexpr int kOffMul = kOffScale + 4 * 8 * 16;  // a factor a row
  static constexpr int kOffSums = kOffMul + kPromptTile * 4;  // second stream's maxima and sums,
                                                              // two items in turn
  static constexpr int kOffMarks = kOffSums + 2 * kPromptTile * 8;
  static constexpr int kMarks = kPromptTile * D / 8;      // of an item; four items
  static constexpr int kOffBar = kOffMarks + 4 * kMarks;
  static constexpr int kBars = 7 * 2 + 3;
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
// The same with A in tensor memory: a lane a row, two elements a column.
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :
      : "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
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
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t* u) {
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
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(u[0]),
      "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]),
      "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(addr)
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
  // two of each, by stream (the parity of the tile)
  uint64_t* k_full = bars;        // widened K tile there (widen warps)
  uint64_t* k_empty = bars + 2;   // its product is done (commit)
  uint64_t* v_full = bars + 4;
  uint64_t* v_empty = bars + 6;
  uint64_t* s_full = bars + 8;    // S is in tensor memory (commit)
  uint64_t* p_full = bars + 10;   // P' is in its place, O is rescaled (softmax warps)
  uint64_t* pv_done = bars + 12;  // P V is done (commit)
  uint64_t* q_full = bars + 14;   // an item's queries are in shared memory (first stream)
  uint64_t* b_done = bars + 15;   // the second stream is through with an item
  uint64_t* o_empty = bars + 16;  // an item's outputs are read (first stream)
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
      mbar_init(&p_full[i], kSoftWarps);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(q_full, kSoftWarps);
    mbar_init(b_done, kSoftWarps);
    mbar_init(o_empty, kSoftWarps);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {  // all of it: two S, two O
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
  const uint32_t tmem_o = tmem + 2 * kPromptTile;  // O of stream u: + 128 u
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
      // O += P V of tile m, the first of its item and stream or not
      auto output = [&](int m, bool first) {
        const int u = m & 1;
        if (!wait(&p_full[u], (m >> 1) & 1) || !wait(&v_full[u], (m >> 1) & 1) ||
            (first && item > 0 && !wait(o_empty, (item - 1) & 1)))
          return false;
        after_sync();
        const uint64_t v_desc = operand_desc(sm + S::kOffV + u * S::kOperand, S::kHalf, 1024);
#pragma unroll
        for (int k = 0; k < kPromptTile / 16; ++k)  // 16 tokens: 8 columns of P, 16 rows of V
          mma_f16_ts(tmem_o + u * kPromptTile, tmem + u * kPromptTile + 8 * k,
                     v_desc + ((k * 16 * 128) >> 4), idesc_o, first && k == 0 ? 0u : 1u);
        __threadfence_block();  // the widen warps' marks, for those who wait for pv_done
        commit_to(&v_empty[u]);
        commit_to(&pv_done[u]);
        return true;
      };
      while (ok && walk.next(p)) {
        if (!(ok = wait(q_full, item & 1))) break;
        const int n0 = n;
        for (int t = walk.t0; t < walk.t1 && ok; ++t, ++n) {
          const int u = n & 1;
          // the stream's last P lies where this S goes
          ok = wait(&k_full[u], (n >> 1) & 1) &&
               (n < 2 || wait(&pv_done[u], ((n >> 1) & 1) ^ 1u));
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
          if (n > n0) ok = output(n - 1, n - 1 - n0 < 2);
        }
        if (ok) ok = output(n - 1, n - 1 - n0 < 2);
        ++item;
      }
    }
  } else if (warp >= kWidenWarp) {
    // ------------------------------------------------------------ widen
    constexpr int CPR = D / 16, RPP = 128 / CPR, NP = kPromptTile / RPP;  // chunks a row, rows a pass
    const int wt = tid - kWidenWarp * 32;
    const int c = wt % CPR, rr = wt / CPR;
    const uint32_t raw_k = sm + S::kOffRaw + 16 * wt, raw_v = raw_k + S::kRaw;  // + 2048 a pass
    const ptrdiff_t v_from_k = p.v - p.k;
    float sc_k = 0.f, sc_v = 0.f;  // scales of block wt of the loaded tile, threads 0 .. 7
    int ids = -1;         // lane 8 j + b: block b of tile t + j, j < 4
    Walk<G> next = walk;  // the item of the tile that is loaded
    bool more = next.next(p);
    int lt = more ? next.t0 : 0, id_at = 4;
    uint32_t real = 0u;   // bit i: the row of pass i has a page and is below the limit
    int64_t offs[NP];     // where its chunk lies
    // The next tile's K codes and its scales on their way, then (load_v) its V codes.
    auto load_k = [&]() {
      if (more) {
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
        if (wt < 8) {
          sc_k = sc_v = 0.f;  // no page
          if (id_b >= 0) {
            const size_t blk = (size_t)id_b * p.kv_heads + next.h;
            sc_k = p.k_scale[blk];
            sc_v = p.v_scale[blk];
          }
        }
        real = 0u;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int row = i * RPP + rr, tok = lt * kPromptTile + row;
          const int id = __shfl_sync(0xffffffffu, ids, 8 * id_at + (row >> 4));
          offs[i] = ((((int64_t)max(id, 0) * p.kv_heads + next.h) << p.page_shift) +
                     (tok & (p.page - 1))) * D + 16 * c;
          const bool is = id >= 0 && tok < next.limit;
          real |= (uint32_t)is << i;
          cp16_if(raw_k + 2048 * i, p.k + offs[i], is);
        }
      }
      cp_commit();
    };
    auto load_v = [&]() {
      if (more) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
          cp16_if(raw_v + 2048 * i, p.k + offs[i] + v_from_k, (real >> i & 1u) != 0u);
        ++id_at;
        if (++lt >= next.t1) {
          more = next.next(p);
          lt = next.t0;
          id_at = 4;
        }
      }
      cp_commit();
    };
    // 16 codes to two chunks of an operand row
    auto widen = [&](uint32_t to, int row, uint32_t from) {
      const uint4 v = lds128(from);
      const uint4 a = make_uint4(e4m3_lo(v.x), e4m3_hi(v.x), e4m3_lo(v.y), e4m3_hi(v.y));
      const uint4 b = make_uint4(e4m3_lo(v.z), e4m3_hi(v.z), e4m3_lo(v.w), e4m3_hi(v.w));
      const uint32_t half = to + (c >> 2) * S::kHalf;
      const int j = 2 * (c & 3), first = c >> 2;  // the halves' lanes write in other orders:
      sts128(half + operand_at(row, j + first), first ? b : a);  // no bank twice
      sts128(half + operand_at(row, j + 1 - first), first ? a : b);
    };
    load_k();
    load_v();
    while (ok && walk.next(p)) {
      const int n_rows = walk.s.n * p.group;
      const int cur_r0 = walk.rt * kRows;
      uint32_t* mine = marks + (item & 3) * (S::kMarks / 4);
      const int low = seen(p, walk.s, cur_r0);  // tokens that the first row sees
      for (int t = walk.t0; t < walk.t1 && ok; ++t, ++n) {
        const int u = n & 1;
        if (n >= 2 && !(ok = wait(&k_empty[u], ((n >> 1) & 1) ^ 1u))) break;
        if (wt < 8)  // the block's K scale, log2 and inverse of its V scale; no page: -inf
          reinterpret_cast<float4*>(base + S::kOffScale)[(n & 3) * 8 + wt] =
              sc_v > 0.f ? make_float4(sc_k, lg2(sc_v), 1.0f / sc_v, 0.f)
                         : make_float4(0.f, -INFINITY, 0.f, 0.f);
        cp_wait<1>();  // K's copies
#pragma unroll
        for (int i = 0; i < NP; ++i)
          widen(sm + S::kOffK + u * S::kOperand, i * RPP + rr, raw_k + 2048 * i);
        to_async_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_full[u]);
        load_k();
        if (n >= 2 && !(ok = wait(&v_empty[u], ((n >> 1) & 1) ^ 1u))) break;
        cp_wait<1>();  // V's
        if ((t + 1) * kPromptTile > low && low < walk.limit) {
          // Rows of the item end at different tokens here, and a NaN that one row
          // sees must not reach a row that does not (0 * NaN): NaN codes leave V,
          // and the outputs that they belong to are marked.
#pragma unroll 1
          for (int i = 0; i < NP; ++i) {
            const int tok = t * kPromptTile + i * RPP + rr;
#pragma unroll 1
            for (int k = 0; k < 4; ++k) {
              const uint32_t at = raw_v + 2048 * i + 4 * k;
              const uint32_t v = lds32(at);
              const uint32_t nan = __vcmpeq4(v & 0x7f7f7f7fu, 0x7f7f7f7fu);
              if (nan == 0u) continue;
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(v & ~nan) : "memory");
              const uint32_t bits = ((nan & 1u) | (nan >> 7 & 2u) | (nan >> 14 & 4u) |
                                     (nan >> 21 & 8u)) << (16 * (c & 1) + 4 * k);
#pragma unroll 1
              for (int r = cur_r0; r < min(n_rows, cur_r0 + kRows); ++r)
                if (tok < seen(p, walk.s, r))
                  atomicOr(mine + (r - cur_r0) * (D / 32) + (c >> 1), bits);
            }
          }
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < NP; ++i)
          widen(sm + S::kOffV + u * S::kOperand, i * RPP + rr, raw_v + 2048 * i);
        to_async_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[u]);
        load_v();
      }
      ++item;
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int stream = warp / kSoftWarps, r = tid % kPromptTile;  // row of the item
    const uint32_t lanes = (uint32_t)(32 * (warp % kSoftWarps)) << 16;  // its lanes of tensor memory
    const uint32_t tmem_s = tmem + lanes + stream * kPromptTile;
    float* mul_s = reinterpret_cast<float*>(base + S::kOffMul);
    float2* sums_s = reinterpret_cast<float2*>(base + S::kOffSums);
    while (ok && walk.next(p)) {
      const int n_rows = walk.s.n * p.group;
      const int row = walk.rt * kRows + r;
      const bool in = row < n_rows;
      const int qi = by_group(p, row);
      const int lim = in ? seen(p, walk.s, row) : 0;
      float q_mul;
      if (stream == 0) {
        // ---- this row's query, scaled to 2^14, as the A operand. The last item's
        // products are done: both streams are through with it.
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
        mul_s[r] = q_mul;
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
        to_async_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      } else {
        if (!(ok = wait(q_full, item & 1))) break;
        q_mul = mul_s[r];
      }
      float m = -INFINITY;  // the running maximum that the stream's O and l are scaled by
      float l = 0.f;
      int last = -1;        // the stream's last tile
      for (int t = walk.t0; t < walk.t1 && ok; ++t, ++n) {
        if ((n & 1) != stream) continue;
        if (!(ok = wait(&s_full[stream], (n >> 1) & 1))) break;
        after_sync();
        const float4* sc = scale_s + (n & 3) * 8;
        const int left = lim - t * kPromptTile;  // tokens of the tile that the row sees
        const bool cut = __any_sync(0xffffffffu, left < kPromptTile);
        // Columns 32 c .. + 31 of S to log2 units with the value scale, masked. Read
        // twice, for the maximum and for P': 128 registers a thread are what two
        // streams leave.
        float x[32];
        auto scores = [&](int c) {
          ld32(tmem_s + 32 * c, x);
          ld_wait();
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const float4 f = sc[2 * c + b];
            const float ks = f.x * q_mul;
#pragma unroll
            for (int k = 0; k < 16; ++k) x[16 * b + k] = fmaf(x[16 * b + k], ks, f.y);
          }
          if (cut) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (32 * c + k >= left) x[k] = -INFINITY;
          }
        };
        float tops[8];  // chains side by side
#pragma unroll
        for (int k = 0; k < 8; ++k) tops[k] = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          scores(c);
#pragma unroll
          for (int k = 0; k < 32; ++k) tops[k & 7] = fmaxf(tops[k & 7], x[k]);
        }
        const float top = fmaxf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])),
                                fmaxf(fmaxf(tops[4], tops[5]), fmaxf(tops[6], tops[7])));
        // ---- a row's maximum much larger: all rows' O and l move to theirs (the
        // stream's last product is done: S came after it)
        if (__any_sync(0xffffffffu, top > m + kGrowth)) {
          const float most = fmaxf(m, top);
          const float al = m == -INFINITY ? 0.f : ex2(m - most);
          m = most;
          l *= al;
          if (last >= 0) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              const uint32_t at = tmem_o + lanes + stream * kPromptTile + 32 * c;
              float o[32];
              ld32(at, o);
              ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] *= al;
              st32(at, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        const float sub = m == -INFINITY ? 0.f : m - kPromptShift;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          scores(c);
          uint32_t w[16];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float a = ex2(x[16 * b + 2 * k] - sub), d = ex2(x[16 * b + 2 * k + 1] - sub);
              sum[k & 3] += a + d;
              w[8 * b + k] = half2_bits(a, d);
            }
            l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), sc[2 * c + b].z, l);
          }
          st16(tmem_s + 16 * c, w);  // over columns that have been read
        }
        st_wait();
        before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[stream]);
        last = n;
      }
      if (!ok || (last >= 0 && !(ok = wait(&pv_done[stream], (last >> 1) & 1)))) break;
      // ---- the streams meet: the second one leaves maximum and sum
      if (stream == 1) {
        sums_s[(item & 1) * kPromptTile + r] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(b_done);
        ++item;
        continue;
      }
      if (!(ok = wait(b_done, item & 1))) break;
      after_sync();
      const float2 other = sums_s[(item & 1) * kPromptTile + r];
      const float most = fmaxf(m, other.x);
      const float fa = m == -INFINITY ? 0.f : ex2(m - most);
      const float fb = other.x == -INFINITY ? 0.f : ex2(other.x - most);
      l = l * fa + other.y * fb;
      const bool has_a = last >= 0, has_b = walk.t1 - walk.t0 > 1 || !has_a;
      uint32_t* mine = marks + (item & 3) * (S::kMarks / 4) + r * (D / 32);  // this thread's alone
      const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
      uint16_t* dst = p.out + (int64_t)(walk.s.first + qi) * p.out_row +
                      (int64_t)(walk.h * p.group + row - qi * p.group) * p.out_head;
      float* part = p.parts + (((size_t)blockIdx.x * 2 + walk.slot(share)) * kRows + r) * S::kPitch;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32], o2[32];
        if (has_a) ld32(tmem_o + lanes + 32 * c, o);
        if (has_b) ld32(tmem_o + lanes + kPromptTile + 32 * c, o2);
        ld_wait();
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = (has_a ? o[k] * fa : 0.f) + (has_b ? o2[k] * fb : 0.f);
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
        if (in) *reinterpret_cast<float2*>(part + D) = make_float2(most, l);
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
