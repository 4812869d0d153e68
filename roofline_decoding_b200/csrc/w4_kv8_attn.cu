// w4_kv8_attn.cu - attention of a step's queries over the paged 8-bit KV cache.
//
//   o_r = sum_j softmax_j(scale q_r . (sk_j k_j)) sv_j v_j,  j < limit(r)
//
// with e4m3 codes k_j, v_j, and sk_j, sv_j the scales of their page and head.
// The query rows of one cache head (G query heads times the sequence's new
// tokens) form tiles of 8 or 16 rows; an item is (sequence, cache head, row
// tile), and its work is its 32-token tiles of the cache.
//
// Bound by the cache's bytes at the small row counts of decoding (2 D bytes a
// token and cache head against 4 D operations a query row), so the design is
// about streaming: every warp runs alone on its own ring of tiles (cp.async,
// 16 bytes a lane, no barrier between warps in the loop) and holds its own
// running maximum, sum and output; the CTA's warps merge once an item.
//
// Work split: the tiles of all items are numbered in one line and every CTA
// takes an equal, contiguous share, found on the device from the lengths: no
// length is needed on the host, a captured launch follows new lengths, and
// ragged sequences balance. An item cut by the border of two shares leaves
// fp32 partials that a second, programmatically dependent launch joins in
// order; nothing is atomic, so results repeat bit for bit.
//
// Arithmetic: mma.sync m16n8k16 in fp16 with fp32 sums, transposed: the cache
// is the 16-wide operand (S^T = K Q^T, O^T = V^T P^T) and the query rows the
// 8-wide one, so that a decoding step's few rows leave little of a product
// unused, every widened K or V register serves all row blocks, and softmax and
// output take half the registers of the 16-row form (some 600 instead of 900
// instructions a tile, all counted). P^T turns from result to operand by movmatrix. e4m3
// widens to fp16 exactly. Queries enter scaled by a power of two a row that
// brings their largest element to 2^14 (bf16 to fp16 is then exact but for
// elements 2^-28 below the row's largest). The page's value scale is folded
// into the exponent: P' = exp2(s + log2 sv - m + 14) with m the running maximum
// of s + log2 sv, so P' is at most 2^14, its rounding to fp16 (11 bits) stays
// relative down to 2^-28 of the largest weight, and the fp32 sum adds
// P' / sv, unrounded (where scales lie so far apart that P' may vanish and
// P' / sv not, exp2(s - m + 14) itself).
//
// 32 sequences of up to 32768 tokens, 32 heads on 8 of 128: 173 us, 6.4 TB/s. A
// single token over 700, 12 heads on 2: 8.6 us, the latency of two launches and of
// length, page number, tile, products and merge.
#include "w4_kv8_attn.cuh"

#include <algorithm>

namespace w4 {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;        // tokens of one ring stage of a warp
constexpr int kCtasPerSm = 2;
constexpr float kShift = 14.0f;  // P' is at most 2^kShift

// From this many query rows of a cache head a sequence (on average) on, the other
// kernel. This one and the other one, 32 heads on 8 of 128: 64 sequences over 1000 tokens
// with 34 rows 68.9 and 82.9 us, with 66 117 and 89; 8 over 2000 with 34 rows 25.7 and
// 29.5, 50 31.2 and 30.5, 66 38.8 and 32.4; one over 2000 with 64 15.9 and 18.3, with 256
// 26.6 and 24.0.
// The average is all that the host knows. A step that mixes is better called in two
// parts, by sequences: 31 of one row and one of 2048 over 4096 tokens 420 us, apart 48 and
// 260; 63 of one row and one of 512 over 1000 118, apart 33 and 34.
constexpr int kPromptRows = 64;

// Every row tile of a sequence counts as long as its last (the few tiles above a
// row tile's own limit are passed over), in tiles.
template <int NT>
struct Rows8 {
  static constexpr int kRows = 8 * NT;
  static constexpr int kTile = w4::kTile;
  static constexpr int kUnit = 1;
  static constexpr int kOver = 12;           // so that a CTA of many short items does not end last
                                             // (64 sequences of 1500 at most: 29 us, with 4 39)
  static constexpr int kMinShare = kWarps;   // below a tile a warp, more CTAs only add partials
  static constexpr int kCut = 0;             // equal shares always
  static __device__ __forceinline__ int tiles(const AttnP& p, const Seq& s, int) {
    return (min(s.past + s.n, p.capacity) + kTile - 1) / kTile;
  }
  static __device__ __forceinline__ int row_tiles(const AttnP& p, const Seq& s) {
    return (s.n * p.group + kRows - 1) / kRows;
  }
  static __device__ __forceinline__ int64_t seq_work(const AttnP& p, const Seq& s) {
    return s.n > 0 ? (int64_t)p.kv_heads * row_tiles(p, s) * (tiles(p, s, 0) + kOver) : 0;
  }
  static __device__ __forceinline__ void locate(const AttnP& p, const Seq& s, int64_t off, int* h,
                                                int* rt, int64_t* at, int64_t* len) {
    const int nrt = row_tiles(p, s);
    *len = tiles(p, s, 0) + kOver;
    const int64_t item = divide(off, *len);
    *h = (int)divide(item, nrt);
    *rt = (int)(item - (int64_t)*h * nrt);
    *at = off - item * *len;
  }
};

// NT: 8-row blocks of an item (1 or 2).
template <int D, int NT>
struct AttnShape {
  static constexpr int kRows = 8 * NT;               // query rows of an item
  static constexpr int kStageBytes = 2 * kTile * D;  // K, then V
  static constexpr int kStages = D == 128 ? 3 : 5;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kScales = kWarps * kStages * 16;  // per stage: K, V scale of two halves
  static constexpr int kPitch = D + 4;                   // floats; the 4 hold maximum and sum
  static constexpr int kMerge = 2 * kRows * kPitch * 4;  // two warps' outputs
  static constexpr int kMarks = kRows * D / 8;  // one bit an output: a NaN value reached it
  static constexpr int kKSteps = D / 16;        // 16-dim steps of K Q^T
  static constexpr int kMTiles = D / 16;        // 16-dim tiles of V^T P^T
  static constexpr int kWords = D / 32;         // 32-bit words of a lane's V chunk
  static constexpr int kSmem = kRing + kScales + kMerge + kMarks;
  static_assert(kCtasPerSm * (kSmem + 1024) <= 228 * 1024, "shared memory of an SM");
};

// Byte offset of 16-byte chunk c of row r in a tile. Chunks are XOR-ed with
// the 128-byte line's number, so that neither the K reads (8 lanes: two rows,
// every second chunk) nor, at D = 128, the V reads (four rows, two chunks) of a
// quarter warp share a bank. The loops use the same map in lane constants: a
// step of 8 rows (D = 128) or of 8 or 16 (D = 64) keeps or flips bit 6.
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  if constexpr (D == 128) {
    return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
  } else {
    const int line = r >> 1, cc = ((r & 1) << 2) | c;
    return (uint32_t)(line * 128 + ((cc ^ (line & 7)) << 4));
  }
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
// The queries of 8 rows as the B operand: row `row` (this lane's, of n_rows) is
// scaled to 2^14, step s of lane t is dims D/4 t + 4 s .. + 3, the order of the
// K words. Returns the factor that turns a sum into log2 units, but for the
// key scale.
template <int D>
__device__ __forceinline__ float load_queries(const AttnP& p, const Seq& s, int h, int row,
                                              int n_rows, int t, uint32_t (&b)[D / 16][2]) {
  const int i = by_group(p, row);
  const bool in = row < n_rows;
  uint4 raw[D / 32];
  const uint16_t* src = p.q + (int64_t)(s.first + i) * p.q_row +
                        (int64_t)(h * p.group + row - i * p.group) * p.q_head + (D / 4) * t;
#pragma unroll
  for (int w = 0; w < D / 32; ++w)
    raw[w] = in ? reinterpret_cast<const uint4*>(src)[w] : make_uint4(0u, 0u, 0u, 0u);
  const uint32_t* rw = reinterpret_cast<const uint32_t*>(raw);
  float f[D / 4];
  float amax = 0.f;
#pragma unroll
  for (int w = 0; w < D / 8; ++w) {
    float2 v;
    if (p.bf16)
      v = make_float2(__uint_as_float(rw[w] << 16), __uint_as_float(rw[w] & 0xffff0000u));
    else
      v = __half22float2(*reinterpret_cast<const __half2*>(&rw[w]));
    f[2 * w] = v.x;
    f[2 * w + 1] = v.y;
    amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
  }
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  // 2^(14 - exponent of amax), within what fp32 holds
  const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 126);
  // (an infinite query has no softmax: NaN, also where its scores are all -inf and would
  // look like a row that sees nothing)
  const float up = amax <= 3.4028234e38f ? __uint_as_float((uint32_t)(14 - e + 127) << 23)
                                         : __int_as_float(0x7fffffff);
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    b[k][0] = half2_bits(f[4 * k] * up, f[4 * k + 1] * up);
    b[k][1] = half2_bits(f[4 * k + 2] * up, f[4 * k + 3] * up);
  }
  return p.scale_log2 * __uint_as_float((uint32_t)(e - 14 + 127) << 23);
}

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) kv8_attention_kernel(const AttnP p) {
  using S = AttnShape<D, NT>;
  using G = Rows8<NT>;
  constexpr int kRows = S::kRows;
  extern __shared__ __align__(128) uint8_t smem_kv8[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem_kv8) + warp * S::kStages * S::kStageBytes;
  float* scales = reinterpret_cast<float*>(smem_kv8 + S::kRing) + warp * S::kStages * 4;
  float* merge = reinterpret_cast<float*>(smem_kv8 + S::kRing + S::kScales);
  uint32_t* marks = reinterpret_cast<uint32_t*>(merge + S::kMerge / 4);

  grid_dependency_wait();
  grid_launch_dependents();
  const Share share = find_share<G>(p);
  if (tid == 0) p.join[blockIdx.x].count = 0;
  if (share.x >= share.end) return;
  for (int i = tid; i < S::kMarks / 4; i += kThreads) marks[i] = 0u;
  __syncthreads();

  // ---- the load side: this warp's tiles, kStages - 1 ahead of the compute side
  Walk<G> lw;
  lw.start(share);
  Walk<G> cw = lw;
  // The queries of an item on their way to the L1 cache while its first tiles are.
  auto prefetch_queries = [&]() {
    constexpr int kLines = D / 64;  // 128-byte lines of a head
    const int row = lw.rt * kRows + tid / kLines;
    if (tid < kRows * kLines && row < lw.s.n * p.group) {
      const int i = by_group(p, row);
      asm volatile("prefetch.global.L1 [%0];" ::"l"(
          p.q + (int64_t)(lw.s.first + i) * p.q_row +
          (int64_t)(lw.h * p.group + row - i * p.group) * p.q_head + 64 * (tid % kLines)));
    }
  };
  bool more = lw.next(p);
  if (more) prefetch_queries();
  int lt = more ? lw.t0 + warp : 0;
  // Page numbers of the warp's next 16 tiles, two halves of 16 tokens each: lane
  // 2 k + half has those of tile k.
  int ids = -1, id_at = 16;
  auto fetch_ids = [&]() {
    const int tile = lt + kWarps * (lane >> 1);
    const int tok = tile * kTile + 16 * (lane & 1);
    ids = -1;
    if (tile < lw.t1 && tok < lw.limit) {
      const int pi = tok >> p.page_shift;
      if (pi < p.max_pages) ids = p.page_table[lw.b * p.table_stride + pi];
      if ((uint32_t)ids >= (uint32_t)p.pages) {
        ids = -1;
        atomicCAS(p.err, 0, kErrKvRange);
      }
    }
    id_at = 0;
  };
  if (more) fetch_ids();
  int issue_slot = 0;
  // this lane's 16 bytes of a 512-byte pass, in global and in shared memory
  const uint32_t src_lane = 16 * lane;
  const uint32_t dst_lane = chunk_at<D>(lane / (D / 16), lane % (D / 16));
  const ptrdiff_t v_from_k = p.v - p.k;
  auto issue = [&]() {
    if (more && lt >= lw.t1) {
      do {
        more = lw.next(p);
        if (more) prefetch_queries();
        lt = lw.t0 + warp;
      } while (more && lt >= lw.t1);
      id_at = 16;
    }
    if (more) {
      if (id_at == 16) fetch_ids();
      const int tok0 = lt * kTile;
      const int id0 = __shfl_sync(0xffffffffu, ids, 2 * id_at);
      const int id1 = __shfl_sync(0xffffffffu, ids, 2 * id_at + 1);
      ++id_at;
      const uint32_t st = ring + issue_slot * S::kStageBytes + dst_lane;
      if (lane < 2) {  // the scales of the halves; a V scale of -1 marks one that is left out
        const int id = lane ? id1 : id0;
        const size_t blk = (size_t)max(id, 0) * p.kv_heads + lw.h;
        float* dst = scales + issue_slot * 4 + lane;
        if (id >= 0) {
          cp4(smem_u32(dst), p.k_scale + blk);
          cp4(smem_u32(dst + 2), p.v_scale + blk);
        } else {
          dst[0] = 0.f;
          dst[2] = -1.f;
        }
      }
      const bool full = tok0 + kTile <= lw.limit && (id0 | id1) >= 0;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int id = max(half ? id1 : id0, 0);
        const uint8_t* src = p.k + src_lane +
                             ((((size_t)id * p.kv_heads + lw.h) << p.page_shift) +
                              ((tok0 + 16 * half) & (p.page - 1))) * D;
        if (full) {
#pragma unroll
          for (int i = 0; i < 16 * D / 512; ++i) {
            const uint32_t dst = (i & 1 ? st ^ 64u : st) + half * 16 * D + i * 512;
            cp16(dst, src + i * 512);
            cp16(dst + kTile * D, src + v_from_k + i * 512);
          }
        } else {  // rows behind the limit, and those of no page, become zeros
          const int valid = (half ? id1 : id0) >= 0 ? lw.limit - tok0 - 16 * half : 0;
#pragma unroll
          for (int i = 0; i < 16 * D / 512; ++i) {
            const uint32_t dst = (i & 1 ? st ^ 64u : st) + half * 16 * D + i * 512;
            const bool real = i * (512 / D) + lane / (D / 16) < valid;
            cp16_if(dst, src + i * 512, real);
            cp16_if(dst + kTile * D, src + v_from_k + i * 512, real);
          }
        }
      }
      lt += kWarps;
    }
    cp_commit();
    issue_slot = issue_slot + 1 == S::kStages ? 0 : issue_slot + 1;
  };
#pragma unroll 1
  for (int i = 0; i < S::kStages - 1; ++i) issue();

  // lane constants of the K reads (token g, chunk c; token g + 8) and V reads
  // (tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9)
  uint32_t k_at[D / 64], k_at8[D / 64], v_at[4];
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    k_at[c] = chunk_at<D>(g, (D / 64) * t + c);
    k_at8[c] = chunk_at<D>(g + 8, (D / 64) * t + c);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v_at[i] = kTile * D + (D == 128 ? chunk_at<D>(2 * t + (i & 1) + 8 * (i >> 1), g)
                                    : chunk_at<D>(2 * t + (i & 1) + 8 * (i >> 1), g >> 1) +
                                          8 * (g & 1));

  int slot = 0;
  while (cw.next(p)) {
    // ---- queries of this item: row 8 n + g as operand, rows 8 n + 2 t and
    // 8 n + 2 t + 1 of the results
    const int n_rows = cw.s.n * p.group;
    const int r0 = cw.rt * kRows;
    uint32_t qf[NT][S::kKSteps][2];
    float q_mul[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float mul = load_queries<D>(p, cw.s, cw.h, r0 + 8 * n + g, n_rows, t, qf[n]);
#pragma unroll
      for (int r = 0; r < 2; ++r)
        q_mul[n][r] = __shfl_sync(0xffffffffu, mul, 4 * (2 * t + r));
    }
    int lim[NT][2];  // tokens that the row sees
    int low = 0x7fffffff;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = r0 + 8 * n + 2 * t + r;
        lim[n][r] = row < n_rows ? seen(p, cw.s, row) : 0;
        if (lim[n][r] > 0) low = min(low, lim[n][r]);
      }
    low = __reduce_min_sync(0xffffffffu, low);

    float o[NT][S::kMTiles][4];
    float m[NT][2], l[NT][2], sub[NT][2];
    float most_lv = -100.0f;  // largest log2 of a V scale so far (of kLeastScale: -80)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < S::kMTiles; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
#pragma unroll
      for (int r = 0; r < 2; ++r) m[n][r] = -INFINITY, l[n][r] = 0.f, sub[n][r] = 0.f;
    }

#pragma unroll 1
    for (int tile = cw.t0 + warp; tile < cw.t1; tile += kWarps) {
      cp_wait<S::kStages - 2>();
      __syncwarp();  // this stage has landed, and the stage before it is read
      issue();
      const uint32_t st = ring + slot * S::kStageBytes;
      // ---- S^T = K Q^T: tokens 16 i + g and + 8, a lane's K words are dims D/4 t ..
      float s[2][NT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        uint4 ka[2], kb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          ka[i] = lds128(st + k_at[c] + i * 16 * D);
          kb[i] = lds128(st + k_at8[c] + i * 16 * D);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int k = 4 * c + w;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t x = reinterpret_cast<const uint32_t*>(&ka[i])[w];
            const uint32_t y = reinterpret_cast<const uint32_t*>(&kb[i])[w];
            const uint32_t a0 = e4m3_lo(x), a1 = e4m3_lo(y), a2 = e4m3_hi(x), a3 = e4m3_hi(y);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma_16816<false>(s[i][n], a0, a1, a2, a3, qf[n][k][0], qf[n][k][1]);
          }
        }
      }
      // ---- scores in log2 units with the value scale, masked
      const float4 sc = *reinterpret_cast<const float4*>(scales + slot * 4);
      const float ks[2] = {sc.x, sc.y};
      const float lv[2] = {sc.z < 0.f ? -INFINITY : lg2(fmaxf(sc.z, kLeastScale)),
                           sc.w < 0.f ? -INFINITY : lg2(fmaxf(sc.w, kLeastScale))};
      most_lv = fmaxf(most_lv, fmaxf(lv[0], lv[1]));
      const int tok0 = tile * kTile;
      const bool cut = tok0 + kTile > low;  // some row ends inside the tile, or before it
      float top[NT][2];  // this lane's largest score of each row
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {  // elements r and r + 2 are row r's
          const float f[2] = {q_mul[n][r] * ks[0], q_mul[n][r] * ks[1]};
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = r; e < 4; e += 2) {
              float& x = s[i][n][e];
              x = fmaf(x, f[i], lv[i]);
              if (cut && tok0 + 16 * i + g + 8 * (e >> 1) >= lim[n][r]) x = -INFINITY;
            }
          top[n][r] = fmaxf(fmaxf(s[0][n][r], s[0][n][r + 2]), fmaxf(s[1][n][r], s[1][n][r + 2]));
        }
      bool larger = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) larger |= top[n][0] > m[n][0] || top[n][1] > m[n][1];
      if (__any_sync(0xffffffffu, larger)) {  // seldom after the first tiles
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float most = top[n][r];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1)
              most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
            most = fmaxf(most, m[n][r]);
            // (l's in two steps: between far scales it is below fp32, the product is not)
            const float root = m[n][r] == -INFINITY ? 0.f : ex2(0.5f * (m[n][r] - most));
            const float al = root * root;
            m[n][r] = most;
            // (rounded up: where the steps of fp32 are coarser than the shift P' stays in range)
            sub[n][r] = most == -INFINITY ? 0.f : __fadd_ru(most, -kShift);
            l[n][r] *= root;
            l[n][r] *= root;
#pragma unroll
            for (int j = 0; j < S::kMTiles; ++j) {
              o[n][j][r] *= al;
              o[n][j][r + 2] *= al;
            }
          }
      }
      if (fminf(lv[0], lv[1]) < most_lv - kFar) {  // (seldom, but at a sequence's end)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (lv[i] < most_lv - kFar && lv[i] > -INFINITY) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                l[n][e & 1] += ex2(s[i][n][e] - sub[n][e & 1] - lv[i]);
          }
      }
      uint32_t pf[2][NT][2];  // P^T as the B operand: 16 tokens a step
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // 1 / sv, or nothing: left out, or in the sum already
        const float inv = lv[i] < most_lv - kFar ? 0.f : ex2(-lv[i]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float(&v)[4] = s[i][n];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = ex2(v[e] - sub[n][e & 1]);
          l[n][0] = fmaf(v[0] + v[2], inv, l[n][0]);
          l[n][1] = fmaf(v[1] + v[3], inv, l[n][1]);
          pf[i][n][0] = transpose8x8(half2_bits(v[0], v[1]));
          pf[i][n][1] = transpose8x8(half2_bits(v[2], v[3]));
        }
      }
      // ---- O^T += V^T P^T: a lane's V chunks are dims D/8 g .. of tokens 2t, 2t+1,
      // 2t+8, 2t+9 of each 16; byte pairs of two tokens make the A operand
      if (cut && low < cw.limit) {
        // Rows of this item end at different tokens here, and a NaN that one row
        // sees must not reach a row that does not (0 * NaN): NaN codes leave the
        // tile, and the outputs that they belong to are marked.
        bool some = false;  // seldom
#pragma unroll
        for (int i = 0; i < kTile * D / 512; ++i)
          some |= any_nan(lds128(st + kTile * D + 512 * i + 16 * lane));
        if (__any_sync(0xffffffffu, some)) {
#pragma unroll 1
          for (int i = lane; i < kTile * D / 16; i += 32) {
            const int tok = tok0 + i / (D / 16), c = i % (D / 16);
            const uint32_t at = st + kTile * D + chunk_at<D>(i / (D / 16), c);
#pragma unroll 1
            for (int w = 0; w < 4; ++w) {
              const uint32_t v = lds32(at + 4 * w);
              const uint32_t nan = nan_codes(v);
              if (nan == 0u) continue;
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + 4 * w), "r"(v & ~nan) : "memory");
              const uint32_t bits = ((nan & 1u) | (nan >> 7 & 2u) | (nan >> 14 & 4u) |
                                     (nan >> 21 & 8u)) << (16 * (c & 1) + 4 * w);
#pragma unroll 1
              for (int r = r0; r < min(n_rows, r0 + kRows); ++r)
                if (tok < seen(p, cw.s, r)) atomicOr(marks + (r - r0) * (D / 32) + (c >> 1), bits);
            }
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t vw[4][S::kWords];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t at = st + v_at[k] + i * 16 * D;
          if constexpr (D == 128) {
            const uint4 w = lds128(at);
            vw[k][0] = w.x, vw[k][1] = w.y, vw[k][2] = w.z, vw[k][3] = w.w;
          } else {
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                         : "=r"(vw[k][0]), "=r"(vw[k][1])
                         : "r"(at));
          }
        }
#pragma unroll
        for (int w = 0; w < S::kWords; ++w) {
          const uint32_t x0 = __byte_perm(vw[0][w], vw[1][w], 0x5140);
          const uint32_t y0 = __byte_perm(vw[0][w], vw[1][w], 0x7362);
          const uint32_t x1 = __byte_perm(vw[2][w], vw[3][w], 0x5140);
          const uint32_t y1 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
          uint32_t a0 = e4m3_lo(x0), a1 = e4m3_hi(x0), a2 = e4m3_lo(x1), a3 = e4m3_hi(x1);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma_16816<false>(o[n][2 * w], a0, a1, a2, a3, pf[i][n][0], pf[i][n][1]);
          a0 = e4m3_lo(y0), a1 = e4m3_hi(y0), a2 = e4m3_lo(y1), a3 = e4m3_hi(y1);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma_16816<false>(o[n][2 * w + 1], a0, a1, a2, a3, pf[i][n][0], pf[i][n][1]);
        }
      }
      slot = slot + 1 == S::kStages ? 0 : slot + 1;
    }

    // ---- merge the warps: 2 and 3 into 0 and 1, then 1 into 0. o[n][j] holds
    // dims D/8 g + 2 j (elements 0, 1) and + 1 (2, 3) of rows 2 t and 2 t + 1.
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
          l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], off);
    // Two rounds and a last one in which warp 0 leaves the sum: one copy of the
    // code for all, since code that runs once an item costs its fetch.
#pragma unroll 1
    for (int step = 2;; step >>= 1) {
      __syncthreads();  // the buffers are free
      if (warp >= step && warp < max(2 * step, 1)) {
        float* buf = merge + (warp - step) * kRows * S::kPitch;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float* row = buf + (8 * n + 2 * t + r) * S::kPitch;
            if (g == 0) row[D] = m[n][r], row[D + 1] = l[n][r];
#pragma unroll
            for (int j = 0; j < S::kMTiles; j += 2)
              *reinterpret_cast<float4*>(row + (D / 8) * g + 2 * j) = make_float4(
                  o[n][j][r], o[n][j][r + 2], o[n][j + 1][r], o[n][j + 1][r + 2]);
          }
      }
      __syncthreads();
      if (step == 0) break;
      if (warp < step) {
        const float* buf = merge + warp * kRows * S::kPitch;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float* row = buf + (8 * n + 2 * t + r) * S::kPitch;
            const float om = row[D], ol = row[D + 1];
            const float nm = fmaxf(m[n][r], om);
            const float ra = m[n][r] == -INFINITY ? 0.f : ex2(0.5f * (m[n][r] - nm)), fa = ra * ra;
            const float rb = om == -INFINITY ? 0.f : ex2(0.5f * (om - nm)), fb = rb * rb;
            m[n][r] = nm;
            l[n][r] = l[n][r] * ra * ra + ol * rb * rb;
#pragma unroll
            for (int j = 0; j < S::kMTiles; j += 2) {
              const float4 v = *reinterpret_cast<const float4*>(row + (D / 8) * g + 2 * j);
              o[n][j][r] = o[n][j][r] * fa + v.x * fb;
              o[n][j][r + 2] = o[n][j][r + 2] * fa + v.y * fb;
              o[n][j + 1][r] = o[n][j + 1][r] * fa + v.z * fb;
              o[n][j + 1][r + 2] = o[n][j + 1][r + 2] * fa + v.w * fb;
            }
          }
      }
    }
    // Eight dims of a row a thread: the output of a whole item, or a part that is
    // left for the second launch.
    float* part =
        p.parts + ((size_t)blockIdx.x * 2 + cw.slot(share)) * kRows * S::kPitch;
#pragma unroll 1
    for (int e = tid; e < kRows * (D / 8); e += kThreads) {
      const int rr = e / (D / 8), d = 8 * (e % (D / 8));
      if (r0 + rr >= n_rows) break;
      const float* src = merge + rr * S::kPitch;
      float v[8];
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src + d);
      *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(src + d + 4);
      uint8_t* mark = reinterpret_cast<uint8_t*>(marks) + e;  // this thread's alone
      if (*mark) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (*mark >> k & 1) v[k] = __int_as_float(0x7fffffff);
        *mark = 0;
      }
      if (cw.whole) {
        const float sum = src[D + 1];
        const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
        const int i = by_group(p, r0 + rr);
        uint16_t* dst = p.out + (int64_t)(cw.s.first + i) * p.out_row +
                        (int64_t)(cw.h * p.group + r0 + rr - i * p.group) * p.out_head + d;
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float a = v[2 * k] * inv, b = v[2 * k + 1] * inv;
          if (p.bf16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            w[k] = *reinterpret_cast<const uint32_t*>(&h);
          } else {
            w[k] = half2_bits(a, b);
          }
        }
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        float* dst = part + rr * S::kPitch;
        *reinterpret_cast<float4*>(dst + d) = *reinterpret_cast<const float4*>(v);
        *reinterpret_cast<float4*>(dst + d + 4) = *reinterpret_cast<const float4*>(v + 4);
        if (d == 0) *reinterpret_cast<float2*>(dst + D) = *reinterpret_cast<const float2*>(src + D);
      }
    }
    if (!cw.whole && tid == 0) cw.describe(p, share);
    __syncthreads();  // marks are read before the next item sets any
  }
}

template <int D, int NT>
int launch(AttnP p, int max_rows, const DeviceInfo& di, cudaStream_t stream) {
  using S = AttnShape<D, NT>;
  p.join = reinterpret_cast<Join*>(p.parts + (size_t)kMaxCtas * 2 * S::kRows * S::kPitch);
  const int ctas = std::min(kMaxCtas, kCtasPerSm * di.sm_count);
  cudaError_t e = launch_overlapped(kv8_attention_kernel<D, NT>, dim3((unsigned)ctas), kThreads,
                                    S::kSmem, stream, p);
  if (e != cudaSuccess) return cuda_fail(e, "w4_kv8_attention launch");
  // Blocks of an item's join. Where the page table has no room for more than a
  // few partials an item, a warp a row. Else a row at a time each: eight blocks
  // when there are few items for all the CTAs (one sequence of 32768 tokens over
  // two heads: 13 us in all, against 16 with four), four otherwise (16 sequences
  // of up to 2000 over four heads: 13.0 us, against 14.7 with eight).
  const int most = ((p.capacity + kTile - 1) / kTile) / Rows8<NT>::kMinShare + 2;
  const bool few_items = (int64_t)ctas > (int64_t)kFew * p.seqs * p.kv_heads;
  const int by = most <= kFew ? (max_rows + kJoinWarps - 1) / kJoinWarps
                              : std::min(max_rows, few_items ? 8 : 4);
  e = launch_overlapped(kv8_join_kernel<D, S::kRows>, dim3((unsigned)ctas, (unsigned)by), kJoinThreads, 0,
                        stream, p);
  return e == cudaSuccess ? W4_OK : cuda_fail(e, "w4_kv8_attention join launch");
}

}  // namespace

size_t kv8_attention_workspace_bytes(int head_dim) {
  return std::max((size_t)kMaxCtas * (2 * 16 * (head_dim + 4) * 4 + sizeof(Join)),  // 16-row items
                  kv8_prompt_workspace_bytes(head_dim));
}

template <int D, int NT>
static int init_attention(const DeviceInfo& di) {
  constexpr int smem = AttnShape<D, NT>::kSmem;
  if (smem > di.max_smem_optin)
    return fail(W4_ERR_UNSUPPORTED, "w4_kv8_attention needs %d B of shared memory", smem);
  cudaError_t e = cudaFuncSetAttribute(kv8_attention_kernel<D, NT>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kv8_attention_kernel<D, NT>,
                             cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared);
  return e == cudaSuccess ? W4_OK : cuda_fail(e, "cudaFuncSetAttribute(kv8 attention)");
}

int kv8_init_device(const DeviceInfo& di) {
  int st = init_attention<64, 1>(di);
  if (st == W4_OK) st = init_attention<64, 2>(di);
  if (st == W4_OK) st = init_attention<128, 1>(di);
  if (st == W4_OK) st = init_attention<128, 2>(di);
  if (st == W4_OK) st = kv8_prompt_init_device(di);
  return st;
}

int launch_kv8_attention(const w4_kv8_cache& c, const w4_kv_batch& bt, const w4_heads& q,
                         const w4_heads& out, int bf16, float scale, void* workspace,
                         const DeviceInfo& di, cudaStream_t stream) {
  AttnP p = {};
  p.k = static_cast<const uint8_t*>(c.k);
  p.v = static_cast<const uint8_t*>(c.v);
  p.k_scale = c.k_scale;
  p.v_scale = c.v_scale;
  p.page_table = bt.page_table;
  p.lengths = bt.lengths;
  p.row_starts = bt.row_starts;
  p.table_stride = bt.table_stride;
  p.pages = c.pages;
  p.page = c.page_size;
  p.page_shift = c.page_size == 16 ? 4 : c.page_size == 32 ? 5 : c.page_size == 64 ? 6 : 7;
  p.max_pages = bt.max_pages;
  // below 2^31 with room for a step's rows and a tile's rounding
  p.capacity = (int)std::min<int64_t>((int64_t)bt.max_pages * c.page_size, 0x70000000);
  p.kv_heads = c.kv_heads;
  p.seqs = bt.seqs;
  p.rows = bt.rows;
  p.group = q.heads / c.kv_heads;
  p.group_mul = p.group > 1 ? (uint32_t)(((1ull << 32) + p.group - 1) / p.group) : 0u;
  p.q = static_cast<const uint16_t*>(q.ptr);
  p.q_row = q.row_stride;
  p.q_head = q.head_stride;
  p.out = static_cast<uint16_t*>(out.ptr);
  p.out_row = out.row_stride;
  p.out_head = out.head_stride;
  p.bf16 = bf16;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.parts = static_cast<float*>(workspace);
  p.err = di.err_word;
  // Rows of an item by the rows that a sequence brings on average. Items of 8 and of 16:
  // 64 sequences of 1500 tokens, 4 rows 28.9 and 36.3 us, 8 of 2000, 16 rows 15.9 and
  // 16.2, 32 rows 21.9 and 20.3; 32 of 1000, 32 rows 39.6 and 33.7. (Items of 32 rows read
  // the cache less often, but 35.1 us there: fewer tiles on their way, longer chains.)
  const int64_t avg = ((int64_t)bt.rows + bt.seqs - 1) / bt.seqs * p.group;
  if (avg >= kPromptRows) return launch_kv8_prompt(p, c.head_dim, di, stream);
  const int rows = avg <= 8 ? 8 : 16;
  const int max_rows = (int)std::min<int64_t>(rows, (int64_t)bt.rows * p.group);
  if (c.head_dim == 128)
    return rows == 8 ? launch<128, 1>(p, max_rows, di, stream)
                     : launch<128, 2>(p, max_rows, di, stream);
  return rows == 8 ? launch<64, 1>(p, max_rows, di, stream)
                   : launch<64, 2>(p, max_rows, di, stream);
}

}  // namespace w4
