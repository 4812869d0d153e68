// w4_kv8_attn.cuh - what the two kernels of attention over the paged 8-bit KV
// cache share: the call's parameters, the split of the work over the CTAs, and
// the join of items that the split cuts.
#pragma once

#include "w4_internal.h"
#include "w4_ptx.cuh"

#include <algorithm>

namespace w4 {

struct AttnP {
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  const int32_t *page_table, *lengths, *row_starts;
  int64_t table_stride;
  int capacity;  // tokens that a row of the page table holds
  int pages, page, page_shift, max_pages, kv_heads, seqs, rows, group;
  uint32_t group_mul;  // ceil(2^32 / group), 0 for group 1
  const uint16_t* q;
  int64_t q_row, q_head;
  uint16_t* out;
  int64_t out_row, out_head;
  int bf16;
  float scale_log2;
  float* parts;       // [CTAs][2][rows of an item][D + 4], maximum and sum behind the outputs
  struct Join* join;  // [CTAs]
  int* err;
};

// What the second launch needs to join an item: written by the CTA whose share
// begins at the item's first inner border, empty (count 0) by every other.
struct Join {
  int count;       // partials, CTAs cta .. cta + count - 1
  int cta, slot;   // the first partial's CTA and slot; the others are in slot 0
  int row0, head0; // first output row of the sequence, first query head
  int r0, rows;    // the tile's first query row, and all query rows of the item's head
  int pad;
};

// Many query rows a sequence (w4_kv8_prompt.cu); p.join is set by the launch.
int launch_kv8_prompt(AttnP p, int head_dim, const DeviceInfo& di, cudaStream_t stream);
int kv8_prompt_init_device(const DeviceInfo& di);
size_t kv8_prompt_workspace_bytes(int head_dim);

namespace {

// CTAs that the workspace has room for: two an SM on the largest sm_100 part.
constexpr int kMaxCtas = 320;

// A value scale below this counts as this: values of 2^-71 at most. Weights over
// scales (the softmax's sums hold P' / sv) then stay inside fp32.
constexpr float kLeastScale = 0x1p-80f;
// Scales this much below the largest so far (in log2) are far: a P' that vanishes then
// still counts in the sum, which is made without it.
constexpr float kFar = 80.0f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two e4m3 codes (the low half of w, or the high) to fp16, exactly.
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}"
      : "=r"(d)
      : "r"(w));
  return d;
}
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}"
      : "=r"(d)
      : "r"(w));
  return d;
}

__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Zeros where it is not `real` (src is a valid address all the same).
__device__ __forceinline__ void cp16_if(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(real ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The bytes of four e4m3 codes that are NaN (0x7f, 0xff): all ones.
__device__ __forceinline__ uint32_t nan_codes(uint32_t v) {
  return (((v & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u) * 0xffu;
}
__device__ __forceinline__ bool any_nan(const uint4& v) {
  return ((((v.x & 0x7f7f7f7fu) + 0x01010101u) | ((v.y & 0x7f7f7f7fu) + 0x01010101u) |
           ((v.z & 0x7f7f7f7fu) + 0x01010101u) | ((v.w & 0x7f7f7f7fu) + 0x01010101u)) &
          0x80808080u) != 0u;
}

// A sequence's rows and tokens. A length that the page table cannot hold is cut
// to what it holds; rows behind a negative one see nothing, and none are counted.
struct Seq {
  int first, n;  // rows
  int past;
  bool bad;      // has rows, and a length that the page table has no room for
};
__device__ __forceinline__ Seq load_seq(const AttnP& p, int b) {
  Seq s;
  const int length = p.lengths[b];
  s.first = min(max(p.row_starts[b], 0), p.rows);
  s.n = min(max(p.row_starts[b + 1], s.first), p.rows) - s.first;
  s.past = min(max(length, 0), p.capacity);
  s.bad = s.n > 0 && (length < 0 || length > p.capacity - s.n);
  if (length < 0) s.n = 0;
  return s;
}
// r / group, for r < 2^28: group_mul * group exceeds 2^32 by less than 16.
__device__ __forceinline__ int by_group(const AttnP& p, int r) {
  return p.group_mul ? (int)__umulhi((uint32_t)r, p.group_mul) : r;
}
// a / b, in 32 bits where a fits them (the 64-bit division is a long call).
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  if (((uint64_t)a | (uint64_t)b) < (1ull << 32)) return (uint32_t)a / (uint32_t)b;
  return a / b;
}
// Tokens that query row r (of n * group) of the sequence sees.
__device__ __forceinline__ int seen(const AttnP& p, const Seq& s, int r) {
  return min(s.past + by_group(p, r) + 1, p.capacity);
}
// ------------------------------------------------------------ the split
//
// Items (a sequence's cache head and tile of query rows) lie in one line, each
// with a length that its geometry G gives: kOver units for what an item costs
// beside its tiles (queries, merge, output), then kUnit units a tile of tokens.
// Every CTA takes an equal, contiguous share of the line.

// The tile at unit v of an item.
template <typename G>
__device__ __forceinline__ int tile_at(int64_t v) {
  return v <= G::kOver ? 0 : (int)((v - G::kOver) / G::kUnit);
}

// `per` units of the line a CTA, the last ones less or none. Every warp works it
// out by itself, up to 128 sequences at a time.
struct Share {
  int64_t x, end;  // this CTA's units
  int64_t per;     // units of a share
  int b;           // the sequence of unit x
  int64_t off;     // x's place in the sequence
};

__device__ __forceinline__ int64_t scan32(int64_t v, int lane) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += up;
  }
  return v;
}

// Item blockIdx.x as this CTA's share.
template <typename G>
__device__ __forceinline__ Share item_share(const AttnP& p, int64_t per) {
  const int lane = threadIdx.x & 31;
  Share f;
  f.x = f.end = f.off = 0;
  f.per = per;
  f.b = 0;
  int left = (int)blockIdx.x;  // items before it, of the sequences from here
#pragma unroll 1
  for (int b0 = 0; b0 < p.seqs; b0 += 32) {
    Seq s;
    s.n = 0;
    if (b0 + lane < p.seqs) s = load_seq(p, b0 + lane);
    const int mine = s.n > 0 ? p.kv_heads * G::row_tiles(p, s) : 0;
    const int upto = (int)scan32(mine, lane);
    const unsigned hit = __ballot_sync(0xffffffffu, upto > left);
    if (hit) {
      const int src = __ffs(hit) - 1;
      f.b = b0 + src;
      left -= __shfl_sync(0xffffffffu, upto - mine, src);
      s = load_seq(p, f.b);
      const int nrt = G::row_tiles(p, s);
      f.off = left / nrt * G::upto(p, s, nrt) + G::upto(p, s, left % nrt);
      f.end = G::length(p, s, left % nrt);
      return f;
    }
    left -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return f;
}

template <typename G>
__device__ __forceinline__ Share find_share(const AttnP& p) {
  const int lane = threadIdx.x & 31;
  Share f;
  // Neighbouring sequences a lane, whose loads go out together: 512 sequences of 300
  // tokens at most 85 us, 100 with one a lane.
  const int each = p.seqs > 32 ? 4 : 1;
  int64_t all = 0, w[4];
  int items = 0;          // of all sequences, and the longest (G::kCut > 0)
  int64_t longest = 0;
  bool bad = false;       // a length that the page table has no room for
  auto load = [&](int b0) {
    Seq s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = b0 + each * lane + i;
      s[i].first = s[i].n = s[i].past = 0;
      s[i].bad = false;
      if (i < each && b < p.seqs) s[i] = load_seq(p, b);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
      if (i >= each) continue;
      w[i] = G::seq_work(p, s[i]);
      bad |= s[i].bad;
      if (s[i].n == 0) continue;
      if constexpr (G::kCut > 0) {
        const int nrt = G::row_tiles(p, s[i]);
        items = (int)min(items + (int64_t)p.kv_heads * nrt, (int64_t)1 << 24);
        longest = max(longest, G::length(p, s[i], nrt - 1));
      }
    }
  };
#pragma unroll 1
  for (int b0 = 0; b0 < p.seqs; b0 += 32 * each) {
    load(b0);
    all += (w[0] + w[1]) + (w[2] + w[3]);
  }
  if (bad) atomicCAS(p.err, 0, kErrKvRange);
#pragma unroll
  for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  f.per = max((int64_t)G::kMinShare, divide(all + gridDim.x - 1, gridDim.x));
  if constexpr (G::kCut > 0) {
    // No more items than CTAs and the longest little longer than a share: an item
    // a CTA, none cut. Only the share's length counts then.
    items = __reduce_add_sync(0xffffffffu, items);
#pragma unroll
    for (int o = 16; o; o >>= 1) longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
    if (items <= (int)gridDim.x && longest <= f.per + G::kCut) return item_share<G>(p, f.per);
  }
  f.x = min(all, f.per * blockIdx.x);
  f.end = min(all, f.x + f.per);
  f.b = 0;
  f.off = 0;
  if (f.x >= f.end) return f;
  int64_t before = 0;
#pragma unroll 1
  for (int b0 = 0;; b0 += 32 * each) {
    if (p.seqs > 32 * each) load(b0);  // else the first pass has left them
    const int64_t mine = (w[0] + w[1]) + (w[2] + w[3]), upto = scan32(mine, lane);
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > f.x);
    if (hit || b0 + 32 * each >= p.seqs) {
      const int src = hit ? __ffs(hit) - 1 : 31;
      int64_t left = f.x - before - (upto - mine);  // lane src's are used
      int at = 0;
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (at == i && i + 1 < each && left >= w[i]) left -= w[i], at = i + 1;
      f.b = min(b0 + each * src + __shfl_sync(0xffffffffu, at, src), p.seqs - 1);
      f.off = __shfl_sync(0xffffffffu, left, src);
      return f;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

// Walks a CTA's share item by item.
template <typename G>
struct Walk {
  int64_t x, end;  // next unit of the line, end of the share
  int b;           // sequence of x
  int64_t off;     // x's place in it
  // the item
  Seq s;
  int h, rt;      // cache head, row tile
  int64_t item0;  // where it begins in the line
  int nt;         // its tiles
  int t0, t1;     // the share's part of them, without those above the rows' limit
  bool whole;     // the part is all of them
  int limit;      // tokens that the row tile's last row sees

  __device__ __forceinline__ void start(const Share& f) { x = f.x, end = f.end, b = f.b, off = f.off; }

  // The next item of which the share has a tile.
  __device__ __forceinline__ bool next(const AttnP& p) {
    while (true) {
      if (x >= end) return false;
      s = load_seq(p, b);
      for (int64_t w; off >= (w = G::seq_work(p, s));) {  // no rows, or just done
        off -= w;
        if (++b >= p.seqs) return false;
        s = load_seq(p, b);
      }
      int64_t at, len;
      G::locate(p, s, off, &h, &rt, &at, &len);
      limit = seen(p, s, min(s.n * p.group, (rt + 1) * G::kRows) - 1);
      nt = G::tiles(p, s, limit);
      const int64_t to = min(len, at + (end - x));
      item0 = x - at;
      x += to - at;
      off += to - at;
      t0 = min(tile_at<G>(at), nt);
      t1 = to == len ? nt : min(tile_at<G>(to), nt);
      if (t0 < t1) break;
    }
    whole = t1 - t0 == nt;
    t1 = min(t1, (limit + G::kTile - 1) / G::kTile);
    return true;
  }

  // Where this CTA leaves its part of a cut item: a share has at most one item
  // that begins before it (or with it) and one that ends behind it.
  __device__ __forceinline__ int slot(const Share& f) const { return f.x >= item0 ? 0 : 1; }

  // Describes the join of a cut item. The CTA whose part is the second one does:
  // its share begins inside the item and the share before at its first tile.
  __device__ __forceinline__ void describe(const AttnP& p, const Share& f) const {
    if (t0 == 0 || tile_at<G>(f.x - f.per - item0) > 0) return;
    const int last = (int)divide(item0 + G::kOver + (int64_t)nt * G::kUnit - 1, f.per);
    Join jn;
    jn.count = last - (int)blockIdx.x + 2;
    jn.cta = (int)blockIdx.x - 1;
    jn.slot = f.x - f.per >= item0 ? 0 : 1;  // as slot() of the share before
    jn.row0 = s.first;
    jn.head0 = h * p.group;
    jn.r0 = rt * G::kRows;
    jn.rows = s.n * p.group;
    jn.pad = 0;
    p.join[blockIdx.x] = jn;
  }
};

// CTAs that a batch can use: a share has kMinShare units at least, and the host
// knows bounds of the items and, by the page table, of their lengths.
template <typename G>
inline int useful_ctas(const AttnP& p, int ctas) {
  const int64_t items = std::min<int64_t>(  // (times 2^31 units at most)
      (int64_t)p.kv_heads * ((int64_t)p.rows * p.group / G::kRows + p.seqs), 1 << 30);
  const int64_t units = G::kOver + G::kMore +
                        G::kUnit * (((int64_t)p.capacity + G::kTile - 1) / G::kTile);
  return (int)std::min<int64_t>(ctas, (items * units + G::kMinShare - 1) / G::kMinShare);
}

// ------------------------------------------------------------ the join

constexpr int kJoinWarps = 8;
constexpr int kJoinThreads = kJoinWarps * 32;
constexpr int kFew = 8;  // partials that a warp joins by itself

// Joins the partials of an item: blockIdx.x the border, blockIdx.y the rows. A
// few partials: a warp a row. Many (a long sequence over many CTAs): the block
// takes one row at a time, first every partial's factor, then the sum of the
// outputs, eight partials side by side and in a fixed order.
template <int D, int kRows>
__global__ void __launch_bounds__(kJoinThreads) kv8_join_kernel(const AttnP p) {
  constexpr int V = D / 32, kPitch = D + 4;
  __shared__ float factor[kMaxCtas];
  __shared__ float sm[kJoinWarps], sl[kJoinWarps], so[kJoinWarps][D];
  grid_dependency_wait();
  grid_launch_dependents();
  const Join jn = p.join[blockIdx.x];
  if (jn.count == 0) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows = min(kRows, jn.rows - jn.r0);
  auto part_of = [&](int c, int ri) {
    return p.parts +
           (((size_t)(jn.cta + c) * 2 + (c == 0 ? jn.slot : 0)) * kRows + ri) * kPitch;
  };
  auto store = [&](int ri, const float (&o)[V], float l) {
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    const int row = jn.r0 + ri, i = by_group(p, row);
    uint16_t* dst = p.out + (int64_t)(jn.row0 + i) * p.out_row +
                    (int64_t)(jn.head0 + row - i * p.group) * p.out_head + V * lane;
    uint32_t w[V / 2];
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      if (p.bf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(o[2 * k] * inv, o[2 * k + 1] * inv);
        w[k] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        w[k] = half2_bits(o[2 * k] * inv, o[2 * k + 1] * inv);
      }
    }
#pragma unroll
    for (int k = 0; k < V / 2; ++k) reinterpret_cast<uint32_t*>(dst)[k] = w[k];
  };
  if (jn.count <= kFew) {
#pragma unroll 1
    for (int ri = blockIdx.y * kJoinWarps + warp; ri < rows; ri += gridDim.y * kJoinWarps) {
      // The sums' factor in two steps: from one scale to another it may leave fp32 alone.
      float m[kFew], l[kFew], v[kFew][V];
      float most = -INFINITY;
#pragma unroll
      for (int c = 0; c < kFew; ++c) {
        m[c] = -INFINITY, l[c] = 0.f;
        if (c < jn.count) {
          const float* part = part_of(c, ri);
          m[c] = part[D], l[c] = part[D + 1];
#pragma unroll
          for (int i = 0; i < V; ++i) v[c][i] = part[V * lane + i];
        }
        most = fmaxf(most, m[c]);
      }
      float sum = 0.f, o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = 0.f;
#pragma unroll
      for (int c = 0; c < kFew; ++c)
        if (c < jn.count) {
          const float h = m[c] == -INFINITY ? 0.f : ex2(0.5f * (m[c] - most)), f = h * h;
          sum += l[c] * h * h;
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] += v[c][i] * f;
        }
      store(ri, o, sum);
    }
    return;
  }
#pragma unroll 1
  for (int ri = blockIdx.y; ri < rows; ri += gridDim.y) {
    constexpr int kMine = (kMaxCtas + kJoinThreads - 1) / kJoinThreads;
    float m[kMine], pl[kMine], most = -INFINITY;
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int c = tid + k * kJoinThreads;
      m[k] = -INFINITY, pl[k] = 0.f;
      if (c < jn.count) {
        const float2 ml = *reinterpret_cast<const float2*>(part_of(c, ri) + D);
        m[k] = ml.x, pl[k] = ml.y;
      }
      most = fmaxf(most, m[k]);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
    if (lane == 0) sm[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) most = fmaxf(most, sm[w]);
    float l = 0.f;
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int c = tid + k * kJoinThreads;
      const float h = m[k] == -INFINITY ? 0.f : ex2(0.5f * (m[k] - most));
      if (c < jn.count) factor[c] = h * h;
      l += pl[k] * h * h;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    if (lane == 0) sl[warp] = l;
    __syncthreads();
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.f;
#pragma unroll 8
    for (int c = warp; c < jn.count; c += kJoinWarps) {
      const float* part = part_of(c, ri) + V * lane;
      const float f = factor[c];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] += part[i] * f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) so[warp][V * lane + i] = o[i];
    __syncthreads();
    if (warp == 0) {
      l = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) {
        l += sl[w];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] += so[w][V * lane + i];
      }
      store(ri, o, l);
    }
    __syncthreads();  // the shared sums are read
  }
}

}  // namespace
}  // namespace w4
