// w4_kv8.cu - per-head norm and rotation of queries and keys, and the write
// side of the paged 8-bit KV cache.
//
//   norm_rope : x' = x * rsqrt(mean(x^2) + eps) * w over one head (skipped
//               without a weight), then the rotate-half rotation
//               y[d]       = x'[d] cos[d] - x'[d + D/2] sin[d]
//               y[d + D/2] = x'[d + D/2] cos[d + D/2] + x'[d] sin[d + D/2],
//               all in fp32 from the 16-bit inputs, one rounding at the store.
//   append    : the same for a step's keys on their way into the cache (and
//               for its queries, in the same launch), values beside them.
//               A block of the cache is one page of one head; K and V have a
//               scale each, a power of two: the smallest s with amax <= 448 s
//               over the rows that this call puts into the block, and no less
//               than the block's scale where the block goes on. A power of two
//               costs e4m3 (4 significand bits, a floating format) nothing in
//               precision, and when a block's scale grows its older rows move
//               to the new one exactly, but for values that become e4m3
//               subnormals.
//
// Both are bound by memory and, at the small end, by launch latency. A head is
// held by D / 16 lanes, each with the two 16-byte chunks that the rotation
// pairs (dims 8l.. and D/2 + 8l..): the rotation needs no exchange, the norm's
// sum three (or two) shuffles, and every access is 16 bytes wide.
//
// norm_rope of 8191 rows of 32 and 8 heads of 128: 33.1 us, 5.3 TB/s (a copy
// reaches 6.45); of 8 rows 2.6 us. append of 3 x 4001 rows of 2 heads with 12 of
// queries: 21 us, 3.8 TB/s: a block's loads, its largest value and its codes follow
// one another, and 21 warps an SM do not hide all of that; of 64 x 1 rows of 8
// heads 3.6 us, the latency of length, page number, scale and row.
#include "w4_internal.h"
#include "w4_ptx.cuh"

#include <cuda_fp8.h>

#include <algorithm>

namespace w4 {

namespace {

constexpr int kMinScaleExp = -32, kMaxScaleExp = 120;

// ------------------------------------------------------------ element types

struct F8 {
  float f[8];
};

// Eight 16-bit elements (16 bytes) to fp32, and back with one rounding.
template <bool BF16>
__device__ __forceinline__ F8 unpack8(const uint4& v) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
  F8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      r.f[2 * i] = __uint_as_float(w[i] << 16);
      r.f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      r.f[2 * i] = h.x;
      r.f[2 * i + 1] = h.y;
    }
  }
  return r;
}

template <bool BF16>
__device__ __forceinline__ uint4 pack8(const F8& r) {
  uint4 v;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(r.f[2 * i], r.f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(r.f[2 * i], r.f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return v;
}

// Eight elements at index i (a multiple of 8) of a table or weight.
__device__ __forceinline__ F8 load8(const void* p, int type, size_t i) {
  if (type == W4_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 b = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i)[1];
    return F8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
  }
  const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
  return type == W4_BF16 ? unpack8<true>(v) : unpack8<false>(v);
}

// Eight fp32 values times mul to e4m3: round to nearest even, +-448 beyond the
// range (infinities too), NaN kept.
__device__ __forceinline__ uint2 to_e4m3x8(const F8& r, float mul) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(
        make_float2(r.f[4 * i] * mul, r.f[4 * i + 1] * mul), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(
        make_float2(r.f[4 * i + 2] * mul, r.f[4 * i + 3] * mul), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// Eight codes times mul, rounded again.
__device__ __forceinline__ uint2 again_e4m3x8(uint2 v, float mul) {
  const uint32_t w[2] = {v.x, v.y};
  F8 f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(
        (__nv_fp8x2_storage_t)((w[j >> 1] >> (16 * (j & 1))) & 0xffffu), __NV_E4M3);
    const float2 f2 = __half22float2(*reinterpret_cast<const __half2*>(&hr));
    f.f[2 * j] = f2.x;
    f.f[2 * j + 1] = f2.y;
  }
  return to_e4m3x8(f, mul);
}

// ------------------------------------------------------------ one head

// What a lane multiplies its two chunks a (dims 8l..) and b (D/2 + 8l..) of a
// normed head by: norm weight and rotation in one,
//   a' = a ac - b bs,  b' = b bc + a as.
struct Turn {
  F8 ac, bs, bc, as;
};

template <int D>
__device__ __forceinline__ void load_turn(const void* cos_t, const void* sin_t, int type,
                                          int64_t pos, int l, Turn& r) {
  const size_t at = (size_t)pos * D + 8 * l;
  r.ac = load8(cos_t, type, at);
  r.bc = load8(cos_t, type, at + D / 2);
  r.bs = load8(sin_t, type, at);
  r.as = load8(sin_t, type, at + D / 2);
}

// Brings the norm's weight into r (r holds cos and sin where `turned`).
template <int D, bool BF16>
__device__ __forceinline__ void weigh(const void* weight, int l, bool turned, Turn& r) {
  const F8 wa = load8(weight, BF16 ? W4_BF16 : W4_F16, 8 * l);
  const F8 wb = load8(weight, BF16 ? W4_BF16 : W4_F16, D / 2 + 8 * l);
  if (!turned) {
    r.ac = wa;
    r.bc = wb;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    r.ac.f[i] *= wa.f[i];
    r.bs.f[i] *= wb.f[i];
    r.bc.f[i] *= wb.f[i];
    r.as.f[i] *= wa.f[i];
  }
}

// A head spread over D / 16 neighbouring lanes: normed, then multiplied out.
// All lanes of the warp take part in the sum's exchange.
template <int D>
__device__ __forceinline__ void norm_turn(F8& a, F8& b, bool normed, float eps, bool turned,
                                          const Turn& r) {
  if (normed) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(a.f[i], a.f[i], fmaf(b.f[i], b.f[i], ss));
#pragma unroll
    for (int off = D / 32; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    const float inv = rsqrtf(ss * (1.0f / D) + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a.f[i] *= inv;
      b.f[i] *= inv;
    }
  }
  if (turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = a.f[i], y = b.f[i];
      a.f[i] = fmaf(x, r.ac.f[i], -(y * r.bs.f[i]));
      b.f[i] = fmaf(y, r.bc.f[i], x * r.as.f[i]);
    }
  } else if (normed) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a.f[i] *= r.ac.f[i];
      b.f[i] *= r.bc.f[i];
    }
  }
}

struct HeadsIn {
  const uint16_t* p;
  int64_t row, head;  // strides in elements
};

struct RopeParams {
  HeadsIn q, k;
  uint16_t *q_out, *k_out;
  int64_t q_out_row, q_out_head, k_out_row, k_out_head;
  const void *q_norm, *k_norm, *cos_t, *sin_t;
  const int64_t* positions;
  int heads, kv_heads, rows, max_pos;
  int table_type;
  float eps;
  int groups_per_warp;
  int* err;
};

// Groups of heads that a warp holds at once, of queries and of keys.
template <int D>
__host__ __device__ __forceinline__ int head_groups(int heads) {
  constexpr int HPW = 32 / (D / 16);
  return (heads + HPW - 1) / HPW;
}

// Head groups [g0, g1) of the queries or keys of one row.
template <int D, bool BF16>
__device__ __forceinline__ void rope_groups(const HeadsIn& x, uint16_t* out, int64_t out_row,
                                            int64_t out_head, int heads, const void* weight,
                                            const RopeParams& p, int64_t row, int64_t pos, int g0,
                                            int g1, int lane) {
  constexpr int L = D / 16, HPW = 32 / L;
  const int l = lane % L;
  const bool turned = p.cos_t != nullptr;
  const uint16_t* src = x.p + row * x.row + 8 * l;
  uint16_t* dst = out + row * out_row + 8 * l;
  auto load = [&](int h, uint4& va, uint4& vb) {
    va = vb = make_uint4(0u, 0u, 0u, 0u);
    if (h < heads) {
      va = *reinterpret_cast<const uint4*>(src + h * x.head);
      vb = *reinterpret_cast<const uint4*>(src + h * x.head + D / 2);
    }
  };
  uint4 va, vb;  // the next group's, on their way while a group is worked on
  load(g0 * HPW + lane / L, va, vb);
  Turn r;
  if (turned) load_turn<D>(p.cos_t, p.sin_t, p.table_type, pos, l, r);
  if (weight) weigh<D, BF16>(weight, l, turned, r);
#pragma unroll 1
  for (int g = g0; g < g1; ++g) {
    const int h = g * HPW + lane / L;
    F8 a = unpack8<BF16>(va), b = unpack8<BF16>(vb);
    if (g + 1 < g1) load(h + HPW, va, vb);
    norm_turn<D>(a, b, weight != nullptr, p.eps, turned, r);
    if (h < heads) {
      *reinterpret_cast<uint4*>(dst + h * out_head) = pack8<BF16>(a);
      *reinterpret_cast<uint4*>(dst + h * out_head + D / 2) = pack8<BF16>(b);
    }
  }
}

// Groups [g0, g1) of a row, the queries' first.
template <int D, bool BF16>
__device__ __forceinline__ void rope_row(const RopeParams& p, int64_t row, int64_t pos, int g0,
                                         int g1, int lane) {
  const int gq = head_groups<D>(p.heads);
  if (g0 < gq)
    rope_groups<D, BF16>(p.q, p.q_out, p.q_out_row, p.q_out_head, p.heads, p.q_norm, p, row, pos, g0,
                   min(g1, gq), lane);
  if (g1 > gq)
    rope_groups<D, BF16>(p.k, p.k_out, p.k_out_row, p.k_out_head, p.kv_heads, p.k_norm, p, row, pos,
                   max(g0 - gq, 0), g1 - gq, lane);
}

// Seven blocks an SM (72 registers): 33.1 us for the 8191 rows, 36.9 with six and 36.6
// with as many registers as it takes (85).
constexpr int kRopeThreads = 128;

template <int D, bool BF16>
__global__ void __launch_bounds__(kRopeThreads, 7) norm_rope_kernel(const RopeParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int groups = head_groups<D>(p.heads) + head_groups<D>(p.kv_heads);
  const int per_row = (groups + p.groups_per_warp - 1) / p.groups_per_warp;
  const int64_t unit = (int64_t)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = unit / per_row;
  if (row >= p.rows) return;
  const int g0 = (int)(unit - row * per_row) * p.groups_per_warp;
  const int64_t pos = p.positions ? p.positions[row] : 0;
  if (p.cos_t && (pos < 0 || pos >= p.max_pos)) {  // no such table row: the row is left as it is
    if (lane == 0) atomicCAS(p.err, 0, kErrKvRange);
    return;
  }
  rope_row<D, BF16>(p, row, pos, g0, min(groups, g0 + p.groups_per_warp), lane);
}

// ------------------------------------------------------------ append

struct AppendParams {
  RopeParams rope;  // q (heads may be 0), tables, k_norm; its k fields are unused
  HeadsIn k, v;
  uint8_t *k_cache, *v_cache;  // e4m3 [pages, kv_heads, page, D]
  float *k_scale, *v_scale;    // [pages, kv_heads]
  const int32_t *page_table, *lengths, *row_starts;
  int64_t table_stride;
  int pages, page, page_shift, max_pages, seqs, rows, kv_heads;
  int kv_units;   // K and V blocks of the (sequence, page) pairs that it may touch
  int kv_blocks;  // CTAs of the cache part; those after them turn queries
};

// First row and number of rows of sequence b, kept inside the buffers.
__device__ __forceinline__ int seq_rows(const AppendParams& p, int b, int* first) {
  const int a = min(max(p.row_starts[b], 0), p.rows);
  const int e = min(max(p.row_starts[b + 1], a), p.rows);
  *first = a;
  return e - a;
}

// Pages that n rows behind `past` tokens touch (behind a negative length: as many at most,
// of which none is written).
__device__ __forceinline__ int touched(int past, int n, int page_shift) {
  return n > 0 ? (((past & ((1 << page_shift) - 1)) + n - 1) >> page_shift) + 1 : 0;
}

constexpr int kAppendThreads = 256;

// One block of the cache, K or V of one head of one page, by W warps. A lane
// group holds NP rows in registers: a whole page with eight warps; one warp
// loads a block of more rows twice, for its largest value and for its codes.
template <int D, bool BF16, int W, int NP>
__device__ __forceinline__ void append_block(const AppendParams& p, int unit) {
  constexpr int L = D / 16, kThreads = W * 32, RPP = kThreads / L;  // rows a turn
  const int tid = threadIdx.x % kThreads, lane = tid & 31, l = tid % L;
  const bool is_v = unit & 1;
  const int h = (unit >> 1) % p.kv_heads;
  int g = (unit >> 1) / p.kv_heads;  // which (sequence, page) pair

  // Every warp finds the pair by a scan over the sequences, four neighbours a lane
  // if there are many: their loads go out together.
  const int each = p.seqs > 32 ? 4 : 1;
  int b = -1, past = 0, n = 0, first = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < p.seqs; b0 += 32 * each) {
    int f[4], m[4], ps[4], cnt[4], mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int bb = b0 + each * lane + i;
      f[i] = m[i] = ps[i] = 0;
      if (i < each && bb < p.seqs) {
        m[i] = seq_rows(p, bb, &f[i]);
        ps[i] = p.lengths[bb];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) mine += cnt[i] = touched(ps[i], m[i], p.page_shift);
    int incl = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, incl > g);
    if (hit) {
      const int src = __ffs(hit) - 1;
      int left = g - (incl - mine), at = 0;  // (lane src's are used)
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (at == i && i + 1 < each && left >= cnt[i]) left -= cnt[i], at = i + 1;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at == i) past = ps[i], n = m[i], first = f[i];
      b = b0 + each * src + __shfl_sync(0xffffffffu, at, src);
      g = __shfl_sync(0xffffffffu, left, src);
      past = __shfl_sync(0xffffffffu, past, src);
      n = __shfl_sync(0xffffffffu, n, src);
      first = __shfl_sync(0xffffffffu, first, src);
      break;
    }
    g -= __shfl_sync(0xffffffffu, incl, 31);
  }
  if (b < 0) return;  // fewer pairs than the bound
  const int64_t slot_page = (past >> p.page_shift) + g;                  // page of the sequence
  const int64_t tok0 = max((int64_t)past, slot_page * p.page);  // its first new token
  // Tokens that the rotation tables have no row for end the step, for K and V alike: a
  // page must not hold the value of a token whose key is missing.
  const int64_t stop = min((int64_t)past + n, (slot_page + 1) * p.page);
  const int64_t upto = p.rope.cos_t ? min(stop, (int64_t)p.rope.max_pos) : stop;
  const int cnt = past < 0 ? 0 : (int)max(upto - tok0, (int64_t)0);
  const int slot0 = (int)(tok0 - slot_page * p.page);
  const int64_t row0 = first + (tok0 - past);
  const int page = past >= 0 && slot_page < p.max_pages
                       ? p.page_table[(int64_t)b * p.table_stride + slot_page]
                       : -1;
  const bool turned = !is_v && p.rope.cos_t != nullptr;
  const HeadsIn& x = is_v ? p.v : p.k;

  F8 a[NP], c[NP];
  auto load = [&](int base) {  // rows base + i RPP + tid / L, normed and turned
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = base + i * RPP + tid / L;
      uint4 va = make_uint4(0u, 0u, 0u, 0u), vb = va;
      if (r < cnt) {
        const uint16_t* src = x.p + (row0 + r) * x.row + h * x.head + 8 * l;
        va = *reinterpret_cast<const uint4*>(src);
        vb = *reinterpret_cast<const uint4*>(src + D / 2);
      }
      a[i] = unpack8<BF16>(va);
      c[i] = unpack8<BF16>(vb);
      if (!is_v) {
        Turn t;
        if (turned)  // a row past the block's: any table row, its zeros stay zeros
          load_turn<D>(p.rope.cos_t, p.rope.sin_t, p.rope.table_type,
                       r < cnt ? tok0 + r : cnt > 0 ? tok0 : 0, l, t);
        if (p.rope.k_norm) weigh<D, BF16>(p.rope.k_norm, l, turned, t);
        norm_turn<D>(a[i], c[i], p.rope.k_norm != nullptr, p.rope.eps, turned, t);
      }
    }
  };
  load(0);  // on its way beside the page's number
  const bool no_page = page < 0 || page >= p.pages;
  if (tid == 0 && (no_page || upto < stop)) atomicCAS(p.rope.err, 0, kErrKvRange);
  if (no_page || cnt == 0) return;  // no such length, page, or position in it: not stored
  const size_t block = (size_t)page * p.kv_heads + h;
  float* scale_at = (is_v ? p.v_scale : p.k_scale) + block;
  uint8_t* codes = (is_v ? p.v_cache : p.k_cache) + block * p.page * D;
  const float old = slot0 > 0 ? *scale_at : 0.f;
  float amax = 0.f;
#pragma unroll 1
  for (int base = 0; base < cnt; base += NP * RPP) {
    if constexpr (W == 1)
      if (base > 0) load(base);
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // infinities and NaN do not set the scale (rows past cnt: 0)
        const float u = fabsf(a[i].f[j]), w = fabsf(c[i].f[j]);
        amax = fmaxf(amax, fmaxf(u <= 3.4028234e38f ? u : 0.f, w <= 3.4028234e38f ? w : 0.f));
      }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  if constexpr (W > 1) {
    __shared__ float red[W];
    if (lane == 0) red[tid >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) amax = fmaxf(amax, red[w]);
  }
  // amax = m 2^e with 1 <= m < 2, and 448 = 1.75 * 2^8: the least power of
  // two is 2^(e - 8), or twice that when m > 1.75
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, kMinScaleExp), kMaxScaleExp);
  const float scale = fmaxf(__uint_as_float((uint32_t)(e + 127) << 23), old);
  const float inv = 1.0f / scale;  // a power of two, unless the block's own scale was none
#pragma unroll 1
  for (int base = 0; base < cnt; base += NP * RPP) {
    if constexpr (W == 1)
      if (cnt > NP * RPP) load(base);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = base + i * RPP + tid / L;
      if (r < cnt) {
        uint8_t* dst = codes + (size_t)(slot0 + r) * D + 8 * l;
        *reinterpret_cast<uint2*>(dst) = to_e4m3x8(a[i], inv);
        *reinterpret_cast<uint2*>(dst + D / 2) = to_e4m3x8(c[i], inv);
      }
    }
  }
  if (scale != old) {
    if (tid == 0) *scale_at = scale;
    const float ratio = old * inv;  // the rows in use, rounded again in the larger scale
    uint4* at = reinterpret_cast<uint4*>(codes);
    const int chunks = slot0 * (D / 16);
#pragma unroll 1
    for (int i0 = tid; i0 < chunks; i0 += 4 * kThreads) {  // four reads on their way
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k * kThreads < chunks) v[k] = at[i0 + k * kThreads];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k * kThreads < chunks) {
          const uint2 lo = again_e4m3x8(make_uint2(v[k].x, v[k].y), ratio);
          const uint2 hi = again_e4m3x8(make_uint2(v[k].z, v[k].w), ratio);
          at[i0 + k * kThreads] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
    }
  }
}

template <int D, bool BF16, int W, int NP>
__global__ void __launch_bounds__(kAppendThreads, W == 1 ? 3 : NP == 4 ? 2 : 3)
    append_kernel(const AppendParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  if ((int)blockIdx.x < p.kv_blocks) {
    const int unit = W == 1 ? (int)blockIdx.x * (kAppendThreads / 32) + (int)(threadIdx.x >> 5)
                            : (int)blockIdx.x;
    if (unit < p.kv_units) append_block<D, BF16, W, NP>(p, unit);
    return;
  }
  // queries: a warp takes a row's heads, or a part of them
  const int lane = threadIdx.x & 31;
  const RopeParams& r = p.rope;
  const int groups = head_groups<D>(r.heads);
  const int per_row = (groups + r.groups_per_warp - 1) / r.groups_per_warp;
  const int64_t unit =
      (int64_t)(blockIdx.x - p.kv_blocks) * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = unit / per_row;
  if (row >= p.rows) return;
  const int g0 = (int)(unit - row * per_row) * r.groups_per_warp;
  const int g1 = min(groups, g0 + r.groups_per_warp);
  {  // the heads on their way while the row's position is looked up
    constexpr int kLanes = D / 64;  // lanes a head: one a 128-byte line
    for (int h = g0 * (32 / (D / 16)) + lane / kLanes; h < min(r.heads, g1 * (32 / (D / 16)));
         h += 32 / kLanes)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(r.q.p + row * r.q.row + h * r.q.head +
                                                    64 * (lane % kLanes)));
  }
  int b = 0;  // the sequence: as many as end at or before this row
#pragma unroll 4
  for (int b0 = 0; b0 < p.seqs; b0 += 32) {
    const int bb = b0 + lane;
    b += __popc(__ballot_sync(0xffffffffu, bb < p.seqs && p.row_starts[bb + 1] <= row));
  }
  if (b >= p.seqs || row < p.row_starts[b]) return;  // a row outside every sequence
  const int length = p.lengths[b];
  const int64_t pos = (int64_t)length + row - max(p.row_starts[b], 0);
  if (length < 0 || (r.cos_t && pos >= r.max_pos)) {
    if (lane == 0) atomicCAS(r.err, 0, kErrKvRange);
    return;
  }
  rope_row<D, BF16>(r, row, pos, g0, g1, lane);
}

template <int D, bool BF16>
auto append_fn(bool by_warp, int np) -> void (*)(AppendParams) {
  if (by_warp) return append_kernel<D, BF16, 1, 1>;
  if (np == 4) return append_kernel<D, BF16, 8, D == 128 ? 4 : 2>;  // pages of 128, D = 128
  return np == 2 ? append_kernel<D, BF16, 8, 2> : append_kernel<D, BF16, 8, 1>;
}

HeadsIn heads_in(const w4_heads& x) {
  return HeadsIn{static_cast<const uint16_t*>(x.ptr), x.row_stride, x.head_stride};
}

// Head groups a warp takes: whole rows (the position's table row is then read
// once) when there are rows enough, else one group a warp, so that a few rows
// still spread over the SMs. Rows of 32 and 8 heads, a group a warp and whole rows:
// 64 rows 2.3 and 5.6 us, 512 5.3 and 5.7, 1024 7.6 and 6.4, 4096 28 and 16.
int groups_per_warp(int64_t rows, int groups, int sms) {
  return rows > 5 * (int64_t)sms ? std::max(groups, 1) : 1;
}

RopeParams rope_params(const w4_rope& r, const DeviceInfo& di) {
  RopeParams p = {};
  p.cos_t = r.cos_table;
  p.sin_t = r.sin_table;
  p.table_type = r.table_dtype;
  p.max_pos = r.max_pos;
  p.q_norm = r.q_norm;
  p.k_norm = r.k_norm;
  p.eps = r.eps;
  p.err = di.err_word;
  return p;
}

void set_queries(RopeParams& p, const w4_heads& q, const w4_heads& q_out) {
  p.q = heads_in(q);
  p.heads = q.heads;
  p.q_out = static_cast<uint16_t*>(q_out.ptr);
  p.q_out_row = q_out.row_stride;
  p.q_out_head = q_out.head_stride;
}

}  // namespace

int launch_norm_rope(const w4_heads& q, const w4_heads& k, const w4_heads& q_out,
                     const w4_heads& k_out, int bf16, int rows, int head_dim, const w4_rope& rope,
                     const int64_t* positions, const DeviceInfo& di, cudaStream_t stream) {
  RopeParams p = rope_params(rope, di);
  set_queries(p, q, q_out);
  p.k = heads_in(k);
  p.kv_heads = k.heads;
  p.k_out = static_cast<uint16_t*>(k_out.ptr);
  p.k_out_row = k_out.row_stride;
  p.k_out_head = k_out.head_stride;
  p.positions = positions;
  p.rows = rows;
  const int groups = head_dim == 128 ? head_groups<128>(p.heads) + head_groups<128>(p.kv_heads)
                                     : head_groups<64>(p.heads) + head_groups<64>(p.kv_heads);
  p.groups_per_warp = groups_per_warp(rows, groups, di.sm_count);
  const int64_t units = (int64_t)rows * ((groups + p.groups_per_warp - 1) / p.groups_per_warp);
  const int64_t blocks = (units + kRopeThreads / 32 - 1) / (kRopeThreads / 32);
  if (blocks > 0x7fffffff) return fail(W4_ERR_UNSUPPORTED, "w4_qk_norm_rope: %d rows", rows);
  void (*fn)(RopeParams) = head_dim == 128
                               ? (bf16 ? norm_rope_kernel<128, true> : norm_rope_kernel<128, false>)
                               : (bf16 ? norm_rope_kernel<64, true> : norm_rope_kernel<64, false>);
  const cudaError_t e =
      launch_overlapped(fn, dim3((unsigned)blocks), kRopeThreads, 0, stream, p);
  return e == cudaSuccess ? W4_OK : cuda_fail(e, "w4_qk_norm_rope launch");
}

int launch_kv8_append(const w4_kv8_cache& c, const w4_kv_batch& bt, const w4_heads& k,
                      const w4_heads& v, const w4_heads& q, const w4_heads& q_out, int bf16,
                      const w4_rope& rope, const DeviceInfo& di, cudaStream_t stream) {
  AppendParams p = {};
  p.rope = rope_params(rope, di);
  set_queries(p.rope, q, q_out);
  p.rope.rows = bt.rows;
  p.k = heads_in(k);
  p.v = heads_in(v);
  p.k_cache = static_cast<uint8_t*>(c.k);
  p.v_cache = static_cast<uint8_t*>(c.v);
  p.k_scale = c.k_scale;
  p.v_scale = c.v_scale;
  p.page_table = bt.page_table;
  p.lengths = bt.lengths;
  p.row_starts = bt.row_starts;
  p.table_stride = bt.table_stride;
  p.pages = c.pages;
  p.page = c.page_size;
  p.page_shift = c.page_size == 16 ? 4 : c.page_size == 32 ? 5 : c.page_size == 64 ? 6 : 7;
  p.kv_heads = c.kv_heads;
  p.max_pages = bt.max_pages;
  p.seqs = bt.seqs;
  p.rows = bt.rows;
  // n rows of a sequence touch at most (n - 1) / page + 2 pages, and no more than n
  const int64_t pairs =
      std::min<int64_t>(bt.rows, (int64_t)bt.rows / c.page_size + 2 * (int64_t)bt.seqs);
  const int64_t kv_units = pairs * c.kv_heads * 2;
  // A warp a block of the cache while sequences bring a few rows each (most threads of
  // a CTA would idle), and for more rows where there are blocks for many waves of
  // CTAs; else a CTA a block. By warps and by CTAs, 8 heads of 128: 64 sequences of 1
  // row 3.6 and 11.6 us, of 8 on average 11.2 and 17.3, of 16 19.0 and 20.0, of 32 39
  // and 25; 32 of 8 (1152 units) 11.1 and 9.4; 8 of 4 3.2 and 5.1, of 8 5.6 and 5.7, of
  // 16 15.9 and 5.7.
  const bool by_warp = bt.rows <= 4 * (int64_t)bt.seqs ||
                       (bt.rows <= 16 * (int64_t)bt.seqs && kv_units >= 10 * (int64_t)di.sm_count);
  const int64_t kv_blocks =
      by_warp ? (kv_units + kAppendThreads / 32 - 1) / (kAppendThreads / 32) : kv_units;
  const int groups = c.head_dim == 128 ? head_groups<128>(q.heads) : head_groups<64>(q.heads);
  p.rope.groups_per_warp = groups_per_warp(bt.rows, groups, di.sm_count);
  const int64_t units =
      (int64_t)bt.rows * ((groups + p.rope.groups_per_warp - 1) / p.rope.groups_per_warp);
  const int64_t blocks = kv_blocks + (units + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  if (blocks > 0x7fffffff || kv_units > 0x7fffffff)
    return fail(W4_ERR_UNSUPPORTED, "w4_kv8_append: %d rows", bt.rows);
  p.kv_units = (int)kv_units;
  p.kv_blocks = (int)kv_blocks;
  const int np = std::max(1, c.page_size * (c.head_dim / 16) / kAppendThreads);
  void (*fn)(AppendParams) = c.head_dim == 128
                                 ? (bf16 ? append_fn<128, true>(by_warp, np)
                                         : append_fn<128, false>(by_warp, np))
                                 : (bf16 ? append_fn<64, true>(by_warp, np)
                                         : append_fn<64, false>(by_warp, np));
  const cudaError_t e =
      launch_overlapped(fn, dim3((unsigned)blocks), kAppendThreads, 0, stream, p);
  return e == cudaSuccess ? W4_OK : cuda_fail(e, "w4_kv8_append launch");
}

}  // namespace w4
