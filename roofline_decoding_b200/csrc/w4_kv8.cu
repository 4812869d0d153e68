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
#include "w4_internal.h"
#include "w4_ptx.cuh"

#include <cuda_fp8.h>

#include <algorithm>

namespace w4 {

namespace {

constexpr int kMinScaleExp = -32, kMaxScaleExp = 120;

// ------------------------------------------------------------ element types

// Eight 16-bit elements (16 bytes) to fp32.
__device__ __forceinline__ void unpack8(const uint4& v, int bf16, float (&f)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (bf16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8], int bf16) {
  uint4 v;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (bf16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return v;
}

// Eight elements at index i (a multiple of 8) of a table or weight.
__device__ __forceinline__ void load8(const void* p, int type, size_t i, float (&f)[8]) {
  if (type == W4_F32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
    const float4 b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i) + 1);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
    f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    unpack8(__ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i)),
            type == W4_BF16, f);
  }
}

// Eight fp32 values to e4m3: round to nearest even, +-448 beyond the range
// (infinities too), NaN kept.
__device__ __forceinline__ uint2 to_e4m3x8(const float (&f)[8], float mul) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(
        make_float2(f[4 * i] * mul, f[4 * i + 1] * mul), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(
        make_float2(f[4 * i + 2] * mul, f[4 * i + 3] * mul), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// ------------------------------------------------------------ one head

// The rotation of one position: this lane's chunks of its cos and sin rows.
struct Turn {
  float c0[8], c1[8], s0[8], s1[8];
};

template <int D>
__device__ __forceinline__ void load_turn(const void* cos_t, const void* sin_t, int type,
                                          int64_t pos, int l, Turn& r) {
  const size_t at = (size_t)pos * D + 8 * l;
  load8(cos_t, type, at, r.c0);
  load8(cos_t, type, at + D / 2, r.c1);
  load8(sin_t, type, at, r.s0);
  load8(sin_t, type, at + D / 2, r.s1);
}

// Norm (where the lane's head has a weight) and rotation of a head spread over
// D / 16 neighbouring lanes. `normed` is the same for the whole warp: every
// lane takes part in the sum's exchange.
template <int D>
__device__ __forceinline__ void norm_turn(float (&a)[8], float (&b)[8], bool normed,
                                          const void* weight, int bf16, float eps, int l,
                                          bool turned, const Turn& r) {
  if (normed) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
#pragma unroll
    for (int off = D / 32; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if (weight) {
      const float inv = rsqrtf(ss / (float)D + eps);
      float w0[8], w1[8];
      load8(weight, bf16 ? W4_BF16 : W4_F16, 8 * l, w0);
      load8(weight, bf16 ? W4_BF16 : W4_F16, D / 2 + 8 * l, w1);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] = a[i] * inv * w0[i];
        b[i] = b[i] * inv * w1[i];
      }
    }
  }
  if (turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = a[i], y = b[i];
      a[i] = fmaf(x, r.c0[i], -(y * r.s0[i]));
      b[i] = fmaf(y, r.c1[i], x * r.s1[i]);
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
  int bf16, table_type;
  float eps;
  int groups_per_warp;
  int* err;
};

// Heads [h_first, h_last) of one row, 32 / (D/16) at a time; the loads of U
// turns go out together.
template <int D, int U>
__device__ __forceinline__ void rope_heads(const RopeParams& p, int64_t row, int64_t pos,
                                           int h_first, int h_last, int lane) {
  constexpr int L = D / 16, HPW = 32 / L;
  const int l = lane % L;
  Turn r;
  if (p.cos_t) load_turn<D>(p.cos_t, p.sin_t, p.table_type, pos, l, r);
#pragma unroll 1
  for (int h0 = h_first; h0 < h_last; h0 += U * HPW) {
    uint4 va[U], vb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * HPW + lane / L;
      va[u] = vb[u] = make_uint4(0u, 0u, 0u, 0u);
      if (h < h_last) {
        const uint16_t* src = (h < p.heads ? p.q.p + row * p.q.row + h * p.q.head
                                           : p.k.p + row * p.k.row + (h - p.heads) * p.k.head) +
                              8 * l;
        va[u] = *reinterpret_cast<const uint4*>(src);
        vb[u] = *reinterpret_cast<const uint4*>(src + D / 2);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * HPW + lane / L;
      const bool is_q = h < p.heads;
      float a[8], b[8];
      unpack8(va[u], p.bf16, a);
      unpack8(vb[u], p.bf16, b);
      // a turn may hold the last query heads and the first key heads: each lane
      // takes its own head's weight
      norm_turn<D>(a, b, p.q_norm || p.k_norm, is_q ? p.q_norm : p.k_norm, p.bf16, p.eps, l,
                   p.cos_t != nullptr, r);
      if (h < h_last) {
        uint16_t* dst = (is_q ? p.q_out + row * p.q_out_row + h * p.q_out_head
                              : p.k_out + row * p.k_out_row + (h - p.heads) * p.k_out_head) +
                        8 * l;
        *reinterpret_cast<uint4*>(dst) = pack8(a, p.bf16);
        *reinterpret_cast<uint4*>(dst + D / 2) = pack8(b, p.bf16);
      }
    }
  }
}

constexpr int kRopeThreads = 128;

template <int D, int U>
__global__ void __launch_bounds__(kRopeThreads) norm_rope_kernel(const RopeParams p) {
  constexpr int HPW = 32 / (D / 16);
  const int lane = threadIdx.x & 31;
  const int all = p.heads + p.kv_heads, groups = (all + HPW - 1) / HPW;
  const int per_row = (groups + p.groups_per_warp - 1) / p.groups_per_warp;
  const int64_t unit = (int64_t)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = unit / per_row;
  if (row >= p.rows) return;
  const int h0 = (int)(unit - row * per_row) * p.groups_per_warp * HPW;
  const int64_t pos = p.positions ? p.positions[row] : 0;
  if (p.cos_t && (pos < 0 || pos >= p.max_pos)) {  // no such table row: the row is left as it is
    if (lane == 0) atomicCAS(p.err, 0, kErrKvRange);
    return;
  }
  rope_heads<D, U>(p, row, pos, h0, min(all, h0 + p.groups_per_warp * HPW), lane);
}

// ------------------------------------------------------------ append

struct AppendParams {
  RopeParams rope;  // q (heads may be 0), tables, k_norm; its k fields are unused
  HeadsIn k, v;
  uint8_t *k_cache, *v_cache;  // e4m3 [pages, kv_heads, page, D]
  float *k_scale, *v_scale;    // [pages, kv_heads]
  const int32_t *page_table, *lengths, *row_starts;
  int64_t table_stride;
  int pages, page, max_pages, seqs, rows, kv_heads;
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

// Pages that n rows behind `past` tokens touch.
__device__ __forceinline__ int touched(int past, int n, int page) {
  return n > 0 ? (past % page + n - 1) / page + 1 : 0;
}

constexpr int kAppendThreads = 256;

// One block of the cache, K or V of one head of one page, by W warps. Each
// pass holds NP rows a lane group in registers; a block of more rows is loaded
// twice, for its largest value and for its codes.
template <int D, int W, int NP>
__device__ __forceinline__ void append_block(const AppendParams& p, int unit) {
  constexpr int L = D / 16, kThreads = W * 32, RPP = kThreads / L;  // rows a turn
  const int tid = threadIdx.x % kThreads, lane = tid & 31, l = tid % L;
  const bool is_v = unit & 1;
  const int h = (unit >> 1) % p.kv_heads;
  int g = (unit >> 1) / p.kv_heads;  // which (sequence, page) pair

  // every warp finds the pair by a scan over the sequences, 32 at a time
  int b = -1, past = 0, n = 0, first = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < p.seqs; b0 += 32) {
    const int bb = b0 + lane;
    int f = 0, m = 0, ps = 0;
    if (bb < p.seqs) {
      m = seq_rows(p, bb, &f);
      ps = max(p.lengths[bb], 0);
    }
    const int cnt = touched(ps, m, p.page);
    int incl = cnt;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, incl > g);
    if (hit) {
      const int src = __ffs(hit) - 1;
      b = b0 + src;
      g -= __shfl_sync(0xffffffffu, incl - cnt, src);
      past = __shfl_sync(0xffffffffu, ps, src);
      n = __shfl_sync(0xffffffffu, m, src);
      first = __shfl_sync(0xffffffffu, f, src);
      break;
    }
    g -= __shfl_sync(0xffffffffu, incl, 31);
  }
  if (b < 0) return;  // fewer pairs than the bound
  const int64_t slot_page = past / p.page + g;                  // page of the sequence
  const int64_t tok0 = max((int64_t)past, slot_page * p.page);  // its first new token
  const int cnt = (int)(min((int64_t)past + n, (slot_page + 1) * p.page) - tok0);
  const int slot0 = (int)(tok0 - slot_page * p.page);
  const int64_t row0 = first + (tok0 - past);
  const int page =
      slot_page < p.max_pages ? p.page_table[(int64_t)b * p.table_stride + slot_page] : -1;
  const bool turned = !is_v && p.rope.cos_t != nullptr;
  if (page < 0 || page >= p.pages || (turned && tok0 + cnt > p.rope.max_pos)) {
    if (tid == 0) atomicCAS(p.rope.err, 0, kErrKvRange);  // no such page or position: not stored
    return;
  }
  const HeadsIn& x = is_v ? p.v : p.k;
  const size_t block = (size_t)page * p.kv_heads + h;
  float* scale_at = (is_v ? p.v_scale : p.k_scale) + block;
  uint8_t* codes = (is_v ? p.v_cache : p.k_cache) + block * p.page * D;
  const float old = slot0 > 0 ? *scale_at : 0.f;

  float a[NP][8], c[NP][8];
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
      unpack8(va, p.rope.bf16, a[i]);
      unpack8(vb, p.rope.bf16, c[i]);
      if (!is_v) {
        Turn t;
        if (turned && r < cnt)
          load_turn<D>(p.rope.cos_t, p.rope.sin_t, p.rope.table_type, tok0 + r, l, t);
        norm_turn<D>(a[i], c[i], p.rope.k_norm != nullptr, p.rope.k_norm, p.rope.bf16, p.rope.eps,
                     l, turned && r < cnt, t);
      }
    }
  };
  float amax = 0.f;
#pragma unroll 1
  for (int base = 0; base < cnt; base += NP * RPP) {
    load(base);
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // infinities and NaN do not set the scale (rows past cnt: 0)
        const float u = fabsf(a[i][j]), w = fabsf(c[i][j]);
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
#pragma unroll 1
    for (int i = tid; i < slot0 * (D / 8); i += kThreads) {
      uint2* at = reinterpret_cast<uint2*>(codes) + i;
      const uint2 v = *at;
      float f[8];
      const uint32_t w[2] = {v.x, v.y};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(
            (__nv_fp8x2_storage_t)((w[j >> 1] >> (16 * (j & 1))) & 0xffffu), __NV_E4M3);
        const float2 f2 = __half22float2(*reinterpret_cast<const __half2*>(&hr));
        f[2 * j] = f2.x;
        f[2 * j + 1] = f2.y;
      }
      *at = to_e4m3x8(f, ratio);
    }
  }
}

template <int D, int W, int NP>
__global__ void __launch_bounds__(kAppendThreads, W == 1 ? 3 : NP == 4 ? 2 : 3)
    append_kernel(const AppendParams p) {
  if ((int)blockIdx.x < p.kv_blocks) {
    const int unit = W == 1 ? (int)blockIdx.x * (kAppendThreads / 32) + (int)(threadIdx.x >> 5)
                            : (int)blockIdx.x;
    if (unit < p.kv_units) append_block<D, W, NP>(p, unit);
    return;
  }
  // queries: a warp takes a row's heads, or a part of them
  constexpr int HPW = 32 / (D / 16);
  const int lane = threadIdx.x & 31;
  const RopeParams& r = p.rope;
  const int groups = (r.heads + HPW - 1) / HPW;
  const int per_row = (groups + r.groups_per_warp - 1) / r.groups_per_warp;
  const int64_t unit =
      (int64_t)(blockIdx.x - p.kv_blocks) * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = unit / per_row;
  if (row >= p.rows) return;
  int b = 0;  // the sequence: as many as end at or before this row
#pragma unroll 1
  for (int b0 = 0; b0 < p.seqs; b0 += 32) {
    const int bb = b0 + lane;
    b += __popc(__ballot_sync(0xffffffffu, bb < p.seqs && p.row_starts[bb + 1] <= row));
  }
  if (b >= p.seqs || row < p.row_starts[b]) return;  // a row outside every sequence
  const int64_t pos = (int64_t)max(p.lengths[b], 0) + row - max(p.row_starts[b], 0);
  if (r.cos_t && pos >= r.max_pos) {
    if (lane == 0) atomicCAS(r.err, 0, kErrKvRange);
    return;
  }
  const int h0 = (int)(unit - row * per_row) * r.groups_per_warp * HPW;
  rope_heads<D, 1>(r, row, pos, h0, min(r.heads, h0 + r.groups_per_warp * HPW), lane);
}

HeadsIn heads_in(const w4_heads& x) {
  return HeadsIn{static_cast<const uint16_t*>(x.ptr), x.row_stride, x.head_stride};
}

// Head groups a warp takes: whole rows (the position's table row is then read
// once) when there are rows enough for about 32 warps an SM, else one group a
// warp, so that a few rows still spread over the SMs.
int groups_per_warp(int64_t rows, int groups, int sms) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(groups, rows * groups / (32 * sms)));
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
  p.bf16 = bf16;
  const int hpw = 32 / (head_dim / 16);
  const int groups = (p.heads + p.kv_heads + hpw - 1) / hpw;
  p.groups_per_warp = groups_per_warp(rows, groups, di.sm_count);
  const int64_t units = (int64_t)rows * ((groups + p.groups_per_warp - 1) / p.groups_per_warp);
  const int64_t blocks = (units + kRopeThreads / 32 - 1) / (kRopeThreads / 32);
  if (blocks > 0x7fffffff) return fail(W4_ERR_UNSUPPORTED, "w4_qk_norm_rope: %d rows", rows);
  void (*fn)(RopeParams) = head_dim == 128 ? norm_rope_kernel<128, 2> : norm_rope_kernel<64, 2>;
  fn<<<(unsigned)blocks, kRopeThreads, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? W4_OK : cuda_fail(e, "w4_qk_norm_rope launch");
}

int launch_kv8_append(const w4_kv8_cache& c, const w4_kv_batch& bt, const w4_heads& k,
                      const w4_heads& v, const w4_heads& q, const w4_heads& q_out, int bf16,
                      const w4_rope& rope, const DeviceInfo& di, cudaStream_t stream) {
  AppendParams p = {};
  p.rope = rope_params(rope, di);
  set_queries(p.rope, q, q_out);
  p.rope.rows = bt.rows;
  p.rope.bf16 = bf16;
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
  p.kv_heads = c.kv_heads;
  p.max_pages = bt.max_pages;
  p.seqs = bt.seqs;
  p.rows = bt.rows;
  // n rows of a sequence touch at most (n - 1) / page + 2 pages, and no more than n
  const int64_t pairs =
      std::min<int64_t>(bt.rows, (int64_t)bt.rows / c.page_size + 2 * (int64_t)bt.seqs);
  const int64_t kv_units = pairs * c.kv_heads * 2;
  // A warp a block of the cache while sequences bring a few rows each: most
  // threads of a CTA would idle on one row. A CTA a block for prompts.
  const bool by_warp = bt.rows <= 4 * (int64_t)bt.seqs;
  const int64_t kv_blocks =
      by_warp ? (kv_units + kAppendThreads / 32 - 1) / (kAppendThreads / 32) : kv_units;
  const int hpw = 32 / (c.head_dim / 16);
  const int groups = (q.heads + hpw - 1) / hpw;
  p.rope.groups_per_warp = groups_per_warp(bt.rows, groups, di.sm_count);
  const int64_t units =
      (int64_t)bt.rows * ((groups + p.rope.groups_per_warp - 1) / p.rope.groups_per_warp);
  const int64_t blocks = kv_blocks + (units + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  if (blocks > 0x7fffffff || kv_units > 0x7fffffff)
    return fail(W4_ERR_UNSUPPORTED, "w4_kv8_append: %d rows", bt.rows);
  p.kv_units = (int)kv_units;
  p.kv_blocks = (int)kv_blocks;
  const int np = std::max(1, c.page_size * (c.head_dim / 16) / kAppendThreads);
  void (*fn)(AppendParams);
  if (c.head_dim == 128)
    fn = by_warp   ? append_kernel<128, 1, 1>
         : np == 4 ? append_kernel<128, 8, 4>
         : np == 2 ? append_kernel<128, 8, 2>
                   : append_kernel<128, 8, 1>;
  else
    fn = by_warp   ? append_kernel<64, 1, 1>
         : np == 2 ? append_kernel<64, 8, 2>
                   : append_kernel<64, 8, 1>;
  fn<<<(unsigned)blocks, kAppendThreads, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? W4_OK : cuda_fail(e, "w4_kv8_append launch");
}

}  // namespace w4
