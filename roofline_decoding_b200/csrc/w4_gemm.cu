// w4_gemm.cu - W4A16 GEMM on the 5th-generation tensor cores (tcgen05) for
// the prefill rows of W4Linear.
//
// Y[M, N] = X[M, K] @ W[K, N], W = dequantize_v1(packed, scales): the
// operation the reference runs for more than 8 rows as dequantize_v1 (an
// fp16 [K, N] copy of the weights, roofline/kernels.py:77-90) followed by an
// fp32 matmul (scripts/decode_loop.py:51-55). Here the dequantised tile never
// leaves shared memory:
//   TMA warps    : one brings X tiles [up to 256 rows x 64 k] (128B swizzle,
//                  the canonical K-major layout the MMA reads), the other the
//                  packed words of the W tile (128 or 256 columns), each
//                  through a ring of its own: words leave as soon as they are
//                  unpacked, so the dequantisation runs ahead of the MMA and
//                  no load's latency waits for an MMA's (2048 x 8960 x 1536:
//                  64 us, 93 with one ring for both);
//   8 dequant warps: expand each packed word into 8 fp16 (q - 8) * s values
//                  - bit-identical to dequantize_v1 - and write them K-major,
//                  128B-swizzled, into one of the B buffers;
//   MMA warp     : one thread issues tcgen05.mma (M = 128, N = 128 or 256,
//                  K = 16, fp32 accumulate in tensor memory), four per 64-k
//                  stage for each of the tile's one or two 128-row halves
//                  (both halves share one dequantised B tile), and commits to
//                  the ring's mbarriers;
//   epilogue     : the dequant warps read the accumulators with tcgen05.ld,
//                  apply bias, activation (or the gated pair of interleaved
//                  gate and up columns) and residual in fp32 where the call
//                  asks for them, and store Y (fp16 or bf16) with one rounding.
// bf16 activations use bf16 weights bf16((q - 8) * s) (one rounding of the
// fp32 product; the reference has no bf16 path). Every wait is bounded; a
// CTA that gives up sets the device error word, drains its copies and
// frees its tensor memory.
//
// Work split: a launch covers a region of output tiles in row-major order
// (blockIdx.x) and may cut K into up to 8 slices (blockIdx.z), the slices of
// a tile forming a thread-block cluster. A sliced CTA leaves its fp32
// accumulators in shared memory (the freed operand rings) and every rank then
// sums a band of the tile's rows over all ranks in rank order (DSMEM), so the
// result does not depend on scheduling. The host uses slices for grids of
// too few tiles, and for the last few tiles of a grid that would otherwise
// leave most SMs idle in a final wave (a second, programmatically dependent
// launch that runs while the first one's last wave finishes).
#include "w4_internal.h"
#include "w4_tcgen05.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace w4 {

namespace {

constexpr int kUM = 128;          // MMA M (rows of one accumulator)
constexpr int kBMMax = 2 * kUM;   // rows of Y per CTA: up to two accumulators share a W tile
constexpr int kBK = 64;           // k per ring stage (one 128-byte swizzle row of fp16)
constexpr int kDqWarps = 8;       // dequant (and epilogue) warps
constexpr int kMmaWarp = 1 + kDqWarps;
constexpr int kPackedWarp = kMmaWarp + 1;
constexpr int kGemmThreads = 32 * (kPackedWarp + 1);  // warp 0 X, 1..8 dequant, 9 MMA, 10 W
constexpr int kErrGemmWait = 7;

struct GemmParams {
  void* y;
  int M, K, N;
  int x_bf16, y_bf16;
  int* err;
  // output tiles of this launch: blockIdx.x = t is tile (m_tile0 + t / ntx,
  // n_tile0 + t % ntx) in units of the instance's rows and columns
  int m_tile0, n_tile0, ntx;
  uint32_t x_bytes;  // of an X tile's copy
  int ksplit;       // K slices (gridDim.z, one cluster per tile when > 1)
  const uint16_t* scales;  // fp16 [K/128, N]
  int act;               // w4_act
  const void* bias;      // [N] of y's type, or null
  const void* residual;  // like y, or null
  int wait_at_end;  // the second launch of a plan runs beside the first and
                    // completes only after it (griddepcontrol.wait at exit);
                    // the first waits before it touches global memory
};

// Tile of BN columns (MMA N = BN, 128 or 256) and its shared memory layout
// (base 1024-aligned): X ring, B buffers, packed ring, then the barriers and the
// tensor-memory address. The rings take what the 227 KB hold.
template <int BN, int NACC>
struct GemmShape {
  // A stage: an X tile and a dequantised W tile. One barrier says that both
  // are there (the X copy's bytes and the dequant warps' arrivals), one that
  // the MMA has read both: the issuing thread's own instructions bound a stage
  // of few MMAs (each wait costs it about 130 clocks, each commit 70).
  static constexpr int kStages = BN == 128 ? (NACC == 1 ? 6 : 4) : (NACC == 1 ? 4 : 3);
  // The dequant warps work as two groups that take the stages in turn: a
  // stage's chain (wait, shared loads, unpack, shared stores, proxy fence,
  // arrival) is latency, not issue slots. The rings are then even, so that a
  // slot belongs to one group, which sees its phases one after another (a
  // parity wait cannot tell a phase from the next but one); three stages of the
  // largest tile are left to all warps together.
  static constexpr int kGroups = kStages % 2 == 0 ? 2 : 1;
  static constexpr int kGroupWarps = kDqWarps / kGroups;
  static constexpr int kPkStages = BN == 128 ? 6 : 4;
  static constexpr int kNumBars = 2 * kStages + 2 * kPkStages + 1;
  static constexpr int kBM = NACC * kUM;                 // rows of Y per CTA
  static constexpr int kXBytes = kBM * kBK * 2;          // 16 or 32 KB
  static constexpr int kBBytes = BN * kBK * 2;           // 16 or 32 KB
  static constexpr int kPkBytes = (kBK / 8) * BN * 4;    // packed words of a stage
  static constexpr int kTmemCols = NACC * BN;            // fp32 accumulators
  static constexpr int kOffX = 0;
  static constexpr int kOffB = kOffX + kStages * kXBytes;
  static constexpr int kOffPk = kOffB + kStages * kBBytes;
  static constexpr int kOffBar = kOffPk + kPkStages * kPkBytes;
  static constexpr int kOffTmem = kOffBar + kNumBars * 8;
  static constexpr int kSmem = 1024 + kOffTmem + 16;
  static constexpr int kColsPerThread = BN / (kGroupWarps * 32);  // of a group's stage
  static_assert(kSmem <= 227 * 1024 && kPkStages % kGroups == 0, "rings");
  static_assert(kOffB % 1024 == 0 && kXBytes % 1024 == 0 && kBBytes % 1024 == 0,
                "swizzled operand tiles start on 1024-byte boundaries");
  static_assert(kOffPk % 128 == 0 && kPkBytes % 128 == 0,
                "tensor-copy destinations are 128-byte aligned");
  static_assert(kTmemCols <= 512 && kColsPerThread * kGroupWarps * 32 == BN, "tile");
  // K slices: the fp32 partial tile (rows padded by 4 floats against bank
  // conflicts) reuses the X and B rings, free once the accumulators are final
  static constexpr int kPitch = BN + 4;
  static constexpr bool kCanSplit = kBM * kPitch * 4 <= kOffPk;
};

// ---------------------------------------------------------------- dequant

// One packed word (8 consecutive k of one column, nibble i = k 8j + i) to 8
// dequantised 16-bit values in k order: pair (q_2i, q_2i+1) is built by one
// byte permute of the word and its 4-bit shift plus one LOP3 into the
// mantissa of 1024 (fp16) or 128 (bf16); then (q - 8) is exact and the
// scale product is rounded once.
template <bool kBF16>
__device__ __forceinline__ uint4 dequant_word(uint32_t w, uint32_t s2, float sf) {
  const uint32_t y = w >> 4;
  uint32_t h[4];
  h[0] = __byte_perm(w, y, 0x4400);
  h[1] = __byte_perm(w, y, 0x5511);
  h[2] = __byte_perm(w, y, 0x6622);
  h[3] = __byte_perm(w, y, 0x7733);
  uint4 out;
  uint32_t* o = reinterpret_cast<uint32_t*>(&out);
  if constexpr (!kBF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = lop3_and_or(h[i], 0x000F000Fu, 0x64006400u);  // 1024 + q
      __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v),
                          __half2half2(__ushort_as_half(0x6408)));   // q - 8 (1032)
      d = __hmul2(d, *reinterpret_cast<const __half2*>(&s2));       // one rounding
      o[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  } else {
    const float off = -136.0f * sf;  // exact: 11 + 5 bits
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = lop3_and_or(h[i], 0x000F000Fu, 0x43004300u);  // 128 + q
      // (128 + q) s - 136 s = (q - 8) s: exact, it has 15 bits
      const float lo = fmaf(__uint_as_float(v << 16), sf, off);
      const float hi = fmaf(__uint_as_float(v & 0xFFFF0000u), sf, off);
      const __nv_bfloat162 d = __floats2bfloat162_rn(lo, hi);  // one rounding
      o[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
  return out;
}

// ---------------------------------------------------------------- epilogue

// Four 16-bit elements (8 bytes) or eight (16 bytes) to fp32.
template <int NV>
__device__ __forceinline__ void load_row(const void* p, size_t at, int bf16, float (&f)[NV]) {
  uint32_t w[NV / 2];
  const uint16_t* src = static_cast<const uint16_t*>(p) + at;
  if constexpr (NV == 8)
    *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(src);
  else
    *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(src);
#pragma unroll
  for (int i = 0; i < NV / 2; ++i) {
    if (bf16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

// NV elements of a row to 16 bits, two a word.
template <int NV>
__device__ __forceinline__ void pack_row(int bf16, const float (&f)[NV], uint32_t (&w)[NV / 2]) {
#pragma unroll
  for (int i = 0; i < NV / 2; ++i) {
    if (bf16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
}

__device__ __forceinline__ uint4 pick(bool first, const uint4& a, const uint4& b) {
  return make_uint4(first ? a.x : b.x, first ? a.y : b.y, first ? a.z : b.z, first ? a.w : b.w);
}
__device__ __forceinline__ uint4 swap_lanes(const uint4& v, int lanes) {
  return make_uint4(__shfl_xor_sync(0xffffffffu, v.x, lanes), __shfl_xor_sync(0xffffffffu, v.y, lanes),
                    __shfl_xor_sync(0xffffffffu, v.z, lanes), __shfl_xor_sync(0xffffffffu, v.w, lanes));
}
// Four lanes with a row of four 16-byte chunks each: chunk j of row t to chunk t of
// row j, and back. A warp then reads and writes 64 bytes of 8 rows at a time instead
// of 16 bytes of 32, each of which costs the L1 cache a line's turn.
__device__ __forceinline__ void transpose4(uint4 (&c)[4], int lane) {
#pragma unroll
  for (int s = 1; s <= 2; s <<= 1) {
    const bool odd = lane & s;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int lo = s == 1 ? 2 * i : i, hi = lo + s;
      const uint4 got = swap_lanes(pick(odd, c[lo], c[hi]), s);
      c[lo] = pick(odd, got, c[lo]);
      c[hi] = pick(odd, c[hi], got);
    }
  }
}

// a / (1 + e^-a), with the exponential of -|a|: that of -a leaves fp32 below -88 (and the
// short division is zero from 2^126 on), where a bf16 result times a large up column is
// still far from zero.
__device__ __forceinline__ float silu(float a) {
  const float e = __expf(-fabsf(a));
  return __fdividef(a < 0.f ? a * e : a, 1.0f + e);
}

// Bias and activation of NV accumulators of columns n.. of a row (u: the up
// columns, 32 further, of a gated pair).
template <int NV>
__device__ __forceinline__ void activate(const GemmParams& p, int n, float (&a)[NV],
                                         float (&u)[NV]) {
  const bool gated = p.act == W4_ACT_SWIGLU;
  if (p.bias) {
    float b[NV];
    load_row(p.bias, (size_t)n, p.y_bf16, b);
#pragma unroll
    for (int i = 0; i < NV; ++i) a[i] += b[i];
    if (gated) {
      load_row(p.bias, (size_t)n + W4B200_SWIGLU_BLOCK, p.y_bf16, b);
#pragma unroll
      for (int i = 0; i < NV; ++i) u[i] += b[i];
    }
  }
  if (gated) {
#pragma unroll
    for (int i = 0; i < NV; ++i) a[i] = silu(a[i]) * u[i];
  } else if (p.act == W4_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < NV; ++i) a[i] = silu(a[i]);
  } else if (p.act == W4_ACT_GELU) {
    // x Phi(x) by the complementary error function: 1 + erf would cancel in
    // the left tail
#pragma unroll
    for (int i = 0; i < NV; ++i) a[i] = 0.5f * a[i] * erfcf(a[i] * -0.70710678118654752f);
  }
}

// Where column n of a row goes: gate column 64 j + i is output column 32 j + i.
__device__ __forceinline__ size_t out_at(const GemmParams& p, int row, int n) {
  const bool gated = p.act == W4_ACT_SWIGLU;
  const int col = gated ? (n >> 6) * W4B200_SWIGLU_BLOCK + (n & (W4B200_SWIGLU_BLOCK - 1)) : n;
  return (size_t)row * (gated ? p.N / 2 : p.N) + col;
}

__device__ __forceinline__ void prefetch_l1(const void* p) {
  asm volatile("prefetch.global.L1 [%0];" ::"l"(p));
}
__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

template <bool kBF16, int BN, int NACC>
__global__ void __launch_bounds__(kGemmThreads, 1)
    w4_gemm_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                   const GemmParams p) {
  using S = GemmShape<BN, NACC>;
  extern __shared__ uint8_t smem_gemm[];
  uint8_t* base = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_gemm) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + S::kOffBar);
  uint64_t* full = bars;                           // X landed, W dequantised
  uint64_t* empty = full + S::kStages;             // the MMA has read both
  uint64_t* full_pk = empty + S::kStages;          // packed words landed
  uint64_t* empty_pk = full_pk + S::kPkStages;     // unpacked
  uint64_t* acc_full = empty_pk + S::kPkStages;    // accumulator final
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base + S::kOffTmem);
  int* abort_flag = reinterpret_cast<int*>(base + S::kOffTmem + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = (int)blockIdx.x;
  const int n0 = (p.n_tile0 + t % p.ntx) * BN, m0 = (p.m_tile0 + t / p.ntx) * S::kBM;
  // this CTA's K slice: 64-k stages [kt0, kt0 + KT)
  const int KT_all = p.K / kBK;
  const int kt0 = (int)((long long)blockIdx.z * KT_all / p.ksplit);
  const int KT = (int)((long long)(blockIdx.z + 1) * KT_all / p.ksplit) - kt0;

  auto load_x = [&](int kt) {
    const int s = kt % S::kStages;
    mbar_arrive_expect_tx(&full[s], p.x_bytes);
    tma_load_2d(base + S::kOffX + s * S::kXBytes, &tm_x, &full[s], (kt0 + kt) * kBK, m0);
  };
  auto load_w = [&](int kt) {
    const int s = kt % S::kPkStages;
    mbar_arrive_expect_tx(&full_pk[s], S::kPkBytes);
    tma_load_2d(base + S::kOffPk + s * S::kPkBytes, &tm_w, &full_pk[s], n0, (kt0 + kt) * (kBK / 8));
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], S::kGroupWarps + 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < S::kPkStages; ++i) {
      mbar_init(&full_pk[i], 1);
      mbar_init(&empty_pk[i], S::kGroupWarps);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
    if (!p.wait_at_end) grid_dependency_wait();  // the inputs are written
    // the first copies go out while the other warps still set up
    for (int kt = 0; kt < min(S::kPkStages, KT); ++kt) load_w(kt);
    for (int kt = 0; kt < min(S::kStages, KT); ++kt) load_x(kt);
  }
  if (warp == kMmaWarp) {  // tensor memory for the accumulators
    tc_alloc(tmem_slot, S::kTmemCols);
    tc_fence_before();
  }
  if (!p.wait_at_end) grid_dependency_wait();
  // A dependent launch may fill the SMs that this grid frees. The second launch
  // of a plan does not wait before it reads, so it must not start before what
  // wrote the inputs has ended: not before this wait.
  grid_launch_dependents();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_d = *tmem_slot;
  auto give_up = [&](int code) {
    if (p.err) atomicCAS(p.err, 0, code);
    *reinterpret_cast<volatile int*>(abort_flag) = 1;
  };
  auto stopped = [&]() { return *reinterpret_cast<volatile int*>(abort_flag) != 0; };

  if (warp == 0) {
    // ------------------------------------------------------------ X
    if (lane == 0) {
      int issued = min(S::kStages, KT);
      for (int kt = issued; kt < KT; ++kt) {
        if (!mbar_wait(&empty[kt % S::kStages], ((kt / S::kStages) & 1) ^ 1u)) {
          give_up(kErrGemmWait);
          break;
        }
        if (stopped()) break;
        load_x(kt);
        ++issued;
      }
      for (int j = max(issued - S::kStages, 0); j < issued; ++j)  // no copy left in flight
        if (!mbar_wait(&full[j % S::kStages], (j / S::kStages) & 1)) give_up(kErrDrainWait);
    }
  } else if (warp == kPackedWarp) {
    // ------------------------------------------------------------ W
    if (lane == 0) {
      int issued = min(S::kPkStages, KT);  // thread 0 issued these
      for (int kt = issued; kt < KT; ++kt) {
        if (!mbar_wait(&empty_pk[kt % S::kPkStages], ((kt / S::kPkStages) & 1) ^ 1u)) {
          give_up(kErrGemmWait);
          break;
        }
        if (stopped()) break;
        load_w(kt);
        ++issued;
      }
      for (int j = max(issued - S::kPkStages, 0); j < issued; ++j)
        if (!mbar_wait(&full_pk[j % S::kPkStages], (j / S::kPkStages) & 1)) give_up(kErrDrainWait);
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA
    if (lane == 0) {
      constexpr uint32_t idesc = tc_idesc(kBF16 ? 1 : 0, 0, BN);
      const uint64_t xd0 = tc_operand(smem_u32(base + S::kOffX), 16, 1024);
      const uint64_t bd0 = tc_operand(smem_u32(base + S::kOffB), 16, 1024);
      for (int kt = 0; kt < KT; ++kt) {
        const int s = kt % S::kStages;
        if (!mbar_wait(&full[s], (kt / S::kStages) & 1)) {
          give_up(kErrGemmWait);
          break;
        }
        tc_fence_after();
        const uint64_t xd = tc_operand_at(xd0, s * S::kXBytes);
        const uint64_t bd = tc_operand_at(bd0, s * S::kBBytes);
#pragma unroll
        for (int kk = 0; kk < kBK / 16; ++kk)  // 16 k = 32 bytes along the swizzled row
          // accumulator a: rows 128a.. (16 KB further per 128 rows), columns a*BN..
#pragma unroll
          for (int a = 0; a < NACC; ++a)
            tc_mma(tmem_d + a * BN, tc_operand_at(xd, a * kUM * 128 + kk * 32),
                   tc_operand_at(bd, kk * 32), idesc, kk > 0 ? 1u : (uint32_t)(kt > 0));
        tc_commit(&empty[s]);
      }
      tc_commit(acc_full);  // after every issued MMA (also when none was issued)
    }
  } else {
    // ------------------------------------------------------------ dequant
    constexpr int kGroupThreads = S::kGroupWarps * 32;
    const int group = (warp - 1) / S::kGroupWarps;
    const int dt = threadIdx.x - 32 - group * kGroupThreads;
    // this thread's scales come straight from global memory, a stage ahead
    uint16_t next[S::kColsPerThread];
    auto load_scales = [&](int kt) {
#pragma unroll
      for (int c = 0; c < S::kColsPerThread; ++c) {
        const int n = n0 + dt + c * kGroupThreads;
        next[c] = kt < KT && n < p.N
                      ? p.scales[(size_t)((kt0 + kt) * kBK / 128) * p.N + n]
                      : (uint16_t)0;
      }
    };
    load_scales(group);
    // the epilogue's bias and residual on their way into the caches
    const int q = warp & 3;           // this warp's 32-lane slice of tensor memory
    const int half = (warp - 1) / 4;  // which accumulator (rows 0..127 or 128..255)
    const int tile_row = half * kUM + 32 * q + lane, row = m0 + tile_row;
    const bool has_row = half < NACC && row < p.M;
    if (p.bias && dt < BN / 64 && n0 + 64 * dt < p.N)
      prefetch_l1(static_cast<const uint16_t*>(p.bias) + n0 + 64 * dt);
    if (p.residual && has_row)
      for (int c = 0; c < BN && n0 + c < p.N; c += p.act == W4_ACT_SWIGLU ? 128 : 64)
        prefetch_l2(static_cast<const uint16_t*>(p.residual) + out_at(p, row, n0 + c));
    for (int kt = group; kt < KT; kt += S::kGroups) {
      const int s = kt % S::kPkStages, sb = kt % S::kStages;
      const bool there =
          mbar_wait(&full_pk[s], (kt / S::kPkStages) & 1) &&
          (kt < S::kStages || mbar_wait(&empty[sb], ((kt / S::kStages) & 1) ^ 1u));
      if (!__all_sync(0xffffffffu, there)) {  // a warp gives up as a whole
        give_up(kErrGemmWait);
        break;
      }
      const uint32_t* pk = reinterpret_cast<const uint32_t*>(base + S::kOffPk + s * S::kPkBytes);
      uint16_t now[S::kColsPerThread];
#pragma unroll
      for (int c = 0; c < S::kColsPerThread; ++c) now[c] = next[c];
      load_scales(kt + S::kGroups);
#pragma unroll
      for (int c = 0; c < S::kColsPerThread; ++c) {
        const int n = dt + c * kGroupThreads;  // column of the tile
        const uint16_t sbits = now[c];
        const uint32_t s2 = (uint32_t)sbits | ((uint32_t)sbits << 16);
        const float sf = __half2float(__ushort_as_half(sbits));
        uint8_t* brow = base + S::kOffB + sb * S::kBBytes + n * 128;  // row n: 64 k of column n
        uint32_t wv[kBK / 8];
#pragma unroll
        for (int j = 0; j < kBK / 8; ++j) wv[j] = pk[j * BN + n];
#pragma unroll
        for (int j = 0; j < kBK / 8; ++j)  // chunk j lands at chunk j ^ (row % 8)
          *reinterpret_cast<uint4*>(brow + ((j ^ (n & 7)) << 4)) =
              dequant_word<kBF16>(wv[j], s2, sf);
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&full[sb]);
        mbar_arrive(&empty_pk[s]);
      }
    }
    // ------------------------------------------------------------ epilogue
    const bool gated = p.act == W4_ACT_SWIGLU;
    const int step = gated ? 2 : 1;  // 32-column blocks a turn
    uint4 res[4] = {};               // the next turn's residual, a turn ahead of its use
    // Chunk k of a lane in memory: chunk t of row k of its quad where tiles have many
    // rows, of its own row otherwise. Turned and not, in the fused loop: 300 x 1536 x 1536 17.0 and 18.2 us,
    // 2048 x 8960 x 1536 65.6 and 68.6, 1709 x 128 x 7296 with a residual 35 and 41; but
    // one accumulator, 17 x 1536 x 2048 14.6 and 13.4, 64 x 4096 x 4096 28.9 and 27.0.
    constexpr bool kTurn = NACC == 2;
    const int t = lane & 3;
    auto row_of = [&](int k) { return kTurn ? row - t + k : row; };
    auto col_of = [&](int k) { return 8 * (kTurn ? t : k); };
    auto load_residual = [&](int c) {
      if (half < NACC && c < BN / 32 && p.residual && n0 + 32 * c < p.N) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (row_of(k) < p.M)
            res[k] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.residual) +
                                                     out_at(p, row_of(k), n0 + 32 * c) + col_of(k));
      }
    };
    auto store = [&](int c, uint4 (&y)[4]) {
      if (kTurn) transpose4(y, lane);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (row_of(k) < p.M)
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) +
                                    out_at(p, row_of(k), n0 + 32 * c) + col_of(k)) = y[k];
    };
    const bool plain = !p.bias && !p.residual && p.act == W4_ACT_NONE;
    if (p.ksplit == 1) load_residual(0);
    if (!mbar_wait(acc_full, 0)) give_up(kErrGemmWait);
    const bool stop = __any_sync(0xffffffffu, stopped());
    tc_fence_after();
    const uint32_t acc = tmem_d + ((uint32_t)(32 * q) << 16) + half * BN;
    if (p.ksplit > 1) {
      // K slice: this warp's 32 rows of its accumulator -> the fp32 partial tile
      if constexpr (S::kCanSplit) {
        if (!stop && half < NACC && m0 + tile_row - lane < p.M) {
          float* prow = reinterpret_cast<float*>(base) + (size_t)tile_row * S::kPitch;
#pragma unroll 1
          for (int c = 0; c < BN / 32; ++c) {
            uint32_t r[32];
            tc_ld32(acc + 32 * c, r);
            if (has_row) {
#pragma unroll
              for (int v = 0; v < 8; ++v)
                *reinterpret_cast<uint4*>(prow + 32 * c + 4 * v) =
                    make_uint4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
            }
          }
        }
      }
    } else if (stop || half >= NACC || m0 + tile_row - lane >= p.M) {
      // no rows
    } else if (plain) {
      // Its own loop: with the activations' code between a turn's steps w4_gemm took 2 us
      // more, all of it the code's fetch (20 x 128 x 128 6.2 us, 4.2 so; 200 x 1024 x 1536
      // 13.7 and 11.8).
#pragma unroll 1
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t r[32];
        tc_ld32(acc + 32 * c, r);
        if (n0 + 32 * c >= p.N) break;
        uint4 y[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          float a[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] = __uint_as_float(r[8 * v + e]);
          uint32_t w[4];
          pack_row(p.y_bf16, a, w);
          y[v] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        store(c, y);
      }
    } else {
#pragma unroll 1
      for (int c = 0; c < BN / 32; c += step) {
        uint32_t r[32], ru[32];
        tc_ld32(acc + 32 * c, r);
        if (gated) tc_ld32(acc + 32 * c + 32, ru);
        uint4 now[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) now[v] = res[v];
        load_residual(c + step);
        if (n0 + 32 * c < p.N) {
          if (kTurn && p.residual) transpose4(now, lane);
          uint4 y[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float a[8], u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              a[e] = __uint_as_float(r[8 * v + e]);
              u[e] = gated ? __uint_as_float(ru[8 * v + e]) : 0.f;
            }
            activate(p, n0 + 32 * c + 8 * v, a, u);
            if (p.residual) {
              float f[8];
              load_row(&now[v], 0, p.y_bf16, f);
#pragma unroll
              for (int e = 0; e < 8; ++e) a[e] += f[e];
            }
            uint32_t w[4];
            pack_row(p.y_bf16, a, w);
            y[v] = make_uint4(w[0], w[1], w[2], w[3]);
          }
          store(c, y);
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if constexpr (S::kCanSplit) {
    if (p.ksplit > 1) {
      // rank r writes rows [r*R/S, (r+1)*R/S) of the tile, each the sum of
      // every rank's partial in rank order
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();
      const int rank = (int)blockIdx.z;
      const int rows = min(S::kBM, p.M - m0);  // of the tile, cut into bands
      const int r0 = rank * rows / p.ksplit, r1 = (rank + 1) * rows / p.ksplit;
      const bool gated = p.act == W4_ACT_SWIGLU;
      const int c4s = gated ? BN / 8 : BN / 4;  // groups of four output columns
      const float* part = reinterpret_cast<const float*>(base);
      for (int i = threadIdx.x; i < (r1 - r0) * c4s; i += kGemmThreads) {
        const int row = r0 + i / c4s;
        int col = 4 * (i - (i / c4s) * c4s);
        if (gated) col = (col >> 5) * 64 + (col & 31);  // the gate column
        if (n0 + col >= p.N) continue;
        const int at = row * S::kPitch + col;
        float4 v[8], w[8];  // every rank's part, all on their way at once
#pragma unroll
        for (int rr = 0; rr < 8; ++rr) {
          v[rr] = w[rr] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (rr < p.ksplit) {
            v[rr] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(part + at, rr));
            if (gated)
              w[rr] = *reinterpret_cast<const float4*>(
                  cluster.map_shared_rank(part + at + W4B200_SWIGLU_BLOCK, rr));
          }
        }
        float a[4] = {0.f, 0.f, 0.f, 0.f}, u[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int rr = 0; rr < 8; ++rr) {
          a[0] += v[rr].x, a[1] += v[rr].y, a[2] += v[rr].z, a[3] += v[rr].w;
          u[0] += w[rr].x, u[1] += w[rr].y, u[2] += w[rr].z, u[3] += w[rr].w;
        }
        activate(p, n0 + col, a, u);
        const size_t to = out_at(p, m0 + row, n0 + col);
        if (p.residual) {
          float f[4];
          load_row(p.residual, to, p.y_bf16, f);
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] += f[e];
        }
        uint32_t packed[2];
        pack_row(p.y_bf16, a, packed);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + to) = make_uint2(packed[0], packed[1]);
      }
      cluster.sync();  // the other ranks' reads of this CTA's partial are done
    }
  }
  if (warp == kMmaWarp) {
    // every MMA has completed (acc_full) before its tensor memory is freed
    if (lane == 0 && !mbar_wait(acc_full, 0)) give_up(kErrGemmWait);
    __syncwarp();
    tc_fence_after();
    tc_dealloc(tmem_d, S::kTmemCols);
  }
  if (p.wait_at_end) grid_dependency_wait();
}

bool encode_2d(CUtensorMap* map, CUtensorMapDataType dt, int elem, const void* gaddr,
               uint64_t inner, uint64_t outer, uint32_t box_inner, uint32_t box_outer,
               CUtensorMapSwizzle swz) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return false;
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {inner * (uint64_t)elem};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t estr[2] = {1, 1};
  return enc(map, dt, 2, const_cast<void*>(gaddr), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

template <bool B, int BN, int NACC>
void* gemm_fn() {
  return reinterpret_cast<void*>(&w4_gemm_kernel<B, BN, NACC>);
}

// Clusters of s CTAs of the 128-column instances that the device holds at once
// (a cluster needs its SMs within one GPC), by device, accumulators and s.
static int g_clusters[64][3][9];

static int count_clusters() {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  for (int nacc = 1; nacc <= 2 && e == cudaSuccess; ++nacc)
    for (int s = 2; s <= 8 && e == cudaSuccess; ++s) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1, 1, (unsigned)s);
      cfg.blockDim = dim3(kGemmThreads);
      cfg.dynamicSmemBytes = nacc == 1 ? GemmShape<128, 1>::kSmem : GemmShape<128, 2>::kSmem;
      cudaLaunchAttribute at;
      at.id = cudaLaunchAttributeClusterDimension;
      at.val.clusterDim.x = at.val.clusterDim.y = 1;
      at.val.clusterDim.z = (unsigned)s;
      cfg.attrs = &at;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(
          &g_clusters[dev & 63][nacc][s],
          nacc == 1 ? gemm_fn<true, 128, 1>() : gemm_fn<true, 128, 2>(), &cfg);
    }
  return e == cudaSuccess ? W4_OK : cuda_fail(e, "cudaOccupancyMaxActiveClusters(w4_gemm)");
}

int gemm_init_device(const DeviceInfo& di) {
  struct K {
    void* fn;
    int smem;
  } ks[8] = {{gemm_fn<false, 128, 1>(), GemmShape<128, 1>::kSmem},
             {gemm_fn<true, 128, 1>(), GemmShape<128, 1>::kSmem},
             {gemm_fn<false, 256, 1>(), GemmShape<256, 1>::kSmem},
             {gemm_fn<true, 256, 1>(), GemmShape<256, 1>::kSmem},
             {gemm_fn<false, 128, 2>(), GemmShape<128, 2>::kSmem},
             {gemm_fn<true, 128, 2>(), GemmShape<128, 2>::kSmem},
             {gemm_fn<false, 256, 2>(), GemmShape<256, 2>::kSmem},
             {gemm_fn<true, 256, 2>(), GemmShape<256, 2>::kSmem}};
  for (const K& k : ks) {
    if ((size_t)k.smem > (size_t)di.max_smem_optin)
      return fail(W4_ERR_UNSUPPORTED, "w4_gemm needs %d B of shared memory", k.smem);
    cudaError_t e = cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(w4_gemm smem)");
    e = cudaFuncSetAttribute(k.fn, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(w4_gemm carveout)");
  }
  return count_clusters();
}

// Tile width: 256 columns halve the re-reads of X per FLOP; 128 when a
// 256-wide grid would not cover the SMs.
// Two accumulators (256 rows) share every dequantised W tile, which halves
// the dequantisation per FLOP; one only when M fits 128 rows.
static int gemm_tile(int M, int N, int sms, int* nacc) {
  const long long m2 = (M + kBMMax - 1) / kBMMax;
  *nacc = M <= kUM ? 1 : 2;
  if (*nacc == 2 && (N % 256 == 0 || N > 1024) && (long long)((N + 255) / 256) * m2 >= sms)
    return 256;
  return 128;
}

namespace {

// One launch of a prepared plan: the instance, its tile region and K slices.
struct GemmLaunch {
  int bn, nacc;
  int m_tile0, n_tile0, ntx, tiles;
  int ksplit;
  bool after_previous;  // programmatic dependent launch, waits for it at exit
};

void* gemm_instance(int bf16, int bn, int nacc, size_t* smem) {
  if (bn == 256 && nacc == 2) {
    *smem = GemmShape<256, 2>::kSmem;
    return bf16 ? gemm_fn<true, 256, 2>() : gemm_fn<false, 256, 2>();
  }
  if (bn == 256) {
    *smem = GemmShape<256, 1>::kSmem;
    return bf16 ? gemm_fn<true, 256, 1>() : gemm_fn<false, 256, 1>();
  }
  if (nacc == 2) {
    *smem = GemmShape<128, 2>::kSmem;
    return bf16 ? gemm_fn<true, 128, 2>() : gemm_fn<false, 128, 2>();
  }
  *smem = GemmShape<128, 1>::kSmem;
  return bf16 ? gemm_fn<true, 128, 1>() : gemm_fn<false, 128, 1>();
}

// The launches of one GEMM (at most two). split_k > 0 forces one launch of
// 128 x 256 tiles (one accumulator) cut into that many K slices. few_tiles lets
// grids that leave SMs idle be cut along K, which w4_gemm's own calls are not
// (their sums keep their order).
int gemm_plan(int M, int K, int N, int sms, int split_k, bool few_tiles, int dev,
              GemmLaunch* out) {
  const int kt = K / kBK;
  const int nt128 = (N + 127) / 128;
  // the K-sliced tile: 128 rows x 256 columns (its partial tile fits the
  // freed rings; two accumulators of 256 columns would not)
  const int nt256 = (N + 255) / 256, mt1 = (M + kUM - 1) / kUM;
  if (split_k > 0) {
    out[0] = GemmLaunch{256, 1, 0, 0, nt256, nt256 * mt1, std::min(split_k, kt), false};
    return 1;
  }
  int nacc = 2;
  const int bn = gemm_tile(M, N, sms, &nacc);
  const int bm = nacc * kUM;
  const int ntx = (N + bn - 1) / bn, mtx = (M + bm - 1) / bm;
  const int tiles = ntx * mtx;
  if (few_tiles && tiles * 2 <= sms) {
    // Half the SMs or more would have no tile: as many K slices as are resident
    // at once, of three stages at least. Whole tiles and slices: 17 x 1536 x 2048
    // 13.7 and 6.5 us, 64 x 4096 x 4096 27 and 12, 511 x 8960 x 1536 66 and 22,
    // 128 x 1536 x 8960 (70 tiles, 2 slices) 14.5 and 11.7.
    for (int s = std::min(8, kt / 3); s >= 2; --s)
      if (tiles <= g_clusters[dev & 63][nacc][s]) {
        out[0] = GemmLaunch{128, nacc, 0, 0, nt128, tiles, s, false};
        return 1;
      }
  }
  // A grid of more tiles than that is not cut along K: slices would share SMs.
  // Measured on 2048 x 8960 x 1536 (96 tiles) when the whole tiles took 96 us
  // (64 by now): three slices over 288 CTAs 118-128 us, each slice's stages at
  // half the rate.
  if (tiles >= sms && bn == 256 && nacc == 2) {
    // a last wave of a few tiles: those tiles go to a second launch as
    // 128-column tiles cut into K slices, spread over the SMs the first
    // launch frees
    const int rem = tiles % sms;
    if (rem > 0 && rem * 4 <= sms && rem <= ntx) {
      const int n_lo = (ntx - rem) * 2;  // first 128-column tile of the remainder
      const int nrx = nt128 - n_lo;
      const int s = std::max(1, std::min(8, std::min(sms / nrx, kt / 4)));
      out[0] = GemmLaunch{256, 2, 0, 0, ntx, tiles - rem, 1, false};
      out[1] = GemmLaunch{128, 2, mtx - 1, n_lo, nrx, nrx, s, true};
      return 2;
    }
  }
  out[0] = GemmLaunch{bn, nacc, 0, 0, ntx, tiles, 1, false};
  return 1;
}

}  // namespace

int launch_gemm(const void* x, int x_bf16, const int32_t* packed, const void* scales, void* y,
                int y_bf16, int M, int K, int N, const w4_gemm_ops& ops, int split_k,
                bool few_tiles, cudaStream_t stream) {
  int dev = 0;
  int st = current_device(&dev);
  if (st != W4_OK) return st;
  const DeviceInfo& di = device_info(dev);
  GemmLaunch plan[2];
  const int n = gemm_plan(M, K, N, di.sm_count > 0 ? di.sm_count : 148, split_k, few_tiles, dev,
                          plan);
  for (int i = 0; i < n; ++i) {
    const GemmLaunch& L = plan[i];
    const int BM = L.nacc * kUM;
    // Rows behind the last are not copied: what lies there reaches sums of its own rows
    // alone. (Zero-filled rows of a tensor below 128 KB cost more than real ones: 1 x
    // 4096 x 14336 39 us with whole boxes, 28 so; 1 x 1536 x 8960 10.7 and 9.0.)
    const int box_rows = std::min(BM, (M + 7) / 8 * 8);
    CUtensorMap tm_x, tm_w;
    if (!encode_2d(&tm_x,
                   x_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                   x, (uint64_t)K, (uint64_t)M, kBK, (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_2d(&tm_w, CU_TENSOR_MAP_DATA_TYPE_INT32, 4, packed, (uint64_t)N,
                   (uint64_t)(K / 8), (uint32_t)L.bn, kBK / 8, CU_TENSOR_MAP_SWIZZLE_NONE))
      return fail(W4_ERR_CUDA, "cuTensorMapEncodeTiled failed for w4_gemm M=%d K=%d N=%d", M, K,
                  N);
    GemmParams p;
    p.y = y;
    p.M = M;
    p.K = K;
    p.N = N;
    p.x_bf16 = x_bf16;
    p.y_bf16 = y_bf16;
    p.scales = static_cast<const uint16_t*>(scales);
    p.act = ops.act;
    p.bias = ops.bias;
    p.residual = ops.residual;
    p.err = di.err_word;
    p.m_tile0 = L.m_tile0;
    p.n_tile0 = L.n_tile0;
    p.ntx = L.ntx;
    p.ksplit = L.ksplit;
    p.x_bytes = (uint32_t)box_rows * kBK * 2;
    p.wait_at_end = L.after_previous ? 1 : 0;
    size_t smem = 0;
    void* fn = gemm_instance(x_bf16, L.bn, L.nacc, &smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)L.tiles, 1, (unsigned)L.ksplit);
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2];
    unsigned na = 0;
    if (L.ksplit > 1) {
      attrs[na].id = cudaLaunchAttributeClusterDimension;
      attrs[na].val.clusterDim.x = 1;
      attrs[na].val.clusterDim.y = 1;
      attrs[na].val.clusterDim.z = (unsigned)L.ksplit;
      ++na;
    }
    if (L.after_previous || few_tiles) {  // the first one waits before it reads anything
      attrs[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attrs[na].val.programmaticStreamSerializationAllowed = 1;
      ++na;
    }
    cfg.attrs = attrs;
    cfg.numAttrs = na;
    void* args[] = {&tm_x, &tm_w, &p};
    cudaError_t e = cudaLaunchKernelExC(&cfg, fn, args);
    if (e != cudaSuccess) return cuda_fail(e, "w4_gemm launch");
  }
  return W4_OK;
}

}  // namespace w4
