// Few tokens times 4-bit weights: C[token][row] = alpha * sum_g s[row, g] sum_{i in g} (q[row][i] - z[row, g]) x[token][i] + beta C.
//
// Bound by the bytes of the weights and, as these come from memory at two thirds of its rate, by the instructions that make operands of them.  Codes go
// from global memory through a ring of bulk copies for each warp into the registers of mma.m16n8k16, in whose order they are stored (tcec_codes.cuh).
// (tcgen05 takes operands from shared memory or TMEM: expanded codes would be written there and read again, and its tiles have no use for eight columns.)
// A few logic instructions make operands of a word of eight codes: a 4-bit code in the low bits of a 16-bit number that is otherwise zero is that code
// (or 16 times it, in the next four bits) times a power of two, subnormal or not; nothing is added or taken off.  The upper ones have an accumulator of
// their own.  What the zero points take off is z times the sum of x over the group, and the power of two goes into the last factor.  (Codes made to
// numbers first, by a magic number and a subtraction: an FP32 token times 16384 x 16384 in groups of 64 49 us instead of 45 at the time.)  How bf16
// operands are kept from products below FP32: tcec_stage.cuh.  Values of 2^122 and more count as infinite, and an infinite value makes NaN of its token's results
// (q inf - z inf).
//
// Columns are tokens; an FP32 token takes three, its bf16 parts of 8 bits each, which together are exactly it.  Every product of a code and a part is
// exact; a group's sum is made in the MMA's FP32 accumulator, then multiplied by its scale and added in FP32, rounded to nearest.  As code and zero
// point are multiplied apart, what is rounded off is relative to scale * (code + zero) * |x|.
//
// A CTA takes up to kStrips strips of 16 rows; its warps divide k block by block and add up through shared memory in a fixed order.  One strip after the other, the
// operands of the columns stay in registers: 16384 x 16384 with 16 tokens 45.6 us, strips side by side 53.8, with one FP32 token (groups of 64) 35 and 42.
//
// Measured, from memory, of calls in a row: one bf16 token times 4096 x 4096 5.3 us (the kernel 4.6, 2.0 TB/s: 32 rows of blocks an SM are over before the copies are up to speed), times
// 16384 x 16384 29.3 (4.9 TB/s), FP32 in groups of 64 33.8 (4.5 TB/s); 8 tokens 28 us, 16 46, 10 of FP32 94.
#pragma once
#include "tcec_gemm_codes.cuh"

namespace tcec_sm100 {

template <bool kF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (kF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Loads that are issued where they stand, ahead of the waits that follow.
__device__ __forceinline__ uint4 ld_ahead128(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// kEights: columns in eights.  kOne: one token, taken from x as it is; else x comes staged (tcec_stage.cuh).
template <int kType, int kGroup, int kEights, int kStrips, bool kOne>
struct GemvQ4Cfg {
  static constexpr int PARTS = kType == kTypeF32 ? 3 : 1;
  static constexpr int ROWS = 16 * kStrips;
  static constexpr int MOST_WARPS = kStrips == 4 || kEights == 4 ? 8 : 16;
  static constexpr int STAGE_BYTES = kStrips * q4_strip_bytes(kGroup);
  // Whether CTAs may have a strip less (one_gemv).  Where nothing comes of it the test costs 3 % (two strips of one token, 4096 x 4096), and in groups of 32 with
  // 9 to 16 columns 8 % (8192 x 8192).
  static constexpr bool SHARED_OUT = kOne ? kStrips == 4 : kEights == 1 || (kEights == 2 && kGroup > 32);
  static constexpr int STAGES = 2;                            // blocks of codes under way, of each warp
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int X_PITCH = 320;                         // of a column in shared memory: two columns' lanes read from all banks
  static constexpr int X_BYTES = kOne ? 8 * X_PITCH : 0;
  static constexpr int SUM_PITCH = kEights * 8 + 1;
  static constexpr int SUM_BYTES = ROWS * SUM_PITCH * 4;      // of a warp
  static constexpr int WARP_BYTES = RING_BYTES + X_BYTES > SUM_BYTES ? RING_BYTES + X_BYTES : SUM_BYTES;
  static constexpr int smem_bytes(int warps) { return warps * WARP_BYTES + 128; }
  // Warps that an SM's registers hold: 64 registers a thread for one token, else what the operands of the columns need.  All of an SM in one CTA where CTAs
  // are no more than SMs (five tokens times 4096 x 16384 11.2 us, with at most eight warps a CTA 17.1).
  static constexpr int WARPS_OF_SM = kOne && kStrips < 4 ? 32 : kEights == 4 ? 8 : 16;
};

template <bool kF16>
__device__ __forceinline__ void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool zero) {
  if (zero) d[0] = d[1] = d[2] = d[3] = 0.f;
  mma16816<kF16>(d, a0, a1, a2, a3, b0, b1);
}

// One strip: operands b of the four panels, `sums` of x over the groups and `unit` for this lane's two columns of each eight.
template <int kType, int kGroup, int kEights>
__device__ __forceinline__ void multiply_strip(float (&acc)[kEights][4], const uint8_t* strip, int lane, const uint4 (&b)[4][kEights],
                                               const float2 (&sums)[kCodeSpan / kGroup][kEights], const float2 (&unit)[kEights]) {
  constexpr bool kF16 = kType == kTypeF16;
  constexpr int kSpans = kCodeSpan / kGroup;
  // In f16 the codes lie three bits higher, which with bit 10, the exponent's last, are as high as numbers grow evenly: the tensor core aligns
  // products by their operands' exponents, and what lies low among the smallest keeps fewer bits.
  constexpr int kUp = kF16 ? 3 : 0;
  constexpr uint32_t kLow = 0x000f000fu << kUp, kHigh = 0x00f000f0u << kUp;
  const uint4 w[2] = {*reinterpret_cast<const uint4*>(strip + lane * 16), *reinterpret_cast<const uint4*>(strip + 512 + lane * 16)};
  const uint32_t* e = reinterpret_cast<const uint32_t*>(strip + kStripCodeBytes) + (lane >> 2);
#pragma unroll
  for (int q = 0; q < kSpans; ++q) {
    float d[kEights][2][4];  // of codes, and of 16 times codes
#pragma unroll
    for (int panel = q * 4 / kSpans; panel < (q + 1) * 4 / kSpans; ++panel) {
      const bool first = panel == q * 4 / kSpans;
      const uint4 pair = w[panel >> 1];
      const uint32_t word0 = panel & 1 ? pair.z : pair.x, word1 = panel & 1 ? pair.w : pair.y;  // of rows g and g + 8
      const uint32_t w0 = word0 << kUp, w1 = word1 << kUp, v0 = word0 >> (8 - kUp), v1 = word1 >> (8 - kUp);
#pragma unroll
      for (int c = 0; c < kEights; ++c) {
        mma16816_zero<kF16>(d[c][0], w0 & kLow, w1 & kLow, v0 & kLow, v1 & kLow, b[panel][c].x, b[panel][c].z, first);
        mma16816_zero<kF16>(d[c][1], w0 & kHigh, w1 & kHigh, v0 & kHigh, v1 & kHigh, b[panel][c].y, b[panel][c].w, first);
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t entry = e[q * 16 + r * 8];
      const float scale = __uint_as_float(entry & ~15u), z = 8388608.0f - __uint_as_float(0x4b000000u | (entry & 15u));  // minus the zero point
#pragma unroll
      for (int c = 0; c < kEights; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float u = j ? unit[c].y : unit[c].x, x = j ? sums[q][c].y : sums[q][c].x;
          const float sum = __fmaf_rn(0.0625f * u, d[c][1][r * 2 + j], u * d[c][0][r * 2 + j]);
          acc[c][r * 2 + j] = __fmaf_rn(scale, __fmaf_rn(z, x, sum), acc[c][r * 2 + j]);
        }
    }
  }
}

template <int kType, int kGroup, int kEights, int kStrips, bool kOne>
__global__ void __launch_bounds__(32 * GemvQ4Cfg<kType, kGroup, kEights, kStrips, kOne>::MOST_WARPS, kOne || kStrips == 4 ? 2 : 1) gemv_q4_kernel(const GemvQ4Params p) {
  using Cfg = GemvQ4Cfg<kType, kGroup, kEights, kStrips, kOne>;
  static_assert(!kOne || kEights == 1, "one token has at most three columns");
  constexpr int kSpans = kCodeSpan / kGroup;
  constexpr bool kF16 = kType == kTypeF16;
  constexpr uint32_t kOnes = kF16 ? 0x04000400u : 0x00800080u;  // 2^7 times a code's 1, the smallest normal number: no bits are lost
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[Cfg::MOST_WARPS][Cfg::STAGES];
  __shared__ uint32_t abort_flag;
  uint8_t* const smem = smem_raw + ((0u - smem_u32(smem_raw)) & 127u);
  const int warp = warp_index(), lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  uint8_t* const ring = smem + warp * Cfg::RING_BYTES;
  [[maybe_unused]] uint8_t* const x_shared = smem + warps * Cfg::RING_BYTES + warp * Cfg::X_BYTES;
  if (lane == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) mbar_init(smem_u32(&bars[warp][s]), 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) abort_flag = 0;
  if constexpr (kOne)  // columns that no part of the token has
    for (int i = lane; i < Cfg::X_BYTES / 16; i += 32) reinterpret_cast<uint4*>(x_shared)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const int cta = blockIdx.x, strip0 = Cfg::SHARED_OUT ? cta * p.strips + min(cta, p.more) : cta * kStrips, row0 = strip0 * 16;
  const int strips = Cfg::SHARED_OUT ? min(p.strips + (cta < p.more), (p.n - row0 - 1) / 16 + 1) : kStrips;
  constexpr size_t kBlockBytes = q4_block_bytes(kGroup);
  // strips of one tile of rows, or the last ones of one and the first ones of the next
  const uint32_t bytes = Cfg::SHARED_OUT ? min(strips, 8 - strip0 % 8) * q4_strip_bytes(kGroup) : Cfg::STAGE_BYTES;
  const uint32_t bytes_next = strips * q4_strip_bytes(kGroup) - bytes;
  const uint8_t* codes_next = p.codes + static_cast<size_t>(strip0 / 8 + 1) * p.blocks * kBlockBytes;
  const uint8_t* codes = p.codes + static_cast<size_t>(strip0 / 8) * p.blocks * kBlockBytes + strip0 % 8 * q4_strip_bytes(kGroup);
  auto fetch = [&](int kb, int stage) {  // lane 0
    if (dev_flag(p.debug_flags, 128) && blockIdx.x == 0 && kb == 0) return;
    const uint32_t bar = smem_u32(&bars[warp][stage]);
    const uint32_t to = smem_u32(ring + stage * Cfg::STAGE_BYTES);
    mbar_arrive_expect_tx(bar, bytes + bytes_next);
    bulk_load(to, codes + kb * kBlockBytes, bytes, bar);
    if (Cfg::SHARED_OUT && bytes_next) bulk_load(to + bytes, codes_next + kb * kBlockBytes, bytes_next, bar);
  };
  // Staged x is written by the kernel before this one, which was through its own wait when this one could start: whatever the codes
  // come from has ended, and they are fetched without waiting for x.
  if constexpr (kOne) wait_for_launch_before();
  if (lane == 0)
    for (int i = 0; i < Cfg::STAGES; ++i)
      if (warp + i * warps < p.blocks) fetch(warp + i * warps, i);
  if constexpr (!kOne) wait_for_launch_before();
  let_next_launch_start();

  float acc[kStrips][kEights][4];
#pragma unroll
  for (int s = 0; s < kStrips; ++s)
#pragma unroll
    for (int c = 0; c < kEights; ++c) acc[s][c][0] = acc[s][c][1] = acc[s][c][2] = acc[s][c][3] = 0.f;

  // x of the next block, on its way while this one is worked on: the token's four values of this lane, or whole operands
  [[maybe_unused]] Four<kType> four;
  [[maybe_unused]] uint4 b_ahead[4][kEights];
  [[maybe_unused]] const void* const token_x = kOne ? after_wait(p.x) : nullptr;
  auto load_four = [&](int kb) {
    const int k0 = kb * kCodeSpan + lane * 4, left = p.k - k0;
    if (p.vec && left >= 4) {
      four.load(token_x, k0);
    } else {
      uint32_t v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long at = min(k0 + j, p.k - 1) * p.x_k;
        if constexpr (kType == kTypeF32) v[j] = ld_operand32(static_cast<const uint32_t*>(token_x) + at);
        else v[j] = ld_operand16(static_cast<const uint16_t*>(token_x) + at);
        if (j >= left) v[j] = 0;
      }
      if constexpr (kType == kTypeF32) four.raw = make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
      else four.raw = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
    }
  };
  const uint8_t* const staged = kOne ? nullptr : after_wait(p.staged) + lane * 16;
  auto load_operands = [&](int kb, int panel) {
#pragma unroll
    for (int c = 0; c < kEights; ++c) b_ahead[panel][c] = ld_ahead128(staged + static_cast<size_t>(kb) * (kEights * 2048) + panel * (kEights * 512) + c * 512);
  };
  // behind the operands of all blocks: what makes products values, and the sums of x over the groups
  [[maybe_unused]] float2 sums_ahead[kSpans][kEights], units_ahead[kEights];
  [[maybe_unused]] const uint8_t* const staged_sums =
      kOne ? nullptr : after_wait(p.staged) + static_cast<size_t>(p.blocks) * (kEights * 2048) + (lane & 3) * 8;
  auto load_sums = [&](int kb) {
    const uint8_t* at = staged_sums + static_cast<size_t>(kb) * staged_sum_bytes(kEights);
#pragma unroll
    for (int c = 0; c < kEights; ++c) {
      const uint2 u = ld_operand64(at + c * 32);
      units_ahead[c] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
#pragma unroll
      for (int q = 0; q < kSpans; ++q) {
        const uint2 v = ld_operand64(at + (q + 1) * kEights * 32 + c * 32);
        sums_ahead[q][c] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
      }
    }
  };
  if (warp < p.blocks) {
    if constexpr (kOne) {
      load_four(warp);
    } else if constexpr (kEights == 1) {
      load_sums(warp);
#pragma unroll
      for (int panel = 0; panel < 4; ++panel) load_operands(warp, panel);
    }
  }
  int stage = 0;
  uint32_t parity = 0;
  bool ok = true;
  int kb = warp;
  for (; kb < p.blocks; kb += warps) {
    const int next = kb + warps;
    [[maybe_unused]] float unit = kUnitF16;
    if constexpr (kOne) {
      uint8_t* to = x_shared + lane * 8;
      float v[4];
      if constexpr (kType != kTypeF16) {
        four.get(v);
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
        const UpX by = up_x(__reduce_max_sync(0xffffffffu, most));
        unit = by.unit;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] *= by.up;
      }
      if constexpr (kType == kTypeF32) {
        uint2 hi, mid, lo;
        split3_bf16(v[0], v[1], hi.x, mid.x, lo.x);
        split3_bf16(v[2], v[3], hi.y, mid.y, lo.y);
        *reinterpret_cast<uint2*>(to) = hi;
        *reinterpret_cast<uint2*>(to + Cfg::X_PITCH) = mid;
        *reinterpret_cast<uint2*>(to + 2 * Cfg::X_PITCH) = lo;
      } else if constexpr (kType == kTypeBf16) {
        *reinterpret_cast<uint2*>(to) = make_uint2(__byte_perm(__float_as_uint(v[0]), __float_as_uint(v[1]), 0x7632),
                                                   __byte_perm(__float_as_uint(v[2]), __float_as_uint(v[3]), 0x7632));
      } else {
        *reinterpret_cast<uint2*>(to) = four.raw;
      }
      if (next < p.blocks) load_four(next);
      __syncwarp();  // what all lanes have written, for all to read
    }
    if constexpr (kEights > 1) {  // more warps instead of operands ahead (16 tokens times 16384 x 16384: 46 us, 54 so)
      load_sums(kb);
#pragma unroll
      for (int panel = 0; panel < 4; ++panel) load_operands(kb, panel);
    }
    ok = mbar_wait_lanes(smem_u32(&bars[warp][stage]), parity, &abort_flag);
    if (!ok) break;
    const uint8_t* const here = ring + stage * Cfg::STAGE_BYTES;
    if constexpr (kOne) {
      // sums of x: the same products with a constant for codes
      uint4 b[4][1];
      float ones[kSpans][4];
      float2 sums[kSpans][1];
#pragma unroll
      for (int panel = 0; panel < 4; ++panel) {
        b[panel][0] = *reinterpret_cast<const uint4*>(x_shared + (lane >> 2) * Cfg::X_PITCH + panel * 64 + (lane & 3) * 16);
        const int q = panel * kSpans / 4;
        mma16816_zero<kF16>(ones[q], kOnes, kOnes, kOnes, kOnes, b[panel][0].x, b[panel][0].z, panel == q * 4 / kSpans);
        mma16816<kF16>(ones[q], kOnes, kOnes, kOnes, kOnes, b[panel][0].y, b[panel][0].w);
      }
#pragma unroll
      for (int q = 0; q < kSpans; ++q) sums[q][0] = make_float2(ones[q][0] * (unit * 0x1p-7f), ones[q][1] * (unit * 0x1p-7f));
      const float2 units[1] = {make_float2(unit, unit)};
#pragma unroll
      for (int s = 0; s < kStrips; ++s)
        if (!Cfg::SHARED_OUT || s < kStrips - 1 || strips == kStrips) multiply_strip<kType, kGroup, 1>(acc[s], here + s * q4_strip_bytes(kGroup), lane, b, sums, units);
    } else if constexpr (kEights > 1) {
#pragma unroll
      for (int c = 0; c < kEights; ++c)
        if constexpr (kF16) units_ahead[c] = make_float2(kUnitF16, kUnitF16);
#pragma unroll
      for (int s = 0; s < kStrips; ++s)
        if (!Cfg::SHARED_OUT || s < kStrips - 1 || strips == kStrips)
          multiply_strip<kType, kGroup, kEights>(acc[s], here + s * q4_strip_bytes(kGroup), lane, b_ahead, sums_ahead, units_ahead);
    } else {
      uint4 b[4][kEights];
      float2 sums[kSpans][kEights], units[kEights];
#pragma unroll
      for (int c = 0; c < kEights; ++c) {
        units[c] = kF16 ? make_float2(kUnitF16, kUnitF16) : units_ahead[c];
#pragma unroll
        for (int panel = 0; panel < 4; ++panel) b[panel][c] = b_ahead[panel][c];
#pragma unroll
        for (int q = 0; q < kSpans; ++q) sums[q][c] = sums_ahead[q][c];
      }
      if (next < p.blocks) {
        load_sums(next);
#pragma unroll
        for (int panel = 0; panel < 4; ++panel) load_operands(next, panel);
      }
#pragma unroll
      for (int s = 0; s < kStrips; ++s)
        if (!Cfg::SHARED_OUT || s < kStrips - 1 || strips == kStrips) multiply_strip<kType, kGroup, kEights>(acc[s], here + s * q4_strip_bytes(kGroup), lane, b, sums, units);
    }
    __syncwarp();  // all have read the stage
    if (lane == 0 && kb + Cfg::STAGES * warps < p.blocks) fetch(kb + Cfg::STAGES * warps, stage);
    if (++stage == Cfg::STAGES) stage = 0, parity ^= 1;
  }
  if (!ok) {
    abort_flag = 1;
    if (lane == 0) {
      atomicCAS(p.status, 0, kErrOperandWait);
      // this warp's own copies land before the CTA gives up its shared memory
      for (int i = 0; i < Cfg::STAGES && kb < p.blocks; ++i, kb += warps) {
        mbar_wait_plain(smem_u32(&bars[warp][stage]), parity);
        if (++stage == Cfg::STAGES) stage = 0, parity ^= 1;
      }
    }
  }

  __syncthreads();  // all codes have been read: sums take their place
  if (abort_flag) return;
  float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int s = 0; s < kStrips; ++s)
#pragma unroll
    for (int c = 0; c < kEights; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sums[(warp * Cfg::ROWS + s * 16 + (lane >> 2) + (j >> 1) * 8) * Cfg::SUM_PITCH + c * 8 + (lane & 3) * 2 + (j & 1)] = acc[s][c][j];
  __syncthreads();
  void* const c = after_wait(p.c);
  for (int i = threadIdx.x; i < Cfg::ROWS * p.tokens; i += blockDim.x) {
    const int r = i % Cfg::ROWS, token = i / Cfg::ROWS, row = row0 + r;
    if (row >= p.n || r >= strips * 16) continue;
    float v = 0.f;
#pragma unroll
    for (int part = Cfg::PARTS - 1; part >= 0; --part)  // the small ones first
#pragma unroll 4
      for (int w = 0; w < warps; ++w) v += sums[(w * Cfg::ROWS + r) * Cfg::SUM_PITCH + token * Cfg::PARTS + part];
    const long long at = token * p.c_token + row * p.c_row;
    v = __fmul_rn(p.alpha, v);
    if (p.beta != 0.f) v = __fmaf_rn(p.beta, ld_element_as(p.c_type, c, at), v);
    st_element_as(p.c_type, c, at, v);
  }
}

}  // namespace tcec_sm100
