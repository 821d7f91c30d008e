// Few tokens times 4-bit weights: C[token][row] = alpha * sum_g s[row, g] sum_{i in g} (q[row][i] - z[row, g]) x[token][i] + beta C.
//
// Bound by the bytes of the weights, which go from global memory into the registers of mma.m16n8k16 and nowhere else: a block
// of codes is stored in the order of those registers (tcec_codes.cuh), so a lane's two 128-bit loads are the operands of eight MMAs once
// the codes are expanded (logic and one exact subtraction for two codes).  The tensor cores of mma.sync are plenty for up to 16 columns, and
// unlike tcgen05.mma they take their operands from registers.
//
// Columns are tokens; an FP32 token takes three, its bf16 parts of 8 bits each, which together are exactly it.  Every product
// of a code and a part is exact; a group's sum is made in the MMA's FP32 accumulator, then multiplied by its scale and added in
// FP32, rounded to nearest.
//
// A CTA takes 16 kStrips rows; its warps divide k block by block and add up through shared memory in a fixed order.
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
  static constexpr int WARPS = 8;
  static constexpr int STAGE_BYTES = kStrips * q4_strip_bytes(kGroup);
  static constexpr int STAGES = 4;                            // blocks of codes under way, of each warp
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int X_PITCH = 320;                         // of a column in shared memory: two columns' lanes read from all banks
  static constexpr int X_BYTES = kOne ? 8 * X_PITCH : 0;
  static constexpr int SUM_PITCH = kEights * 8 + 1;
  static constexpr int SUM_BYTES = WARPS * ROWS * SUM_PITCH * 4;
  static constexpr int USED = WARPS * (RING_BYTES + X_BYTES);
  static constexpr int SMEM_BYTES = (USED > SUM_BYTES ? USED : SUM_BYTES) + 128;
};

// The codes of a block, a strip at a time, times the operands b(panel, eight); sums folded into acc.
template <int kType, int kGroup, int kEights, int kStrips, class B>
__device__ __forceinline__ void multiply_block(float (&acc)[kStrips][kEights][4], const uint8_t* stage, int lane, const B& operands) {
  constexpr bool kF16 = kType == kTypeF16;
  constexpr int kSpans = kCodeSpan / kGroup;
  uint4 w[kStrips][2];  // rows g and g + 8, of two panels each
#pragma unroll
  for (int s = 0; s < kStrips; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h) w[s][h] = *reinterpret_cast<const uint4*>(stage + s * q4_strip_bytes(kGroup) + h * 512 + lane * 16);
#pragma unroll
  for (int q = 0; q < kSpans; ++q) {
    float d[kStrips][kEights][4];
    uint32_t entry[kStrips][2];
#pragma unroll
    for (int s = 0; s < kStrips; ++s) {
      const uint32_t* e = reinterpret_cast<const uint32_t*>(stage + s * q4_strip_bytes(kGroup) + kStripCodeBytes) + q * 16 + (lane >> 2);
      entry[s][0] = e[0];
      entry[s][1] = e[8];
#pragma unroll
      for (int c = 0; c < kEights; ++c) d[s][c][0] = d[s][c][1] = d[s][c][2] = d[s][c][3] = 0.f;
    }
#pragma unroll
    for (int panel = q * 4 / kSpans; panel < (q + 1) * 4 / kSpans; ++panel) {
      uint4 b[kEights];
      operands(panel, b);
#pragma unroll
      for (int s = 0; s < kStrips; ++s) {
        const uint4 pair = w[s][panel >> 1];
        const uint4 r0 = q4_expand<kF16>(panel & 1 ? pair.z : pair.x, q4_zero<kF16>(entry[s][0] & 15u));
        const uint4 r1 = q4_expand<kF16>(panel & 1 ? pair.w : pair.y, q4_zero<kF16>(entry[s][1] & 15u));
#pragma unroll
        for (int c = 0; c < kEights; ++c) {
          mma16816<kF16>(d[s][c], r0.x, r1.x, r0.y, r1.y, b[c].x, b[c].y);
          mma16816<kF16>(d[s][c], r0.z, r1.z, r0.w, r1.w, b[c].z, b[c].w);
        }
      }
    }
#pragma unroll
    for (int s = 0; s < kStrips; ++s) {
      const float s0 = __uint_as_float(entry[s][0] & ~15u), s1 = __uint_as_float(entry[s][1] & ~15u);
#pragma unroll
      for (int c = 0; c < kEights; ++c) {
        acc[s][c][0] = __fmaf_rn(s0, d[s][c][0], acc[s][c][0]);
        acc[s][c][1] = __fmaf_rn(s0, d[s][c][1], acc[s][c][1]);
        acc[s][c][2] = __fmaf_rn(s1, d[s][c][2], acc[s][c][2]);
        acc[s][c][3] = __fmaf_rn(s1, d[s][c][3], acc[s][c][3]);
      }
    }
  }
}

template <int kType, int kGroup, int kEights, int kStrips, bool kOne>
__global__ void __launch_bounds__(256) gemv_q4_kernel(const GemvQ4Params p) {
  using Cfg = GemvQ4Cfg<kType, kGroup, kEights, kStrips, kOne>;
  static_assert(!kOne || kEights == 1, "one token has at most three columns");
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[Cfg::WARPS][Cfg::STAGES];
  __shared__ uint32_t abort_flag;
  uint8_t* const smem = smem_raw + ((0u - smem_u32(smem_raw)) & 127u);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  uint8_t* const ring = smem + warp * Cfg::RING_BYTES;
  [[maybe_unused]] uint8_t* const x_shared = smem + Cfg::WARPS * Cfg::RING_BYTES + warp * Cfg::X_BYTES;
  if (lane == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) mbar_init(smem_u32(&bars[warp][s]), 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) abort_flag = 0;
  if constexpr (kOne)  // columns that no part of the token has
    for (int i = lane; i < Cfg::X_BYTES / 16; i += 32) reinterpret_cast<uint4*>(x_shared)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const int row0 = blockIdx.x * Cfg::ROWS;
  constexpr size_t kBlockBytes = q4_block_bytes(kGroup);
  const uint8_t* codes = p.codes + static_cast<size_t>(row0 / kCodeRows) * p.blocks * kBlockBytes + row0 % kCodeRows / 16 * q4_strip_bytes(kGroup);
  auto fetch = [&](int kb, int stage) {  // lane 0
    const uint32_t bar = smem_u32(&bars[warp][stage]);
    mbar_arrive_expect_tx(bar, Cfg::STAGE_BYTES);
    bulk_load(smem_u32(ring + stage * Cfg::STAGE_BYTES), codes + kb * kBlockBytes, Cfg::STAGE_BYTES, bar);
  };
  // Staged x is written by the kernel before this one, which was through its own wait when this one could start: whatever the codes
  // come from has ended, and they are fetched without waiting for x.
  if constexpr (kOne) wait_for_launch_before();
  if (lane == 0)
    for (int i = 0; i < Cfg::STAGES; ++i)
      if (warp + i * Cfg::WARPS < p.blocks) fetch(warp + i * Cfg::WARPS, i);
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
  auto load_four = [&](int kb) {
    const int k0 = kb * kCodeSpan + lane * 4, left = p.k - k0;
    if (p.vec && left >= 4) {
      four.load(p.x, k0);
    } else {
      uint32_t v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long at = min(k0 + j, p.k - 1) * p.x_k;
        if constexpr (kType == kTypeF32) v[j] = ld_operand32(static_cast<const uint32_t*>(p.x) + at);
        else v[j] = ld_operand16(static_cast<const uint16_t*>(p.x) + at);
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
  if (warp < p.blocks) {
    if constexpr (kOne) {
      load_four(warp);
    } else {
#pragma unroll
      for (int panel = 0; panel < 4; ++panel) load_operands(warp, panel);
    }
  }
  int stage = 0;
  uint32_t parity = 0;
  bool ok = true;
  int kb = warp;
  for (; kb < p.blocks; kb += Cfg::WARPS) {
    const int next = kb + Cfg::WARPS;
    if constexpr (kOne) {
      uint8_t* to = x_shared + lane * 8;
      if constexpr (kType == kTypeF32) {
        uint2 hi, mid, lo;
        split3_bf16(four.raw.x, four.raw.y, hi.x, mid.x, lo.x);
        split3_bf16(four.raw.z, four.raw.w, hi.y, mid.y, lo.y);
        *reinterpret_cast<uint2*>(to) = hi;
        *reinterpret_cast<uint2*>(to + Cfg::X_PITCH) = mid;
        *reinterpret_cast<uint2*>(to + 2 * Cfg::X_PITCH) = lo;
      } else {
        *reinterpret_cast<uint2*>(to) = four.raw;
      }
      if (next < p.blocks) load_four(next);
    }
    ok = mbar_wait_lanes(smem_u32(&bars[warp][stage]), parity, &abort_flag);  // brings the lanes together, too
    if (!ok) break;
    const uint8_t* const here = ring + stage * Cfg::STAGE_BYTES;
    if constexpr (kOne) {
      multiply_block<kType, kGroup, kEights, kStrips>(acc, here, lane, [&](int panel, uint4(&b)[kEights]) {
        b[0] = *reinterpret_cast<const uint4*>(x_shared + (lane >> 2) * Cfg::X_PITCH + panel * 64 + (lane & 3) * 16);
      });
    } else {
      multiply_block<kType, kGroup, kEights, kStrips>(acc, here, lane, [&](int panel, uint4(&b)[kEights]) {
#pragma unroll
        for (int c = 0; c < kEights; ++c) b[c] = b_ahead[panel][c];
        if (next < p.blocks) load_operands(next, panel);
      });
    }
    __syncwarp();  // all have read the stage
    if (lane == 0 && kb + Cfg::STAGES * Cfg::WARPS < p.blocks) fetch(kb + Cfg::STAGES * Cfg::WARPS, stage);
    if (++stage == Cfg::STAGES) stage = 0, parity ^= 1;
  }
  if (!ok) {
    abort_flag = 1;
    if (lane == 0) {
      atomicCAS(p.status, 0, kErrOperandWait);
      // this warp's own copies land before the CTA gives up its shared memory
      for (int i = 0; i < Cfg::STAGES && kb < p.blocks; ++i, kb += Cfg::WARPS) {
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
  for (int i = threadIdx.x; i < Cfg::ROWS * p.tokens; i += 256) {
    const int r = i % Cfg::ROWS, token = i / Cfg::ROWS, row = row0 + r;
    if (row >= p.n) continue;
    float v = 0.f;
#pragma unroll
    for (int part = Cfg::PARTS - 1; part >= 0; --part)  // the small ones first
#pragma unroll
      for (int w = 0; w < Cfg::WARPS; ++w) v += sums[(w * Cfg::ROWS + r) * Cfg::SUM_PITCH + token * Cfg::PARTS + part];
    const long long at = token * p.c_token + row * p.c_row;
    v = __fmul_rn(p.alpha, v);
    if (p.beta != 0.f) v = __fmaf_rn(p.beta, ld_element_as(p.c_type, p.c, at), v);
    st_element_as(p.c_type, p.c, at, v);
  }
}

}  // namespace tcec_sm100
