// Few columns of a gradient from activations in 8 bits: C[col][feature] = alpha * sum_b s[feature, b] sum_{i in b} code[feature][i] dy[i][col] + beta C, where a
// block b is 128 tokens.
//
// Bound by the bytes of the activations, as the product of few tokens with 4-bit weights (tcec_gemv_q4.cuh), and made like it: a warp takes a block
// of 16 kStrips features at a time through a ring of bulk copies, codes become operands of mma.m16n8k16 without arithmetic (sign and magnitude are
// those of a 16-bit number, the magnitude in its lowest bits; in f16 four bits higher, where the tensor core keeps them all), columns come staged
// (tcec_stage.cuh), and the power of two goes into the factor that makes the sums of a block values.  (In tiles on tcgen05 codes are converted, written to
// shared memory and read again for columns of which most do not exist: 8192 x 4096 of rank 16 18.7 us.)
//
// Measured, from memory, with the staging: 8192 x 4096 of rank 16 12.9 us (2.7 TB/s), of rank 4 10.2; 4096 x 16384 of rank 16 18.5 (3.8 TB/s); 1024 x 1024 4.2.
#pragma once
#include "tcec_gemv_q4.cuh"

namespace tcec_sm100 {

template <int kEights, int kStrips>
struct GemvQ8Cfg {
  static constexpr int ROWS = 16 * kStrips;
  static constexpr int MOST_WARPS = kEights == 4 ? 8 : 16;
  static constexpr int CHUNK_PITCH = ROWS * 16 + 64;          // 16 tokens; eight lanes' halves of two chunks lie in different banks
  static constexpr int STAGE_BYTES = 8 * CHUNK_PITCH + ROWS * 4;
  static constexpr int COPIED_BYTES = 8 * ROWS * 16 + ROWS * 4;
  static constexpr int STAGES = kStrips == 1 ? 4 : 2;        // 16384 x 2048 of rank 4: 11.9 us, with two 18.1; of two strips more than two do not fit
  static constexpr int RING_BYTES = (STAGES * STAGE_BYTES + 127) / 128 * 128;
  static constexpr int SUM_PITCH = kEights * 8 + 1;
  static constexpr int SUM_BYTES = ROWS * SUM_PITCH * 4;      // of a warp
  static constexpr int WARP_BYTES = RING_BYTES > SUM_BYTES ? RING_BYTES : SUM_BYTES;
  static constexpr int smem_bytes(int warps) { return warps * WARP_BYTES + 128; }
  static constexpr int WARPS_OF_SM = kEights == 1 ? 20 : kEights == 2 ? 16 : 8;
};

// Two of four codes (tokens 0 2 1 3, sign and magnitude) as operands: tokens 0 and 1, or 2 and 3.
template <bool kF16, bool kSecond>
__device__ __forceinline__ uint32_t q8_operand(uint32_t w) {
  constexpr int kUp = kF16 ? 4 : 0;
  constexpr uint32_t kSize = 0x007f007fu << kUp, kSign = 0x80008000u;
  if constexpr (kSecond) return ((w >> (8 - kUp)) & kSize) | (w & kSign);
  else return ((w << kUp) & kSize) | ((w << 8) & kSign);
}

template <int kType, int kEights, int kStrips>
__global__ void __launch_bounds__(32 * GemvQ8Cfg<kEights, kStrips>::MOST_WARPS, 1) gemv_q8_kernel(const GemvQ8Params p) {
  using Cfg = GemvQ8Cfg<kEights, kStrips>;
  constexpr int kParts = kType == kTypeF32 ? 3 : 1;
  constexpr bool kF16 = kType == kTypeF16;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[Cfg::MOST_WARPS][Cfg::STAGES];
  __shared__ uint32_t abort_flag;
  uint8_t* const smem = smem_raw + ((0u - smem_u32(smem_raw)) & 127u);
  const int warp = warp_index(), lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  uint8_t* const ring = smem + warp * Cfg::RING_BYTES;
  if (lane == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) mbar_init(smem_u32(&bars[warp][s]), 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) abort_flag = 0;
  __syncthreads();
  const int row0 = (p.first + blockIdx.x) * Cfg::ROWS;
  const uint8_t* codes = p.codes + static_cast<size_t>(row0 / kCodeRows) * p.blocks * kQ8BlockBytes;
  auto fetch = [&](int kb, int stage) {  // a chunk a lane, and the scales
    if (dev_flag(p.debug_flags, 128) && blockIdx.x == 0 && kb == 0) return;
    const uint32_t bar = smem_u32(&bars[warp][stage]), to = smem_u32(ring + stage * Cfg::STAGE_BYTES);
    const uint8_t* from = codes + static_cast<size_t>(kb) * kQ8BlockBytes;
    if (lane == 0) mbar_arrive_expect_tx(bar, Cfg::COPIED_BYTES);
    __syncwarp();
    if (lane < 8) bulk_load(to + lane * Cfg::CHUNK_PITCH, from + lane * 2048 + row0 % kCodeRows * 16, Cfg::ROWS * 16, bar);
    else if (lane == 8) bulk_load(to + 8 * Cfg::CHUNK_PITCH, from + kQ8CodeBytes + row0 % kCodeRows * 4, Cfg::ROWS * 4, bar);
  };
  // The kernel before stages dY and has itself waited for whatever wrote the codes: they are fetched without waiting for it.
  for (int i = 0; i < Cfg::STAGES; ++i)
    if (warp + i * warps < p.blocks) fetch(warp + i * warps, i);
  wait_for_launch_before();
  let_next_launch_start();

  float acc[kStrips][kEights][4];
#pragma unroll
  for (int s = 0; s < kStrips; ++s)
#pragma unroll
    for (int c = 0; c < kEights; ++c) acc[s][c][0] = acc[s][c][1] = acc[s][c][2] = acc[s][c][3] = 0.f;
  const uint8_t* const staged = after_wait(p.staged) + lane * 16;
  const uint8_t* const staged_units = after_wait(p.staged) + static_cast<size_t>(p.blocks) * (kEights * 2048) + (lane & 3) * 8;
  const int at = (lane >> 2) * 16 + ((lane >> 1) & 1) * Cfg::CHUNK_PITCH + (lane & 1) * 8;  // of this lane's tokens of a panel, in a strip
  int stage = 0;
  uint32_t parity = 0;
  bool ok = true;
  int kb = warp;
  for (; kb < p.blocks; kb += warps) {
    uint4 b[4][kEights];
    float2 unit[kEights];
#pragma unroll
    for (int c = 0; c < kEights; ++c) {
      unit[c] = make_float2(0x1p20f, 0x1p20f);
      if constexpr (!kF16) {
        const uint2 u = ld_operand64(staged_units + static_cast<size_t>(kb) * staged_sum_bytes(kEights) + c * 32);
        unit[c] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
      }
#pragma unroll
      for (int panel = 0; panel < 4; ++panel)
        b[panel][c] = ld_ahead128(staged + static_cast<size_t>(kb) * (kEights * 2048) + panel * (kEights * 512) + c * 512);
    }
    ok = mbar_wait_lanes(smem_u32(&bars[warp][stage]), parity, &abort_flag);
    if (!ok) break;
    const uint8_t* const here = ring + stage * Cfg::STAGE_BYTES;
#pragma unroll
    for (int s = 0; s < kStrips; ++s) {
      float d[kEights][4];
#pragma unroll
      for (int panel = 0; panel < 4; ++panel) {
        const uint8_t* from = here + panel * 2 * Cfg::CHUNK_PITCH + s * 256 + at;
        const uint2 w0 = *reinterpret_cast<const uint2*>(from), w1 = *reinterpret_cast<const uint2*>(from + 128);  // of rows g and g + 8
#pragma unroll
        for (int c = 0; c < kEights; ++c) {
          mma16816_zero<kF16>(d[c], q8_operand<kF16, false>(w0.x), q8_operand<kF16, false>(w1.x), q8_operand<kF16, true>(w0.x),
                              q8_operand<kF16, true>(w1.x), b[panel][c].x, b[panel][c].y, panel == 0);
          mma16816<kF16>(d[c], q8_operand<kF16, false>(w0.y), q8_operand<kF16, false>(w1.y), q8_operand<kF16, true>(w0.y),
                         q8_operand<kF16, true>(w1.y), b[panel][c].z, b[panel][c].w);
        }
      }
      const float* scales = reinterpret_cast<const float*>(here + 8 * Cfg::CHUNK_PITCH) + s * 16 + (lane >> 2);
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < kEights; ++c) {
          acc[s][c][r * 2] = __fmaf_rn(scales[r * 8], unit[c].x * d[c][r * 2], acc[s][c][r * 2]);
          acc[s][c][r * 2 + 1] = __fmaf_rn(scales[r * 8], unit[c].y * d[c][r * 2 + 1], acc[s][c][r * 2 + 1]);
        }
    }
    __syncwarp();  // all have read the stage
    if (kb + Cfg::STAGES * warps < p.blocks) fetch(kb + Cfg::STAGES * warps, stage);
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
  for (int i = threadIdx.x; i < Cfg::ROWS * p.cols; i += blockDim.x) {
    const int r = i % Cfg::ROWS, col = i / Cfg::ROWS, row = row0 + r;
    if (row >= p.rows) continue;
    float v = 0.f;
#pragma unroll
    for (int part = kParts - 1; part >= 0; --part)  // the small ones first
#pragma unroll 4
      for (int w = 0; w < warps; ++w) v += sums[(w * Cfg::ROWS + r) * Cfg::SUM_PITCH + col * kParts + part];
    const long long to = row * p.c_row + col * p.c_col;
    v = __fmul_rn(p.alpha, v);
    if (p.beta != 0.f) v = __fmaf_rn(p.beta, ld_element_as(p.c_type, c, to), v);
    st_element_as(p.c_type, c, to, v);
  }
}

}  // namespace tcec_sm100
