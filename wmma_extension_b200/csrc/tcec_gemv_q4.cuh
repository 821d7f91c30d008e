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

struct GemvQ4Params {
  const uint8_t* codes;
  const void* x;              // element (token, i) at token * x_token + i * x_k
  long long x_token, x_k;
  int n, k, tokens, blocks;
  int vec;                    // x_k 1 and aligned for 16 bytes
  float alpha, beta;
  void* c;                    // element (token, row) at token * c_token + row * c_row
  long long c_token, c_row;
  int c_type;
};

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

// Eight consecutive values of a column's token from k0 on, as 16-bit operands.
template <int kType>
__device__ __forceinline__ uint4 load_column8(const GemvQ4Params& p, int col, int k0) {
  constexpr int kParts = kType == kTypeF32 ? 3 : 1;
  const int token = col / kParts;
  uint4 o = make_uint4(0, 0, 0, 0);
  if (token >= p.tokens) return o;
  const long long at = token * p.x_token + k0 * p.x_k;
  if constexpr (kType == kTypeF32) {
    const int part = col - token * kParts;
    float v[8] = {};
    if (p.vec && k0 + 8 <= p.k) {
      const float4 a = ld_operand(reinterpret_cast<const float4*>(static_cast<const float*>(p.x) + at));
      const float4 b = ld_operand(reinterpret_cast<const float4*>(static_cast<const float*>(p.x) + at + 4));
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k0 + j < p.k) v[j] = ld_operand(static_cast<const float*>(p.x) + at + j * p.x_k);
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t hi, mid, lo;
      split3_bf16(v[2 * j], v[2 * j + 1], hi, mid, lo);
      w[j] = part == 0 ? hi : part == 1 ? mid : lo;
    }
    o = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    const uint16_t* x = static_cast<const uint16_t*>(p.x);
    if (p.vec && k0 + 8 <= p.k) {
      o = ld_operand128(x + at);
    } else {
      uint32_t w[8] = {};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k0 + j < p.k) w[j] = ld_operand16(x + at + j * p.x_k);
      o = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
  }
  return o;
}

// kCols: columns in eights.
template <int kType, int kGroup, int kCols, int kStrips>
__global__ void __launch_bounds__(256) gemv_q4_kernel(const GemvQ4Params p) {
  constexpr bool kF16 = kType == kTypeF16;
  constexpr int kParts = kType == kTypeF32 ? 3 : 1, kSpans = kCodeSpan / kGroup, kWarps = 8;
  constexpr int kRows = 16 * kStrips, kWidth = kCols * 8;
  __shared__ float sums[kWarps][kRows][kWidth + 1];
  wait_for_launch_before();
  let_next_launch_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * kRows;
  const size_t block_bytes = q4_block_bytes(kGroup);
  const uint8_t* base = p.codes + static_cast<size_t>(row0 / kCodeRows) * p.blocks * block_bytes;
  const int in_tile = row0 % kCodeRows;

  float acc[kStrips][kCols][4];
#pragma unroll
  for (int s = 0; s < kStrips; ++s)
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[s][c][0] = acc[s][c][1] = acc[s][c][2] = acc[s][c][3] = 0.f;

  for (int kb = warp; kb < p.blocks; kb += kWarps) {
    const uint8_t* block = base + kb * block_bytes;
    uint4 w[kStrips][2];
    uint32_t entries[kStrips][kSpans][2];
#pragma unroll
    for (int s = 0; s < kStrips; ++s) {
      const uint8_t* strip = block + (in_tile / 16 + s) * 1024 + lane * 16;
      w[s][0] = ld_once128(strip);
      w[s][1] = ld_once128(strip + 512);
#pragma unroll
      for (int q = 0; q < kSpans; ++q) {
        const uint8_t* e = block + kQ4CodeBytes + q * kEntryBytes + (in_tile + s * 16 + g) * 4;
        entries[s][q][0] = ld_operand32(e);
        entries[s][q][1] = ld_operand32(e + 32);
      }
    }
    uint4 x[kCols][4];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int panel = 0; panel < 4; ++panel) x[c][panel] = load_column8<kType>(p, c * 8 + g, kb * kCodeSpan + panel * 32 + t * 8);
#pragma unroll
    for (int s = 0; s < kStrips; ++s)
#pragma unroll
      for (int q = 0; q < kSpans; ++q) {
        const uint32_t zero0 = q4_zero<kF16>(entries[s][q][0] & 15u), zero1 = q4_zero<kF16>(entries[s][q][1] & 15u);
        const float s0 = __uint_as_float(entries[s][q][0] & ~15u), s1 = __uint_as_float(entries[s][q][1] & ~15u);
        float d[kCols][4];
#pragma unroll
        for (int c = 0; c < kCols; ++c) d[c][0] = d[c][1] = d[c][2] = d[c][3] = 0.f;
#pragma unroll
        for (int panel = q * 4 / kSpans; panel < (q + 1) * 4 / kSpans; ++panel) {
          const uint4 pair = w[s][panel >> 1];
          const uint4 a = q4_expand<kF16>(panel & 1 ? pair.z : pair.x, zero0), b = q4_expand<kF16>(panel & 1 ? pair.w : pair.y, zero1);
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            mma16816<kF16>(d[c], a.x, b.x, a.y, b.y, x[c][panel].x, x[c][panel].y);
            mma16816<kF16>(d[c], a.z, b.z, a.w, b.w, x[c][panel].z, x[c][panel].w);
          }
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          acc[s][c][0] = __fmaf_rn(s0, d[c][0], acc[s][c][0]);
          acc[s][c][1] = __fmaf_rn(s0, d[c][1], acc[s][c][1]);
          acc[s][c][2] = __fmaf_rn(s1, d[c][2], acc[s][c][2]);
          acc[s][c][3] = __fmaf_rn(s1, d[c][3], acc[s][c][3]);
        }
      }
  }

#pragma unroll
  for (int s = 0; s < kStrips; ++s)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[warp][s * 16 + g + (j >> 1) * 8][c * 8 + t * 2 + (j & 1)] = acc[s][c][j];
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * p.tokens; i += 256) {
    const int r = i % kRows, token = i / kRows, row = row0 + r;
    if (row >= p.n) continue;
    float v = 0.f;
#pragma unroll
    for (int part = kParts - 1; part >= 0; --part)  // the small ones first
#pragma unroll
      for (int wq = 0; wq < kWarps; ++wq) v += sums[wq][r][token * kParts + part];
    const long long at = token * p.c_token + row * p.c_row;
    v = __fmul_rn(p.alpha, v);
    if (p.beta != 0.f) v = __fmaf_rn(p.beta, ld_element_as(p.c_type, p.c, at), v);
    st_element_as(p.c_type, p.c, at, v);
  }
}

}  // namespace tcec_sm100
