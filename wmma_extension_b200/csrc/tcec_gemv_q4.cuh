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
  int vec;                    // x_k 1 and four values at a time aligned
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

// A warp's x of one block in shared memory: columns of 128 values in 16 bits, 320 bytes apart, so that lanes of two columns and four
// times 16 bytes read from all banks at once.
constexpr int kXPitch = 320;

template <int kType, int kGroup, int kCols, int kStrips>
struct GemvQ4Cfg {
  static constexpr int PARTS = kType == kTypeF32 ? 3 : 1;
  static constexpr int WIDTH = kCols * 8;                     // columns
  static constexpr int TOKENS = WIDTH / PARTS;
  static constexpr int ROWS = 16 * kStrips;
  static constexpr int WARPS = 8;
  static constexpr int AHEAD = kCols == 1 ? 2 : 1;            // blocks loaded ahead of the one at work
  static constexpr int X_BYTES = WIDTH * kXPitch;             // of a warp
  static constexpr int SUM_PITCH = WIDTH + 1;
  static constexpr int SUM_BYTES = WARPS * ROWS * SUM_PITCH * 4;
  static constexpr int SMEM_BYTES = WARPS * X_BYTES > SUM_BYTES ? WARPS * X_BYTES : SUM_BYTES;
};

// What a lane holds of one block: codes and entries of its rows, and four values of every token.
template <int kType, int kGroup, int kCols, int kStrips>
struct GemvQ4Block {
  using Cfg = GemvQ4Cfg<kType, kGroup, kCols, kStrips>;
  static constexpr int kSpans = kCodeSpan / kGroup;
  uint4 w[kStrips][2];
  uint32_t entry[kStrips][kSpans][2];
  Four<kType> x[Cfg::TOKENS];

  __device__ __forceinline__ void load(const GemvQ4Params& p, const uint8_t* block, int kb, int in_tile, int lane) {
    const uint8_t* strip = block + in_tile * 64 + lane * 16;
    const uint8_t* e = block + kQ4CodeBytes + (in_tile + (lane >> 2)) * 4;
#pragma unroll
    for (int s = 0; s < kStrips; ++s) {
      w[s][0] = ld_once128(strip + s * 1024);
      w[s][1] = ld_once128(strip + s * 1024 + 512);
#pragma unroll
      for (int q = 0; q < kSpans; ++q) {
        entry[s][q][0] = ld_operand32(e + q * kEntryBytes + s * 64);
        entry[s][q][1] = ld_operand32(e + q * kEntryBytes + s * 64 + 32);
      }
    }
    const int k0 = kb * kCodeSpan + lane * 4, left = p.k - k0;
    if (p.vec && (kb + 1) * kCodeSpan <= p.k) {
#pragma unroll
      for (int i = 0; i < Cfg::TOKENS; ++i)
        if (i < p.tokens) x[i].load(p.x, i * p.x_token + k0);
    } else {
#pragma unroll
      for (int i = 0; i < Cfg::TOKENS; ++i)
        if (i < p.tokens) {
          uint32_t v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const long long at = i * p.x_token + min(k0 + j, p.k - 1) * p.x_k;
            if constexpr (kType == kTypeF32) v[j] = ld_operand32(static_cast<const uint32_t*>(p.x) + at);
            else v[j] = ld_operand16(static_cast<const uint16_t*>(p.x) + at);
            if (j >= left) v[j] = 0;
          }
          if constexpr (kType == kTypeF32) x[i].raw = make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
          else x[i].raw = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
        }
    }
  }
  // x in its columns, for the lanes that need it as operand.
  __device__ __forceinline__ void share_x(const GemvQ4Params& p, uint8_t* mine, int lane) const {
#pragma unroll
    for (int i = 0; i < Cfg::TOKENS; ++i)
      if (i < p.tokens) {
        uint8_t* to = mine + i * Cfg::PARTS * kXPitch + lane * 8;
        if constexpr (kType == kTypeF32) {
          uint2 hi, mid, lo;
          split3_bf16(x[i].raw.x, x[i].raw.y, hi.x, mid.x, lo.x);
          split3_bf16(x[i].raw.z, x[i].raw.w, hi.y, mid.y, lo.y);
          *reinterpret_cast<uint2*>(to) = hi;
          *reinterpret_cast<uint2*>(to + kXPitch) = mid;
          *reinterpret_cast<uint2*>(to + 2 * kXPitch) = lo;
        } else {
          *reinterpret_cast<uint2*>(to) = x[i].raw;
        }
      }
  }
  __device__ __forceinline__ void multiply(float (&acc)[kStrips][kCols][4], const uint8_t* mine, int lane) const {
    constexpr bool kF16 = kType == kTypeF16;
#pragma unroll
    for (int q = 0; q < kSpans; ++q) {
      float d[kStrips][kCols][4];
#pragma unroll
      for (int s = 0; s < kStrips; ++s)
#pragma unroll
        for (int c = 0; c < kCols; ++c) d[s][c][0] = d[s][c][1] = d[s][c][2] = d[s][c][3] = 0.f;
#pragma unroll
      for (int panel = q * 4 / kSpans; panel < (q + 1) * 4 / kSpans; ++panel) {
        uint4 b[kCols];
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          b[c] = *reinterpret_cast<const uint4*>(mine + (c * 8 + (lane >> 2)) * kXPitch + panel * 64 + (lane & 3) * 16);
#pragma unroll
        for (int s = 0; s < kStrips; ++s) {
          const uint4 pair = w[s][panel >> 1];
          const uint4 r0 = q4_expand<kF16>(panel & 1 ? pair.z : pair.x, q4_zero<kF16>(entry[s][q][0] & 15u));
          const uint4 r1 = q4_expand<kF16>(panel & 1 ? pair.w : pair.y, q4_zero<kF16>(entry[s][q][1] & 15u));
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            mma16816<kF16>(d[s][c], r0.x, r1.x, r0.y, r1.y, b[c].x, b[c].y);
            mma16816<kF16>(d[s][c], r0.z, r1.z, r0.w, r1.w, b[c].z, b[c].w);
          }
        }
      }
#pragma unroll
      for (int s = 0; s < kStrips; ++s) {
        const float s0 = __uint_as_float(entry[s][q][0] & ~15u), s1 = __uint_as_float(entry[s][q][1] & ~15u);
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          acc[s][c][0] = __fmaf_rn(s0, d[s][c][0], acc[s][c][0]);
          acc[s][c][1] = __fmaf_rn(s0, d[s][c][1], acc[s][c][1]);
          acc[s][c][2] = __fmaf_rn(s1, d[s][c][2], acc[s][c][2]);
          acc[s][c][3] = __fmaf_rn(s1, d[s][c][3], acc[s][c][3]);
        }
      }
    }
  }
};

// kCols: columns in eights.
template <int kType, int kGroup, int kCols, int kStrips>
__global__ void __launch_bounds__(256) gemv_q4_kernel(const GemvQ4Params p) {
  using Cfg = GemvQ4Cfg<kType, kGroup, kCols, kStrips>;
  using Block = GemvQ4Block<kType, kGroup, kCols, kStrips>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* mine = smem + warp * Cfg::X_BYTES;
  for (int i = lane; i < Cfg::X_BYTES / 16; i += 32) reinterpret_cast<uint4*>(mine)[i] = make_uint4(0, 0, 0, 0);  // columns that nobody has
  const int row0 = blockIdx.x * Cfg::ROWS, in_tile = row0 % kCodeRows;
  constexpr size_t kBlockBytes = q4_block_bytes(kGroup);
  const uint8_t* base = p.codes + static_cast<size_t>(row0 / kCodeRows) * p.blocks * kBlockBytes;
  __syncwarp();
  wait_for_launch_before();
  let_next_launch_start();

  float acc[kStrips][kCols][4];
#pragma unroll
  for (int s = 0; s < kStrips; ++s)
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[s][c][0] = acc[s][c][1] = acc[s][c][2] = acc[s][c][3] = 0.f;

  constexpr int kHeld = Cfg::AHEAD + 1;
  Block held[kHeld];
#pragma unroll
  for (int i = 0; i < Cfg::AHEAD; ++i)
    if (warp + i * Cfg::WARPS < p.blocks) held[i].load(p, base + (warp + i * Cfg::WARPS) * kBlockBytes, warp + i * Cfg::WARPS, in_tile, lane);
  for (int kb = warp; kb < p.blocks; kb += kHeld * Cfg::WARPS) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int now = kb + i * Cfg::WARPS, next = now + Cfg::AHEAD * Cfg::WARPS;
      if (now >= p.blocks) break;
      if (next < p.blocks) held[(i + Cfg::AHEAD) % kHeld].load(p, base + next * kBlockBytes, next, in_tile, lane);
      held[i].share_x(p, mine, lane);
      __syncwarp();
      held[i].multiply(acc, mine, lane);
      __syncwarp();
    }
  }

  __syncthreads();  // x is read, sums take its place
  float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int s = 0; s < kStrips; ++s)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
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
