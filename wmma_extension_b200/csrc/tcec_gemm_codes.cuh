// Products of a dense operand with an operand kept as codes (tcec_codes.cuh), on tcgen05 tensor cores:
//
//   D[row][col] = sum_g s[row, g] * sum_{i in g} code[row][i] * dense[col][i]
//
// rows: the outputs of 4-bit weights, or the features of 8-bit activations; cols: tokens, or the outputs of a weight gradient;
// i: k, or tokens; g: the codes that share a scale.
//
// Codes are whole numbers of at most 7 bits and a sign, which f16 and bf16 hold exactly, so the tensor cores multiply them with the
// dense operand as it is: f16 or bf16, or FP32 in three bf16 parts of 8 bits each, which are exactly it.  The sum of a group is made
// in the tensor core's FP32 accumulator, and is then multiplied by its scale and added in FP32 registers, rounded to nearest: scales
// never meet 16 bits, and the accumulator, which truncates, never holds more than 128 (FP32: 3 x 128) products.  Rows are the lanes of
// TMEM, so a scale is one register of the thread that holds the row.
//
// The dense operand is first laid out in panels (stage_panels_kernel), whatever its type, order and alignment: 128 columns x 32 of the
// sum x 2 bytes in the core-matrix order that the MMA reads, so that the product brings them in with linear bulk copies.
#pragma once
#include "tcec_codes.cuh"
#include "tcec_gemm_panels.cuh"
#include "tcec_gemm_roles.cuh"

namespace tcec_sm100 {

// ---------------------------------------------------------------- the dense operand in panels
constexpr int kSpanPanels = kCodeSpan / 32;                  // panels of one block and part
constexpr int kSpanBytes = kSpanPanels * kPanelBytes;        // 32 KB
struct StagePanelsParams {
  const void* src;            // element (col, i) at col * col_step + i * sum_step
  long long col_step, sum_step;
  int cols, sum;
  int blocks;                 // along the sum
  uint8_t* panels;            // [128 columns][block][part][panel]
  int vec;                    // sum_step 1 and aligned for 16 bytes
};
// x = hi + mid + lo, 8 bits each, two values at a time.  Exactly so unless lo falls below the smallest bf16 number; what is not finite
// stays in hi alone.
__device__ __forceinline__ void split3_bf16(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  const uint32_t bx = x != x ? 0x7fc00000u : __float_as_uint(x), by = y != y ? 0x7fc00000u : __float_as_uint(y);
  float rx = x - __uint_as_float(bx & 0xffff0000u), ry = y - __uint_as_float(by & 0xffff0000u);
  if (not_finite(x)) rx = 0.f;
  if (not_finite(y)) ry = 0.f;
  hi = __byte_perm(bx, by, 0x7632);
  const uint32_t mx = __float_as_uint(rx), my = __float_as_uint(ry);
  mid = __byte_perm(mx, my, 0x7632);
  const float lx = rx - __uint_as_float(mx & 0xffff0000u), ly = ry - __uint_as_float(my & 0xffff0000u);
  lo = __byte_perm(__float_as_uint(lx), __float_as_uint(ly), 0x7632);
}

// One CTA a block of 128 columns x 128 of the sum; an item is 16 bytes of a panel, eight consecutive values of one column.
template <int kType>
__global__ void __launch_bounds__(256) stage_panels_kernel(const StagePanelsParams p) {
  constexpr int kParts = kType == kTypeF32 ? 3 : 1;
  wait_for_launch_before();
  const int kb = blockIdx.x % p.blocks, cb = blockIdx.x / p.blocks;
  uint8_t* out = p.panels + static_cast<size_t>(blockIdx.x) * kParts * kSpanBytes;
  const int cols = min(kCodeRows, (p.cols - cb * kCodeRows + 15) & ~15);  // columns that an MMA may read
#pragma unroll 2
  for (int it = 0; it < 8; ++it) {
    const int item = threadIdx.x + it * 256;
    int r, c, panel;
    if (p.sum_step == 1) {  // a warp: 8 columns x 64 bytes
      r = (item & 7) + ((item >> 5) & 15) * 8;
      c = (item >> 3) & 3;
      panel = item >> 9;
    } else {                // a warp: 32 columns
      r = item & 127;
      c = (item >> 7) & 3;
      panel = item >> 9;
    }
    if (r >= cols) continue;
    const int col = cb * kCodeRows + r, i0 = kb * kCodeSpan + panel * 32 + c * 8;
    const long long at = col * p.col_step + i0 * p.sum_step;
    uint8_t* to = out + panel * kPanelBytes + (r >> 3) * 512 + c * 128 + (r & 7) * 16;
    const bool whole = col < p.cols && i0 + 8 <= p.sum;
    if constexpr (kType == kTypeF32) {
      float v[8] = {};
      if (whole && p.vec) {
        const float4 a = ld_operand(reinterpret_cast<const float4*>(static_cast<const float*>(p.src) + at));
        const float4 b = ld_operand(reinterpret_cast<const float4*>(static_cast<const float*>(p.src) + at + 4));
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col < p.cols && i0 + j < p.sum) v[j] = ld_operand(static_cast<const float*>(p.src) + at + j * p.sum_step);
      }
      uint32_t part[3][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) split3_bf16(v[2 * j], v[2 * j + 1], part[0][j], part[1][j], part[2][j]);
#pragma unroll
      for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4*>(to + q * kSpanBytes) = make_uint4(part[q][0], part[q][1], part[q][2], part[q][3]);
    } else {
      uint4 o = make_uint4(0, 0, 0, 0);
      const uint16_t* src = static_cast<const uint16_t*>(p.src);
      if (whole && p.vec) {
        o = ld_operand128(src + at);
      } else {
        uint32_t w[8] = {};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col < p.cols && i0 + j < p.sum) w[j] = ld_operand16(src + at + j * p.sum_step);
        o = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
      }
      *reinterpret_cast<uint4*>(to) = o;
    }
  }
  let_next_launch_start();
}

// ---------------------------------------------------------------- codes to 16-bit operands
__device__ __forceinline__ uint32_t sub16x2(uint32_t a, uint32_t b, bool f16) {
  uint32_t d;
  if (f16) asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// A whole number below the step of the last place of `magic` is put into its low bits, and magic (with the zero point) is taken off again.
template <bool kF16>
__device__ __forceinline__ uint32_t q4_zero(int z) {
  const uint32_t one = (kF16 ? 0x6400u : 0x4300u) | static_cast<uint32_t>(z);  // 1024 + z, 128 + z
  return one | one << 16;
}
// Eight 4-bit codes to code - zero point, in order.
template <bool kF16>
__device__ __forceinline__ uint4 q4_expand(uint32_t w, uint32_t zero) {
  constexpr uint32_t kMagic = kF16 ? 0x64006400u : 0x43004300u, kMask = 0x000f000fu;
  return make_uint4(sub16x2((w & kMask) | kMagic, zero, kF16), sub16x2(((w >> 4) & kMask) | kMagic, zero, kF16),
                    sub16x2(((w >> 8) & kMask) | kMagic, zero, kF16), sub16x2(((w >> 12) & kMask) | kMagic, zero, kF16));
}
// Two codes of 8 bits (sign and magnitude) in bits 0-7 and 16-23: +-(magic + magnitude) -+ magic.
template <bool kF16>
__device__ __forceinline__ uint32_t q8_expand2(uint32_t x) {
  constexpr uint32_t kMagic = kF16 ? 0x64006400u : 0x43004300u;
  const uint32_t base = ((x << 8) & 0x80008000u) | kMagic;
  return sub16x2(base | (x & 0x007f007fu), base, kF16);
}
template <bool kF16>
__device__ __forceinline__ uint4 q8_expand(uint2 w) {
  return make_uint4(q8_expand2<kF16>(__byte_perm(w.x, 0, 0x4140)), q8_expand2<kF16>(__byte_perm(w.x, 0, 0x4342)),
                    q8_expand2<kF16>(__byte_perm(w.y, 0, 0x4140)), q8_expand2<kF16>(__byte_perm(w.y, 0, 0x4342)));
}

// ---------------------------------------------------------------- the product
struct GemmCodesParams {
  const uint8_t* codes;       // [row tile][block]
  const uint8_t* panels;      // [128 columns][block][part]
  int rows, cols, blocks;     // blocks along the sum
  int parts;                  // of the dense operand: 1, or 3 (FP32)
  int row_tiles, col_tiles;
  float alpha, beta;
  void* c;
  long long c_row, c_col;     // steps between elements of C along rows and columns of this product
  int c_type;
  int* status;
};

// kSpans: groups of 4-bit codes in a block (1, 2 or 4); 0: 8-bit codes, one group a block.
template <int BN, int kSpans>
struct GemmCodesCfg {
  static constexpr bool Q8 = kSpans == 0;
  static constexpr int GROUPS = Q8 ? 1 : kSpans;
  static constexpr int THREADS = 512;
  static constexpr int CODE_BYTES = Q8 ? kQ8CodeBytes : kQ4CodeBytes;
  static constexpr int BLOCK_BYTES = CODE_BYTES + kEntryBytes * GROUPS;
  // Expanded codes: a chunk of 8 along the sum is 128 rows x 16 bytes, in core matrices of 8 rows; the chunks lie 32 bytes off a
  // multiple of 128, so that lanes with rows g, g + 1 of four chunks write to all banks at once.
  static constexpr int CHUNK_BYTES = 128 * 16 + 32;
  static constexpr int A_BYTES = 16 * CHUNK_BYTES;
  static constexpr int A_STAGES = 2;
  static constexpr int B_BYTES = BN * 128;                    // 64 of the sum, one part
  static constexpr int B_STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr int B_OFFSET = 0;
  static constexpr int A_OFFSET = B_STAGES * B_BYTES;
  static constexpr int SMEM_BYTES = A_OFFSET + A_STAGES * A_BYTES + 1024;
  static_assert(SMEM_BYTES <= 232448 - 512, "dynamic + static shared memory exceed an SM");
  static_assert(B_STAGES * B_BYTES >= 128 * BN * 4, "partial results go where the dense operand was");
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int NC = BN / 2;                           // columns of an epilogue thread
  // 512 threads x 128 registers at launch: 128 x (40 + 72) + 2 x 128 x 200 = 65536
  static constexpr bool REBALANCE = BN == 256;
};

__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float s) {
  asm("{\n\t.reg .b64 d, v, m;\n\t"
      "mov.b64 d, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 m, {%4, %4};\n\t"
      "fma.rn.f32x2 d, v, m, d;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b), "f"(s));
}
// Loads that are issued where they stand, ahead of the waits that follow.
__device__ __forceinline__ uint32_t ld_ahead32(const void* p) {
  uint32_t v;
  asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_ahead64(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 ld_ahead128(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// What a converter thread holds of one block: the codes of 16 chunks, one block ahead of the one it expands.
template <bool kF16, int kSpans>
struct Converter {  // 4 bits: two strips of 16 rows, lane 4 g + t has rows g and g + 8 of both
  uint4 w[2][2];
  uint32_t entry[kSpans][2][2];
  int code_at, entry_at, out_at;
  __device__ __forceinline__ Converter(int warp, int lane) {
    code_at = warp * 2048 + lane * 16;
    entry_at = kQ4CodeBytes + (warp * 32 + (lane >> 2)) * 4;
    out_at = (lane & 3) * GemmCodesCfg<128, kSpans>::CHUNK_BYTES + warp * 512 + (lane >> 2) * 16;
  }
  __device__ __forceinline__ void load_strip(const uint8_t* block, int s) {
    w[s][0] = ld_ahead128(block + code_at + s * 1024);
    w[s][1] = ld_ahead128(block + code_at + s * 1024 + 512);
#pragma unroll
    for (int q = 0; q < kSpans; ++q) {
      entry[q][s][0] = ld_ahead32(block + entry_at + q * kEntryBytes + s * 64);
      entry[q][s][1] = ld_ahead32(block + entry_at + q * kEntryBytes + s * 64 + 32);
    }
  }
  __device__ __forceinline__ void load(const uint8_t* block) {
    load_strip(block, 0);
    load_strip(block, 1);
  }
  // Expands what it holds to `out` and loads from `next` in its place.
  __device__ __forceinline__ void expand(uint8_t* out, const uint8_t* next) {
    constexpr int kChunk = GemmCodesCfg<128, kSpans>::CHUNK_BYTES;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int panel = 0; panel < 4; ++panel) {
        const uint4 pair = w[s][panel >> 1];
        uint8_t* to = out + out_at + panel * 4 * kChunk + s * 256;
        const int q = panel * kSpans / 4;
        *reinterpret_cast<uint4*>(to) = q4_expand<kF16>(panel & 1 ? pair.z : pair.x, q4_zero<kF16>(entry[q][s][0] & 15u));
        *reinterpret_cast<uint4*>(to + 128) = q4_expand<kF16>(panel & 1 ? pair.w : pair.y, q4_zero<kF16>(entry[q][s][1] & 15u));
      }
      if (next) load_strip(next, s);
    }
  }
};
template <bool kF16>
struct Converter<kF16, 0> {  // 8 bits: one row
  uint2 w[16];
  int code_at, out_at;
  __device__ __forceinline__ Converter(int warp, int lane) {
    code_at = (warp * 32 + lane) * 8;
    out_at = (warp * 32 + lane) * 16;
  }
  __device__ __forceinline__ void load(const uint8_t* block) {
#pragma unroll
    for (int c = 0; c < 16; ++c) w[c] = ld_ahead64(block + code_at + c * 1024);
  }
  __device__ __forceinline__ void expand(uint8_t* out, const uint8_t* next) {
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      *reinterpret_cast<uint4*>(out + out_at + c * GemmCodesCfg<128, 0>::CHUNK_BYTES) = q8_expand<kF16>(w[c]);
      if (next) w[c] = ld_ahead64(next + code_at + c * 1024);
    }
  }
};

// Launched with clusters of 1, 2, 4 or 8 CTAs (256 columns: 1): one tile of 128 rows x BN columns a cluster, whose CTAs divide the sum and add up through
// shared memory, in the order of the sum.
template <int BN, bool kF16, int kSpans>
__global__ void __launch_bounds__(512, 1) tcec_gemm_codes_kernel(const GemmCodesParams p) {
  using Cfg = GemmCodesCfg<BN, kSpans>;
  constexpr int kGroups = Cfg::GROUPS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_a_full[Cfg::A_STAGES], bar_a_empty[Cfg::A_STAGES];
  __shared__ uint64_t bar_b_full[Cfg::B_STAGES], bar_b_empty[Cfg::B_STAGES];
  __shared__ uint64_t bar_acc_full[2], bar_acc_free[2], bar_drain[1];
  __shared__ uint32_t tmem_base_s;
  __shared__ uint32_t abort_flag;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int shares = static_cast<int>(cluster_nctarank()), share = static_cast<int>(cluster_ctarank());
  const int tile = blockIdx.x / shares;
  const int rt = tile % p.row_tiles, ct = tile / p.row_tiles;
  const int kb_first = static_cast<int>(static_cast<long long>(p.blocks) * share / shares);
  const int kb_end = static_cast<int>(static_cast<long long>(p.blocks) * (share + 1) / shares);
  const uint8_t* codes = p.codes + static_cast<size_t>(rt) * p.blocks * Cfg::BLOCK_BYTES;
  const int cols = min(BN, p.cols - ct * BN), cols16 = (cols + 15) & ~15;

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::A_STAGES; ++s) {
      mbar_init(smem_u32(&bar_a_full[s]), 4);
      mbar_init(smem_u32(&bar_a_empty[s]), 1);
    }
    for (int s = 0; s < Cfg::B_STAGES; ++s) {
      mbar_init(smem_u32(&bar_b_full[s]), 1);
      mbar_init(smem_u32(&bar_b_empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 1);
      mbar_init(smem_u32(&bar_acc_free[i]), 8);
    }
    mbar_init(smem_u32(&bar_drain[0]), 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_base_s), Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if (shares > 1) cluster_sync_all();  // the others' shared memory exists before anything is written to it
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  volatile uint32_t* abortp = &abort_flag;
  wait_for_launch_before();

  float acc[Cfg::NC];

  if (warp < 4) {
    if constexpr (Cfg::REBALANCE) setmaxnreg_dec<40>();
    if (warp == 0) {
      // ---------------------------------------------------------- copies of the dense operand
      if (elect_one()) {
        uint32_t bs = 0, bph = 0, armed = 0, armed_parity = 0;
        bool ok = true;
        const uint8_t* src0 = p.panels + (static_cast<size_t>(ct * BN >> 7) * p.blocks + kb_first) * p.parts * kSpanBytes + (ct * BN & 127) * 64;
        const uint8_t* src1 = src0 + static_cast<size_t>(p.blocks) * p.parts * kSpanBytes;  // the second 128 columns of 256
        const uint32_t rows0 = min(128, cols16) * 64, rows1 = cols16 > 128 ? (cols16 - 128) * 64 : 0;
        for (int left = (kb_end - kb_first) * p.parts * 2; left > 0; --left) {  // a half of a block and part
          if (!mbar_wait(smem_u32(&bar_b_empty[bs]), bph ^ 1, abortp)) {
            ok = false;
            break;
          }
          const uint32_t bfull = smem_u32(&bar_b_full[bs]);
          mbar_arrive_expect_tx(bfull, 2 * (rows0 + rows1));
          armed |= 1u << bs;
          armed_parity = (armed_parity & ~(1u << bs)) | (bph << bs);
          const uint32_t dst = smem_base + Cfg::B_OFFSET + bs * Cfg::B_BYTES;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            bulk_load(dst + q * (BN * 64), src0 + q * kPanelBytes, rows0, bfull);
            if (BN > 128 && rows1) bulk_load(dst + q * (BN * 64) + kPanelBytes, src1 + q * kPanelBytes, rows1, bfull);
          }
          src0 += 2 * kPanelBytes;
          src1 += 2 * kPanelBytes;
          if (++bs == Cfg::B_STAGES) bs = 0, bph ^= 1;
        }
        if (!ok) {
          abort_flag = 1;
          atomicCAS(p.status, 0, kErrProducerWait);
          // this thread's own copies land before the CTA gives up its shared memory
          for (uint32_t q = 0; q < Cfg::B_STAGES; ++q)
            if (armed & (1u << q)) mbar_wait_plain(smem_u32(&bar_b_full[q]), (armed_parity >> q) & 1);
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- MMAs
      if (elect_one()) {
        const uint64_t a_const = umma_desc_kmajor_noswizzle(0, Cfg::CHUNK_BYTES, 128), b_const = umma_desc_kmajor_noswizzle(0, 128, 512);
        const uint32_t idesc = umma_idesc(kF16 ? 0u : 1u, 128, cols16);
        const uint32_t a16 = ((smem_base + Cfg::A_OFFSET) & 0x3ffff) >> 4, b16 = ((smem_base + Cfg::B_OFFSET) & 0x3ffff) >> 4;
        uint32_t as = 0, aph = 0, bs = 0, bph = 0, fold = 0;
        bool ok = true;
        for (int kb = kb_first; kb < kb_end && ok; ++kb) {
          if (!mbar_wait(smem_u32(&bar_a_full[as]), aph, abortp, 0)) {
            ok = false;
            break;
          }
          const uint32_t a_here = a16 + as * (Cfg::A_BYTES >> 4);
          for (int part = 0; part < p.parts && ok; ++part) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (!mbar_wait(smem_u32(&bar_b_full[bs]), bph, abortp, 0)) {
                ok = false;
                break;
              }
              tc_fence_after();
              const uint32_t b_here = b16 + bs * (Cfg::B_BYTES >> 4);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int step = h * 4 + j;  // of 16 along the sum
                // an accumulator holds one group; where a block is one, all parts of it
                const bool first = step % (8 / kGroups) == 0 && (kGroups > 1 || part == 0);
                const bool last = step % (8 / kGroups) == 8 / kGroups - 1 && (kGroups > 1 || part == p.parts - 1);
                if (first) {
                  if (!mbar_wait(smem_u32(&bar_acc_free[fold & 1]), ((fold >> 1) & 1) ^ 1, abortp, 0)) {
                    ok = false;
                    break;
                  }
                  tc_fence_after();
                }
                umma_ss<false>(tmem + (fold & 1) * BN, a_const | (a_here + step * (2 * Cfg::CHUNK_BYTES >> 4)),
                               b_const | (b_here + (j >> 1) * (BN * 64 >> 4) + (j & 1) * 16), idesc, first ? 0u : 1u);
                if (last) {
                  umma_commit(smem_u32(&bar_acc_full[fold & 1]));
                  ++fold;
                }
              }
              if (!ok) break;
              umma_commit(smem_u32(&bar_b_empty[bs]));
              if (++bs == Cfg::B_STAGES) bs = 0, bph ^= 1;
            }
          }
          if (!ok) break;
          umma_commit(smem_u32(&bar_a_empty[as]));
          if (++as == Cfg::A_STAGES) as = 0, aph ^= 1;
        }
        if (!ok) mma_thread_gave_up<false>(&abort_flag, p.status, kErrMmaWait, &bar_drain[0]);
      }
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ codes to operands
    if constexpr (Cfg::REBALANCE) setmaxnreg_dec<72>();
    Converter<kF16, kSpans> held(warp - 4, lane);
    uint32_t as = 0, aph = 0;
    bool ok = true;
    if (kb_first < kb_end) held.load(codes + static_cast<size_t>(kb_first) * Cfg::BLOCK_BYTES);
    for (int kb = kb_first; kb < kb_end; ++kb) {
      if (!mbar_wait_warp(smem_u32(&bar_a_empty[as]), aph ^ 1, abortp, 64)) {
        ok = false;
        break;
      }
      held.expand(smem_gen + Cfg::A_OFFSET + as * Cfg::A_BYTES, kb + 1 < kb_end ? codes + static_cast<size_t>(kb + 1) * Cfg::BLOCK_BYTES : nullptr);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_a_full[as]));
      if (++as == Cfg::A_STAGES) as = 0, aph ^= 1;
    }
    if (!ok) {
      abort_flag = 1;
      if (lane == 0) atomicCAS(p.status, 0, kErrOperandWait);
    }
  } else {
    // ------------------------------------------------------------ scales
    if constexpr (Cfg::REBALANCE) setmaxnreg_inc<200>();
#pragma unroll
    for (int i = 0; i < Cfg::NC; ++i) acc[i] = 0.f;
    const int q = warp & 3, r = q * 32 + lane, first_col = (warp >= 12 ? Cfg::NC : 0);
    const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + first_col;
    const bool any = first_col < cols;
    const int rounds = kGroups > 1 ? p.parts : 1;  // of the groups of a block
    uint32_t fold = 0;
    bool ok = true;
    float scale[kGroups], next[kGroups];
    auto load_scales = [&](int kb) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        next[g] = __uint_as_float(ld_ahead32(codes + static_cast<size_t>(kb) * Cfg::BLOCK_BYTES + Cfg::CODE_BYTES + g * kEntryBytes + r * 4) &
                                  (Cfg::Q8 ? ~0u : ~15u));
    };
    if (kb_first < kb_end) load_scales(kb_first);
    for (int kb = kb_first; kb < kb_end && ok; ++kb) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) scale[g] = next[g];
      if (kb + 1 < kb_end) load_scales(kb + 1);
      for (int round = 0; round < rounds && ok; ++round) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g, ++fold) {
          if (!mbar_wait_warp(smem_u32(&bar_acc_full[fold & 1]), (fold >> 1) & 1, abortp, 64)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (any) {
            uint32_t v[2][16];
            tmem_ld_32x32b_x16(taddr + (fold & 1) * BN, v[0]);
#pragma unroll
            for (int i = 0; i < Cfg::NC; i += 16) {
              tmem_ld_wait();
              if (i + 16 < Cfg::NC) tmem_ld_32x32b_x16(taddr + (fold & 1) * BN + i + 16, v[(i / 16 + 1) & 1]);
#pragma unroll
              for (int j = 0; j < 16; j += 2)
                fma2(acc[i + j], acc[i + j + 1], __uint_as_float(v[(i / 16) & 1][j]), __uint_as_float(v[(i / 16) & 1][j + 1]), scale[g]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_acc_free[fold & 1]));
        }
      }
    }
    if (!ok) {
      abort_flag = 1;
      if (lane == 0) atomicCAS(p.status, 0, kErrEpilogueWait);
    }
    if (shares == 1 && ok) {
      const int row = rt * 128 + r;
      if (row < p.rows) {
        const long long base = row * p.c_row + static_cast<long long>(ct * BN + first_col) * p.c_col;
#pragma unroll
        for (int i = 0; i < Cfg::NC; ++i)
          if (first_col + i < cols) {
            const long long at = base + i * p.c_col;
            float v = __fmul_rn(p.alpha, acc[i]);
            if (p.beta != 0.f) v = __fmaf_rn(p.beta, ld_element_as(p.c_type, p.c, at), v);
            st_element_as(p.c_type, p.c, at, v);
          }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, Cfg::TMEM_COLS);
  if constexpr (!Cfg::REBALANCE) {
    if (shares > 1) {
      cluster_sync_all();  // nobody reads operands any more where the partial results go
      const int per = BN / shares;  // columns that a CTA adds up and stores
      if (warp >= 8) {
        const int r = (warp & 3) * 32 + lane, first_col = (warp >= 12 ? Cfg::NC : 0);
#pragma unroll
        for (int i = 0; i < Cfg::NC; ++i) {
          const int col = first_col + i, to = col / per;
          const uint32_t at = smem_base + Cfg::B_OFFSET + ((share * per + col - to * per) * 128 + r) * 4;
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_cta(at, to)), "f"(acc[i]) : "memory");
        }
      }
      // A CTA whose wait ran out has no share: it tells the others, and none of them stores its part of the tile.
      if (static_cast<int>(threadIdx.x) < shares && *abortp) raise_abort_in(&abort_flag, threadIdx.x);
      __syncwarp();
      cluster_sync_all();
      if (warp >= 8 && !*abortp) {
        const int t = threadIdx.x - 256, r = t & 127, row = rt * 128 + r;
        if (row < p.rows) {
          const float* parts = reinterpret_cast<const float*>(smem_gen + Cfg::B_OFFSET) + r;
          for (int i = t >> 7; i < per; i += 2) {
            const int col = share * per + i;
            if (col >= cols) break;
            float v = parts[i * 128];
            for (int s = 1; s < shares; ++s) v += parts[(s * per + i) * 128];
            const long long at = row * p.c_row + static_cast<long long>(ct * BN + col) * p.c_col;
            v = __fmul_rn(p.alpha, v);
            if (p.beta != 0.f) v = __fmaf_rn(p.beta, ld_element_as(p.c_type, p.c, at), v);
            st_element_as(p.c_type, p.c, at, v);
          }
        }
      }
    }
  }
}

}  // namespace tcec_sm100
