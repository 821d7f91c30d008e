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
//
// A block of 128 x 128 codes and 128 columns moves 64 KB through shared memory to the MMAs, 33 of expanded codes and 40 of copies in, and 8 out to the
// converters, 1130 cycles at 128 bytes each, while its MMAs take 520; tiles of 256 x 256 on two SMs do twice as many products with the same (1024 cycles of
// MMAs).  That is not all that bounds the pairs: by counters the 8192 x 4096 x 4096 gradient keeps the tensor pipe busy for half of the time and no other unit for
// longer, 1000 tokens times 4096 x 4096 for a third, so what is left lies between the roles below.  Measured in a row, with the staging: 512 tokens times 4096 x 4096,
// 128 tiles of 32 blocks, 25.2 us (680 TFLOP/s), 1000 tokens on pairs 39.5 (850), 8192 x 4096 x 4096 gradient 308 at the power cap (890; the kernel alone 280).
// Groups of 32 have four accumulators a block to fold, FP32 three times as many: 512 tokens 44 us, FP32 103, in groups of 128 56.
// Few columns: by the codes' way from memory to operands; 8192 x 4096 gradient of rank 48 18.7 us (1.8 TB/s), 64 tokens times 4096 x 4096 12.9.
#pragma once
#include "tcec_codes.cuh"
#include "tcec_codes_launch.h"
#include "tcec_gemm_panels.cuh"
#include "tcec_gemm_roles.cuh"
#include "tcec_stage.cuh"

namespace tcec_sm100 {

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
// (a & b) | c in one instruction; the compiler makes two of it when b and c are both constants.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// Eight 4-bit codes to code - zero point, in order.
template <bool kF16>
__device__ __forceinline__ uint4 q4_expand(uint32_t w, uint32_t zero) {
  constexpr uint32_t mask = 0x000f000fu, magic = kF16 ? 0x64006400u : 0x43004300u;
  return make_uint4(sub16x2(and_or(w, mask, magic), zero, kF16), sub16x2(and_or(w >> 4, mask, magic), zero, kF16),
                    sub16x2(and_or(w >> 8, mask, magic), zero, kF16), sub16x2(and_or(w >> 12, mask, magic), zero, kF16));
}
// Eight 8-bit codes (sign and magnitude) in the bytes 0 2, 1 3 of two words, to operands in order: +-(magic + magnitude) -+ magic.
template <bool kF16>
__device__ __forceinline__ uint4 q8_expand(uint32_t w0, uint32_t w1) {
  constexpr uint32_t kMagic = kF16 ? 0x64006400u : 0x43004300u, kSign = 0x80008000u, kSize = 0x007f007fu;
  const uint32_t a = ((w0 << 8) & kSign) | kMagic, b = (w0 & kSign) | kMagic, c = ((w1 << 8) & kSign) | kMagic, d = (w1 & kSign) | kMagic;
  return make_uint4(sub16x2((w0 & kSize) | a, a, kF16), sub16x2(((w0 >> 8) & kSize) | b, b, kF16), sub16x2((w1 & kSize) | c, c, kF16),
                    sub16x2(((w1 >> 8) & kSize) | d, d, kF16));
}

// ---------------------------------------------------------------- the product
// kSpans: groups of 4-bit codes in a block (1, 2 or 4); 0: 8-bit codes, one group a block.
template <int BN, int kSpans>
struct GemmCodesCfg {
  static constexpr bool Q8 = kSpans == 0;
  static constexpr bool PAIR = BN == 256;                     // 256 x 256 tiles on two SMs
  static constexpr int GROUPS = Q8 ? 1 : kSpans;
  static constexpr int CONVERTERS = 8, FOLDERS = 8;           // warps
  static constexpr int TEAMS = BN == 64 && !Q8 ? 4 : PAIR && kSpans != 1 ? 1 : 2, TEAM = CONVERTERS / TEAMS;  // of converters: each takes a block in turn, with TEAM warps
  static constexpr int THREADS = 32 * (4 + CONVERTERS + FOLDERS);
  static constexpr int CODE_BYTES = Q8 ? kQ8CodeBytes : kQ4CodeBytes;
  static constexpr int BLOCK_BYTES = CODE_BYTES + kEntryBytes * GROUPS;
  // Expanded codes: a chunk of 8 along the sum is 128 rows x 16 bytes, in core matrices of 8 rows; the chunks lie 32 bytes off a
  // multiple of 128, so that lanes with rows g, g + 1 of four chunks write to all banks at once.
  static constexpr int CHUNK_BYTES = 128 * 16 + 32;
  static constexpr int A_BYTES = 16 * CHUNK_BYTES;
  static constexpr int A_STAGES = BN == 64 && !Q8 ? 4 : 3;
  static constexpr int BC = PAIR ? 128 : BN;                  // columns of the dense operand that a CTA brings in
  static constexpr int B_HALF = BC * 128;                     // 64 of the sum, one part
  static constexpr int B_STAGES = (BN == 64 && kSpans < 4) || (PAIR && kSpans == 1) ? 3 : 2;  // of two halves, which are filled and given back one by one
  static constexpr int CODE_STAGES = PAIR ? (kSpans == 1 ? 2 : 3) : Q8 && BN == 128 ? 2 : 4;
  static constexpr int ACCS = BN == 256 ? 2 : 4;              // accumulators
  static constexpr int SCALE_SLOTS = ACCS + A_STAGES + 1;     // blocks; see the converters
  static constexpr int B_OFFSET = 0;
  static constexpr int A_OFFSET = B_STAGES * 2 * B_HALF;
  static constexpr int CODE_OFFSET = A_OFFSET + A_STAGES * A_BYTES;
  static constexpr int SCALE_OFFSET = CODE_OFFSET + CODE_STAGES * BLOCK_BYTES;
  static constexpr int SMEM_BYTES = SCALE_OFFSET + SCALE_SLOTS * GROUPS * 512 + 1024;
  static_assert(TEAMS <= A_STAGES && CODE_STAGES % TEAMS == 0, "a team may not wait for a phase that is two ahead");
  static_assert(SMEM_BYTES <= 232448 - 512, "dynamic + static shared memory exceed an SM");
  static_assert(PAIR || A_OFFSET >= 128 * BN * 4, "partial results go where the dense operand was");
  static constexpr int TMEM_COLS = ACCS * BN;
  static constexpr int NC = BN / 2;                           // columns of a folding thread
  static constexpr int LOAD_COLS = BN == 256 ? 16 : 32;       // of them at a time, twice
  // 640 threads x 96 registers at launch: 128 x 40 + 256 x 32 + 256 x 184 = 60416 of 61440
  static constexpr int REGS_LAUNCH = 96, REGS_CONTROL = 40, REGS_CONVERT = 32, REGS_FOLD = 184;
  static_assert(128 * REGS_CONTROL + 32 * CONVERTERS * REGS_CONVERT + 32 * FOLDERS * REGS_FOLD <= THREADS * REGS_LAUNCH, "register shares");
};

__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float s) {
  asm("{\n\t.reg .b64 d, v, m;\n\t"
      "mov.b64 d, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 m, {%4, %4};\n\t"
      "fma.rn.f32x2 d, v, m, d;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b), "f"(s));
}
__device__ __forceinline__ void tmem_ld_32x32b(uint32_t taddr, uint32_t (&v)[32]) { tmem_ld_32x32b_x32(taddr, v); }
__device__ __forceinline__ void tmem_ld_32x32b(uint32_t taddr, uint32_t (&v)[16]) { tmem_ld_32x32b_x16(taddr, v); }
// What the MMAs of a block wait for, asked for at once: one after the other the answers of barriers that are ready took the issuing thread 100
// to 300 cycles each, more than the MMAs themselves.
__device__ __forceinline__ bool mbar_wait_three(uint32_t a, uint32_t pa, uint32_t b, uint32_t pb, uint32_t c, uint32_t pc, volatile uint32_t* abortp) {
  for (uint32_t i = 0; i < TCEC_WAIT_LIMIT; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred P, Q, R;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 Q, [%3], %4;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 R, [%5], %6;\n\t"
        "and.pred P, P, Q;\n\tand.pred P, P, R;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t}"
        : "=r"(ok)
        : "r"(a), "r"(pa), "r"(b), "r"(pb), "r"(c), "r"(pc)
        : "memory");
    if (__all_sync(0xffffffffu, ok)) return true;
    if ((i & 0x3ff) == 0x3ff && __any_sync(0xffffffffu, *abortp)) return false;
  }
  return false;
}
// All lanes poll: one lane that tells the others costs 10 % (8192 x 4096 x 4096 gradient 268 us, 299 so).
__device__ __forceinline__ bool mbar_wait_lanes(uint32_t bar, uint32_t parity, volatile uint32_t* abortp) {
  bool ok = false;
  for (uint32_t i = 0; !ok && i < TCEC_WAIT_LIMIT; ++i) {
    ok = mbar_try_wait(bar, parity);
    if ((i & 0x3ff) == 0x3ff && *abortp) break;
  }
  return __all_sync(0xffffffffu, ok);
}

// Expands a part of the codes of one block (shared memory) to 16-bit operands: part `index` of kParts, a warp.
template <bool kF16, int kSpans, int kParts>
struct Converter {  // 4 bits: strips of 16 rows, lane 4 g + t has rows g and g + 8
  static __device__ __forceinline__ void expand(const uint8_t* block, uint8_t* out, int index, int lane) {
    constexpr int kChunk = GemmCodesCfg<128, kSpans>::CHUNK_BYTES, kStrips = 8 / kParts, kStripBytes = q4_strip_bytes(128 / kSpans);
    const uint8_t* codes = block + index * kStrips * kStripBytes + lane * 16;
    const uint32_t* entries = reinterpret_cast<const uint32_t*>(block + index * kStrips * kStripBytes + kStripCodeBytes) + (lane >> 2);
    uint8_t* to = out + (lane & 3) * kChunk + index * kStrips * 256 + (lane >> 2) * 16;
#pragma unroll 1
    for (int s = 0; s < kStrips; ++s) {
      const uint4 w[2] = {*reinterpret_cast<const uint4*>(codes + s * kStripBytes), *reinterpret_cast<const uint4*>(codes + s * kStripBytes + 512)};
#pragma unroll
      for (int q = 0; q < kSpans; ++q) {
        const uint32_t zero0 = q4_zero<kF16>(entries[s * (kStripBytes / 4) + q * 16] & 15u);
        const uint32_t zero1 = q4_zero<kF16>(entries[s * (kStripBytes / 4) + q * 16 + 8] & 15u);
#pragma unroll
        for (int panel = q * 4 / kSpans; panel < (q + 1) * 4 / kSpans; ++panel) {
          const uint4 pair = w[panel >> 1];
          uint8_t* at = to + panel * 4 * kChunk + s * 256;
          *reinterpret_cast<uint4*>(at) = q4_expand<kF16>(panel & 1 ? pair.z : pair.x, zero0);
          *reinterpret_cast<uint4*>(at + 128) = q4_expand<kF16>(panel & 1 ? pair.w : pair.y, zero1);
        }
      }
    }
  }
};
template <bool kF16, int kParts>
struct Converter<kF16, 0, kParts> {  // 8 bits: 32 rows at a time, a lane each; of eight warps two share them, half of the sum each
  static __device__ __forceinline__ void expand(const uint8_t* block, uint8_t* out, int index, int lane) {
    constexpr int kChunk = GemmCodesCfg<128, 0>::CHUNK_BYTES;
#pragma unroll
    for (int r = 0; r < (kParts < 4 ? 4 / kParts : 1); ++r) {
      const int rows = kParts < 4 ? index * (4 / kParts) + r : index & 3, half = kParts == 8 ? index >> 2 : 0;
      const int at = (rows * 32 + lane) * 16;  // of this row, among 16 tokens of codes and among 8 of operands
#pragma unroll 1
      for (int c = half * 4; c < half * 4 + (kParts == 8 ? 4 : 8); c += 2) {
        const uint4 v = *reinterpret_cast<const uint4*>(block + c * 2048 + at), w = *reinterpret_cast<const uint4*>(block + (c + 1) * 2048 + at);
        *reinterpret_cast<uint4*>(out + (2 * c) * kChunk + at) = q8_expand<kF16>(v.x, v.y);
        *reinterpret_cast<uint4*>(out + (2 * c + 1) * kChunk + at) = q8_expand<kF16>(v.z, v.w);
        *reinterpret_cast<uint4*>(out + (2 * c + 2) * kChunk + at) = q8_expand<kF16>(w.x, w.y);
        *reinterpret_cast<uint4*>(out + (2 * c + 3) * kChunk + at) = q8_expand<kF16>(w.z, w.w);
      }
    }
  }
};

// Columns of one row of C, `step` bytes apart: alpha * acc + beta * C.  Each of these loops is gone through once a tile, and what it costs is to fetch
// its instructions (element by element with the type, the stride and beta looked at each time, a tile of 64 columns took 1.7 us to store), so
// the common one is kept short.
template <int kType, int N>
__device__ __forceinline__ void store_columns(const float (&acc)[N], uint8_t* at, long long step, int cols, float alpha, float beta) {
  typedef typename Element<kType>::type T;
  if (beta == 0.f && cols >= N) {
#pragma unroll
    for (int i = 0; i < N; ++i, at += step) *reinterpret_cast<T*>(at) = Element<kType>::put(__fmul_rn(alpha, acc[i]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i, at += step)
      if (i < cols) {
        float v = __fmul_rn(alpha, acc[i]);
        if (beta != 0.f) v = __fmaf_rn(beta, Element<kType>::get(*reinterpret_cast<T*>(at)), v);
        *reinterpret_cast<T*>(at) = Element<kType>::put(v);
      }
  }
}
template <int N>
__device__ __forceinline__ void store_columns_as(const GemmCodesParams& p, const float (&acc)[N], long long row, long long col, int cols) {
  const int size = p.c_type == kTypeF32 ? 4 : 2;
  uint8_t* const at = static_cast<uint8_t*>(p.c) + (row * p.c_row + col * p.c_col) * size;
  if (p.c_type == kTypeF32) store_columns<kTypeF32>(acc, at, p.c_col * size, cols, p.alpha, p.beta);
  else if (p.c_type == kTypeF16) store_columns<kTypeF16>(acc, at, p.c_col * size, cols, p.alpha, p.beta);
  else store_columns<kTypeBf16>(acc, at, p.c_col * size, cols, p.alpha, p.beta);
}

// Which rows and columns a tile is.  Sixteen rows of tiles at a time go through all columns: what is on at a time shares its operands.
struct CodeTile {
  int row, col;
};
__device__ __forceinline__ CodeTile code_tile(int tile, int rows, int cols) {
  const int width = 16 * cols, group = tile / width, in = tile - group * width, size = min(16, rows - group * 16);
  return {group * 16 + in % size, in / size};
}

// A cluster works on a tile at a time.
//   BN = 64, 128: tiles of 128 x BN, clusters of 1, 2, 4 or 8 CTAs, which divide the sum and add up through shared memory, in its order.
//   BN = 256: tiles of 256 x 256 on CTA pairs (tcgen05 cta_group::2), each with its 128 rows of codes and half of the columns of the dense
//   operand; the leader issues the MMAs of both.  The peer's operands are announced to the leader by a relay thread.
template <int BN, bool kF16, int kSpans>
__global__ void __launch_bounds__(GemmCodesCfg<BN, kSpans>::THREADS, 1) tcec_gemm_codes_kernel(const GemmCodesParams p) {
  using Cfg = GemmCodesCfg<BN, kSpans>;
  constexpr int kGroups = Cfg::GROUPS;
  constexpr bool kPair = Cfg::PAIR;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_code_full[Cfg::CODE_STAGES], bar_code_empty[Cfg::CODE_STAGES];
  __shared__ uint64_t bar_a_full[Cfg::A_STAGES], bar_a_empty[Cfg::A_STAGES];
  __shared__ uint64_t bar_b_full[Cfg::B_STAGES], bar_b_empty[2 * Cfg::B_STAGES];
  __shared__ uint64_t bar_acc_full[Cfg::ACCS], bar_acc_free[Cfg::ACCS], bar_drain[1];
  __shared__ uint32_t tmem_base_s;
  __shared__ uint32_t abort_flag;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int ctas = kPair ? 2 : static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  const bool leader = !kPair || rank == 0;
  const int shares = kPair ? 1 : ctas;  // of the sum
  const int first_tile = blockIdx.x / ctas, stride = gridDim.x / ctas;
  const int tile_rows = kPair ? (p.row_tiles + 1) / 2 : p.row_tiles, ntiles = tile_rows * p.col_tiles;
  const int kb_first = kPair ? 0 : static_cast<int>(static_cast<long long>(p.blocks) * rank / shares);
  const int kb_end = kPair ? p.blocks : static_cast<int>(static_cast<long long>(p.blocks) * (rank + 1) / shares);
  const int nkb = kb_end - kb_first;
  auto row_tile = [&](const CodeTile& t) { return kPair ? t.row * 2 + rank : t.row; };

  if (warp == 0) {  // a barrier or two a lane
    if (lane < Cfg::CODE_STAGES) {
      mbar_init(smem_u32(&bar_code_full[lane]), 1);
      mbar_init(smem_u32(&bar_code_empty[lane]), Cfg::TEAM);
    } else if (lane >= 8 && lane < 8 + Cfg::A_STAGES) {
      mbar_init(smem_u32(&bar_a_full[lane - 8]), Cfg::TEAM + (kPair && leader));  // in a leader the peer's relay too
      mbar_init(smem_u32(&bar_a_empty[lane - 8]), 1);
    } else if (lane >= 16 && lane < 16 + Cfg::B_STAGES) {
      mbar_init(smem_u32(&bar_b_full[lane - 16]), 2 + (kPair && leader));
      mbar_init(smem_u32(&bar_b_empty[2 * (lane - 16)]), 1);
      mbar_init(smem_u32(&bar_b_empty[2 * (lane - 16) + 1]), 1);
    } else if (lane >= 24 && lane < 24 + Cfg::ACCS) {
      mbar_init(smem_u32(&bar_acc_full[lane - 24]), 1);
      mbar_init(smem_u32(&bar_acc_free[lane - 24]), (kPair ? 2 : 1) * Cfg::FOLDERS);  // of a pair the leader's is used
    } else if (lane == 31) {
      mbar_init(smem_u32(&bar_drain[0]), 1);
      abort_flag = 0;
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_pair(smem_u32(&tmem_base_s), Cfg::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(&tmem_base_s), Cfg::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (ctas > 1) cluster_sync_all();  // the others' barriers and shared memory exist before anything is written to them
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  volatile uint32_t* abortp = &abort_flag;
  // Only what touches the dense operand or C waits for the kernel before, which stages the dense operand: that was through its own wait when
  // this one could start, so whatever the codes come from has ended, and they are fetched and expanded meanwhile.
  auto give_up = [&](int code) {
    if constexpr (kPair) raise_abort_pair(&abort_flag);
    else abort_flag = 1;
    atomicCAS(p.status, 0, code);
  };

  if (warp < 4) {
    setmaxnreg_dec<Cfg::REGS_CONTROL>();
    if (warp == 0) {
      // ---------------------------------------------------------- copies of the dense operand
      wait_for_launch_before();
      if (elect_one()) {
        uint32_t half = 0, ph = 0, armed = 0, armed_parity = 0;  // halves of stages
        bool ok = true;
        for (int tile = first_tile; tile < ntiles && ok; tile += stride) {
          const CodeTile ti = code_tile(tile, tile_rows, p.col_tiles);
          const int col = ti.col * BN + (kPair ? rank * 128 : 0);
          const uint32_t bytes = max(0, min(Cfg::BC, (p.cols - col + 15) & ~15)) * 64;  // a pair's second half may have no columns
          const uint8_t* src = after_wait(p.panels) + (static_cast<size_t>(col >> 7) * p.blocks + kb_first) * p.parts * kSpanBytes + (col & 127) * 64;
          for (int left = nkb * p.parts * 2; left > 0; --left) {  // a half of a block and part
            if (!mbar_wait(smem_u32(&bar_b_empty[half]), ph ^ 1, abortp)) {
              ok = false;
              break;
            }
            const uint32_t full = smem_u32(&bar_b_full[half >> 1]);
            if (bytes) {
              mbar_arrive_expect_tx(full, 2 * bytes);
              armed |= 1u << half;
              armed_parity = (armed_parity & ~(1u << half)) | (ph << half);
              const uint32_t dst = smem_base + Cfg::B_OFFSET + half * Cfg::B_HALF;
              bulk_load(dst, src, bytes, full);
              bulk_load(dst + Cfg::BC * 64, src + kPanelBytes, bytes, full);
            } else {
              mbar_arrive(full);
            }
            src += 2 * kPanelBytes;
            if (++half == 2 * Cfg::B_STAGES) half = 0, ph ^= 1;
          }
        }
        if (!ok) {
          give_up(kErrProducerWait);
          // This thread's own copies land before the CTA gives up its shared memory.  A stage of which only the first half was asked for
          // does not become full: its second half is arrived for.
          if (half & 1) mbar_arrive(smem_u32(&bar_b_full[half >> 1]));
          for (uint32_t q = 0; q < 2 * Cfg::B_STAGES; ++q)
            if (armed & (1u << q)) mbar_wait_plain(smem_u32(&bar_b_full[q >> 1]), (armed_parity >> q) & 1);
        }
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------- copies of the codes
      if (elect_one()) {
        uint32_t cs = 0, cph = 0, armed = 0, armed_parity = 0;
        bool ok = true;
        for (int tile = first_tile; tile < ntiles && ok; tile += stride) {
          const int rt = min(row_tile(code_tile(tile, tile_rows, p.col_tiles)), p.row_tiles - 1);  // the last pair may have one row of tiles
          const uint8_t* src = p.codes + (static_cast<size_t>(rt) * p.blocks + kb_first) * Cfg::BLOCK_BYTES;
          for (int kb = 0; kb < nkb; ++kb, src += Cfg::BLOCK_BYTES) {
            if (!mbar_wait(smem_u32(&bar_code_empty[cs]), cph ^ 1, abortp)) {
              ok = false;
              break;
            }
            const uint32_t full = smem_u32(&bar_code_full[cs]);
            if (!(dev_flag(p.debug_flags, 128) && static_cast<int>(blockIdx.x) == ctas - 1 && kb == nkb / 2)) {
              mbar_arrive_expect_tx(full, Cfg::BLOCK_BYTES);
              armed |= 1u << cs;
              armed_parity = (armed_parity & ~(1u << cs)) | (cph << cs);
              bulk_load(smem_base + Cfg::CODE_OFFSET + cs * Cfg::BLOCK_BYTES, src, Cfg::BLOCK_BYTES, full);
            }
            if (++cs == Cfg::CODE_STAGES) cs = 0, cph ^= 1;
          }
        }
        if (!ok) {
          give_up(kErrProducerWait);
          for (uint32_t q = 0; q < Cfg::CODE_STAGES; ++q)
            if (armed & (1u << q)) mbar_wait_plain(smem_u32(&bar_code_full[q]), (armed_parity >> q) & 1);
        }
      }
    } else if (warp == 1) {
      const bool one = elect_one();  // which issues; all lanes go along, so that what it needs is the warp's
      uint32_t as = 0, aph = 0, bs = 0, bph = 0;
      bool ok = true;
      if (!leader && one) {
        // -------------------------------------------------------- peer: "my operands are there"
        for (int tile = first_tile; tile < ntiles && ok; tile += stride)
          for (int kb = 0; kb < nkb && ok; ++kb) {
            if (!mbar_wait(smem_u32(&bar_a_full[as]), aph, abortp, 0)) {
              ok = false;
              break;
            }
            mbar_arrive_cluster(map_to_cta(smem_u32(&bar_a_full[as]), 0));
            if (++as == Cfg::A_STAGES) as = 0, aph ^= 1;
            for (int part = 0; part < p.parts; ++part) {
              if (!mbar_wait(smem_u32(&bar_b_full[bs]), bph, abortp, 0)) {
                ok = false;
                break;
              }
              mbar_arrive_cluster(map_to_cta(smem_u32(&bar_b_full[bs]), 0));
              if (++bs == Cfg::B_STAGES) bs = 0, bph ^= 1;
            }
          }
        if (!ok) give_up(kErrMmaWait);
      } else if (leader) {
        // -------------------------------------------------------- MMAs
        const uint64_t a_const = umma_desc_kmajor_noswizzle(0, Cfg::CHUNK_BYTES, 128), b_const = umma_desc_kmajor_noswizzle(0, 128, 512);
        const uint32_t a16 = ((smem_base + Cfg::A_OFFSET) & 0x3ffff) >> 4, b16 = ((smem_base + Cfg::B_OFFSET) & 0x3ffff) >> 4;
        uint32_t x = 0, xph = 0;  // the accumulator, and how often they all have been used
        auto commit = [&](uint64_t* bar) {
          if (!one) return;
          if constexpr (kPair) umma_commit_pair(smem_u32(bar));
          else umma_commit(smem_u32(bar));
        };
        for (int tile = first_tile; tile < ntiles && ok; tile += stride) {
          const int cols = p.cols - code_tile(tile, tile_rows, p.col_tiles).col * BN;
          const uint32_t idesc = umma_idesc(kF16 ? 0u : 1u, kPair ? 256 : 128, kPair ? 256 : min(BN, (cols + 15) & ~15));
          for (int kb = 0; kb < nkb && ok; ++kb) {
            const uint32_t a_here = a16 + as * (Cfg::A_BYTES >> 4);
            for (int part = 0; part < p.parts; ++part) {
              // the codes (waited for before), the dense operand, and the first accumulator if a new one begins
              const uint32_t bfull = smem_u32(&bar_b_full[bs]);
              const bool begins = kGroups > 1 || part == 0;
              if (!mbar_wait_three(smem_u32(&bar_a_full[as]), aph, bfull, bph, begins ? smem_u32(&bar_acc_free[x]) : bfull,
                                   begins ? xph ^ 1 : bph, abortp)) {
                ok = false;
                break;
              }
              tc_fence_after();
              // Short loops: the issuing thread shares its instruction cache with four warps that are busy elsewhere, and unrolled what it
              // does for a block took longer than the MMAs.
              uint32_t da = a_here, db = b16 + bs * (2 * Cfg::B_HALF >> 4);
              uint32_t more = kGroups == 1 && part > 0;  // an accumulator holds one group; where a block is one, all parts of it
#pragma unroll 1
              for (int h = 0; h < 2; ++h) {
#pragma unroll 1
                for (int j = 0; j < 2; ++j) {  // 32 of the sum
                  if (kGroups == 4 && h + j > 0 || kGroups == 2 && h > 0 && j == 0) {
                    if (!mbar_wait_lanes(smem_u32(&bar_acc_free[x]), xph ^ 1, abortp)) {
                      ok = false;
                      break;
                    }
                    tc_fence_after();
                    more = 0;
                  }
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
                    if (one) {
                      if constexpr (kPair) umma_ss_pair<false>(tmem + x * BN, a_const | da, b_const | (db + i * 16), idesc, more);
                      else umma_ss<false>(tmem + x * BN, a_const | da, b_const | (db + i * 16), idesc, more);
                    }
                    da += 2 * Cfg::CHUNK_BYTES >> 4;
                    more = 1;
                  }
                  db += Cfg::BC * 64 >> 4;
                  if (kGroups == 4 || kGroups == 2 && j == 1) {
                    commit(&bar_acc_full[x]);
                    if (++x == Cfg::ACCS) x = 0, xph ^= 1;
                  }
                }
                if (!ok) break;
                if (h == 0) commit(&bar_b_empty[2 * bs]);
              }
              if (!ok) break;
              commit(&bar_b_empty[2 * bs + 1]);
              if (++bs == Cfg::B_STAGES) bs = 0, bph ^= 1;
            }
            if (!ok) break;
            if (kGroups == 1) {
              commit(&bar_acc_full[x]);
              if (++x == Cfg::ACCS) x = 0, xph ^= 1;
            }
            commit(&bar_a_empty[as]);
            if (++as == Cfg::A_STAGES) as = 0, aph ^= 1;
          }
        }
        if (!ok && one) mma_thread_gave_up<kPair>(&abort_flag, p.status, kErrMmaWait, &bar_drain[0]);
      }
    }
  } else if (warp < 4 + Cfg::CONVERTERS) {
    // ------------------------------------------------------------ codes to operands
    setmaxnreg_dec<Cfg::REGS_CONVERT>();
    // The teams take the blocks in turn, so that one waits and passes its block on while another expands.  A team that waits for a phase must
    // know that the one before is over, as the next but one has the same parity.  A stage of codes is always the same team's, and of the stages of
    // operands, whose MMAs come in order, there are no fewer than teams.
    const int team = (warp - 4) / Cfg::TEAM, index = (warp - 4) % Cfg::TEAM;
    const int total = first_tile < ntiles ? ((ntiles - first_tile + stride - 1) / stride) * nkb : 0;  // blocks, of all tiles
    uint32_t cs = team, cph = 0, as = team, aph = 0, slot = team;
    bool ok = true;
    for (int i = team; i < total; i += Cfg::TEAMS) {
      if (!mbar_wait_lanes(smem_u32(&bar_code_full[cs]), cph, abortp) || !mbar_wait_lanes(smem_u32(&bar_a_empty[as]), aph ^ 1, abortp)) {
        ok = false;
        break;
      }
      const uint8_t* block = smem_gen + Cfg::CODE_OFFSET + cs * Cfg::BLOCK_BYTES;
      // The scales, for those who come to them when the products are made.  The stage just waited for says that the MMAs of A_STAGES
      // blocks before are done, for which all but the last ACCS accumulators had been folded: a slot is written again later than that.
      float* scales = reinterpret_cast<float*>(smem_gen + Cfg::SCALE_OFFSET) + slot * (kGroups * 128);
#pragma unroll
      for (int t = index * 32 + lane; t < 128; t += Cfg::TEAM * 32)
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
          if constexpr (Cfg::Q8) scales[t] = reinterpret_cast<const float*>(block + Cfg::CODE_BYTES)[t];
          else scales[g * 128 + t] = __uint_as_float(reinterpret_cast<const uint32_t*>(block)[q4_entry_word<128 / (Cfg::Q8 ? 1 : kSpans)>(t, g)] & ~15u);
      Converter<kF16, kSpans, Cfg::TEAM>::expand(block, smem_gen + Cfg::A_OFFSET + as * Cfg::A_BYTES, index, lane);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&bar_a_full[as]));
        mbar_arrive(smem_u32(&bar_code_empty[cs]));
      }
      if ((cs += Cfg::TEAMS) >= Cfg::CODE_STAGES) cs -= Cfg::CODE_STAGES, cph ^= 1;
      if ((as += Cfg::TEAMS) >= Cfg::A_STAGES) as -= Cfg::A_STAGES, aph ^= 1;
      if ((slot += Cfg::TEAMS) >= Cfg::SCALE_SLOTS) slot -= Cfg::SCALE_SLOTS;
    }
    if (!ok && lane == 0) give_up(kErrOperandWait);
  } else {
    // ------------------------------------------------------------ scales
    setmaxnreg_inc<Cfg::REGS_FOLD>();
    wait_for_launch_before();
    const int fw = warp - 4 - Cfg::CONVERTERS, q = warp & 3, r = q * 32 + lane, first_col = fw >= 4 ? Cfg::NC : 0;
    const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + first_col;
    const float* scales = reinterpret_cast<const float*>(smem_gen + Cfg::SCALE_OFFSET) + r;
    const int rounds = kGroups > 1 ? p.parts : 1;  // of the groups of a block
    uint32_t x = 0, xph = 0, slot = 0;
    bool ok = true;
    float acc[Cfg::NC];
    for (int tile = first_tile; tile < ntiles && ok; tile += stride) {
      const CodeTile ti = code_tile(tile, tile_rows, p.col_tiles);
      const int col0 = ti.col * BN + first_col, cols = p.cols - col0;  // from this warp's first column on
#pragma unroll
      for (int i = 0; i < Cfg::NC; ++i) acc[i] = 0.f;
      for (int kb = 0; kb < nkb && ok; ++kb) {
        for (int round = 0; round < rounds && ok; ++round) {
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            if (!mbar_wait_lanes(smem_u32(&bar_acc_full[x]), xph, abortp)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const float s = scales[(slot * kGroups + g) * 128];
            const uint32_t from = taddr + x * BN;
            constexpr int kAtOnce = Cfg::LOAD_COLS;
            uint32_t v[2][kAtOnce];
            tmem_ld_32x32b(from, v[0]);
#pragma unroll
            for (int i = 0; i < Cfg::NC; i += kAtOnce) {
              tmem_ld_wait();
              if (i + kAtOnce < Cfg::NC) {
                tmem_ld_32x32b(from + i + kAtOnce, v[(i / kAtOnce + 1) & 1]);
              } else {  // all of it is in registers: the next products may go there
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                  if constexpr (kPair) mbar_arrive_cluster(map_to_cta(smem_u32(&bar_acc_free[x]), 0));
                  else mbar_arrive(smem_u32(&bar_acc_free[x]));
                }
              }
#pragma unroll
              for (int j = 0; j < kAtOnce; j += 2)
                fma2(acc[i + j], acc[i + j + 1], __uint_as_float(v[(i / kAtOnce) & 1][j]), __uint_as_float(v[(i / kAtOnce) & 1][j + 1]), s);
            }
            if (++x == Cfg::ACCS) x = 0, xph ^= 1;
          }
        }
        if (++slot == Cfg::SCALE_SLOTS) slot = 0;
      }
      const int row = row_tile(ti) * 128 + r;
      if (shares == 1 && ok && row < p.rows && cols > 0) store_columns_as(p, acc, row, col0, cols);
    }
    if (!ok && lane == 0) give_up(kErrEpilogueWait);
    if constexpr (!kPair) {
      if (shares > 1) {  // then a cluster has one tile
        cluster_sync_all();  // nobody reads operands any more where the partial results go
        const CodeTile ti = code_tile(first_tile, tile_rows, p.col_tiles);
        // The columns go to the CTAs in turn, four at a time: what a CTA adds up is the fours rank, rank + shares, ...
        const uint32_t mine = smem_base + Cfg::B_OFFSET + r * 16;
#pragma unroll
        for (int i = 0; i < Cfg::NC / 4; ++i) {
          const uint32_t four = (first_col >> 2) + i;
          const uint32_t at = mine + (rank * (BN / 4 / shares) + four / shares) * 2048;
          st_cluster_v4(map_to_cta(at, four & (shares - 1)), acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
        }
        cluster_sync_all();
        const int row = ti.row * 128 + r;
        if (row < p.rows && !*abortp) {
          const uint32_t fours = BN / 4 / shares;
#pragma unroll 1
          for (uint32_t f = fw >> 2; f < fours; f += 2) {
            const int col = ti.col * BN + (f * shares + rank) * 4;
            if (col >= p.cols) break;
            float4 v[8];
#pragma unroll
            for (int s = 0; s < 8; ++s)
              if (s < shares) v[s] = ld_shared_v4(mine + (s * fours + f) * 2048);
            float sum[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
            for (int s = 1; s < 8; ++s)
              if (s < shares) sum[0] += v[s].x, sum[1] += v[s].y, sum[2] += v[s].z, sum[3] += v[s].w;
            store_columns_as(p, sum, row, col, p.cols - col);
          }
        }
      }
    }
  }

  // (The warps that gave registers away come here too: next to nothing is done.)
  if constexpr (!kPair) {
    if (shares > 1 && warp < 4 + Cfg::CONVERTERS) {
      __syncwarp();
      cluster_sync_all();
      // A CTA whose wait ran out has no share: it tells the others, and none of them stores its part of the tile.
      if (static_cast<int>(threadIdx.x) < shares && *abortp) raise_abort_in(&abort_flag, threadIdx.x);
      __syncwarp();
      cluster_sync_all();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) {
    cluster_sync_all();  // neither CTA leaves while the other may still signal it or read its operands
    if (warp == 1) tmem_dealloc_pair(tmem, Cfg::TMEM_COLS);
  } else {
    if (warp == 1) tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
}

}  // namespace tcec_sm100
