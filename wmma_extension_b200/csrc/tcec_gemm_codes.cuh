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

// Eight FP32 values to an item of each part; the small parts first, so that the accumulator, which truncates, cuts off less.
template <class Put>
__device__ __forceinline__ void put_split(const Put& put, int it, const float (&v)[8], bool none) {
  uint32_t part[3][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) split3_bf16(none ? 0.f : v[2 * j], none ? 0.f : v[2 * j + 1], part[0][j], part[1][j], part[2][j]);
#pragma unroll
  for (int q = 0; q < 3; ++q) put(it, q, make_uint4(part[2 - q][0], part[2 - q][1], part[2 - q][2], part[2 - q][3]));
}

// One CTA a block of 128 columns x 128 of the sum; an item is 16 bytes of a panel, eight consecutive values of one column.  Addresses stay
// among the elements that exist, so that all loads of some items go out before the first is waited for.
template <int kType>
__global__ void __launch_bounds__(256) stage_panels_kernel(const StagePanelsParams p) {
  constexpr int kParts = kType == kTypeF32 ? 3 : 1;
  wait_for_launch_before();
  const int kb = blockIdx.x % p.blocks, cb = blockIdx.x / p.blocks;
  uint8_t* out = p.panels + static_cast<size_t>(blockIdx.x) * kParts * kSpanBytes;
  const int cols = min(kCodeRows, (p.cols - cb * kCodeRows + 15) & ~15);  // columns that an MMA may read
  const int first = threadIdx.x;
  // Item `it` of a thread: column r, chunk c of panel it / 2.
  const bool along = p.sum_step == 1;
  const int r0 = along ? (first & 7) + ((first >> 5) & 7) * 8 : first & 127;   // a warp: 8 columns x 64 bytes, or 32 columns
  const int c0 = along ? (first >> 3) & 3 : first >> 7;
  auto column = [&](int it) { return along ? r0 + (it & 1) * 64 : r0; };
  auto chunk = [&](int it) { return along ? c0 : c0 + (it & 1) * 2; };
  auto put = [&](int it, int part, const uint4& v) {
    const int r = column(it);
    if (r < cols)
      *reinterpret_cast<uint4*>(out + part * kSpanBytes + (it >> 1) * kPanelBytes + (r >> 3) * 512 + chunk(it) * 128 + (r & 7) * 16) = v;
  };
  constexpr int kAtOnce = kType == kTypeF32 ? 2 : 4;  // items whose loads are under way together
  const int cols_here = p.cols - cb * kCodeRows, sum_here = p.sum - kb * kCodeSpan;
  const long long origin = static_cast<long long>(cb) * kCodeRows * p.col_step + static_cast<long long>(kb) * kCodeSpan * p.sum_step;
#pragma unroll 1
  for (int it0 = 0; it0 < 8; it0 += kAtOnce) {
    if (p.vec && sum_here >= kCodeSpan) {
      uint4 raw[kAtOnce][kType == kTypeF32 ? 2 : 1];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int it = it0 + i;
        const long long at = origin + min(column(it), cols_here - 1) * p.col_step + (it >> 1) * 32 + chunk(it) * 8;
        if constexpr (kType == kTypeF32) {
          raw[i][0] = ld_operand128(static_cast<const float*>(p.src) + at);
          raw[i][1] = ld_operand128(static_cast<const float*>(p.src) + at + 4);
        } else {
          raw[i][0] = ld_operand128(static_cast<const uint16_t*>(p.src) + at);
        }
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const bool none = column(it0 + i) >= cols_here;
        if constexpr (kType == kTypeF32) {
          const float v[8] = {__uint_as_float(raw[i][0].x), __uint_as_float(raw[i][0].y), __uint_as_float(raw[i][0].z), __uint_as_float(raw[i][0].w),
                              __uint_as_float(raw[i][1].x), __uint_as_float(raw[i][1].y), __uint_as_float(raw[i][1].z), __uint_as_float(raw[i][1].w)};
          put_split(put, it0 + i, v, none);
        } else {
          put(it0 + i, 0, none ? make_uint4(0, 0, 0, 0) : raw[i][0]);
        }
      }
    } else {
      typename std::conditional<kType == kTypeF32, float, uint32_t>::type w[kAtOnce][8];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int it = it0 + i, at_sum = (it >> 1) * 32 + chunk(it) * 8 + j;
          const long long at = origin + min(column(it), cols_here - 1) * p.col_step + min(at_sum, sum_here - 1) * p.sum_step;
          if constexpr (kType == kTypeF32) w[i][j] = ld_operand(static_cast<const float*>(p.src) + at);
          else w[i][j] = ld_operand16(static_cast<const uint16_t*>(p.src) + at);
        }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int it = it0 + i, at_sum = (it >> 1) * 32 + chunk(it) * 8;
        const bool none = column(it) >= cols_here;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (none || at_sum + j >= sum_here) w[i][j] = 0;
        if constexpr (kType == kTypeF32) put_split(put, it, w[i], false);
        else put(it, 0, make_uint4(w[i][0] | w[i][1] << 16, w[i][2] | w[i][3] << 16, w[i][4] | w[i][5] << 16, w[i][6] | w[i][7] << 16));
      }
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
// Eight 8-bit codes (sign and magnitude) in the bytes 0 2, 1 3 of two words, to operands in order: +-(magic + magnitude) -+ magic.
template <bool kF16>
__device__ __forceinline__ uint4 q8_expand(uint32_t w0, uint32_t w1) {
  constexpr uint32_t kMagic = kF16 ? 0x64006400u : 0x43004300u, kSign = 0x80008000u, kSize = 0x007f007fu;
  const uint32_t a = ((w0 << 8) & kSign) | kMagic, b = (w0 & kSign) | kMagic, c = ((w1 << 8) & kSign) | kMagic, d = (w1 & kSign) | kMagic;
  return make_uint4(sub16x2((w0 & kSize) | a, a, kF16), sub16x2(((w0 >> 8) & kSize) | b, b, kF16), sub16x2((w1 & kSize) | c, c, kF16),
                    sub16x2(((w1 >> 8) & kSize) | d, d, kF16));
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
  static constexpr bool PAIR = BN == 256;                     // 256 x 256 tiles on two SMs
  static constexpr int GROUPS = Q8 ? 1 : kSpans;
  static constexpr int THREADS = 512;
  static constexpr int CODE_BYTES = Q8 ? kQ8CodeBytes : kQ4CodeBytes;
  static constexpr int BLOCK_BYTES = CODE_BYTES + kEntryBytes * GROUPS;
  // Expanded codes: a chunk of 8 along the sum is 128 rows x 16 bytes, in core matrices of 8 rows; the chunks lie 32 bytes off a
  // multiple of 128, so that lanes with rows g, g + 1 of four chunks write to all banks at once.
  static constexpr int CHUNK_BYTES = 128 * 16 + 32;
  static constexpr int A_BYTES = 16 * CHUNK_BYTES;
  static constexpr int A_STAGES = 3;
  static constexpr int BC = PAIR ? 128 : BN;                  // columns of the dense operand that a CTA brings in
  static constexpr int B_BYTES = BC * 128;                    // 64 of the sum, one part
  static constexpr int B_STAGES = BN == 64 ? 6 : 4;
  static constexpr int CODE_STAGES = 3;
  static constexpr int SCALE_SLOTS = 6;                       // blocks; see the converters
  static constexpr int B_OFFSET = 0;
  static constexpr int A_OFFSET = B_STAGES * B_BYTES;
  static constexpr int CODE_OFFSET = A_OFFSET + A_STAGES * A_BYTES;
  static constexpr int SCALE_OFFSET = CODE_OFFSET + CODE_STAGES * BLOCK_BYTES;
  static constexpr int SMEM_BYTES = SCALE_OFFSET + SCALE_SLOTS * GROUPS * 512 + 1024;
  static_assert(SMEM_BYTES <= 232448 - 512, "dynamic + static shared memory exceed an SM");
  static_assert(PAIR || B_STAGES * B_BYTES >= 128 * BN * 4, "partial results go where the dense operand was");
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int NC = BN / 2;                           // columns of an epilogue thread
  static constexpr int LOAD_COLS = PAIR ? 16 : 32;            // of them at a time, twice
  // 512 threads x 128 registers at launch: 128 x (40 + 56) + 2 x 128 x 208 = 65536
  static constexpr bool REBALANCE = PAIR;
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
// All lanes poll, which they notice sooner than one lane that tells the others.
__device__ __forceinline__ bool mbar_wait_lanes(uint32_t bar, uint32_t parity, volatile uint32_t* abortp) {
  const bool ok = mbar_wait(bar, parity, abortp, 0);
  return __all_sync(0xffffffffu, ok);
}

// Expands the codes of one block (shared memory) to 16-bit operands and hands its scales on.
template <bool kF16, int kSpans>
struct Converter {  // 4 bits: two strips of 16 rows a warp, lane 4 g + t has rows g and g + 8 of both
  static __device__ __forceinline__ void expand(const uint8_t* block, uint8_t* out, int warp, int lane) {
    constexpr int kChunk = GemmCodesCfg<128, kSpans>::CHUNK_BYTES;
    const uint8_t* codes = block + warp * 2048 + lane * 16;
    const uint32_t* entries = reinterpret_cast<const uint32_t*>(block + kQ4CodeBytes) + warp * 32 + (lane >> 2);
    uint8_t* to = out + (lane & 3) * kChunk + warp * 512 + (lane >> 2) * 16;
    uint4 w[2][2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) w[s][h] = *reinterpret_cast<const uint4*>(codes + s * 1024 + h * 512);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int q = 0; q < kSpans; ++q) {
        const uint32_t zero0 = q4_zero<kF16>(entries[q * 128 + s * 16] & 15u), zero1 = q4_zero<kF16>(entries[q * 128 + s * 16 + 8] & 15u);
#pragma unroll
        for (int panel = q * 4 / kSpans; panel < (q + 1) * 4 / kSpans; ++panel) {
          const uint4 pair = w[s][panel >> 1];
          uint8_t* at = to + panel * 4 * kChunk + s * 256;
          *reinterpret_cast<uint4*>(at) = q4_expand<kF16>(panel & 1 ? pair.z : pair.x, zero0);
          *reinterpret_cast<uint4*>(at + 128) = q4_expand<kF16>(panel & 1 ? pair.w : pair.y, zero1);
        }
      }
  }
};
template <bool kF16>
struct Converter<kF16, 0> {  // 8 bits: a lane a row
  static __device__ __forceinline__ void expand(const uint8_t* block, uint8_t* out, int warp, int lane) {
    constexpr int kChunk = GemmCodesCfg<128, 0>::CHUNK_BYTES;
    const int at = (warp * 32 + lane) * 16;  // of this row, among 16 tokens of codes and among 8 of operands
#pragma unroll
    for (int c = 0; c < 8; c += 2) {
      const uint4 v = *reinterpret_cast<const uint4*>(block + c * 2048 + at), w = *reinterpret_cast<const uint4*>(block + (c + 1) * 2048 + at);
      *reinterpret_cast<uint4*>(out + (2 * c) * kChunk + at) = q8_expand<kF16>(v.x, v.y);
      *reinterpret_cast<uint4*>(out + (2 * c + 1) * kChunk + at) = q8_expand<kF16>(v.z, v.w);
      *reinterpret_cast<uint4*>(out + (2 * c + 2) * kChunk + at) = q8_expand<kF16>(w.x, w.y);
      *reinterpret_cast<uint4*>(out + (2 * c + 3) * kChunk + at) = q8_expand<kF16>(w.z, w.w);
    }
  }
};

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
__global__ void __launch_bounds__(512, 1) tcec_gemm_codes_kernel(const GemmCodesParams p) {
  using Cfg = GemmCodesCfg<BN, kSpans>;
  constexpr int kGroups = Cfg::GROUPS;
  constexpr bool kPair = Cfg::PAIR;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_code_full[Cfg::CODE_STAGES], bar_code_empty[Cfg::CODE_STAGES];
  __shared__ uint64_t bar_a_full[Cfg::A_STAGES], bar_a_empty[Cfg::A_STAGES];
  __shared__ uint64_t bar_b_full[Cfg::B_STAGES], bar_b_empty[Cfg::B_STAGES];
  __shared__ uint64_t bar_acc_full[2], bar_acc_free[2], bar_drain[1];
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

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::CODE_STAGES; ++s) {
      mbar_init(smem_u32(&bar_code_full[s]), 1);
      mbar_init(smem_u32(&bar_code_empty[s]), 4);
    }
    for (int s = 0; s < Cfg::A_STAGES; ++s) {
      mbar_init(smem_u32(&bar_a_full[s]), kPair && leader ? 5 : 4);  // the converters; in a leader the peer's relay too
      mbar_init(smem_u32(&bar_a_empty[s]), 1);
    }
    for (int s = 0; s < Cfg::B_STAGES; ++s) {
      mbar_init(smem_u32(&bar_b_full[s]), kPair && leader ? 2 : 1);
      mbar_init(smem_u32(&bar_b_empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 1);
      mbar_init(smem_u32(&bar_acc_free[i]), kPair ? 16 : 8);  // of a pair the leader's is used
    }
    mbar_init(smem_u32(&bar_drain[0]), 1);
    abort_flag = 0;
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
  wait_for_launch_before();
  auto give_up = [&](int code) {
    if constexpr (kPair) raise_abort_pair(&abort_flag);
    else abort_flag = 1;
    atomicCAS(p.status, 0, code);
  };

  float acc[Cfg::NC];

  if (warp < 4) {
    if constexpr (Cfg::REBALANCE) setmaxnreg_dec<40>();
    if (warp == 0) {
      // ---------------------------------------------------------- copies of the dense operand
      if (elect_one()) {
        uint32_t bs = 0, bph = 0, armed = 0, armed_parity = 0;
        bool ok = true;
        for (int tile = first_tile; tile < ntiles && ok; tile += stride) {
          const CodeTile ti = code_tile(tile, tile_rows, p.col_tiles);
          const int col = ti.col * BN + (kPair ? rank * 128 : 0);
          const uint32_t bytes = max(0, min(Cfg::BC, (p.cols - col + 15) & ~15)) * 64;  // a pair's second half may have no columns
          const uint8_t* src = p.panels + (static_cast<size_t>(col >> 7) * p.blocks + kb_first) * p.parts * kSpanBytes + (col & 127) * 64;
          for (int left = nkb * p.parts * 2; left > 0; --left) {  // a half of a block and part
            if (!mbar_wait(smem_u32(&bar_b_empty[bs]), bph ^ 1, abortp)) {
              ok = false;
              break;
            }
            const uint32_t bfull = smem_u32(&bar_b_full[bs]);
            if (bytes) {
              mbar_arrive_expect_tx(bfull, 2 * bytes);
              armed |= 1u << bs;
              armed_parity = (armed_parity & ~(1u << bs)) | (bph << bs);
              const uint32_t dst = smem_base + Cfg::B_OFFSET + bs * Cfg::B_BYTES;
              bulk_load(dst, src, bytes, bfull);
              bulk_load(dst + Cfg::BC * 64, src + kPanelBytes, bytes, bfull);
            } else {
              mbar_arrive(bfull);
            }
            src += 2 * kPanelBytes;
            if (++bs == Cfg::B_STAGES) bs = 0, bph ^= 1;
          }
        }
        if (!ok) {
          give_up(kErrProducerWait);
          // this thread's own copies land before the CTA gives up its shared memory
          for (uint32_t q = 0; q < Cfg::B_STAGES; ++q)
            if (armed & (1u << q)) mbar_wait_plain(smem_u32(&bar_b_full[q]), (armed_parity >> q) & 1);
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
            mbar_arrive_expect_tx(full, Cfg::BLOCK_BYTES);
            armed |= 1u << cs;
            armed_parity = (armed_parity & ~(1u << cs)) | (cph << cs);
            bulk_load(smem_base + Cfg::CODE_OFFSET + cs * Cfg::BLOCK_BYTES, src, Cfg::BLOCK_BYTES, full);
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
      if (elect_one()) {
        uint32_t as = 0, aph = 0, bs = 0, bph = 0, fold = 0;
        bool ok = true;
        if (!leader) {
          // -------------------------------------------------------- peer: "my operands are there"
          for (int tile = first_tile; tile < ntiles && ok; tile += stride)
            for (int kb = 0; kb < nkb && ok; ++kb) {
              if (!mbar_wait(smem_u32(&bar_a_full[as]), aph, abortp, 0)) {
                ok = false;
                break;
              }
              mbar_arrive_cluster(map_to_cta(smem_u32(&bar_a_full[as]), 0));
              if (++as == Cfg::A_STAGES) as = 0, aph ^= 1;
              for (int h = 0; h < 2 * p.parts; ++h) {
                if (!mbar_wait(smem_u32(&bar_b_full[bs]), bph, abortp, 0)) {
                  ok = false;
                  break;
                }
                mbar_arrive_cluster(map_to_cta(smem_u32(&bar_b_full[bs]), 0));
                if (++bs == Cfg::B_STAGES) bs = 0, bph ^= 1;
              }
            }
          if (!ok) give_up(kErrMmaWait);
        } else {
          // -------------------------------------------------------- MMAs
          const uint64_t a_const = umma_desc_kmajor_noswizzle(0, Cfg::CHUNK_BYTES, 128), b_const = umma_desc_kmajor_noswizzle(0, 128, 512);
          const uint32_t a16 = ((smem_base + Cfg::A_OFFSET) & 0x3ffff) >> 4, b16 = ((smem_base + Cfg::B_OFFSET) & 0x3ffff) >> 4;
          auto commit = [&](uint64_t* bar) {
            if constexpr (kPair) umma_commit_pair(smem_u32(bar));
            else umma_commit(smem_u32(bar));
          };
          for (int tile = first_tile; tile < ntiles && ok; tile += stride) {
            const int cols = p.cols - code_tile(tile, tile_rows, p.col_tiles).col * BN;
            const uint32_t idesc = umma_idesc(kF16 ? 0u : 1u, kPair ? 256 : 128, kPair ? 256 : min(BN, (cols + 15) & ~15));
            for (int kb = 0; kb < nkb && ok; ++kb) {
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
                    const uint64_t da = a_const | (a_here + step * (2 * Cfg::CHUNK_BYTES >> 4));
                    const uint64_t db = b_const | (b_here + (j >> 1) * (Cfg::BC * 64 >> 4) + (j & 1) * 16);
                    if constexpr (kPair) umma_ss_pair<false>(tmem + (fold & 1) * BN, da, db, idesc, first ? 0u : 1u);
                    else umma_ss<false>(tmem + (fold & 1) * BN, da, db, idesc, first ? 0u : 1u);
                    if (last) {
                      commit(&bar_acc_full[fold & 1]);
                      ++fold;
                    }
                  }
                  if (!ok) break;
                  commit(&bar_b_empty[bs]);
                  if (++bs == Cfg::B_STAGES) bs = 0, bph ^= 1;
                }
              }
              if (!ok) break;
              commit(&bar_a_empty[as]);
              if (++as == Cfg::A_STAGES) as = 0, aph ^= 1;
            }
          }
          if (!ok) mma_thread_gave_up<kPair>(&abort_flag, p.status, kErrMmaWait, &bar_drain[0]);
        }
      }
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ codes to operands
    if constexpr (Cfg::REBALANCE) setmaxnreg_dec<56>();
    uint32_t cs = 0, cph = 0, as = 0, aph = 0, slot = 0;
    const int t = threadIdx.x - 128;
    bool ok = true;
    for (int tile = first_tile; tile < ntiles && ok; tile += stride)
      for (int kb = 0; kb < nkb; ++kb) {
        if (!mbar_wait_lanes(smem_u32(&bar_code_full[cs]), cph, abortp) || !mbar_wait_lanes(smem_u32(&bar_a_empty[as]), aph ^ 1, abortp)) {
          ok = false;
          break;
        }
        const uint8_t* block = smem_gen + Cfg::CODE_OFFSET + cs * Cfg::BLOCK_BYTES;
        // The scales, for those who come to them when the products are made.  A slot is written again six blocks later; the stage just
        // waited for says that the MMAs of three blocks before are done, for which the accumulators of five blocks before were free.
        float* scales = reinterpret_cast<float*>(smem_gen + Cfg::SCALE_OFFSET) + slot * (kGroups * 128) + t;
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
          scales[g * 128] = __uint_as_float(reinterpret_cast<const uint32_t*>(block + Cfg::CODE_BYTES)[g * 128 + t] & (Cfg::Q8 ? ~0u : ~15u));
        Converter<kF16, kSpans>::expand(block, smem_gen + Cfg::A_OFFSET + as * Cfg::A_BYTES, warp - 4, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&bar_a_full[as]));
          mbar_arrive(smem_u32(&bar_code_empty[cs]));
        }
        if (++cs == Cfg::CODE_STAGES) cs = 0, cph ^= 1;
        if (++as == Cfg::A_STAGES) as = 0, aph ^= 1;
        if (++slot == Cfg::SCALE_SLOTS) slot = 0;
      }
    if (!ok && lane == 0) give_up(kErrOperandWait);
  } else {
    // ------------------------------------------------------------ scales
    if constexpr (Cfg::REBALANCE) setmaxnreg_inc<208>();
    const int q = warp & 3, r = q * 32 + lane, first_col = (warp >= 12 ? Cfg::NC : 0);
    const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + first_col;
    const float* scales = reinterpret_cast<const float*>(smem_gen + Cfg::SCALE_OFFSET) + r;
    const int rounds = kGroups > 1 ? p.parts : 1;  // of the groups of a block
    uint32_t fold = 0, slot = 0;
    bool ok = true;
    for (int tile = first_tile; tile < ntiles && ok; tile += stride) {
      const CodeTile ti = code_tile(tile, tile_rows, p.col_tiles);
      const int col0 = ti.col * BN + first_col, cols = p.cols - col0;  // from this warp's first column on
#pragma unroll
      for (int i = 0; i < Cfg::NC; ++i) acc[i] = 0.f;
      for (int kb = 0; kb < nkb && ok; ++kb) {
        for (int round = 0; round < rounds && ok; ++round) {
#pragma unroll
          for (int g = 0; g < kGroups; ++g, ++fold) {
            if (!mbar_wait_lanes(smem_u32(&bar_acc_full[fold & 1]), (fold >> 1) & 1, abortp)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const float s = scales[(slot * kGroups + g) * 128];
            const uint32_t from = taddr + (fold & 1) * BN;
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
                  if constexpr (kPair) mbar_arrive_cluster(map_to_cta(smem_u32(&bar_acc_free[fold & 1]), 0));
                  else mbar_arrive(smem_u32(&bar_acc_free[fold & 1]));
                }
              }
#pragma unroll
              for (int j = 0; j < kAtOnce; j += 2)
                fma2(acc[i + j], acc[i + j + 1], __uint_as_float(v[(i / kAtOnce) & 1][j]), __uint_as_float(v[(i / kAtOnce) & 1][j + 1]), s);
            }
          }
        }
        if (++slot == Cfg::SCALE_SLOTS) slot = 0;
      }
      const int row = row_tile(ti) * 128 + r;
      if (shares == 1 && ok && row < p.rows) {
        const long long base = row * p.c_row + col0 * p.c_col;
#pragma unroll
        for (int i = 0; i < Cfg::NC; ++i)
          if (i < cols) {
            const long long at = base + i * p.c_col;
            float v = __fmul_rn(p.alpha, acc[i]);
            if (p.beta != 0.f) v = __fmaf_rn(p.beta, ld_element_as(p.c_type, p.c, at), v);
            st_element_as(p.c_type, p.c, at, v);
          }
      }
    }
    if (!ok && lane == 0) give_up(kErrEpilogueWait);
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) {
    cluster_sync_all();  // neither CTA leaves while the other may still signal it or read its operands
    if (warp == 1) tmem_dealloc_pair(tmem, Cfg::TMEM_COLS);
  } else {
    if (warp == 1) tmem_dealloc(tmem, Cfg::TMEM_COLS);
    if (shares > 1) {  // then a cluster has one tile
      cluster_sync_all();  // nobody reads operands any more where the partial results go
      const CodeTile ti = code_tile(first_tile, tile_rows, p.col_tiles);
      const int per = BN / shares;  // columns that a CTA adds up and stores
      if (warp >= 8) {
        const int r = (warp & 3) * 32 + lane, first_col = (warp >= 12 ? Cfg::NC : 0);
#pragma unroll
        for (int i = 0; i < Cfg::NC; ++i) {
          const int col = first_col + i, to = col / per;
          const uint32_t at = smem_base + Cfg::B_OFFSET + ((rank * per + col - to * per) * 128 + r) * 4;
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_cta(at, to)), "f"(acc[i]) : "memory");
        }
      }
      // A CTA whose wait ran out has no share: it tells the others, and none of them stores its part of the tile.
      if (static_cast<int>(threadIdx.x) < shares && *abortp) raise_abort_in(&abort_flag, threadIdx.x);
      __syncwarp();
      cluster_sync_all();
      if (warp >= 8 && !*abortp) {
        const int t = threadIdx.x - 256, r = t & 127, row = ti.row * 128 + r;
        if (row < p.rows) {
          const float* parts = reinterpret_cast<const float*>(smem_gen + Cfg::B_OFFSET) + r;
          for (int i = t >> 7; i < per; i += 2) {
            const int col = ti.col * BN + rank * per + i;
            if (col >= p.cols) break;
            float v = parts[i * 128];
            for (int s = 1; s < shares; ++s) v += parts[(s * per + i) * 128];
            const long long at = row * p.c_row + col * p.c_col;
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
