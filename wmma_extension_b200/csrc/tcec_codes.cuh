// Operands held in few bits: weights W (n x k) as 4-bit codes with a scale and a zero point for every `group` of k, and
// activations X (m x k) as 8-bit codes with a scale for every 128 tokens of a feature.
//
//   4 bits:  lo = min(0, min w), hi = max(0, max w) over the group; s = RN16(RN32(RN32(hi - lo) / 15)), f16 or bf16;
//            z = clamp(rint(-lo / s), 0, 15);  q = clamp(rint(w / s) + z, 0, 15);  w^ = s (q - z)
//   8 bits:  s = max(RN32(max |x| / 127), 2^-120);  q = rint(x / s);  x^ = s q
//
// rint is of the exact quotient, ties to even (Quotient).  A group with a value that is not finite (or, with f16 scales,
// whose scale would not be) has the scale NaN, and so has all that is computed from it.
//
// Both are kept in blocks of 128 rows x 128 of the axis that the products sum over ("rows": n for weights, features for
// activations; the sum runs over k or over tokens).  The scale of a code is then the same for a whole row of a tensor-core tile, and
// is applied to the FP32 sum of a group: the tensor cores multiply whole numbers, which bf16 and f16 hold exactly.
//
//   4-bit block: 8 strips of 16 rows, each 256 words of 8 codes and then 128 / group x 16 entries.  A word holds 8 consecutive k of one row,
//   nibble j of them k = 2 j (j < 4) and 2 (j - 4) + 1, so that (w >> 4 i) & 0x000f000f is the pair (2 i, 2 i + 1).  Words are in the
//   order of the registers of mma.m16n8k16: lane 4 g + t of a warp finds rows g and g + 8, k = 8 t .. 8 t + 7 of each 32, in two
//   128-bit loads.  An entry is the scale as FP32 (its low 12 bits or more are zero) with the zero point in the low 4 bits.
//   8-bit block: 8 x 16 tokens x 128 features x 16 bytes (sign and magnitude; tokens 0 2 1 3 of each four), then 128 FP32 scales.
//
// Packing and unpacking are bound by memory: every value is read once and written once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "sm100_ptx.cuh"

namespace tcec_sm100 {

enum : int { kTypeF32 = 0, kTypeF16 = 1, kTypeBf16 = 2 };
constexpr int kCodeRows = 128, kCodeSpan = 128;      // rows of a block, and how far it goes along the sum
constexpr int kQ4CodeBytes = 8192, kQ8CodeBytes = 16384, kEntryBytes = 512;  // 128 entries of one group
__host__ __device__ constexpr int q4_block_bytes(int group) { return kQ4CodeBytes + kEntryBytes * (kCodeSpan / group); }
constexpr int kQ8BlockBytes = kQ8CodeBytes + kEntryBytes;

constexpr int kStripCodeBytes = 1024;
__host__ __device__ constexpr int q4_strip_bytes(int group) { return kStripCodeBytes + 64 * (kCodeSpan / group); }
// Where the word of (row, chunk of 8 k), and the entry of (row, group), lie in a 4-bit block, in words.
template <int kGroup>
__host__ __device__ __forceinline__ int q4_word(int row, int chunk) {
  const int lane = (row & 7) * 4 + (chunk & 3), panel = chunk >> 2;
  return (row >> 4) * (q4_strip_bytes(kGroup) / 4) + (panel >> 1) * 128 + lane * 4 + (panel & 1) * 2 + ((row >> 3) & 1);
}
template <int kGroup>
__host__ __device__ __forceinline__ int q4_entry_word(int row, int group) {
  return (row >> 4) * (q4_strip_bytes(kGroup) / 4) + kStripCodeBytes / 4 + group * 16 + (row & 15);
}

// ---------------------------------------------------------------- typed elements
template <int kType>
struct Element;
template <>
struct Element<kTypeF32> {
  typedef float type;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Element<kTypeF16> {
  typedef __half type;
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Element<kTypeBf16> {
  typedef __nv_bfloat16 type;
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
// Operands of kernels that start early: ordinary coherent loads (see ld_operand in sm100_ptx.cuh).
__device__ __forceinline__ uint16_t ld_operand16(const void* p) {
  uint16_t v;
  asm("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_operand64(const void* p) {
  uint2 v;
  asm("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 ld_operand128(const void* p) {
  uint4 v;
  asm("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_operand32(const void* p) {
  uint32_t v;
  asm("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
template <int kType>
__device__ __forceinline__ float ld_element(const void* base, long long at) {
  if constexpr (kType == kTypeF32) {
    return ld_operand(static_cast<const float*>(base) + at);
  } else if constexpr (kType == kTypeF16) {
    return __half2float(__ushort_as_half(ld_operand16(static_cast<const uint16_t*>(base) + at)));
  } else {
    return __uint_as_float(static_cast<uint32_t>(ld_operand16(static_cast<const uint16_t*>(base) + at)) << 16);
  }
}
// Four elements as they come, to be widened later: loads that are widened behind a branch wait for one another.
template <int kType>
struct Four {
  typename std::conditional<kType == kTypeF32, float4, uint2>::type raw;
  // Consecutive ones, of an address that is aligned for them.
  __device__ __forceinline__ void load(const void* base, long long at) {
    if constexpr (kType == kTypeF32) raw = ld_operand(reinterpret_cast<const float4*>(static_cast<const float*>(base) + at));
    else raw = ld_operand64(static_cast<const uint16_t*>(base) + at);
  }
  __device__ __forceinline__ void get(float (&v)[4]) const {
    if constexpr (kType == kTypeF32) {
      v[0] = raw.x, v[1] = raw.y, v[2] = raw.z, v[3] = raw.w;
    } else if constexpr (kType == kTypeF16) {
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
      v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    } else {
      v[0] = __uint_as_float(raw.x << 16), v[1] = __uint_as_float(raw.x & 0xffff0000u);
      v[2] = __uint_as_float(raw.y << 16), v[3] = __uint_as_float(raw.y & 0xffff0000u);
    }
  }
};
// kLines x 4 elements: line i < lines_left at base + i * line_step, in it element j < left at + j * step; zeros for those beyond.  Addresses stay
// among the elements that exist.  `wide`: four elements lie side by side, aligned.
template <int kType, int kLines>
__device__ __forceinline__ void ld_lines4(const void* base, long long at, long long line_step, long long step, int lines_left, int left, bool wide,
                                          float (&v)[kLines][4]) {
  if (lines_left <= 0 || left <= 0) {
#pragma unroll
    for (int i = 0; i < kLines; ++i) v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
  } else if (wide && left >= 4) {
    Four<kType> f[kLines];
#pragma unroll
    for (int i = 0; i < kLines; ++i) f[i].load(base, at + min(i, lines_left - 1) * line_step);
#pragma unroll
    for (int i = 0; i < kLines; ++i) {
      f[i].get(v[i]);
      if (i >= lines_left) v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kLines; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = ld_element<kType>(base, at + min(i, lines_left - 1) * line_step + min(j, left - 1) * step);
#pragma unroll
    for (int i = 0; i < kLines; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i >= lines_left || j >= left) v[i][j] = 0.f;
  }
}
template <int kType>
__device__ __forceinline__ void st_element(void* base, long long at, float v) {
  static_cast<typename Element<kType>::type*>(base)[at] = Element<kType>::put(v);
}
__device__ __forceinline__ void st_element_as(int type, void* base, long long at, float v) {
  if (type == kTypeF32) st_element<kTypeF32>(base, at, v);
  else if (type == kTypeF16) st_element<kTypeF16>(base, at, v);
  else st_element<kTypeBf16>(base, at, v);
}
__device__ __forceinline__ float ld_element_as(int type, const void* base, long long at) {
  if (type == kTypeF32) return ld_element<kTypeF32>(base, at);
  if (type == kTypeF16) return ld_element<kTypeF16>(base, at);
  return ld_element<kTypeBf16>(base, at);
}

// ---------------------------------------------------------------- arithmetic of the codes
// rint(x / s) of the exact quotient, ties to even, for |x / s| below 2^8, without a branch: of values of few bits, as bf16 has, one quotient in
// some hundred is a tie or next to one, so hardly a warp would go without it (8192 x 4096 bf16 to 8 bits: 125 us with the exact way in a branch for
// 16 values, 50 for four).
//
// q = (x - s / 4) * (1 / s) + 1.5 * 2^23, whose last place is 1, is the number wanted or one below it.  The remainder r = x - q s is exact in FP32: x
// and q s are both multiples of half the last place of s whenever |x| is at least s / 2, and |r| stays below 2 s; where |x| is smaller, q is 0 or -1.
// The sign of 2 r - s decides; a tie (0) of an odd q does too, as the number whose bits are that one bit.  Logic and comparisons, which run at half the
// rate of multiply-adds, are what packing is bound by: three of them here, five with a q to either side (8192 x 4096 to 8 bits and back 54 and 60 us).
constexpr float kRintBase = 12582912.0f;
struct Quotient {
  float s, inv;
  __device__ __forceinline__ explicit Quotient(float scale) {
    s = scale;
    inv = scale < 0x1p-126f ? 0.0f : __fdiv_rn(1.0f, scale);
  }
  __device__ __forceinline__ Quotient(float scale, float inverse) {
    s = scale;
    inv = inverse;
  }
  // A scale below the normal numbers, whose inverse may overflow, is not for nearest().
  __device__ __forceinline__ bool tiny() const { return inv == 0.0f; }
  // kRintBase + rint(x / s), as bits.
  __device__ __forceinline__ int nearest(float x) const { return decide(__fmaf_rn(__fmaf_rn(s, -0.25f, x), inv, kRintBase), x); }
  __device__ __forceinline__ int nearest_of_tiny(float x) const { return decide(floorf(__fdiv_rn(x, s)) + kRintBase, x); }

 private:
  __device__ __forceinline__ int decide(float q, float x) const {
    const float r = __fmaf_rn(kRintBase - q, s, x);
    int bits = __float_as_int(q);
    if (__fmaf_rn(2.0f, r, -s) + __int_as_float(bits & 1) > 0.0f) ++bits;
    return bits;
  }
};
__device__ __forceinline__ bool not_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ float nan32() { return __uint_as_float(0x7fc00000u); }

// ---------------------------------------------------------------- 4-bit weights
// Element (row, i) of a dense matrix lies at row * row_step + i * k_step.
struct PackQ4Params {
  const void* w;
  long long row_step, k_step;
  int n, k;
  int scale_bf16;             // scales of the codes: 0 f16, 1 bf16
  uint8_t* packed;
  int blocks;                 // along k
  int vec;                    // rows of consecutive elements, aligned for four at a time
  // codes that the caller has (pack_q4_codes_kernel)
  const uint8_t* codes;       // n x ceil(k / 2), two a byte, the even k in the low half
  long long codes_ld;
  const void* scales;         // n x groups, 16 bits each
  const uint8_t* zeros;       // n x groups, or null: 8
  int groups;
};

__device__ __forceinline__ uint32_t q4_entry(float s, int z) { return (__float_as_uint(s) & ~15u) | static_cast<uint32_t>(z); }

// One CTA a block.  A warp takes eight rows at a time, four lanes a row: lane 4 g + t has k = 16 j + 4 t .. + 3 of row g for j < 8, so a
// group is two exchanges away at most.  Words gather in shared memory and leave together.  Of few blocks a warp takes eight rows, of many (up to 592 are
// under way at a time) two times eight, in CTAs of which more fit an SM: 1000 x 1024 in groups of 32 4.2 us, 5.5 with sixteen rows a warp, 2048 x 2048 6.9 and 8.0,
// 4096 x 4096 in groups of 128 27 and 24.5.
template <int kType, int kGroup, int kHalves>
__global__ void __launch_bounds__(512 / kHalves) pack_q4_kernel(const PackQ4Params p) {
  constexpr int kSpans = kCodeSpan / kGroup;
  __shared__ __align__(16) uint32_t words[2048 + 128 * kSpans];
  wait_for_launch_before();
  const void* const w = after_wait(p.w);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kb = blockIdx.x % p.blocks, tile = blockIdx.x / p.blocks;
#pragma unroll
  for (int half = 0; half < kHalves; ++half) {
    const int r = warp * 8 * kHalves + half * 8 + g, row = tile * kCodeRows + r, k0 = kb * kCodeSpan + t * 4;
    float v[8][4];
    const int left = row < p.n ? p.k - k0 : 0;
    if (p.vec && left >= 7 * 16 + 4) {
      Four<kType> f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j].load(w, row * p.row_step + k0 + j * 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j].get(v[j]);
    } else if (left > 0) {  // unaligned, column-major or at the edge: addresses stay inside the row
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j][i] = ld_element<kType>(w, row * p.row_step + (k0 + min(j * 16 + i, left - 1)) * p.k_step);
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j * 16 + i >= left) v[j][i] = 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j][0] = v[j][1] = v[j][2] = v[j][3] = 0.f;
    }
    if (half == kHalves - 1) let_next_launch_start();
#pragma unroll
    for (int q = 0; q < kSpans; ++q) {  // groups; 128 / kSpans = 16 * 8 / kSpans
      float lo = 0.f, hi = 0.f;
      float none = 0.f;  // NaN if a value is not finite
#pragma unroll
      for (int j = q * 8 / kSpans; j < (q + 1) * 8 / kSpans; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo = fminf(lo, v[j][i]);
          hi = fmaxf(hi, v[j][i]);
          none = __fmaf_rn(v[j][i], 0.0f, none);
        }
#pragma unroll
      for (int d = 1; d <= 2; d <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        none += __shfl_xor_sync(0xffffffffu, none, d);
      }
      const float want = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
      const float s = p.scale_bf16 ? __bfloat162float(__float2bfloat16_rn(want)) : __half2float(__float2half_rn(want));
      const bool bad = none != 0.f || not_finite(s), some = !bad && s > 0.f;
      const Quotient by(some ? s : 1.0f);
      const int base = __float_as_int(kRintBase), z = !some ? 0 : min((by.tiny() ? by.nearest_of_tiny(-lo) : by.nearest(-lo)) - base, 15);
      uint32_t code[8 / kSpans];
      auto make_codes = [&](auto nearest) {
#pragma unroll
        for (int j = 0; j < 8 / kSpans; ++j) {
          code[j] = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i)  // half of a word
            code[j] |= static_cast<uint32_t>(min(max(nearest(v[q * 8 / kSpans + j][i]) + (z - base), 0), 15)) << ((i & 1) * 16 + (i >> 1) * 4);
        }
      };
      if (!by.tiny()) make_codes([&](float x) { return by.nearest(x); });
      else make_codes([&](float x) { return by.nearest_of_tiny(x); });
#pragma unroll
      for (int j = 0; j < 8 / kSpans; ++j) {
        const uint32_t mine = some ? code[j] : 0, other = __shfl_xor_sync(0xffffffffu, mine, 1);  // the odd lane's half is 8 bits higher
        if ((t & 1) == 0) words[q4_word<kGroup>(r, (q * 8 / kSpans + j) * 2 + (t >> 1))] = mine | (other << 8);
      }
      if (t == 0) words[q4_entry_word<kGroup>(r, q)] = q4_entry(bad ? nan32() : s, z);
    }
  }
  __syncthreads();
  uint4* out = reinterpret_cast<uint4*>(p.packed + (static_cast<size_t>(tile) * p.blocks + kb) * q4_block_bytes(kGroup));
  for (int i = threadIdx.x; i < q4_block_bytes(kGroup) / 16; i += 512 / kHalves) out[i] = reinterpret_cast<const uint4*>(words)[i];
}

// Lays out codes that the caller has.
template <int kGroup>
__global__ void __launch_bounds__(256) pack_q4_codes_kernel(const PackQ4Params p) {
  __shared__ __align__(16) uint32_t words[2048 + 128 * (kCodeSpan / kGroup)];
  wait_for_launch_before();
  const uint8_t *const codes = after_wait(p.codes), *const zeros = after_wait(p.zeros);
  const void* const scales = after_wait(p.scales);
  const int kb = blockIdx.x % p.blocks, tile = blockIdx.x / p.blocks;
  constexpr int kSpans = kCodeSpan / kGroup;
  for (int i = threadIdx.x; i < 128 * kSpans; i += 256) {
    const int r = i & 127, row = tile * kCodeRows + r, g = kb * kSpans + (i >> 7);
    uint32_t entry = 0;
    if (row < p.n && g < p.groups) {
      const long long at = static_cast<long long>(row) * p.groups + g;
      const float s = p.scale_bf16 ? ld_element<kTypeBf16>(scales, at) : ld_element<kTypeF16>(scales, at);
      entry = q4_entry(not_finite(s) ? nan32() : s, zeros ? (zeros[at] & 15) : 8);
    }
    words[q4_entry_word<kGroup>(r, i >> 7)] = entry;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2048; i += 256) {
    const int r = i >> 4, chunk = i & 15, row = tile * kCodeRows + r, k0 = kb * kCodeSpan + chunk * 8;
    const uint32_t z = words[q4_entry_word<kGroup>(r, chunk * 8 / kGroup)] & 15u;  // what is beyond the matrix stands for zero
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t lo = z, hi = z;
      if (row < p.n && k0 + 2 * j < p.k) {
        const uint32_t b = codes[row * p.codes_ld + (k0 >> 1) + j];
        lo = b & 15u;
        if (k0 + 2 * j + 1 < p.k) hi = b >> 4;
      }
      w |= lo << (4 * j) | hi << (4 * j + 16);
    }
    words[q4_word<kGroup>(r, chunk)] = w;
  }
  let_next_launch_start();
  __syncthreads();
  uint4* out = reinterpret_cast<uint4*>(p.packed + (static_cast<size_t>(tile) * p.blocks + kb) * q4_block_bytes(kGroup));
  for (int i = threadIdx.x; i < q4_block_bytes(kGroup) / 16; i += 256) out[i] = reinterpret_cast<const uint4*>(words)[i];
}

// The values that packed operands stand for.  Element (row, i) of the result lies at row * row_step + i * sum_step.
struct UnpackParams {
  const uint8_t* packed;
  void* out;
  long long row_step, sum_step;
  int rows, sum;              // extents: n and k of weights, features and tokens of activations
  int blocks;                 // along the sum
  int vec;                    // results lie in a row as they are computed, aligned for 16 bytes
};

template <int kType, int kGroup>
__global__ void __launch_bounds__(256) unpack_q4_kernel(const UnpackParams p) {
  __shared__ __align__(16) uint32_t words[2048 + 128 * (kCodeSpan / kGroup)];
  wait_for_launch_before();
  const int kb = blockIdx.x % p.blocks, tile = blockIdx.x / p.blocks;
  const uint8_t* in = after_wait(p.packed) + (static_cast<size_t>(tile) * p.blocks + kb) * q4_block_bytes(kGroup);
  for (int i = threadIdx.x; i < q4_block_bytes(kGroup) / 16; i += 256) reinterpret_cast<uint4*>(words)[i] = ld_operand128(in + i * 16);
  let_next_launch_start();
  __syncthreads();
#pragma unroll 2
  for (int i = threadIdx.x; i < 4096; i += 256) {  // four values at a time
    const int r = i >> 5, part = i & 31, chunk = part >> 1, row = tile * kCodeRows + r, k0 = kb * kCodeSpan + part * 4;
    if (row >= p.rows || k0 >= p.sum) continue;
    const uint32_t w = words[q4_word<kGroup>(r, chunk)] >> ((part & 1) * 8);
    const uint32_t entry = words[q4_entry_word<kGroup>(r, chunk * 8 / kGroup)];
    const float s = __uint_as_float(entry & ~15u);
    const int z = static_cast<int>(entry & 15u);
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = s * static_cast<float>(static_cast<int>((w >> ((j & 1) * 16 + (j >> 1) * 4)) & 15u) - z);
    const long long at = row * p.row_step + k0 * p.sum_step;
    if (p.vec && p.sum - k0 >= 4) {
      typename Element<kType>::type o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = Element<kType>::put(v[j]);
      if constexpr (kType == kTypeF32) *reinterpret_cast<uint4*>(static_cast<float*>(p.out) + at) = *reinterpret_cast<const uint4*>(o);
      else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = *reinterpret_cast<const uint2*>(o);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k0 + j < p.sum) st_element<kType>(p.out, at + j * p.sum_step, v[j]);
    }
  }
}

// ---------------------------------------------------------------- 8-bit activations
struct PackQ8Params {
  const void* x;
  long long token_step, feature_step;
  int tokens, features;
  int token_blocks;
  uint8_t* packed;
  int vec;
};

// One CTA a block of 128 tokens x 128 features: a warp takes 16 tokens, a lane four consecutive features of each, all of it in
// registers; the warps' maxima meet in shared memory.
template <int kType>
__global__ void __launch_bounds__(256, 3) pack_q8_kernel(const PackQ8Params p) {
  __shared__ float4 most[8][32], scales[32], inverses[32];
  wait_for_launch_before();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = (p.features - 1) / kCodeRows + 1, tile = blockIdx.x % tiles, tb = blockIdx.x / tiles;  // whole rows at a time
  const int f0 = tile * kCodeRows + lane * 4, t0 = tb * kCodeSpan + warp * 16;
  float v[16][4];
  ld_lines4<kType, 16>(after_wait(p.x), t0 * p.token_step + f0 * p.feature_step, p.token_step, p.feature_step, p.tokens - t0, p.features - f0, p.vec, v);
  let_next_launch_start();
  float m[4];  // the largest magnitude, or NaN if a value is not finite
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float none = 0.f;
    m[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      m[j] = fmaxf(m[j], fabsf(v[i][j]));
      none = __fmaf_rn(v[i][j], 0.0f, none);
    }
    if (none != 0.f) m[j] = nan32();
  }
  most[warp][lane] = make_float4(m[0], m[1], m[2], m[3]);
  __syncthreads();
  uint8_t* block = p.packed + (static_cast<size_t>(tile) * p.token_blocks + tb) * kQ8BlockBytes;
  if (threadIdx.x < 128) {  // a feature each: divisions are long
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) top = max(top, __float_as_uint(reinterpret_cast<const float*>(most[w])[threadIdx.x]));
    const bool bad = top >= 0x7f800000u;
    const Quotient by(bad ? 1.0f : fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), 0x1p-120f));
    reinterpret_cast<float*>(scales)[threadIdx.x] = by.s;
    reinterpret_cast<float*>(inverses)[threadIdx.x] = bad ? nan32() : by.inv;
    reinterpret_cast<float*>(block + kQ8CodeBytes)[threadIdx.x] = bad ? nan32() : by.s;
  }
  __syncthreads();
  const float4 s4 = scales[lane], i4 = inverses[lane];
  const float scale[4] = {s4.x, s4.y, s4.z, s4.w}, inverse[4] = {i4.x, i4.y, i4.z, i4.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool bad = inverse[j] != inverse[j];
    const Quotient by(scale[j], inverse[j]);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // tokens 0 2 1 3 of each four, and their signs
      int q[4];  // magnitudes, in the low bytes
#pragma unroll
      for (int t = 0; t < 4; ++t) q[t] = by.nearest(fabsf(v[4 * i + t][j]));
      const uint32_t size = __byte_perm(__byte_perm(q[0], q[2], 0x0040), __byte_perm(q[1], q[3], 0x0040), 0x5410);
      const uint32_t sign = __byte_perm(__byte_perm(__float_as_uint(v[4 * i][j]), __float_as_uint(v[4 * i + 2][j]), 0x0073),
                                        __byte_perm(__float_as_uint(v[4 * i + 1][j]), __float_as_uint(v[4 * i + 3][j]), 0x0073), 0x5410);
      w[i] = bad ? 0 : (size & 0x7f7f7f7fu) | (sign & 0x80808080u);
    }
    *reinterpret_cast<uint4*>(block + warp * 2048 + (lane * 4 + j) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A lane takes four features of 16 tokens.
template <int kType>
__global__ void __launch_bounds__(256) unpack_q8_kernel(const UnpackParams p) {
  wait_for_launch_before();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = (p.rows - 1) / kCodeRows + 1, tile = blockIdx.x % tiles, tb = blockIdx.x / tiles;
  const uint8_t* block = after_wait(p.packed) + (static_cast<size_t>(tile) * p.blocks + tb) * kQ8BlockBytes;
  const int f0 = tile * kCodeRows + lane * 4, t0 = tb * kCodeSpan + warp * 16;
  const uint4 sc = ld_operand128(block + kQ8CodeBytes + lane * 16);
  const float s[4] = {__uint_as_float(sc.x), __uint_as_float(sc.y), __uint_as_float(sc.z), __uint_as_float(sc.w)};
  uint32_t w[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 in = ld_operand128(block + warp * 2048 + (lane * 4 + j) * 16);
    w[j][0] = in.x, w[j][1] = in.y, w[j][2] = in.z, w[j][3] = in.w;
  }
  let_next_launch_start();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int token = t0 + i;
    if (token >= p.sum) continue;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t code = w[j][i >> 2] >> ((i & 1) * 16 + (i & 2) * 4);
      const float q = __uint_as_float(0x4b000000u | (code & 127u)) - 8388608.0f;  // 2^23 + the magnitude
      v[j] = __fmaf_rn(s[j], code & 128u ? -q : q, 0.0f);  // no negative zeros
    }
    const long long at = f0 * p.row_step + token * p.sum_step;
    if (p.vec && p.rows - f0 >= 4) {
      typename Element<kType>::type o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = Element<kType>::put(v[j]);
      if constexpr (kType == kTypeF32) *reinterpret_cast<uint4*>(static_cast<float*>(p.out) + at) = *reinterpret_cast<const uint4*>(o);
      else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = *reinterpret_cast<const uint2*>(o);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (f0 + j < p.rows) st_element<kType>(p.out, at + j * p.row_step, v[j]);
    }
  }
}

}  // namespace tcec_sm100
