// Operands held in few bits: weights W (n x k) as 4-bit codes with a scale and a zero point for every `group` of k, and
// activations X (m x k) as 8-bit codes with a scale for every 128 tokens of a feature.
//
//   4 bits:  lo = min(0, min w), hi = max(0, max w) over the group; s = RN16(RN32(RN32(hi - lo) / 15)), f16 or bf16;
//            z = clamp(rint(-lo / s), 0, 15);  q = clamp(rint(w / s) + z, 0, 15);  w^ = s (q - z)
//   8 bits:  s = max(RN32(max |x| / 127), 2^-120);  q = rint(x / s);  x^ = s q
//
// rint is of the exact quotient, ties to even (rint_quotient).  A group with a value that is not finite (or, with f16 scales,
// whose scale would not be) has the scale NaN, and so has all that is computed from it.
//
// Both are kept in blocks of 128 rows x 128 of the axis that the products sum over ("rows": n for weights, features for
// activations; the sum runs over k or over tokens).  The scale of a code is then the same for a whole row of a tensor-core tile, and
// is applied to the FP32 sum of a group: the tensor cores multiply whole numbers, which bf16 and f16 hold exactly.
//
//   4-bit block: 8 strips of 16 rows x 256 words of 8 codes, then 128 / group x 128 entries.  A word holds 8 consecutive k of one row,
//   nibble j of them k = 2 j (j < 4) and 2 (j - 4) + 1, so that (w >> 4 i) & 0x000f000f is the pair (2 i, 2 i + 1).  Words are in the
//   order of the registers of mma.m16n8k16: lane 4 g + t of a warp finds rows g and g + 8, k = 8 t .. 8 t + 7 of each 32, in two
//   128-bit loads.  An entry is the scale as FP32 (its low 12 bits or more are zero) with the zero point in the low 4 bits.
//   8-bit block: 16 chunks of 8 tokens x 128 features x 8 bytes (sign and magnitude), then 128 FP32 scales.
//
// Packing and unpacking are bound by memory: every value is read once and written once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace tcec_sm100 {

enum : int { kTypeF32 = 0, kTypeF16 = 1, kTypeBf16 = 2 };
constexpr int kCodeRows = 128, kCodeSpan = 128;      // rows of a block, and how far it goes along the sum
constexpr int kQ4CodeBytes = 8192, kQ8CodeBytes = 16384, kEntryBytes = 512;  // 128 entries of one group
__host__ __device__ constexpr int q4_block_bytes(int group) { return kQ4CodeBytes + kEntryBytes * (kCodeSpan / group); }
constexpr int kQ8BlockBytes = kQ8CodeBytes + kEntryBytes;

// Where the word of (row, chunk of 8 k) lies in a 4-bit block.
__host__ __device__ __forceinline__ int q4_word(int row, int chunk) {
  const int lane = (row & 7) * 4 + (chunk & 3), panel = chunk >> 2;
  return (row >> 4) * 256 + (panel >> 1) * 128 + lane * 4 + (panel & 1) * 2 + ((row >> 3) & 1);
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
// Bytes that one launch reads once: not kept in L1, where the operand that all of it is multiplied with stays.
__device__ __forceinline__ uint4 ld_once128(const void* p) {
  uint4 v;
  asm("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
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
// Four consecutive elements of an address that is aligned for them.
template <int kType>
__device__ __forceinline__ void ld_elements4(const void* base, long long at, float (&v)[4]) {
  if constexpr (kType == kTypeF32) {
    const float4 f = ld_operand(reinterpret_cast<const float4*>(static_cast<const float*>(base) + at));
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
  } else {
    const uint2 w = ld_operand64(static_cast<const uint16_t*>(base) + at);
    if constexpr (kType == kTypeF16) {
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
      v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    } else {
      v[0] = __uint_as_float(w.x << 16), v[1] = __uint_as_float(w.x & 0xffff0000u);
      v[2] = __uint_as_float(w.y << 16), v[3] = __uint_as_float(w.y & 0xffff0000u);
    }
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
// rint(x / s) of the exact quotient, ties to even, for |x / s| below 2^8.
//
// q0 = rint(x * (1 / s)) is off by at most one (a scale below the normal numbers, whose inverse may overflow, is divided by).  The
// remainder r = x - q0 s is exact in FP32: x and q0 s are both multiples of half the last place of s whenever |x| is at least s / 2, and
// |r| stays below 2 s; where |x| is smaller, q0 is 0 or +-1.  Comparing 2 r with s decides.
struct Quotient {
  float s, inv;
  __device__ __forceinline__ explicit Quotient(float scale) {
    s = scale;
    inv = scale < 0x1p-126f ? 0.0f : __fdiv_rn(1.0f, scale);
  }
  __device__ __forceinline__ float rint_of(float x) const {
    float q = rintf(inv != 0.0f ? x * inv : __fdiv_rn(x, s));
    const float r = __fmaf_rn(-q, s, x), r2 = r + r;
    const bool odd = (static_cast<int>(q) & 1) != 0;
    if (r2 > s || (r2 == s && odd)) q += 1.0f;
    else if (r2 < -s || (r2 == -s && odd)) q -= 1.0f;
    return q;
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

// One CTA a block: a warp takes a row at a time, a lane four consecutive k of it; words gather in shared memory and leave together.
template <int kType, int kGroup>
__global__ void __launch_bounds__(256) pack_q4_kernel(const PackQ4Params p) {
  __shared__ __align__(16) uint32_t words[2048 + 128 * (kCodeSpan / kGroup)];
  wait_for_launch_before();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kb = blockIdx.x % p.blocks, tile = blockIdx.x / p.blocks;
  const int k0 = kb * kCodeSpan + lane * 4;
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int r = warp * 16 + i, row = tile * kCodeRows + r;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (row < p.n) {
      const long long at = row * p.row_step + k0 * p.k_step;
      if (p.vec && k0 + 4 <= p.k) {
        ld_elements4<kType>(p.w, at, v);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (k0 + j < p.k) v[j] = ld_element<kType>(p.w, at + j * p.k_step);
      }
    }
    float lo = 0.f, hi = 0.f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lo = fminf(lo, v[j]);
      hi = fmaxf(hi, v[j]);
      bad |= not_finite(v[j]);
    }
#pragma unroll
    for (int d = kGroup / 8; d >= 1; d >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    }
    const uint32_t bads = __ballot_sync(0xffffffffu, bad);
    constexpr uint32_t kOfGroup = kGroup == 128 ? 0xffffffffu : kGroup == 64 ? 0xffffu : 0xffu;
    bad = ((bads >> (lane & ~(kGroup / 4 - 1))) & kOfGroup) != 0;
    const float want = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
    const float s = p.scale_bf16 ? __bfloat162float(__float2bfloat16_rn(want)) : __half2float(__float2half_rn(want));
    bad |= not_finite(s);
    uint32_t code = 0;
    float z = 0.f;
    if (!bad && s > 0.f) {
      const Quotient by(s);
      z = fminf(by.rint_of(-lo), 15.0f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int q = static_cast<int>(fminf(fmaxf(by.rint_of(v[j]) + z, 0.0f), 15.0f));
        code |= static_cast<uint32_t>(q) << ((j & 1) * 16 + (j >> 1) * 4);  // the first half of a word; the odd lane's is 8 higher
      }
    }
    const uint32_t other = __shfl_xor_sync(0xffffffffu, code, 1);
    if ((lane & 1) == 0) words[q4_word(r, lane >> 1)] = code | (other << 8);
    if ((lane & (kGroup / 4 - 1)) == 0)
      words[2048 + (lane / (kGroup / 4)) * 128 + r] = q4_entry(bad ? nan32() : s, static_cast<int>(z));
  }
  let_next_launch_start();
  __syncthreads();
  uint4* out = reinterpret_cast<uint4*>(p.packed + (static_cast<size_t>(tile) * p.blocks + kb) * q4_block_bytes(kGroup));
  for (int i = threadIdx.x; i < q4_block_bytes(kGroup) / 16; i += 256) out[i] = reinterpret_cast<const uint4*>(words)[i];
}

// Lays out codes that the caller has.
template <int kGroup>
__global__ void __launch_bounds__(256) pack_q4_codes_kernel(const PackQ4Params p) {
  __shared__ __align__(16) uint32_t words[2048 + 128 * (kCodeSpan / kGroup)];
  wait_for_launch_before();
  const int kb = blockIdx.x % p.blocks, tile = blockIdx.x / p.blocks;
  constexpr int kSpans = kCodeSpan / kGroup;
  for (int i = threadIdx.x; i < 128 * kSpans; i += 256) {
    const int r = i & 127, row = tile * kCodeRows + r, g = kb * kSpans + (i >> 7);
    uint32_t entry = 0;
    if (row < p.n && g < p.groups) {
      const long long at = static_cast<long long>(row) * p.groups + g;
      const float s = p.scale_bf16 ? ld_element<kTypeBf16>(p.scales, at) : ld_element<kTypeF16>(p.scales, at);
      entry = q4_entry(not_finite(s) ? nan32() : s, p.zeros ? (p.zeros[at] & 15) : 8);
    }
    words[2048 + i] = entry;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2048; i += 256) {
    const int r = i >> 4, chunk = i & 15, row = tile * kCodeRows + r, k0 = kb * kCodeSpan + chunk * 8;
    const uint32_t z = words[2048 + (chunk * 8 / kGroup) * 128 + r] & 15u;  // what is beyond the matrix stands for zero
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t lo = z, hi = z;
      if (row < p.n && k0 + 2 * j < p.k) {
        const uint32_t b = p.codes[row * p.codes_ld + (k0 >> 1) + j];
        lo = b & 15u;
        if (k0 + 2 * j + 1 < p.k) hi = b >> 4;
      }
      w |= lo << (4 * j) | hi << (4 * j + 16);
    }
    words[q4_word(r, chunk)] = w;
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
  const uint8_t* in = p.packed + (static_cast<size_t>(tile) * p.blocks + kb) * q4_block_bytes(kGroup);
  for (int i = threadIdx.x; i < q4_block_bytes(kGroup) / 16; i += 256) reinterpret_cast<uint4*>(words)[i] = ld_operand128(in + i * 16);
  let_next_launch_start();
  __syncthreads();
#pragma unroll 2
  for (int i = threadIdx.x; i < 4096; i += 256) {  // four values at a time
    const int r = i >> 5, part = i & 31, chunk = part >> 1, row = tile * kCodeRows + r, k0 = kb * kCodeSpan + part * 4;
    if (row >= p.rows || k0 >= p.sum) continue;
    const uint32_t w = words[q4_word(r, chunk)] >> ((part & 1) * 8);
    const uint32_t entry = words[2048 + (chunk * 8 / kGroup) * 128 + r];
    const float s = __uint_as_float(entry & ~15u);
    const int z = static_cast<int>(entry & 15u);
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = s * static_cast<float>(static_cast<int>((w >> ((j & 1) * 16 + (j >> 1) * 4)) & 15u) - z);
    const long long at = row * p.row_step + k0 * p.sum_step;
    if (p.vec && k0 + 4 <= p.sum) {
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
__global__ void __launch_bounds__(256) pack_q8_kernel(const PackQ8Params p) {
  __shared__ float4 most[8][32];
  wait_for_launch_before();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x / p.token_blocks, tb = blockIdx.x % p.token_blocks;
  const int f0 = tile * kCodeRows + lane * 4, t0 = tb * kCodeSpan + warp * 16;
  float v[16][4];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
    if (t0 + i < p.tokens) {
      const long long at = (t0 + i) * p.token_step + f0 * p.feature_step;
      if (p.vec && f0 + 4 <= p.features) {
        ld_elements4<kType>(p.x, at, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (f0 + j < p.features) v[i][j] = ld_element<kType>(p.x, at + j * p.feature_step);
      }
    }
  }
  let_next_launch_start();
  float m[4] = {0.f, 0.f, 0.f, 0.f};  // the largest magnitude as bits, among which infinities and NaN come last
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = __uint_as_float(max(__float_as_uint(m[j]), __float_as_uint(v[i][j]) & 0x7fffffffu));
  most[warp][lane] = make_float4(m[0], m[1], m[2], m[3]);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const float4 o = most[w][lane];
    m[0] = __uint_as_float(max(__float_as_uint(m[0]), __float_as_uint(o.x)));
    m[1] = __uint_as_float(max(__float_as_uint(m[1]), __float_as_uint(o.y)));
    m[2] = __uint_as_float(max(__float_as_uint(m[2]), __float_as_uint(o.z)));
    m[3] = __uint_as_float(max(__float_as_uint(m[3]), __float_as_uint(o.w)));
  }
  uint8_t* block = p.packed + (static_cast<size_t>(tile) * p.token_blocks + tb) * kQ8BlockBytes;
  float scale[4];
  uint32_t w[2][4][2] = {};  // chunk of eight tokens, feature, half of the chunk
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool bad = not_finite(m[j]);
    const float s = fmaxf(__fdiv_rn(m[j], 127.0f), 0x1p-120f);
    scale[j] = bad ? nan32() : s;
    if (bad) continue;
    const Quotient by(s);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int q = static_cast<int>(by.rint_of(v[i][j]));
      const uint32_t code = static_cast<uint32_t>(q < 0 ? 128 - q : q);
      w[i >> 3][j][(i >> 2) & 1] |= code << ((i & 3) * 8);
    }
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint4* to = reinterpret_cast<uint4*>(block + (warp * 2 + c) * 1024 + lane * 32);
    to[0] = make_uint4(w[c][0][0], w[c][0][1], w[c][1][0], w[c][1][1]);
    to[1] = make_uint4(w[c][2][0], w[c][2][1], w[c][3][0], w[c][3][1]);
  }
  if (warp == 0) reinterpret_cast<float4*>(block + kQ8CodeBytes)[lane] = make_float4(scale[0], scale[1], scale[2], scale[3]);
}

// A lane takes four features of eight tokens.
template <int kType>
__global__ void __launch_bounds__(256) unpack_q8_kernel(const UnpackParams p) {
  wait_for_launch_before();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x / p.blocks, tb = blockIdx.x % p.blocks;
  const uint8_t* block = p.packed + (static_cast<size_t>(tile) * p.blocks + tb) * kQ8BlockBytes;
  const int f0 = tile * kCodeRows + lane * 4;
  const uint4 sc = ld_operand128(block + kQ8CodeBytes + lane * 16);
  const float s[4] = {__uint_as_float(sc.x), __uint_as_float(sc.y), __uint_as_float(sc.z), __uint_as_float(sc.w)};
  uint4 in[2][2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    in[c][0] = ld_operand128(block + (warp * 2 + c) * 1024 + lane * 32);
    in[c][1] = ld_operand128(block + (warp * 2 + c) * 1024 + lane * 32 + 16);
  }
  let_next_launch_start();
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const uint32_t w[4][2] = {{in[c][0].x, in[c][0].y}, {in[c][0].z, in[c][0].w}, {in[c][1].x, in[c][1].y}, {in[c][1].z, in[c][1].w}};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int token = tb * kCodeSpan + (warp * 2 + c) * 8 + i;
      if (token >= p.sum) continue;
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t code = (w[j][i >> 2] >> ((i & 3) * 8)) & 255u;
        const float q = static_cast<float>(code & 127u);
        v[j] = s[j] * (code & 128u ? -q : q);
      }
      const long long at = f0 * p.row_step + token * p.sum_step;
      if (p.vec && f0 + 4 <= p.rows) {
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
}

}  // namespace tcec_sm100
