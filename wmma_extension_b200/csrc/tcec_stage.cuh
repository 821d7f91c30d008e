// The dense operand of a product with codes, whatever its type, order and alignment, laid out for the tensor cores: 16-bit values, FP32 in three
// bf16 parts of 8 bits each, which together are exactly it; what is beyond the matrix is zero.
//
// Bound by memory: every value is read once and written once (FP32: 6 bytes for 4).
#pragma once
#include "tcec_codes.cuh"
#include "tcec_panels.cuh"

namespace tcec_sm100 {

constexpr int kSpanPanels = kCodeSpan / 32;                  // panels of one block and part
constexpr int kSpanBytes = kSpanPanels * kPanelBytes;        // 32 KB
struct StagePanelsParams {
  const void* src;            // element (col, i) at col * col_step + i * sum_step
  long long col_step, sum_step;
  int cols, sum;
  int blocks;                 // along the sum
  uint8_t* panels;            // [128 columns][block][part][panel]
  int vec;                    // sum_step 1 and aligned for 16 bytes
  int pairs;                  // 16 bits, col_step 1, an even number of columns, aligned for two
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

// Two CTAs a block of 128 columns x 128 of the sum; an item is 16 bytes of a panel, eight consecutive values of one column.  Addresses stay
// among the elements that exist, so that all loads of some items go out before the first is waited for.
template <int kType>
__global__ void __launch_bounds__(256) stage_panels_kernel(const StagePanelsParams p) {
  constexpr int kParts = kType == kTypeF32 ? 3 : 1;
  wait_for_launch_before();
  const void* const operand = after_wait(p.src);
  let_next_launch_start();  // the product: its CTAs take whole SMs, and fetch and expand codes
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
  if constexpr (kType != kTypeF32) {
    if (p.pairs) {  // two columns at a time, eight of the sum, of two panels
      const int r = (first & 63) * 2, c = first >> 6, col = min(r, cols_here - 2);
      const bool none = r >= cols_here;
      uint32_t w[2][8];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          w[h][j] = ld_operand32(static_cast<const uint16_t*>(operand) + origin + col + min((blockIdx.y * 2 + h) * 32 + c * 8 + j, sum_here - 1) * p.sum_step);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int panel = blockIdx.y * 2 + h;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (none || panel * 32 + c * 8 + j >= sum_here) w[h][j] = 0;
        if (r < cols) {  // which is a multiple of 16
          uint4* const to = reinterpret_cast<uint4*>(out + panel * kPanelBytes + (r >> 3) * 512 + c * 128 + (r & 7) * 16);
          to[0] = make_uint4(__byte_perm(w[h][0], w[h][1], 0x5410), __byte_perm(w[h][2], w[h][3], 0x5410), __byte_perm(w[h][4], w[h][5], 0x5410),
                             __byte_perm(w[h][6], w[h][7], 0x5410));
          to[1] = make_uint4(__byte_perm(w[h][0], w[h][1], 0x7632), __byte_perm(w[h][2], w[h][3], 0x7632), __byte_perm(w[h][4], w[h][5], 0x7632),
                             __byte_perm(w[h][6], w[h][7], 0x7632));
        }
      }
      return;
    }
  }
#pragma unroll 1
  for (int it0 = blockIdx.y * 4; it0 < blockIdx.y * 4 + 4; it0 += kAtOnce) {
    if (p.vec && sum_here >= kCodeSpan) {
      uint4 raw[kAtOnce][kType == kTypeF32 ? 2 : 1];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int it = it0 + i;
        const long long at = origin + min(column(it), cols_here - 1) * p.col_step + (it >> 1) * 32 + chunk(it) * 8;
        if constexpr (kType == kTypeF32) {
          raw[i][0] = ld_operand128(static_cast<const float*>(operand) + at);
          raw[i][1] = ld_operand128(static_cast<const float*>(operand) + at + 4);
        } else {
          raw[i][0] = ld_operand128(static_cast<const uint16_t*>(operand) + at);
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
          if constexpr (kType == kTypeF32) w[i][j] = ld_operand(static_cast<const float*>(operand) + at);
          else w[i][j] = ld_operand16(static_cast<const uint16_t*>(operand) + at);
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
}

// Codes that are operands as they are, in the lowest bits of 16 (tcec_gemv_q4.cuh), are multiples of 2^-21 (f16) or 2^-133 (bf16).  f16 products are
// normal FP32 numbers all the same.  bf16 operands come times a power of two, so that their products do not fall below what FP32 holds, 2^-149: 2^100,
// or what suits the largest of a token's 128 values in a block: 2^6 from 2^27 on, 2^127 below 2^-60.  So what is lost lies below 2^-116, 2^-49 times the largest
// value, or 2^-143.  The unit makes the product of a code 1 and such an operand the operand's value.
constexpr float kUnitF16 = 0x1p21f;
struct UpX {
  float up, unit, down;  // down: 1 / up
};
__device__ __forceinline__ UpX up_x(uint32_t most) {  // the bits of the largest magnitude
  if (most >= 0x4d000000u) return {0x1p6f, 0x1p127f, 0x1p-6f};  // 2^27
  if (most < 0x21800000u) return {0x1p127f, 0x1p6f, 0x1p-127f};  // 2^-60
  return {0x1p100f, 0x1p33f, 0x1p-100f};
}

// Columns of mma.m16n8k16: for each block of 128 of the sum, 32 of it and eight columns, lane 4 g + t has 8 values of column g from
// 8 t on, 16 bytes.  A column is a token, or a part of one (FP32).  Behind the operands of all blocks, for each block: the columns'
// units, and the sums over each group (of 32: four, of 64: two) for all columns.
struct StageColumnsParams {
  const void* src;
  long long col_step, sum_step;
  int tokens, sum, blocks;
  int eights;                 // of columns
  int group;
  uint8_t* out;
  int vec;                    // sum_step 1 and aligned for 16 bytes
};
__host__ __device__ constexpr int staged_sum_bytes(int eights) { return (1 + 4) * eights * 32; }
__host__ __device__ constexpr long long staged_bytes(long long blocks, int eights) { return blocks * (eights * 2048 + staged_sum_bytes(eights)); }

// One CTA a block; 16 threads a token, eight values each.
template <int kType>
__global__ void __launch_bounds__(512) stage_columns_kernel(const StageColumnsParams p) {
  constexpr int kParts = kType == kTypeF32 ? 3 : 1;
  wait_for_launch_before();
  const void* const operand = after_wait(p.src);
  let_next_launch_start();
  const int kb = blockIdx.x, chunk = threadIdx.x & 15, token = threadIdx.x >> 4, sum_here = p.sum - kb * kCodeSpan - chunk * 8;
  const long long at = token * p.col_step + (static_cast<long long>(kb) * kCodeSpan + chunk * 8) * p.sum_step;
  float v[8] = {};
  if (token < p.tokens && sum_here > 0) {
    if constexpr (kType == kTypeF32) {
      const float* src = static_cast<const float*>(operand) + at;
      if (p.vec && sum_here >= 8) {
        const float4 a = ld_operand(reinterpret_cast<const float4*>(src)), b = ld_operand(reinterpret_cast<const float4*>(src + 4));
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = ld_operand(src + min(j, sum_here - 1) * p.sum_step);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j >= sum_here) v[j] = 0.f;
      }
    } else {
      const uint16_t* src = static_cast<const uint16_t*>(operand) + at;
      uint32_t w[4];
      if (p.vec && sum_here >= 8) {
        const uint4 o = ld_operand128(src);
        w[0] = o.x, w[1] = o.y, w[2] = o.z, w[3] = o.w;
      } else {
        uint32_t h[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = ld_operand16(src + min(j, sum_here - 1) * p.sum_step);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j >= sum_here) h[j] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = h[2 * j] | h[2 * j + 1] << 16;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kType == kTypeF16) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          v[2 * j] = f.x, v[2 * j + 1] = f.y;
        } else {
          v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
      }
    }
  }
  UpX by = {1.f, kUnitF16, 1.f};
  if constexpr (kType != kTypeF16) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
    by = up_x(most);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= by.up;
  }
  uint32_t part[kParts][4];
  if constexpr (kType == kTypeF32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) split3_bf16(v[2 * j], v[2 * j + 1], part[0][j], part[1][j], part[2][j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (kType == kTypeF16) {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        part[0][j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        part[0][j] = __byte_perm(__float_as_uint(v[2 * j]), __float_as_uint(v[2 * j + 1]), 0x7632);
      }
    }
  }
  const int columns = p.eights * 8;
  uint8_t* out = p.out + static_cast<size_t>(kb) * p.eights * 2048 + (chunk >> 2) * p.eights * 512 + (chunk & 3) * 16;
  uint8_t* sums = p.out + static_cast<size_t>(p.blocks) * p.eights * 2048 + static_cast<size_t>(kb) * staged_sum_bytes(p.eights);
#pragma unroll
  for (int q = 0; q < kParts; ++q) {
    const int col = token * kParts + q;
    if (col < columns) *reinterpret_cast<uint4*>(out + (col >> 3) * 512 + (col & 7) * 64) = make_uint4(part[q][0], part[q][1], part[q][2], part[q][3]);
    float sum = 0.f;
    if constexpr (kType == kTypeF16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)  // the values themselves, as the sum of scaled ones may be 2^28 * 2^100; exact, as their parts are FP32 numbers
        sum += by.down * __uint_as_float(part[q][j] << 16) + by.down * __uint_as_float(part[q][j] & 0xffff0000u);
    }
    for (int d = 1; d < p.group / 8; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const int of_group = p.group / 8;  // threads
    if (col < columns) {
      if ((chunk & (of_group - 1)) == 0)
        *reinterpret_cast<float*>(sums + ((1 + chunk / of_group) * columns + col) * 4) = sum;
      if (chunk == 0) *reinterpret_cast<float*>(sums + col * 4) = by.unit;
    }
  }
}

}  // namespace tcec_sm100
