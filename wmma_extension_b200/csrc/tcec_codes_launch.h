// What the host side of the products with codes hands to their kernels, and the launches, each in a translation unit of its own.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace tcec_sm100 {

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
  int debug_flags;            // develop builds only: bit 7 = a block of codes is never filled, in the last CTA of the first cluster
};

struct GemvQ4Params {
  const uint8_t* codes;
  const uint8_t* staged;      // x as operands of the MMAs (stage_columns_kernel), or null: one token, from x
  const void* x;              // one token: element i at i * x_k
  long long x_k;
  int n, k, tokens, blocks;
  int strips, more;           // strips of 16 rows of a CTA, and how many CTAs, the first ones, have one more (set by the launch)
  int vec;                    // x_k 1 and x aligned for four values at a time
  float alpha, beta;
  void* c;                    // element (token, row) at token * c_token + row * c_row
  long long c_token, c_row;
  int c_type;
  int* status;
  int debug_flags;            // develop builds only: bit 7 = the first block of codes is never filled, in the first CTA
};

struct GemvQ8Params {
  const uint8_t* codes;       // [row tile][block]
  const uint8_t* staged;      // dY as operands of the MMAs (stage_columns_kernel)
  int rows, cols, blocks;     // features, outputs, blocks of tokens
  int first;                  // CTAs of the launches before this one (set by the launch)
  float alpha, beta;
  void* c;
  long long c_row, c_col;
  int c_type;
  int* status;
  int debug_flags;            // as GemvQ4Params
};

}  // namespace tcec_sm100

namespace tcec_host {

// As many warps divide the k of a CTA's rows as let all CTAs run at a time: a second round of them would leave SMs idle at its end, and as every CTA
// goes through all of k it is long (13 tokens times 5000 x 7001: 16.7 us, 19.8 with eight warps whatever the rows).  So many SMs are assumed whatever
// the device has, so that the order of the sums follows from sizes.
inline int warps_of(int ctas, int warps_of_sm, int least, int most) {
  const int warps = warps_of_sm / ((ctas + 147) / 148);
  return warps < least ? most / 2 > least ? most / 2 : most : warps > most ? most : warps;  // too many for one round: then not too few warps
}

cudaError_t set_gemm_codes_attrs();
// eights: of columns (1, 2 or 4), which staged x has.
void launch_gemv_q4(int type, int group, int eights, const tcec_sm100::GemvQ4Params& p, cudaStream_t stream);
// spans: groups of 4-bit codes in a block, 0: 8-bit codes.  ctas: of a cluster.
void launch_gemm_codes(bool f16, int spans, int bn, const tcec_sm100::GemmCodesParams& gp, int ctas, int grid, cudaStream_t stream);
cudaError_t set_gemv_q4_attrs();
// most_ctas > 0: no more than so many at a time.
void launch_gemv_q8(int type, int eights, int most_ctas, const tcec_sm100::GemvQ8Params& p, cudaStream_t stream);
cudaError_t set_gemv_q8_attrs();

}  // namespace tcec_host
