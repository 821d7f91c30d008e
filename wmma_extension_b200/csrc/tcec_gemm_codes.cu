// Launches of the tensor-core products of codes (tcec_gemm_codes.cuh).
#include "tcec_gemm_codes.cuh"

#include "tcec_codes_launch.h"
#include "tcec_launch.h"

using namespace tcec_sm100;

namespace tcec_host {
namespace {

template <int BN, bool F, int S>
cudaError_t set_codes_attr() {
  const cudaError_t e = cudaFuncSetAttribute(tcec_gemm_codes_kernel<BN, F, S>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             GemmCodesCfg<BN, S>::SMEM_BYTES);
  if (e != cudaSuccess) return e;
  cudaFuncAttributes a{};  // the split of the registers among the warps is made for a launch with so many a thread
  const cudaError_t got = cudaFuncGetAttributes(&a, tcec_gemm_codes_kernel<BN, F, S>);
  return got != cudaSuccess ? got : a.numRegs == GemmCodesCfg<BN, S>::REGS_LAUNCH ? cudaSuccess : cudaErrorInvalidConfiguration;
}
template <bool F, int S>
cudaError_t set_codes_attrs() {
  cudaError_t e = set_codes_attr<64, F, S>();
  if (e == cudaSuccess) e = set_codes_attr<128, F, S>();
  if (e == cudaSuccess) e = set_codes_attr<256, F, S>();
  return e;
}
template <bool F>
cudaError_t set_all_codes_attrs() {
  cudaError_t e = set_codes_attrs<F, 0>();
  if (e == cudaSuccess) e = set_codes_attrs<F, 1>();
  if (e == cudaSuccess) e = set_codes_attrs<F, 2>();
  if (e == cudaSuccess) e = set_codes_attrs<F, 4>();
  return e;
}

template <int BN, bool F, int S>
void launch_codes_as(const GemmCodesParams& gp, int shares, int grid, cudaStream_t stream) {
  launch_clusters(tcec_gemm_codes_kernel<BN, F, S>, shares, grid, GemmCodesCfg<BN, S>::THREADS, GemmCodesCfg<BN, S>::SMEM_BYTES, stream, gp);
}
template <bool F, int S>
void launch_codes_of(int bn, const GemmCodesParams& gp, int shares, int grid, cudaStream_t stream) {
  if (bn == 64) launch_codes_as<64, F, S>(gp, shares, grid, stream);
  else if (bn == 128) launch_codes_as<128, F, S>(gp, shares, grid, stream);
  else launch_codes_as<256, F, S>(gp, shares, grid, stream);
}
template <bool F>
void launch_codes(int spans, int bn, const GemmCodesParams& gp, int shares, int grid, cudaStream_t stream) {
  if (spans == 0) launch_codes_of<F, 0>(bn, gp, shares, grid, stream);
  else if (spans == 1) launch_codes_of<F, 1>(bn, gp, shares, grid, stream);
  else if (spans == 2) launch_codes_of<F, 2>(bn, gp, shares, grid, stream);
  else launch_codes_of<F, 4>(bn, gp, shares, grid, stream);
}

}  // namespace

cudaError_t set_gemm_codes_attrs() {
  const cudaError_t e = set_all_codes_attrs<false>();
  return e != cudaSuccess ? e : set_all_codes_attrs<true>();
}
void launch_gemm_codes(bool f16, int spans, int bn, const GemmCodesParams& gp, int ctas, int grid, cudaStream_t stream) {
  if (f16) launch_codes<true>(spans, bn, gp, ctas, grid, stream);
  else launch_codes<false>(spans, bn, gp, ctas, grid, stream);
}

}  // namespace tcec_host
