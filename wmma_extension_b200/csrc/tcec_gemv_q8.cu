// Launches of gradients of few columns from activations in 8 bits (tcec_gemv_q8.cuh).
#include "tcec_gemv_q8.cuh"

#include "tcec_codes_launch.h"
#include "tcec_launch.h"

using namespace tcec_sm100;

namespace tcec_host {
namespace {

// Launches, or (p null) allows the kernel its shared memory.  Where SMs are left to others a launch has no more CTAs than there are SMs for it, and those of
// the next one come when all of them have ended.
template <int T, int E, int S>
cudaError_t one_gemv(const GemvQ8Params* p, int most_ctas, cudaStream_t stream) {
  using Cfg = GemvQ8Cfg<E, S>;
  if (!p) return cudaFuncSetAttribute(gemv_q8_kernel<T, E, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::smem_bytes(Cfg::MOST_WARPS));
  const int ctas = (p->rows - 1) / Cfg::ROWS + 1, most = most_ctas > 0 && most_ctas < ctas ? most_ctas : ctas;
  const int warps = warps_of(most, Cfg::WARPS_OF_SM, 4, Cfg::MOST_WARPS);
  GemvQ8Params q = *p;
  for (q.first = 0; q.first < ctas; q.first += most) {
    const int here = ctas - q.first < most ? ctas - q.first : most;
    if (q.first == 0) launch_early(gemv_q8_kernel<T, E, S>, here, 32 * warps, Cfg::smem_bytes(warps), stream, q);
    else launch_late(gemv_q8_kernel<T, E, S>, here, 32 * warps, Cfg::smem_bytes(warps), stream, q);
  }
  return cudaSuccess;
}
template <int T, int S>
cudaError_t of_strips(int eights, const GemvQ8Params* p, int most_ctas, cudaStream_t stream) {
  return eights == 1   ? one_gemv<T, 1, S>(p, most_ctas, stream)
         : eights == 2 ? one_gemv<T, 2, S>(p, most_ctas, stream)
                       : one_gemv<T, 4, S>(p, most_ctas, stream);
}
template <int T>
void of_type(int eights, int most_ctas, const GemvQ8Params& p, cudaStream_t stream) {
  // One strip a CTA while such CTAs fit the SMs, else two, which share what is done for the columns (rank 16, 8192 tokens: 2368 features 8.7 us with one,
  // 10.5 with two; 3000 12.6 and 11.2; 8192 26.9 and 19.6).
  if (p.rows <= 148 * 16) of_strips<T, 1>(eights, &p, most_ctas, stream);
  else of_strips<T, 2>(eights, &p, most_ctas, stream);
}
template <int T>
cudaError_t set_type() {
  cudaError_t e = cudaSuccess;
  for (int eights = 1; eights <= 4 && e == cudaSuccess; eights *= 2) {
    e = of_strips<T, 1>(eights, nullptr, 0, nullptr);
    if (e == cudaSuccess) e = of_strips<T, 2>(eights, nullptr, 0, nullptr);
  }
  return e;
}

}  // namespace

cudaError_t set_gemv_q8_attrs() {
  cudaError_t e = set_type<kTypeF32>();
  if (e == cudaSuccess) e = set_type<kTypeF16>();
  if (e == cudaSuccess) e = set_type<kTypeBf16>();
  return e;
}
void launch_gemv_q8(int type, int eights, int most_ctas, const GemvQ8Params& p, cudaStream_t stream) {
  if (type == kTypeF32) of_type<kTypeF32>(eights, most_ctas, p, stream);
  else if (type == kTypeF16) of_type<kTypeF16>(eights, most_ctas, p, stream);
  else of_type<kTypeBf16>(eights, most_ctas, p, stream);
}

}  // namespace tcec_host
