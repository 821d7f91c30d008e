// Launches of the product of few tokens with 4-bit weights (tcec_gemv_q4.cuh).
#include "tcec_gemv_q4.cuh"

#include "tcec_codes_launch.h"
#include "tcec_launch.h"

using namespace tcec_sm100;

namespace tcec_host {
namespace {

int ceil_div(int a, int b) { return (a + b - 1) / b; }
// Launches for so many eights of columns and strips of rows a CTA, or (launch false) allows the kernel its shared memory.
template <int T, int G, int E, int S, bool One>
cudaError_t one_gemv(const GemvQ4Params* p, cudaStream_t stream) {
  using Cfg = GemvQ4Cfg<T, G, E, S, One>;
  if (!p) return cudaFuncSetAttribute(gemv_q4_kernel<T, G, E, S, One>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES);
  launch_early(gemv_q4_kernel<T, G, E, S, One>, ceil_div(p->n, Cfg::ROWS), 32 * Cfg::WARPS, Cfg::SMEM_BYTES, stream, *p);
  return cudaSuccess;
}
template <int T, int G>
cudaError_t gemv_of(int eights, const GemvQ4Params& p, cudaStream_t stream) {
  if (!p.staged && p.n <= 8192) return one_gemv<T, G, 1, 1, true>(&p, stream);
  if (!p.staged) return one_gemv<T, G, 1, 2, true>(&p, stream);
  if (eights == 1) return one_gemv<T, G, 1, 2, false>(&p, stream);
  if (eights == 2) return one_gemv<T, G, 2, 2, false>(&p, stream);
  return one_gemv<T, G, 4, 2, false>(&p, stream);
}
template <int T, int G>
cudaError_t set_attrs() {
  cudaError_t e = one_gemv<T, G, 1, 1, true>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 1, 2, true>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 1, 2, false>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 2, 2, false>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 4, 2, false>(nullptr, nullptr);
  return e;
}
template <int T>
struct GemvQ4 {
  static void go(int group, int eights, const GemvQ4Params& p, cudaStream_t stream) {
    if (group == 32) gemv_of<T, 32>(eights, p, stream);
    else if (group == 64) gemv_of<T, 64>(eights, p, stream);
    else gemv_of<T, 128>(eights, p, stream);
  }
  static cudaError_t set() {
    cudaError_t e = set_attrs<T, 32>();
    if (e == cudaSuccess) e = set_attrs<T, 64>();
    if (e == cudaSuccess) e = set_attrs<T, 128>();
    return e;
  }
};

}  // namespace

cudaError_t set_gemv_q4_attrs() {
  cudaError_t e = GemvQ4<kTypeF32>::set();
  if (e == cudaSuccess) e = GemvQ4<kTypeF16>::set();
  if (e == cudaSuccess) e = GemvQ4<kTypeBf16>::set();
  return e;
}
void launch_gemv_q4(int type, int group, int eights, const GemvQ4Params& p, cudaStream_t stream) {
  if (type == kTypeF32) GemvQ4<kTypeF32>::go(group, eights, p, stream);
  else if (type == kTypeF16) GemvQ4<kTypeF16>::go(group, eights, p, stream);
  else GemvQ4<kTypeBf16>::go(group, eights, p, stream);
}

}  // namespace tcec_host
