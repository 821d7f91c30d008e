// Launches of the product of few tokens with 4-bit weights (tcec_gemv_q4.cuh).
#include "tcec_gemv_q4.cuh"

#include "tcec_codes_launch.h"
#include "tcec_launch.h"

using namespace tcec_sm100;

namespace tcec_host {
namespace {

int ceil_div(int a, int b) { return (a - 1) / b + 1; }  // a > 0
// Launches for so many eights of columns and strips of rows a CTA, or (p null) allows the kernel its shared memory.
template <int T, int G, int E, int S, bool One>
cudaError_t one_gemv(const GemvQ4Params* p, cudaStream_t stream) {
  using Cfg = GemvQ4Cfg<T, G, E, S, One>;
  constexpr int kMost = Cfg::MOST_WARPS;
  if (!p) return cudaFuncSetAttribute(gemv_q4_kernel<T, G, E, S, One>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::smem_bytes(kMost));
  // CTAs that are more than the SMs are made as many for each of these, with a strip more or less: 16384 rows are 256 times four strips, eight for some
  // SMs and four for others, or 136 times four and 160 times three, seven for an SM (one FP32 token, groups of 64: 33.9 us, 36.7 so; 10000 x 10000 20.4
  // and 23.6; 5 bf16 tokens times 5000 x 7001 8.0 and 9.4).
  GemvQ4Params q = *p;
  const int strips = ceil_div(p->n, 16), least = ceil_div(strips, S), per_sm = Cfg::SHARED_OUT ? ceil_div(least, 148) : 1;
  const int ctas = per_sm == 1 ? least : 148 * per_sm < strips ? 148 * per_sm : strips;
  q.strips = per_sm == 1 ? S : strips / ctas;
  q.more = per_sm == 1 ? 0 : strips % ctas;
  const int warps = warps_of(ctas, Cfg::WARPS_OF_SM, 4, kMost);
  launch_early(gemv_q4_kernel<T, G, E, S, One>, ctas, 32 * warps, Cfg::smem_bytes(warps), stream, q);
  return cudaSuccess;
}
template <int T, int G>
cudaError_t gemv_of(int eights, const GemvQ4Params& p, cudaStream_t stream) {
  // What is done for x a CTA does once for all its strips.  One token: one strip while such CTAs fit the SMs, two likewise, then four, whose warps need
  // blocks to divide, though (bf16, with one, two and four: 2048 x 4096 3.5, 4.1, 5.7 us; 4096 x 4096 5.3, 4.9, 6.1; 5120 x 5120 8.1, 7.8, 7.2;
  // 8192 x 8192 14.3, 11.7, 10.6; 16384 x 16384 51, 37, 31; 12288 x 1024 4.8, 4.1, 4.2).
  if (!p.staged && p.n <= 148 * 16) return one_gemv<T, G, 1, 1, true>(&p, stream);
  if (!p.staged) return p.n <= 148 * 32 || p.blocks < 16 ? one_gemv<T, G, 1, 2, true>(&p, stream) : one_gemv<T, G, 1, 4, true>(&p, stream);
  // Five tokens, likewise: 2048 x 4096 5.3, 5.1, 6.4 us; 8192 x 8192 13.8, 11.0, 15.4; 12288 x 1024 5.9, 6.2, 5.1; 16384 x 16384 36, 37, 29.
  if (eights == 1) return p.n <= 148 * 64 ? one_gemv<T, G, 1, 2, false>(&p, stream) : one_gemv<T, G, 1, 4, false>(&p, stream);
  // A CTA of two strips does for its columns once what two of one strip do twice, but its SMs may stay idle at the end.  The work of a strip grows
  // with its groups, and a strip of two groups costs about what the columns do (12 tokens, groups of 128: 2048 rows of 4096 5.4 us with one strip,
  // 6.5 with two; 5000 rows of 7001 13.6 and 12.4; in groups of 32 15.9 and 17.8).
  constexpr int kSpans = kCodeSpan / G;
  const bool two = ceil_div(ceil_div(p.n, 32), 148) * (2 * kSpans + 2) <= ceil_div(ceil_div(p.n, 16), 148) * (kSpans + 2);
  if (eights == 2) return two ? one_gemv<T, G, 2, 2, false>(&p, stream) : one_gemv<T, G, 2, 1, false>(&p, stream);
  return two ? one_gemv<T, G, 4, 2, false>(&p, stream) : one_gemv<T, G, 4, 1, false>(&p, stream);
}
template <int T, int G>
cudaError_t set_attrs() {
  cudaError_t e = one_gemv<T, G, 1, 1, true>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 1, 2, true>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 1, 4, true>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 1, 2, false>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 1, 4, false>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 2, 2, false>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 4, 2, false>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 2, 1, false>(nullptr, nullptr);
  if (e == cudaSuccess) e = one_gemv<T, G, 4, 1, false>(nullptr, nullptr);
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
