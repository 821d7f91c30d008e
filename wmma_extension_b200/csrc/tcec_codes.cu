// Host side of the entry points for operands held in few bits (include/tcec.h): argument checks, kernel selection and launches.
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <mutex>

#include "tcec_codes.cuh"
#include "tcec_codes_launch.h"
#include "tcec_internal.h"
#include "tcec_launch.h"
#include "tcec_stage.cuh"

using namespace tcec_sm100;

namespace tcec_host {
namespace {

static_assert(TCEC_TYPE_F32 == kTypeF32 && TCEC_TYPE_F16 == kTypeF16 && TCEC_TYPE_BF16 == kTypeBf16, "types of tcec.h");

constexpr long long kMostBlocks = 0x7fffffffll;  // CTAs of a grid

bool bad_type(int t) { return t < 0 || t > 2; }
bool bad_group(int g) { return g != 32 && g != 64 && g != 128; }
int type_bytes(int t) { return t == TCEC_TYPE_F32 ? 4 : 2; }
long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// A dense matrix of the caller.
struct Dense {
  int layout, rows, cols;
  const void* p;
  long long ld;
  int type;
  long long row_step() const { return layout == TCEC_ROW_MAJOR ? ld : 1; }
  long long col_step() const { return layout == TCEC_ROW_MAJOR ? 1 : ld; }
  bool bad() const { return bad_layout(layout) || bad_type(type) || rows < 0 || cols < 0; }
  bool empty() const { return rows == 0 || cols == 0; }
  // Only of one that holds elements.
  bool bad_memory() const { return !p || !aligned(p, type_bytes(type)) || ld < (layout == TCEC_ROW_MAJOR ? cols : rows); }
  size_t extent() const {
    if (empty()) return 0;
    const long long outer = layout == TCEC_ROW_MAJOR ? rows : cols, inner = layout == TCEC_ROW_MAJOR ? cols : rows;
    return static_cast<size_t>((outer - 1) * ld + inner) * type_bytes(type);
  }
  // Whether its elements may be read or written `bytes` at a time from every multiple of that along a line.
  bool wide(size_t bytes) const { return aligned(p, bytes) && (ld * type_bytes(type)) % static_cast<long long>(bytes) == 0; }
};
bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na && nb && x < y + nb && y < x + na;
}
// Lines of one matrix may lie between those of another, as parts of a wider one.
bool overlap(const Dense& a, const Dense& b) {
  if (!overlap(a.p, a.extent(), b.p, b.extent())) return false;
  const size_t pitch = static_cast<size_t>(a.ld) * type_bytes(a.type);
  if (pitch != static_cast<size_t>(b.ld) * type_bytes(b.type)) return true;
  auto line = [](const Dense& d) { return static_cast<size_t>(d.layout == TCEC_ROW_MAJOR ? d.cols : d.rows) * type_bytes(d.type); };
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  const size_t off = x <= y ? (y - x) % pitch : (pitch - (x - y) % pitch) % pitch;  // of b's lines behind a's
  return off < line(a) || off + line(b) > pitch;
}

size_t q4_bytes(int n, int k, int group) {
  return static_cast<size_t>(ceil_div(n, kCodeRows)) * ceil_div(k, kCodeSpan) * q4_block_bytes(group);
}
size_t q8_bytes(int m, int k) { return static_cast<size_t>(ceil_div(k, kCodeRows)) * ceil_div(m, kCodeSpan) * kQ8BlockBytes; }
// Panels of a dense operand: `cols` columns, `sum` along the sum.
size_t panel_bytes(int cols, int sum, int type) {
  return static_cast<size_t>(ceil_div(cols, kCodeRows)) * ceil_div(sum, kCodeSpan) * (type == TCEC_TYPE_F32 ? 3 : 1) * kSpanBytes;
}

// What a launch needs to know of the current device, and of the options.
struct Here {
  int* status;
  int sm_count;
  int reserve_sms, debug_flags;
};
int get_here(Here* out) {
  const Options opt = snapshot_options();
  std::lock_guard<std::mutex> lock(state_mutex());
  DeviceState* st = nullptr;
  const int rc = get_device_state(&st);
  if (rc != TCEC_OK) return rc;
  if (!st->codes_attrs_done) {
    TCEC_CUDA(set_gemm_codes_attrs());
    TCEC_CUDA(set_gemv_q4_attrs());
    TCEC_CUDA(set_gemv_q8_attrs());
    st->codes_attrs_done = true;
  }
  *out = {st->status, st->sm_count, opt.reserve_sms, opt.debug_flags};
  return TCEC_OK;
}

// No exception leaves the library.
template <class Body>
int guarded(Body body) {
  try {
    return body();
  } catch (...) {
    return TCEC_ERR_ALLOC;
  }
}
int launched() { return cudaGetLastError() == cudaSuccess ? TCEC_OK : TCEC_ERR_CUDA; }

template <template <int> class Launch, class... Args>
void by_type(int type, const Args&... args) {
  if (type == TCEC_TYPE_F32) Launch<kTypeF32>::go(args...);
  else if (type == TCEC_TYPE_F16) Launch<kTypeF16>::go(args...);
  else Launch<kTypeBf16>::go(args...);
}

template <int T>
struct PackQ4 {
  template <int G>
  static void of(int grid, cudaStream_t stream, const PackQ4Params& p) {
    if (grid <= 148 * 4) launch_early(pack_q4_kernel<T, G, 1>, grid, 512, 0, stream, p);
    else launch_early(pack_q4_kernel<T, G, 2>, grid, 256, 0, stream, p);
  }
  static void go(int group, int grid, cudaStream_t stream, const PackQ4Params& p) {
    if (group == 32) of<32>(grid, stream, p);
    else if (group == 64) of<64>(grid, stream, p);
    else of<128>(grid, stream, p);
  }
};
template <int T>
struct UnpackQ4 {
  static void go(int group, int grid, cudaStream_t stream, const UnpackParams& p) {
    if (group == 32) launch_early(unpack_q4_kernel<T, 32>, grid, 256, 0, stream, p);
    else if (group == 64) launch_early(unpack_q4_kernel<T, 64>, grid, 256, 0, stream, p);
    else launch_early(unpack_q4_kernel<T, 128>, grid, 256, 0, stream, p);
  }
};
template <int T>
struct PackQ8 {
  static void go(int grid, cudaStream_t stream, const PackQ8Params& p) { launch_early(pack_q8_kernel<T>, grid, 256, 0, stream, p); }
};
template <int T>
struct UnpackQ8 {
  static void go(int grid, cudaStream_t stream, const UnpackParams& p) { launch_early(unpack_q8_kernel<T>, grid, 256, 0, stream, p); }
};
template <int T>
struct StageColumns {
  static void go(cudaStream_t stream, const StageColumnsParams& p) {
    const int parts = T == kTypeF32 ? 3 : 1, tokens = static_cast<int>(ceil_div(p.eights * 8, parts));
    launch_early(stage_columns_kernel<T>, p.blocks, (tokens * 16 + 31) / 32 * 32, 0, stream, p);
  }
};
template <int T>
struct StagePanels {
  static void go(int grid, cudaStream_t stream, const StagePanelsParams& p) { launch_early(stage_panels_kernel<T>, dim3(grid, 2), 256, 0, stream, p); }
};

// D[row][col] of tcec_gemm_codes.cuh for an operand of codes (spans: groups of 4-bit codes in a block, 0: 8-bit codes) and a dense one whose
// columns and sum lie at the given steps.
int gemm_codes(const void* codes, int spans, int rows, int cols, int sum, const void* dense, long long col_step, long long sum_step,
               int type, bool vec, float alpha, float beta, void* c, long long c_row, long long c_col, int c_type, void* workspace,
               const Here& here, cudaStream_t stream) {
  const int parts = type == TCEC_TYPE_F32 ? 3 : 1, blocks = static_cast<int>(ceil_div(sum, kCodeSpan));
  if (blocks) {
    StagePanelsParams sp{};
    sp.src = dense;
    sp.col_step = col_step;
    sp.sum_step = sum_step;
    sp.cols = cols;
    sp.sum = sum;
    sp.blocks = blocks;
    sp.panels = static_cast<uint8_t*>(workspace);
    sp.vec = vec;
    sp.pairs = type != TCEC_TYPE_F32 && col_step == 1 && !vec && cols % 2 == 0 && sum_step % 2 == 0 && aligned(dense, 4);
    by_type<StagePanels>(type, static_cast<int>(ceil_div(cols, kCodeRows) * blocks), stream, sp);
  }
  GemmCodesParams gp{};
  gp.codes = static_cast<const uint8_t*>(codes);
  gp.panels = static_cast<const uint8_t*>(workspace);
  gp.rows = rows;
  gp.cols = cols;
  gp.blocks = blocks;
  gp.parts = parts;
  gp.row_tiles = static_cast<int>(ceil_div(rows, 128));
  gp.alpha = alpha;
  gp.beta = beta;
  gp.c = c;
  gp.c_row = c_row;
  gp.c_col = c_col;
  gp.c_type = c_type;
  gp.status = here.status;
  gp.debug_flags = here.debug_flags;
  // Pairs of SMs with 256 columns make the most of each converted weight, but are half as many: they are taken where tiles of 128 columns would be
  // more than the SMs (4096 x 4096: 512 tokens, 128 such tiles, 25.8 us, in pairs 36.0; 768 tokens, 192 tiles, 43.4 and 35.7; 1000 45.2 and 38.9).
  int bn = cols <= 64 ? 64 : 128;
  if (cols > 128 && gp.row_tiles * ceil_div(cols, 128) > 148) bn = 256;
  gp.col_tiles = static_cast<int>(ceil_div(cols, bn));
  const long long tiles = (bn == 256 ? ceil_div(gp.row_tiles, 2) : gp.row_tiles) * static_cast<long long>(gp.col_tiles);
  if (tiles > kMostBlocks) return TCEC_ERR_UNSUPPORTED;
  int ctas = bn == 256 ? 2 : 1;  // of a cluster
  // Tiles too few for the SMs divide the sum among the CTAs of clusters.  Only as many clusters as surely run at a time: SMs that a GPC has over stay idle, and
  // 16 clusters of eight took two rounds where 15 took one (64 columns of 4096: 2048 rows 17.5 us, 1920 rows 9.8; with clusters of four 11.0);
  // of four, 35 did and 33 did not (4480 rows 22.1, 4224 rows 12.8).  Constants, as the order of the sums is to follow from sizes alone.
  constexpr long long kMostClusters[4] = {0, 74, 32, 14};  // of 2, 4 and 8 CTAs
  while (bn < 256 && ctas < 8 && !here.reserve_sms && tiles <= kMostClusters[ctas == 1 ? 1 : ctas == 2 ? 2 : 3] && blocks >= 4 * ctas) ctas *= 2;
  // One cluster a tile where the sum is divided; else as many as run at a time.
  const int sms = here.sm_count - here.reserve_sms;
  const long long most = bn == 256 ? sms / 2 : ctas > 1 ? tiles : sms;
  const int grid = static_cast<int>(tiles < most ? tiles : most) * ctas;
  launch_gemm_codes(type == TCEC_TYPE_F16, spans, bn, gp, ctas, grid, stream);
  return launched();
}

// Columns of the tensor-core operand that this many tokens take, and whether they are so few that the weights are streamed through registers
// (tcec_gemv_q4.cuh).  Up to 16 columns always: 16 tokens times 16384 x 16384 46 us, 17 74.  Up to 32 while the rows are few, as tiles of 128 rows then
// leave SMs idle: 24 tokens times 4096 x 4096 10.7 us, in tiles 12.7; 8192 x 4096 15.8 and 16.9; but 16384 x 1024 15.8 and 10.8.  FP32 in
// tiles has three parts to bring in: 10 tokens times 16384 x 16384 94 us, 11 160.
long long columns_of(int m, int type) { return static_cast<long long>(m) * (type == TCEC_TYPE_F32 ? 3 : 1); }
bool streamed(int m, int n, int type) { return columns_of(m, type) <= (n <= 8192 || type == TCEC_TYPE_F32 ? 32 : 16); }
// Whether a gradient has so few columns that the activations are streamed (tcec_gemv_q8.cuh), by the same reasons: 8192 x 4096 of rank 16 12.8 us, in
// tiles 18.3; of rank 32 20.5 and 18.6, 8192 x 1024 13.2 and 13.1, 1024 x 1024 5.4 and 7.8; FP32 of rank 10 18.8 and 29.3, 4096 x 16384 36 and 47.
bool few_columns(int n, int k, int type) { return columns_of(n, type) <= (k <= 148 * 16 || type == TCEC_TYPE_F32 ? 32 : 16); }
int eights_of(int m, int type) { return columns_of(m, type) <= 8 ? 1 : columns_of(m, type) <= 16 ? 2 : 4; }

}  // namespace
}  // namespace tcec_host

using namespace tcec_host;

extern "C" {

size_t tcec_q4_bytes(int n, int k, int group) { return n < 0 || k < 0 || bad_group(group) ? 0 : q4_bytes(n, k, group); }

int tcec_pack_q4(int layout_w, int n, int k, const void* w, long long ldw, int type_w, int group, int type_scale, void* packed, void* stream) {
  return guarded([&]() -> int {
    const Dense d{layout_w, n, k, w, ldw, type_w};
    if (d.bad() || bad_group(group) || (type_scale != TCEC_TYPE_F16 && type_scale != TCEC_TYPE_BF16)) return TCEC_ERR_INVALID_ARGUMENT;
    if (d.empty()) return TCEC_OK;
    if (d.bad_memory() || !packed || !aligned(packed, 16) || overlap(w, d.extent(), packed, q4_bytes(n, k, group))) return TCEC_ERR_INVALID_ARGUMENT;
    const long long tiles = ceil_div(n, kCodeRows), blocks = ceil_div(k, kCodeSpan);
    if (tiles * blocks > kMostBlocks) return TCEC_ERR_UNSUPPORTED;
    Here here;
    const int rc = get_here(&here);
    if (rc != TCEC_OK) return rc;
    PackQ4Params p{};
    p.w = w;
    p.row_step = d.row_step();
    p.k_step = d.col_step();
    p.n = n;
    p.k = k;
    p.scale_bf16 = type_scale == TCEC_TYPE_BF16;
    p.packed = static_cast<uint8_t*>(packed);
    p.blocks = static_cast<int>(blocks);
    p.vec = layout_w == TCEC_ROW_MAJOR && d.wide(4 * type_bytes(type_w));
    by_type<PackQ4>(type_w, group, static_cast<int>(tiles * blocks), static_cast<cudaStream_t>(stream), p);
    return launched();
  });
}

int tcec_pack_q4_codes(int n, int k, const unsigned char* codes, long long ld_codes, const void* scales, int type_scale,
                       const unsigned char* zeros, int group, void* packed, void* stream) {
  return guarded([&]() -> int {
    if (n < 0 || k < 0 || bad_group(group) || (type_scale != TCEC_TYPE_F16 && type_scale != TCEC_TYPE_BF16)) return TCEC_ERR_INVALID_ARGUMENT;
    if (n == 0 || k == 0) return TCEC_OK;
    if (!codes || !scales || !aligned(scales, 2) || ld_codes < ceil_div(k, 2) || !packed || !aligned(packed, 16)) return TCEC_ERR_INVALID_ARGUMENT;
    const long long tiles = ceil_div(n, kCodeRows), blocks = ceil_div(k, kCodeSpan), groups = ceil_div(k, group);
    const size_t out = q4_bytes(n, k, group);
    if (overlap(codes, static_cast<size_t>((n - 1) * ld_codes + ceil_div(k, 2)), packed, out) ||
        overlap(scales, static_cast<size_t>(n) * groups * 2, packed, out) ||
        (zeros && overlap(zeros, static_cast<size_t>(n) * groups, packed, out)))
      return TCEC_ERR_INVALID_ARGUMENT;
    if (tiles * blocks > kMostBlocks) return TCEC_ERR_UNSUPPORTED;
    Here here;
    const int rc = get_here(&here);
    if (rc != TCEC_OK) return rc;
    PackQ4Params p{};
    p.n = n;
    p.k = k;
    p.scale_bf16 = type_scale == TCEC_TYPE_BF16;
    p.packed = static_cast<uint8_t*>(packed);
    p.blocks = static_cast<int>(blocks);
    p.codes = codes;
    p.codes_ld = ld_codes;
    p.scales = scales;
    p.zeros = zeros;
    p.groups = static_cast<int>(groups);
    const int grid = static_cast<int>(tiles * blocks);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (group == 32) launch_early(pack_q4_codes_kernel<32>, grid, 256, 0, s, p);
    else if (group == 64) launch_early(pack_q4_codes_kernel<64>, grid, 256, 0, s, p);
    else launch_early(pack_q4_codes_kernel<128>, grid, 256, 0, s, p);
    return launched();
  });
}

int tcec_unpack_q4(int layout_w, int n, int k, const void* packed, int group, void* w, long long ldw, int type_w, void* stream) {
  return guarded([&]() -> int {
    const Dense d{layout_w, n, k, w, ldw, type_w};
    if (d.bad() || bad_group(group)) return TCEC_ERR_INVALID_ARGUMENT;
    if (d.empty()) return TCEC_OK;
    if (d.bad_memory() || !packed || !aligned(packed, 16) || overlap(w, d.extent(), packed, q4_bytes(n, k, group))) return TCEC_ERR_INVALID_ARGUMENT;
    const long long tiles = ceil_div(n, kCodeRows), blocks = ceil_div(k, kCodeSpan);
    if (tiles * blocks > kMostBlocks) return TCEC_ERR_UNSUPPORTED;
    Here here;
    const int rc = get_here(&here);
    if (rc != TCEC_OK) return rc;
    UnpackParams p{};
    p.packed = static_cast<const uint8_t*>(packed);
    p.out = w;
    p.row_step = d.row_step();
    p.sum_step = d.col_step();
    p.rows = n;
    p.sum = k;
    p.blocks = static_cast<int>(blocks);
    p.vec = layout_w == TCEC_ROW_MAJOR && d.wide(4 * type_bytes(type_w));
    by_type<UnpackQ4>(type_w, group, static_cast<int>(tiles * blocks), static_cast<cudaStream_t>(stream), p);
    return launched();
  });
}

size_t tcec_gemm_q4_workspace_bytes(int m, int n, int k, int type_x) {
  if (m < 0 || n < 0 || k < 0 || bad_type(type_x) || m <= 1) return 0;
  if (streamed(m, n, type_x)) return static_cast<size_t>(staged_bytes(ceil_div(k, kCodeSpan), eights_of(m, type_x)));
  return panel_bytes(m, k, type_x);
}

int tcec_gemm_q4(int layout_x, int layout_c, int m, int n, int k, float alpha, const void* x, long long ldx, int type_x, const void* packed,
                 int group, float beta, void* c, long long ldc, int type_c, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    const Dense dx{layout_x, m, k, x, ldx, type_x}, dc{layout_c, m, n, c, ldc, type_c};
    if (dx.bad() || dc.bad() || bad_group(group) || (type_c != type_x && type_c != TCEC_TYPE_F32)) return TCEC_ERR_INVALID_ARGUMENT;
    if (dc.empty()) return TCEC_OK;
    if (dc.bad_memory()) return TCEC_ERR_INVALID_ARGUMENT;
    const int sum = alpha == 0.f ? 0 : k;  // as without a product, X and W are then not read
    if (!sum) alpha = 0.f;                 // which may be no number, and times a sum over nothing is to be nothing
    const size_t scratch = sum ? tcec_gemm_q4_workspace_bytes(m, n, sum, type_x) : 0;
    if (sum) {
      if (dx.bad_memory() || !packed || !aligned(packed, 16) || workspace_bytes < scratch || (scratch && (!workspace || !aligned(workspace, 16))))
        return TCEC_ERR_INVALID_ARGUMENT;
      if (overlap(dc, dx) || overlap(c, dc.extent(), packed, q4_bytes(n, k, group)) ||
          overlap(workspace, scratch, x, dx.extent()) || overlap(workspace, scratch, c, dc.extent()) ||
          overlap(workspace, scratch, packed, q4_bytes(n, k, group)))
        return TCEC_ERR_INVALID_ARGUMENT;
    }
    if (ceil_div(m, kCodeRows) * ceil_div(k, kCodeSpan) > kMostBlocks) return TCEC_ERR_UNSUPPORTED;
    Here here;
    const int rc = get_here(&here);
    if (rc != TCEC_OK) return rc;
    if (!streamed(m, n, type_x) || (m > 1 && !sum))  // without a sum there is no workspace to stage tokens in
      return gemm_codes(packed, kCodeSpan / group, n, m, sum, x, dx.row_step(), dx.col_step(), type_x, layout_x == TCEC_ROW_MAJOR && dx.wide(16), alpha,
                        beta, c, dc.col_step(), dc.row_step(), type_c, workspace, here, static_cast<cudaStream_t>(stream));
    const cudaStream_t on = static_cast<cudaStream_t>(stream);
    const int blocks = static_cast<int>(ceil_div(sum, kCodeSpan)), eights = eights_of(m, type_x);
    if (m > 1) {
      StageColumnsParams sp{};
      sp.src = x;
      sp.col_step = dx.row_step();
      sp.sum_step = dx.col_step();
      sp.tokens = m;
      sp.sum = sum;
      sp.blocks = blocks;
      sp.eights = eights;
      sp.group = group;
      sp.out = static_cast<uint8_t*>(workspace);
      sp.vec = layout_x == TCEC_ROW_MAJOR && dx.wide(16);
      by_type<StageColumns>(type_x, on, sp);
    }
    GemvQ4Params p{};
    p.codes = static_cast<const uint8_t*>(packed);
    p.staged = m > 1 ? static_cast<const uint8_t*>(workspace) : nullptr;
    p.x = x;
    p.x_k = dx.col_step();
    p.n = n;
    p.k = sum;
    p.tokens = m;
    p.blocks = blocks;
    p.vec = layout_x == TCEC_ROW_MAJOR && dx.wide(4 * type_bytes(type_x));
    p.alpha = alpha;
    p.beta = beta;
    p.c = c;
    p.c_token = dc.row_step();
    p.c_row = dc.col_step();
    p.c_type = type_c;
    p.status = here.status;
    p.debug_flags = here.debug_flags;
    launch_gemv_q4(type_x, group, eights, p, on);
    return launched();
  });
}

size_t tcec_q8_bytes(int m, int k) { return m < 0 || k < 0 ? 0 : q8_bytes(m, k); }

int tcec_pack_q8(int layout_x, int m, int k, const void* x, long long ldx, int type_x, void* packed, void* stream) {
  return guarded([&]() -> int {
    const Dense d{layout_x, m, k, x, ldx, type_x};
    if (d.bad()) return TCEC_ERR_INVALID_ARGUMENT;
    if (d.empty()) return TCEC_OK;
    if (d.bad_memory() || !packed || !aligned(packed, 16) || overlap(x, d.extent(), packed, q8_bytes(m, k))) return TCEC_ERR_INVALID_ARGUMENT;
    const long long tiles = ceil_div(k, kCodeRows), blocks = ceil_div(m, kCodeSpan);
    if (tiles * blocks > kMostBlocks) return TCEC_ERR_UNSUPPORTED;
    Here here;
    const int rc = get_here(&here);
    if (rc != TCEC_OK) return rc;
    PackQ8Params p{};
    p.x = x;
    p.token_step = d.row_step();
    p.feature_step = d.col_step();
    p.tokens = m;
    p.features = k;
    p.token_blocks = static_cast<int>(blocks);
    p.packed = static_cast<uint8_t*>(packed);
    p.vec = layout_x == TCEC_ROW_MAJOR && d.wide(4 * type_bytes(type_x));
    by_type<PackQ8>(type_x, static_cast<int>(tiles * blocks), static_cast<cudaStream_t>(stream), p);
    return launched();
  });
}

int tcec_unpack_q8(int layout_x, int m, int k, const void* packed, void* x, long long ldx, int type_x, void* stream) {
  return guarded([&]() -> int {
    const Dense d{layout_x, m, k, x, ldx, type_x};
    if (d.bad()) return TCEC_ERR_INVALID_ARGUMENT;
    if (d.empty()) return TCEC_OK;
    if (d.bad_memory() || !packed || !aligned(packed, 16) || overlap(x, d.extent(), packed, q8_bytes(m, k))) return TCEC_ERR_INVALID_ARGUMENT;
    const long long tiles = ceil_div(k, kCodeRows), blocks = ceil_div(m, kCodeSpan);
    if (tiles * blocks > kMostBlocks) return TCEC_ERR_UNSUPPORTED;
    Here here;
    const int rc = get_here(&here);
    if (rc != TCEC_OK) return rc;
    UnpackParams p{};
    p.packed = static_cast<const uint8_t*>(packed);
    p.out = x;
    p.row_step = d.col_step();  // rows of the codes are features
    p.sum_step = d.row_step();
    p.rows = k;
    p.sum = m;
    p.blocks = static_cast<int>(blocks);
    p.vec = layout_x == TCEC_ROW_MAJOR && d.wide(4 * type_bytes(type_x));
    by_type<UnpackQ8>(type_x, static_cast<int>(tiles * blocks), static_cast<cudaStream_t>(stream), p);
    return launched();
  });
}

size_t tcec_wgrad_q8_workspace_bytes(int m, int n, int k, int type_dy) {
  if (m < 0 || n < 0 || k < 0 || bad_type(type_dy)) return 0;
  if (few_columns(n, k, type_dy)) return static_cast<size_t>(staged_bytes(ceil_div(m, kCodeSpan), eights_of(n, type_dy)));
  return panel_bytes(n, m, type_dy);
}

int tcec_wgrad_q8(int layout_dy, int layout_c, int m, int n, int k, float alpha, const void* dy, long long lddy, int type_dy, const void* packed,
                  float beta, void* c, long long ldc, int type_c, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    const Dense dd{layout_dy, m, n, dy, lddy, type_dy}, dc{layout_c, n, k, c, ldc, type_c};
    if (dd.bad() || dc.bad() || (type_c != type_dy && type_c != TCEC_TYPE_F32)) return TCEC_ERR_INVALID_ARGUMENT;
    if (dc.empty()) return TCEC_OK;
    if (dc.bad_memory()) return TCEC_ERR_INVALID_ARGUMENT;
    const int sum = alpha == 0.f ? 0 : m;
    if (!sum) alpha = 0.f;
    const size_t scratch = sum ? tcec_wgrad_q8_workspace_bytes(sum, n, k, type_dy) : 0;
    if (sum) {
      if (dd.bad_memory() || !packed || !aligned(packed, 16) || workspace_bytes < scratch || !workspace || !aligned(workspace, 16))
        return TCEC_ERR_INVALID_ARGUMENT;
      if (overlap(dc, dd) || overlap(c, dc.extent(), packed, q8_bytes(m, k)) ||
          overlap(workspace, scratch, dy, dd.extent()) || overlap(workspace, scratch, c, dc.extent()) ||
          overlap(workspace, scratch, packed, q8_bytes(m, k)))
        return TCEC_ERR_INVALID_ARGUMENT;
    }
    if (ceil_div(n, kCodeRows) * ceil_div(m, kCodeSpan) > kMostBlocks) return TCEC_ERR_UNSUPPORTED;
    Here here;
    const int rc = get_here(&here);
    if (rc != TCEC_OK) return rc;
    // columns: the outputs of the layer; the sum: tokens
    if (sum && few_columns(n, k, type_dy)) {
      const cudaStream_t on = static_cast<cudaStream_t>(stream);
      const int blocks = static_cast<int>(ceil_div(sum, kCodeSpan)), eights = eights_of(n, type_dy);
      StageColumnsParams sp{};
      sp.src = dy;
      sp.col_step = dd.col_step();
      sp.sum_step = dd.row_step();
      sp.tokens = n;
      sp.sum = sum;
      sp.blocks = blocks;
      sp.eights = eights;
      sp.group = kCodeSpan;
      sp.out = static_cast<uint8_t*>(workspace);
      sp.vec = layout_dy == TCEC_COL_MAJOR && dd.wide(16);
      by_type<StageColumns>(type_dy, on, sp);
      GemvQ8Params p{};
      p.codes = static_cast<const uint8_t*>(packed);
      p.staged = static_cast<const uint8_t*>(workspace);
      p.rows = k;
      p.cols = n;
      p.blocks = blocks;
      p.alpha = alpha;
      p.beta = beta;
      p.c = c;
      p.c_row = dc.col_step();
      p.c_col = dc.row_step();
      p.c_type = type_c;
      p.status = here.status;
      p.debug_flags = here.debug_flags;
      launch_gemv_q8(type_dy, eights, here.reserve_sms ? here.sm_count - here.reserve_sms : 0, p, on);
      return launched();
    }
    return gemm_codes(packed, 0, k, n, sum, dy, dd.col_step(), dd.row_step(), type_dy, layout_dy == TCEC_COL_MAJOR && dd.wide(16), alpha,
                      beta, c, dc.col_step(), dc.row_step(), type_c, workspace, here, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
