// block_capi.cu — the extern "C" entry points of the block operators (layer
// norm, linears with adapters): argument validation, workspace carving and
// launch sequences.
#include <climits>
#include <cmath>

#include "attn_common.h"
#include "gemm.h"

namespace fa {

#define FA_TRY(expr)              \
  do {                            \
    int _rc = (expr);             \
    if (_rc != FA_OK) return _rc; \
  } while (0)

static int check_dtype(int dtype) {
  return dtype == FA_DTYPE_F32 || dtype == FA_DTYPE_BF16 ? FA_OK : FA_ERR_UNSUPPORTED;
}

constexpr int kMaxNormDim = 16384;

static int check_norm(int dtype, int groups, int rows, int dim, int par_dtype, int64_t ps) {
  FA_TRY(check_dtype(dtype));
  FA_TRY(check_dtype(par_dtype));
  if (groups < 0 || rows < 0 || dim <= 0 || ps < 0) return FA_ERR_INVALID_ARG;
  if (dim > kMaxNormDim || groups > 65535 || (int64_t)groups * rows >= INT32_MAX)
    return FA_ERR_TOO_LARGE;
  return FA_OK;
}

// element-aligned, contiguous last dimension (the kernels pick the access width)
static int check_rows(const fa_tensor_t* t, int es) {
  if (t == nullptr || t->data == nullptr) return FA_ERR_INVALID_ARG;
  if (t->stride_d != 1 || reinterpret_cast<uintptr_t>(t->data) % es != 0) return FA_ERR_ALIGNMENT;
  return FA_OK;
}

// (rows, cols) with rows that start on 16 bytes and do not overlap (a TMA
// descriptor's strides span their dimension)
static int check_matrix(const fa_matrix_t* m, int64_t rows, int64_t cols) {
  if (m == nullptr || m->data == nullptr) return FA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(m->data) % 16 != 0 || m->stride_row % 8 != 0 ||
      m->stride_batch % 8 != 0 || m->stride_row < 0 || m->stride_batch < 0)
    return FA_ERR_ALIGNMENT;
  return rows > 1 && m->stride_row < cols ? FA_ERR_ALIGNMENT : FA_OK;
}

constexpr int kMaxRank = 256;
constexpr int kMaxSteps = 64;
// Rows that another request's broken factor reached are multiplied again under the
// next tile's bounded wait (2e9 cycles): 430 cycles a tile and column of x with
// all SMs at it, a quarter of the wait at this width.
constexpr int kMaxInMany = 1 << 20;

static int check_lora(int dtype, int rows, int in_dim, int out_dim, int rank, float scale) {
  if (dtype != FA_DTYPE_BF16) return FA_ERR_UNSUPPORTED;
  if (rows < 0 || in_dim <= 0 || out_dim <= 0 || rank <= 0) return FA_ERR_INVALID_ARG;
  if (rank > kMaxRank) return FA_ERR_UNSUPPORTED;
  if (!std::isfinite(scale)) return FA_ERR_INVALID_ARG;
  if (rows > (1 << 30) || in_dim > (1 << 24) || out_dim > (1 << 24)) return FA_ERR_TOO_LARGE;
  return FA_OK;
}

static Mat3 mat(const fa_matrix_t* m, int64_t batch, int64_t rows, int64_t cols) {
  return Mat3{m->data, batch, rows, cols, m->stride_batch, m->stride_row, 1};
}

static Mat3 dense(const void* p, int64_t rows, int64_t cols, int64_t ld) {
  return Mat3{const_cast<void*>(p), 1, rows, cols, rows * ld, ld, 1};
}

static int low_dim(int rank) { return (rank + 15) / 16 * 16; }
static size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

static const __nv_bfloat16* bfp(const void* p) { return reinterpret_cast<const __nv_bfloat16*>(p); }

// Up to 64 rows four warps per inner product beat the tensor-core form's fixed
// cost (at 4096, rank 16: 64 rows 4.4 us against 8.3 us). With many adapters
// the other form also needs a plan of the rows first: up to 256 there.
constexpr int kDotRows = 64;
constexpr int kDotRowsMany = 256;

}  // namespace fa

using namespace fa;

extern "C" {

int fa_layer_norm_fwd(int dtype, int groups, int rows, int dim, const fa_tensor_t* x,
                      const void* weight, const void* bias, int par_dtype, int64_t param_stride,
                      int unit_offset, float eps, const fa_tensor_t* y, float* stats,
                      void* stream) {
  FA_TRY(check_norm(dtype, groups, rows, dim, par_dtype, param_stride));
  if (!(eps >= 0.f) || !std::isfinite(eps)) return FA_ERR_INVALID_ARG;
  if ((int64_t)groups * rows == 0) return FA_OK;
  const int es = dtype == FA_DTYPE_BF16 ? 2 : 4, ps = par_dtype == FA_DTYPE_BF16 ? 2 : 4;
  FA_TRY(check_rows(x, es));
  FA_TRY(check_rows(y, es));
  for (const void* p : {weight, bias, (const void*)stats})
    if (reinterpret_cast<uintptr_t>(p) % (p == stats ? 4 : ps) != 0) return FA_ERR_ALIGNMENT;
  FA_TRY(check_sm100());
  return launch_layer_norm_fwd(dtype, groups, rows, dim, x, weight, bias, par_dtype, param_stride,
                               unit_offset, eps, y, stats, reinterpret_cast<cudaStream_t>(stream));
}

size_t fa_layer_norm_bwd_workspace_bytes(int groups, int rows, int dim) {
  if (groups <= 0 || rows < 0 || dim <= 0) return 0;
  return layer_norm_bwd_workspace(groups, rows, dim);
}

int fa_layer_norm_bwd(int dtype, int groups, int rows, int dim, const fa_tensor_t* x,
                      const void* weight, int par_dtype, int64_t param_stride, int unit_offset,
                      const fa_tensor_t* dy, const float* stats, const fa_tensor_t* dx,
                      float* dweight, float* dbias, void* workspace, size_t workspace_bytes,
                      void* stream) {
  FA_TRY(check_norm(dtype, groups, rows, dim, par_dtype, param_stride));
  const int es = dtype == FA_DTYPE_BF16 ? 2 : 4, ps = par_dtype == FA_DTYPE_BF16 ? 2 : 4;
  if ((int64_t)groups * rows > 0) {
    FA_TRY(check_rows(x, es));
    FA_TRY(check_rows(dy, es));
    FA_TRY(check_rows(dx, es));
    if (stats == nullptr) return FA_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(weight) % ps != 0 ||
        reinterpret_cast<uintptr_t>(stats) % 4 != 0)
      return FA_ERR_ALIGNMENT;
  }
  for (const void* p : {(const void*)dweight, (const void*)dbias, (const void*)workspace})
    if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return FA_ERR_ALIGNMENT;
  FA_TRY(check_sm100());
  const size_t need = fa_layer_norm_bwd_workspace_bytes(groups, rows, dim);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return FA_ERR_WORKSPACE;
  const fa_tensor_t none{};
  if ((int64_t)groups * rows == 0) x = dy = dx = &none;  // nothing is read: only sums of nothing
  return launch_layer_norm_bwd(dtype, groups, rows, dim, x, weight, par_dtype, param_stride,
                               unit_offset, dy, stats, dx, dweight, dbias, param_stride == 0,
                               workspace, reinterpret_cast<cudaStream_t>(stream));
}

int fa_lora_linear_fwd(int dtype, int rows, int in_dim, int out_dim, int rank,
                       const fa_matrix_t* x, const fa_matrix_t* w, const fa_matrix_t* a,
                       const fa_matrix_t* b, float scale, const void* bias,
                       const fa_matrix_t* y, void* low, void* stream) {
  FA_TRY(check_lora(dtype, rows, in_dim, out_dim, rank, scale));
  if (rows == 0) return FA_OK;
  FA_TRY(check_matrix(x, rows, in_dim));
  FA_TRY(check_matrix(w, out_dim, in_dim));
  FA_TRY(check_matrix(a, rank, in_dim));
  FA_TRY(check_matrix(b, out_dim, rank));
  FA_TRY(check_matrix(y, rows, out_dim));
  if (low == nullptr) return FA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(low) % 16 != 0 || reinterpret_cast<uintptr_t>(bias) % 2 != 0)
    return FA_ERR_ALIGNMENT;
  FA_TRY(check_sm100());
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int ld = low_dim(rank);
  __nv_bfloat16* lw = reinterpret_cast<__nv_bfloat16*>(low);
  // the product starts while the low-rank factor's kernel runs (which itself
  // starts when all earlier work is done) and waits for it where it needs it
  if (rows <= kDotRows) {
    FA_TRY(launch_low_rows(bfp(x->data), x->stride_row, bfp(a->data), 0, a->stride_row, nullptr, 1,
                           nullptr, scale, rows, in_dim, rank, ld, lw, 2 * ld, ld, st));
  } else {
    SkinnyParams s;
    s.rows = rows;
    s.cols = s.n = s.low_ld = ld;
    s.rank = rank;
    s.K = in_dim;
    s.out = lw;
    s.out_ld = 2 * ld;
    s.lo_at = ld;
    s.scale = scale;
    FA_TRY(launch_gemm_skinny(mat(x, 1, rows, in_dim), false, mat(a, 1, rank, in_dim), false, s,
                              kSkinnyLow, false, st));
  }
  if (linear_as_columns(out_dim, in_dim, rows)) {
    SkinnyParams s;
    s.rows = out_dim;
    s.cols = rows;
    s.K = in_dim;
    s.out = reinterpret_cast<__nv_bfloat16*>(y->data);
    s.out_ld = y->stride_row;
    s.bias = bfp(bias);
    s.low = lw;
    s.low_ld = ld;
    s.low_stride = 2 * ld;
    s.rank = rank;
    return launch_gemm_skinny(mat(w, 1, out_dim, in_dim), false, mat(x, 1, rows, in_dim), false, s,
                              kSkinnyCols, true, st, mat(b, 1, out_dim, rank));
  }
  WideOperands o;
  o.a = mat(x, 1, rows, in_dim);
  o.b = mat(w, 1, out_dim, in_dim);
  o.e = mat(b, 1, out_dim, rank);
  o.d = mat(y, 1, rows, out_dim);
  WideParams p;
  p.M = rows;
  p.N = out_dim;
  p.K = in_dim;
  p.low = lw;
  p.low_ld = ld;
  p.low_stride = 2 * ld;
  p.rank = rank;
  p.early = 1;
  p.bias = bfp(bias);
  return launch_gemm_wide(o, p, kEpiLinear, st);
}

size_t fa_lora_linear_bwd_workspace_bytes(int rows, int rank) {
  if (rows <= 0 || rank <= 0) return 0;
  return (size_t)rows * low_dim(rank) * 4;
}

int fa_lora_linear_bwd(int dtype, int rows, int in_dim, int out_dim, int rank,
                       const fa_matrix_t* x, const fa_matrix_t* w, const fa_matrix_t* a,
                       const fa_matrix_t* b, float scale, const void* low,
                       const fa_matrix_t* dy, const fa_matrix_t* dx, void* da, void* db,
                       void* workspace, size_t workspace_bytes, void* stream) {
  FA_TRY(check_lora(dtype, rows, in_dim, out_dim, rank, scale));
  if ((da == nullptr) != (db == nullptr)) return FA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(da) % 2 != 0 || reinterpret_cast<uintptr_t>(db) % 2 != 0)
    return FA_ERR_ALIGNMENT;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {  // sums of nothing
    FA_TRY(check_sm100());
    if (da != nullptr) {
      FA_TRY(record_cuda_error(cudaMemsetAsync(da, 0, (size_t)rank * in_dim * 2, st)));
      FA_TRY(record_cuda_error(cudaMemsetAsync(db, 0, (size_t)rank * out_dim * 2, st)));
    }
    return FA_OK;
  }
  FA_TRY(check_matrix(b, out_dim, rank));
  FA_TRY(check_matrix(dy, rows, out_dim));
  if (dx != nullptr) {
    FA_TRY(check_matrix(w, out_dim, in_dim));
    FA_TRY(check_matrix(a, rank, in_dim));
    FA_TRY(check_matrix(dx, rows, in_dim));
  }
  if (da != nullptr) {
    FA_TRY(check_matrix(x, rows, in_dim));
    if (low == nullptr) return FA_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(low) % 16 != 0) return FA_ERR_ALIGNMENT;
  }
  const size_t need = fa_lora_linear_bwd_workspace_bytes(rows, rank);
  if (workspace == nullptr || workspace_bytes < need) return FA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return FA_ERR_ALIGNMENT;
  FA_TRY(check_sm100());
  const int ld = low_dim(rank);
  __nv_bfloat16* u = reinterpret_cast<__nv_bfloat16*>(workspace);
  // every kernel after the first starts early and waits for the one before it
  {  // U = scale dy B
    SkinnyParams s;
    s.rows = rows;
    s.cols = s.n = s.low_ld = ld;
    s.rank = rank;
    s.K = out_dim;
    s.out = u;
    s.out_ld = 2 * ld;
    s.lo_at = ld;
    s.scale = scale;
    FA_TRY(launch_gemm_skinny(mat(dy, 1, rows, out_dim), false, mat(b, 1, out_dim, rank), true, s,
                              kSkinnyLow, false, st));
  }
  if (da != nullptr) {
    SkinnyParams s;
    s.cols = rank;
    s.n = ld;
    s.K = rows;
    s.rows = in_dim;  // da = (x^T U)^T
    s.out = reinterpret_cast<__nv_bfloat16*>(da);
    s.out_ld = 1;
    s.out_j = in_dim;
    s.rows2 = out_dim;  // db = dy^T low
    s.out2 = reinterpret_cast<__nv_bfloat16*>(db);
    s.out_ld2 = rank;
    s.out_j2 = 1;
    const Mat3 big[2] = {mat(x, 1, rows, in_dim), mat(dy, 1, rows, out_dim)};
    const Mat3 small[2] = {dense(u, rows, ld, 2 * ld), dense(low, rows, ld, 2 * ld)};
    const Mat3 rest[2] = {dense(u + ld, rows, ld, 2 * ld), dense(bfp(low) + ld, rows, ld, 2 * ld)};
    FA_TRY(launch_skinny_grads(big, small, rest, s, st));
  }
  if (dx == nullptr) return FA_OK;
  if (linear_as_columns(in_dim, out_dim, rows)) {
    SkinnyParams s;
    s.rows = in_dim;
    s.cols = rows;
    s.K = out_dim;
    s.out = reinterpret_cast<__nv_bfloat16*>(dx->data);
    s.out_ld = dx->stride_row;
    s.low = u;
    s.low_ld = ld;
    s.low_stride = 2 * ld;
    s.rank = rank;
    return launch_gemm_skinny(mat(w, 1, out_dim, in_dim), true, mat(dy, 1, rows, out_dim), false, s,
                              kSkinnyCols, true, st, mat(a, 1, rank, in_dim));
  }
  WideOperands o;
  o.b_mn = true;
  o.a = mat(dy, 1, rows, out_dim);
  o.b = mat(w, 1, out_dim, in_dim);
  o.e = mat(a, 1, rank, in_dim);
  o.d = mat(dx, 1, rows, in_dim);
  WideParams p;
  p.M = rows;
  p.N = in_dim;
  p.K = out_dim;
  p.low = u;
  p.low_ld = ld;
  p.low_stride = 2 * ld;
  p.rank = rank;
  p.early = 1;
  return launch_gemm_wide(o, p, kEpiLinear, st);
}

int fa_pad_rows(int64_t rows, int cols, const void* src, int64_t src_stride, void* dst,
                int64_t dst_stride, void* stream) {
  if (rows < 0 || cols <= 0 || src_stride < 0 || dst_stride < cols) return FA_ERR_INVALID_ARG;
  if (rows == 0) return FA_OK;
  if (src == nullptr || dst == nullptr) return FA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(src) % 2 != 0 || reinterpret_cast<uintptr_t>(dst) % 2 != 0)
    return FA_ERR_ALIGNMENT;
  if (rows * cols >= (int64_t)1 << 38) return FA_ERR_TOO_LARGE;
  FA_TRY(check_sm100());
  return launch_pad_rows(rows, cols, src, src_stride, dst, dst_stride,
                         reinterpret_cast<cudaStream_t>(stream));
}

// [low (rows, low_dim) bf16 | per-256-row counts | their adapters | slots]
size_t fa_lora_linear_many_workspace_bytes(int rows, int rank) {
  if (rows <= 0 || rank <= 0) return 0;
  size_t total = align256((size_t)rows * low_dim(rank) * 2);
  const size_t blocks = ((size_t)rows + 255) / 256;
  total += align256(blocks * 4) + align256(blocks * 256 * 4) + align256((size_t)rows * 4);
  return total;
}

int fa_lora_linear_many(int dtype, int rows, int in_dim, int out_dim, int rank, int n_adapters,
                        const fa_matrix_t* x, const fa_matrix_t* w, const fa_matrix_t* a,
                        const fa_matrix_t* b, const int32_t* ids, const float* scales,
                        const void* bias, const fa_matrix_t* y, void* workspace,
                        size_t workspace_bytes, void* stream) {
  FA_TRY(check_lora(dtype, rows, in_dim, out_dim, rank, 1.f));
  if (n_adapters <= 0) return FA_ERR_INVALID_ARG;
  if (in_dim > kMaxInMany) return FA_ERR_TOO_LARGE;
  if (rows == 0) return FA_OK;
  FA_TRY(check_matrix(x, rows, in_dim));
  FA_TRY(check_matrix(w, out_dim, in_dim));
  FA_TRY(check_matrix(a, rank, in_dim));
  FA_TRY(check_matrix(b, out_dim, rank));
  FA_TRY(check_matrix(y, rows, out_dim));
  if (ids == nullptr || scales == nullptr) return FA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(ids) % 4 != 0 || reinterpret_cast<uintptr_t>(scales) % 4 != 0 ||
      reinterpret_cast<uintptr_t>(bias) % 2 != 0)
    return FA_ERR_ALIGNMENT;
  const size_t need = fa_lora_linear_many_workspace_bytes(rows, rank);
  if (workspace == nullptr || workspace_bytes < need) return FA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return FA_ERR_ALIGNMENT;
  if (n_adapters > 1 && (a->stride_batch < in_dim || b->stride_batch < rank))
    return FA_ERR_ALIGNMENT;
  FA_TRY(check_sm100());
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int ld = low_dim(rank);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  __nv_bfloat16* low = reinterpret_cast<__nv_bfloat16*>(ws);
  ws += align256((size_t)rows * ld * 2);
  const size_t blocks = ((size_t)rows + 255) / 256;
  int* cnt = reinterpret_cast<int*>(ws);
  ws += align256(blocks * 4);
  int* list = reinterpret_cast<int*>(ws);
  ws += align256(blocks * 256 * 4);
  int* slot = reinterpret_cast<int*>(ws);
  const bool dots = rows <= kDotRowsMany;
  const bool columns = linear_as_columns(out_dim, in_dim, rows, n_adapters, rank);
  if (!dots || !columns) FA_TRY(launch_adapter_plan(ids, rows, n_adapters, cnt, list, slot, st));
  if (dots) {
    FA_TRY(launch_low_rows(bfp(x->data), x->stride_row, bfp(a->data), a->stride_batch,
                           a->stride_row, ids, n_adapters, scales, 1.f, rows, in_dim, rank, ld, low,
                           ld, 0, st));
  } else {
    SkinnyParams s;
    s.rows = rows;
    s.cols = s.n = s.low_ld = ld;
    s.rank = rank;
    s.K = in_dim;
    s.E = n_adapters;
    s.out = low;
    s.out_ld = ld;
    s.scales = scales;
    s.list_cnt = cnt;
    s.list_ids = list;
    s.slot = slot;
    FA_TRY(launch_gemm_skinny(mat(x, 1, rows, in_dim), false, mat(a, n_adapters, rank, in_dim),
                              false, s, kSkinnyLow, false, st));
  }
  if (columns) {
    SkinnyParams s;
    s.rows = out_dim;
    s.cols = rows;
    s.K = in_dim;
    s.out = reinterpret_cast<__nv_bfloat16*>(y->data);
    s.out_ld = y->stride_row;
    s.bias = bfp(bias);
    s.low = low;
    s.low_ld = ld;
    s.low_stride = ld;
    s.rank = rank;
    s.E = n_adapters;
    s.ids = ids;
    s.raw_x = bfp(x->data);
    s.raw_ldx = x->stride_row;
    s.raw_w = bfp(w->data);
    s.raw_ldw = w->stride_row;
    s.raw_f = bfp(b->data);
    s.raw_fe = b->stride_batch;
    s.raw_ldf = b->stride_row;
    return launch_gemm_skinny(mat(w, 1, out_dim, in_dim), false, mat(x, 1, rows, in_dim), false, s,
                              kSkinnyCols, true, st, mat(b, n_adapters, out_dim, rank));
  }
  WideOperands o;
  o.a = mat(x, 1, rows, in_dim);
  o.b = mat(w, 1, out_dim, in_dim);
  o.e = mat(b, n_adapters, out_dim, rank);
  o.d = mat(y, 1, rows, out_dim);
  WideParams p;
  p.M = rows;
  p.N = out_dim;
  p.K = in_dim;
  p.low = low;
  p.low_ld = ld;
  p.low_stride = ld;
  p.rank = rank;
  p.list_cnt = cnt;
  p.list_ids = list;
  p.slot = slot;
  p.early = 1;
  p.raw_x = bfp(x->data);
  p.raw_ldx = x->stride_row;
  p.raw_w = bfp(w->data);
  p.raw_ldw = w->stride_row;
  p.raw_f = bfp(b->data);
  p.raw_fe = b->stride_batch;
  p.raw_ldf = b->stride_row;
  p.bias = bfp(bias);
  return launch_gemm_wide(o, p, kEpiLinear, st);
}

size_t fa_orthogonalize_workspace_bytes(int batch, int rows, int cols, int steps) {
  if (batch <= 0 || rows <= 0 || cols <= 0 || steps < 1 || steps > kMaxSteps) return 0;
  return orthogonalize_workspace(batch, rows, cols, steps);
}

int fa_orthogonalize(int dtype, int batch, int rows, int cols, const void* g, int64_t g_stride_batch,
                     int64_t g_stride_row, void* o, int64_t o_stride_batch, int64_t o_stride_row,
                     int steps, float a, float b, float c, float eps, void* workspace,
                     size_t workspace_bytes, void* stream) {
  FA_TRY(check_dtype(dtype));
  if (batch < 0 || rows <= 0 || cols <= 0 || steps < 1) return FA_ERR_INVALID_ARG;
  if (steps > kMaxSteps || batch > 65535 || rows > (1 << 20) || cols > (1 << 20) ||
      (int64_t)batch * ((rows + 255) / 256) * ((cols + 255) / 256) >= INT32_MAX)
    return FA_ERR_TOO_LARGE;
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c) || !(eps >= 0.f) ||
      !std::isfinite(eps))
    return FA_ERR_INVALID_ARG;
  const float coef[3] = {a, b, c};
  if (!orthogonalize_in_range(rows, cols, steps, coef)) return FA_ERR_UNSUPPORTED;
  if (batch == 0) return FA_OK;
  if (g == nullptr || o == nullptr) return FA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(g) % (dtype == FA_DTYPE_BF16 ? 2 : 4) != 0 ||
      reinterpret_cast<uintptr_t>(o) % 16 != 0 || o_stride_row % 8 != 0 || o_stride_batch % 8 != 0)
    return FA_ERR_ALIGNMENT;
  const size_t need = fa_orthogonalize_workspace_bytes(batch, rows, cols, steps);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return FA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return FA_ERR_ALIGNMENT;
  FA_TRY(check_sm100());
  return launch_orthogonalize(dtype, batch, rows, cols, g, g_stride_batch, g_stride_row, o,
                              o_stride_batch, o_stride_row, steps, coef, eps, workspace,
                              reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
