// gemm.h — host interface of the matrix-product kernels (gemm_wide_sm100.cu,
// gemm_skinny_sm100.cu) that the adapter linears and the orthogonalisation use.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attn_common.h"

namespace fa {

// A 16-bit (batch, rows, cols) matrix, cols contiguous; strides in elements.
struct Mat3 {
  const void* p = nullptr;
  int64_t batch = 1, rows = 0, cols = 0;
  int64_t stride_batch = 0, stride_row = 0;
  int bf16 = 1;  // else fp16
};

// 3-D TMA descriptor over `m`, box (inner, rows, 1), swizzled over the box's
// inner width (32, 64 or 128 bytes), zero fill.
int make_tmap_3d(CUtensorMap* map, const Mat3& m, int box_inner, int box_rows);

enum WideEpi {
  kEpiLinear = 0,  // bf16 D (+ bias)
  kEpiGram = 1,    // fp16 D = alpha acc, mirrored (symmetric)
  kEpiPoly = 2,    // fp16 D = c0 in + c1 acc, mirrored (symmetric)
  kEpiUpdate = 3,  // D = c0 (hi + lo) + c1 acc as fp16 hi and lo
  kEpiLast = 4     // the same, as bf16 alpha D, straight or transposed
};

// e: the adapters, or the X that an update reads back as hi (d2: its lo, read
// back and written).
struct WideOperands {
  Mat3 a, b, e, d, d2;
  bool b_mn = false;
};

struct WideParams {
  int M = 0, N = 0, K = 0, batch = 1;
  int fmt = 1;  // 0 fp16, 1 bf16 operands
  int tiles_m = 0, tiles_n = 0, tiles_per_batch = 0, symmetric = 0;
  int split = 1;  // kEpiGram in narrow tiles: CTAs (a cluster) that share a tile's contraction
  // adapters: low (M, low_ld) bf16 of rows low_stride apart, low_ld = the rank
  // rounded up to 16;
  // per 256-row block the adapters in use and their count, per row its slot
  // (no lists: adapter 0 for every row)
  const __nv_bfloat16* low = nullptr;
  int low_ld = 0, rank = 0;
  int64_t low_stride = 0;  // elements from row to row of low
  const int* list_cnt = nullptr;
  const int* list_ids = nullptr;
  const int* slot = nullptr;
  // Programmatic dependent launch. 1: of what this product reads only `low`
  // may come from the previous kernel (all older work is complete when that
  // one starts); 2: anything may.
  int early = 0;
  // plain views of A, B and the adapters (E, N, rank), for blocks of several
  const __nv_bfloat16* raw_x = nullptr;
  const __nv_bfloat16* raw_w = nullptr;
  const __nv_bfloat16* raw_f = nullptr;
  int64_t raw_ldx = 0, raw_ldw = 0, raw_fe = 0, raw_ldf = 0;
  const __nv_bfloat16* bias = nullptr;
  // orthogonalisation
  float alpha = 1.f;
  const float* coef = nullptr;
  const __half* in_hi = nullptr;
  const __half* in_lo = nullptr;
  int64_t in_batch = 0;
  int in_ld = 0;
  uint16_t* out_t = nullptr;
  int64_t out_t_batch = 0, out_t_ld = 0;
};

// out[i, j] = sum_k Big[i, k] Small[j, k], j < n <= 256 (token columns: any
// number, in blocks)
constexpr int kMaxColumns = 256;
enum SkinnyOut {
  kSkinnyCols = 0,  // out[j, i] bf16 + bias[i] + the adapters' term of row j
  kSkinnyLow = 1,   // out[i, j] bf16, scaled: a row's own adapter's columns
  kSkinnyGrad = 2   // out[j out_j + i out_ld] bf16, Small with its remainders
};

struct SkinnyParams {
  int rows = 0;  // i
  int cols = 0;  // j that are stored
  int n = 0;     // cols rounded up to 16
  int K = 0;
  __nv_bfloat16* out = nullptr;
  int64_t out_ld = 0, out_j = 0;
  const __nv_bfloat16* bias = nullptr;
  // adapters: low as in WideParams; per token its adapter (none: 0 for all)
  const __nv_bfloat16* low = nullptr;
  int low_ld = 0, rank = 0, E = 1;
  int64_t low_stride = 0;
  // kSkinnyLow: where each row's remainders (what rounding to bf16 dropped, as
  // bf16) go behind its values; 0: nowhere
  int lo_at = 0;
  // kSkinnyGrad: the second product
  int rows2 = 0;
  __nv_bfloat16* out2 = nullptr;
  int64_t out_ld2 = 0, out_j2 = 0;
  const int* ids = nullptr;
  // plain views of Small, Big and the adapters, for tokens of several
  const __nv_bfloat16* raw_x = nullptr;
  const __nv_bfloat16* raw_w = nullptr;
  const __nv_bfloat16* raw_f = nullptr;
  int64_t raw_ldx = 0, raw_ldw = 0, raw_fe = 0, raw_ldf = 0;
  float scale = 1.f;
  const float* scales = nullptr;
  const int* list_cnt = nullptr;
  const int* list_ids = nullptr;
  const int* slot = nullptr;
  int slots_per_pass = 1;
};

// fac: the adapters of a linear for tokens, (E, i, rank) as Big is stored, or
// (E, rank, i) with big_mn.
// early: the launch may start before its predecessor ends (programmatic
// dependent launch); only `low` may then come from that predecessor.
int launch_gemm_skinny(const Mat3& big, bool big_mn, const Mat3& small, bool small_mn,
                       SkinnyParams p, int out, bool early, cudaStream_t st,
                       const Mat3& fac = Mat3{});
// Both factors' gradients in one launch (kSkinnyGrad): Big (K, rows) and Small
// with its remainders (K, n), each stored with its short side contiguous.
int launch_skinny_grads(const Mat3* big, const Mat3* small, const Mat3* small_lo, SkinnyParams p,
                        cudaStream_t st);
// whether a linear of `rows` tokens runs as kSkinnyCols rather than wide
bool linear_as_columns(int64_t out, int64_t K, int rows, int adapters = 0, int rank = 0);
int launch_low_rows(const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* a, int64_t a_e,
                    int64_t a_r, const int* ids, int E, const float* scales, float scale, int rows,
                    int K, int rank, int low_ld, __nv_bfloat16* low, int64_t low_stride, int lo_at,
                    cudaStream_t st);
int launch_pad_rows(int64_t rows, int cols, const void* src, int64_t src_stride, void* dst,
                    int64_t dst_stride, cudaStream_t st);
int launch_adapter_plan(const int* ids, int rows, int E, int* cnt, int* list, int* slot,
                        cudaStream_t st);
int skinny_device_status();

// The descriptors of one call's matrices (each pointer has one shape in it),
// for a sequence of products over the same few: encoding five per launch costs
// as much as the launch.
struct TmapMemo {
  static constexpr int kMost = 12;
  const void* p[kMost];
  int box[kMost];
  CUtensorMap maps[kMost];
  int n = 0;
  int get(CUtensorMap* map, const Mat3& m, int rows);
};

int launch_gemm_wide(const WideOperands& o, WideParams p, int epi, cudaStream_t st,
                     TmapMemo* maps = nullptr);
int wide_device_status();

}  // namespace fa
