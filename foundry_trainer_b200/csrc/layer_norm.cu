// layer_norm.cu — layer norm with an affine or adaptive (modulated) output,
// forward and backward.
//
// Reference: layer_norm_mod (crates/foundry-spike/src/lib.rs:60-71): per row
// mean and variance in fp32, h = (x - mean) / sqrt(var + eps), y = h (1 +
// scale) + shift, cast. Here y = h (off + w) + b with off 0 or 1 and w, b
// shared by all rows or one pair per group of rows (a sample's modulation).
// With t = dy (off + w) the gradients are
//   dx = (t - mean(t) - h mean(t h)) / sqrt(var + eps),
//   dw = sum over rows of dy h,  db = sum over rows of dy.
//
// Bound by memory: the forward reads x once and writes y once (the row is
// held in registers between its statistics and its output, so the variance is
// the exact two-pass one); the backward reads x and dy once and writes dx
// once. dw and db are summed in registers by the thread that owns the column,
// over the rows of its block, and joined in block order by a second kernel:
// the same bits every time. All sums are fp32.
#include <cuda_bf16.h>

#include <algorithm>

#include "attn_common.h"
#include "sm100_ptx.cuh"

namespace fa {
namespace ln {

struct Mat {  // (groups, rows, dim), dim contiguous
  void* p;
  int64_t sg, sr;
};

struct Par {  // weight and bias: rows of `dim`, `stride` apart per group (0: shared)
  const void* w;
  const void* b;
  int64_t stride;
  int bf16;
  float off;
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// E consecutive elements at p: one 16-byte access when E > 1, one element else
template <typename T, int E>
__device__ __forceinline__ void load_e(const T* p, float* e) {
  if constexpr (E == 1) {
    e[0] = to_f<T>(*p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    e[0] = v.x; e[1] = v.y; e[2] = v.z; e[3] = v.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    e[0] = bf16_lo(v.x); e[1] = bf16_hi(v.x); e[2] = bf16_lo(v.y); e[3] = bf16_hi(v.y);
    e[4] = bf16_lo(v.z); e[5] = bf16_hi(v.z); e[6] = bf16_lo(v.w); e[7] = bf16_hi(v.w);
  }
}

template <typename T, int E>
__device__ __forceinline__ void store_e(T* p, const float* e) {
  if constexpr (E == 1) {
    if constexpr (sizeof(T) == 4) *p = e[0];
    else *p = __float2bfloat16_rn(e[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(e[0], e[1], e[2], e[3]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]),
                                              pack_bf16(e[4], e[5]), pack_bf16(e[6], e[7]));
  }
}

// E parameters from column c (fp32 or bf16; vector loads when E > 1)
template <int E>
__device__ __forceinline__ void load_par(const void* base, int64_t at, int bf16, float none, float* e) {
  if (base == nullptr) {
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = none;
  } else if (bf16) {
    const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(base) + at;
    if constexpr (E == 8) {
      load_e<__nv_bfloat16, 8>(p, e);
    } else if constexpr (E == 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      e[0] = bf16_lo(v.x); e[1] = bf16_hi(v.x); e[2] = bf16_lo(v.y); e[3] = bf16_hi(v.y);
    } else {
      e[0] = __bfloat162float(*p);
    }
  } else {
    const float* p = reinterpret_cast<const float*>(base) + at;
    if constexpr (E == 1) {
      e[0] = *p;
    } else {
#pragma unroll
      for (int i = 0; i < E; i += 4) load_e<float, 4>(p + i, e + i);
    }
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the team that owns a row: one warp, or the whole block (through
// `red`, one float per warp; the barrier pair makes `red` reusable).
template <bool WARP>
__device__ __forceinline__ float team_sum(float v, float* red) {
  v = warp_sum(v);
  if constexpr (WARP) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  float s = (threadIdx.x & 31) < nw ? red[threadIdx.x & 31] : 0.f;
  return warp_sum(s);
}

// One row per warp (WARP) or per block; thread t of the row's `team` threads
// owns vectors t, t + team, ... (V of them, E elements each).
template <typename T, int E, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512)
fwd_kernel(Mat x, Mat y, Par par, int64_t n_rows, int rows, int dim, float eps, float* stats) {
  __shared__ float red[32];
  const int team = WARP ? 32 : blockDim.x;
  const int t = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)
                           : (int64_t)blockIdx.x;
  if (row >= n_rows) return;  // uniform over the team
  const int64_t g = row / rows, r = row - g * rows;
  const T* xr = reinterpret_cast<const T*>(x.p) + g * x.sg + r * x.sr;
  float e[V][E];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (t + v * team) * E;
    if (c < dim) {
      load_e<T, E>(xr + c, e[v]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) e[v][i] = 0.f;
    }
  }
  float s = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < E; ++i) s += e[v][i];
  const float mean = team_sum<WARP>(s, red) / (float)dim;
  float q = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const bool in = (t + v * team) * E < dim;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      e[v][i] -= mean;
      if (in) q = fmaf(e[v][i], e[v][i], q);
    }
  }
  const float var = team_sum<WARP>(q, red) / (float)dim;
  const float rstd = 1.f / sqrtf(var + eps);
  if (stats != nullptr && t == 0) {
    stats[row] = mean;
    stats[n_rows + row] = rstd;
  }
  T* yr = reinterpret_cast<T*>(y.p) + g * y.sg + r * y.sr;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (t + v * team) * E;
    if (c < dim) {
      float w[E], b[E], o[E];
      load_par<E>(par.w, g * par.stride + c, par.bf16, 1.f - par.off, w);
      load_par<E>(par.b, g * par.stride + c, par.bf16, 0.f, b);
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] = fmaf(e[v][i] * rstd, par.off + w[i], b[i]);
      store_e<T, E>(yr + c, o);
    }
  }
}

// Sums of K values over the warp, every lane gets all K.
template <int K>
__device__ __forceinline__ void warp_sums(float* v) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
}

// Block (chunk) `blockIdx.x` of group blockIdx.y: rows [chunk * per, ...). R
// rows are in flight at a time; a thread keeps V vectors of E columns of dw
// and db in registers across its rows. part: (groups * chunks, 2, dim) fp32.
// WARP: each of the block's warps is a team of its own and takes rows
// warp, warp + warps, ...; their sums join in warp order at the end.
template <typename T, int E, int V, int R, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512)
bwd_kernel(Mat x, Mat dy, Mat dx, Par par, const float* stats, int64_t n_rows, int rows, int dim,
           int per, int chunks, float* part) {
  extern __shared__ float sm[];
  __shared__ float red[2][32][2 * R];
  const int team = WARP ? 32 : blockDim.x;
  const int t = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int nteam = WARP ? (int)(blockDim.x >> 5) : 1;
  const int me = WARP ? (int)(threadIdx.x >> 5) : 0;
  const int g = blockIdx.x / chunks, chunk = blockIdx.x - g * chunks;
  const int r0 = chunk * per, r1 = min(rows, r0 + per);
  // off + w stays in registers, except at 32 columns a thread (dim > 8192),
  // where it is read again for every row
  constexpr bool kKeepW = V * E < 32;
  float w[kKeepW ? V : 1][E], aw[V][E], ab[V][E];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (t + v * team) * E;
#pragma unroll
    for (int i = 0; i < E; ++i) aw[v][i] = ab[v][i] = 0.f;
    if constexpr (kKeepW) {
#pragma unroll
      for (int i = 0; i < E; ++i) w[v][i] = 0.f;
      if (c < dim) {
        load_par<E>(par.w, (int64_t)g * par.stride + c, par.bf16, 1.f - par.off, w[v]);
#pragma unroll
        for (int i = 0; i < E; ++i) w[v][i] += par.off;
      }
    }
  }
  const T* xg = reinterpret_cast<const T*>(x.p) + (int64_t)g * x.sg;
  const T* dyg = reinterpret_cast<const T*>(dy.p) + (int64_t)g * dy.sg;
  T* dxg = reinterpret_cast<T*>(dx.p) + (int64_t)g * dx.sg;
  const float inv = 1.f / (float)dim;
  int flip = 0;
  for (int rb = r0 + me * R; rb < r1; rb += nteam * R) {
    float h[R][V][E], d[R][V][E], rs[R], s[2 * R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const bool live = rb + k < r1;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = (t + v * team) * E;
        if (live && c < dim) {
          load_e<T, E>(xg + (int64_t)(rb + k) * x.sr + c, h[k][v]);
          load_e<T, E>(dyg + (int64_t)(rb + k) * dy.sr + c, d[k][v]);
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i) h[k][v][i] = d[k][v][i] = 0.f;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const bool live = rb + k < r1;
      const int64_t row = (int64_t)g * rows + rb + k;
      const float mean = live ? stats[row] : 0.f;
      rs[k] = live ? stats[n_rows + row] : 0.f;
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const bool in = live && (t + v * team) * E < dim;
        float* wv = w[kKeepW ? v : 0];
        if constexpr (!kKeepW) {
          if (in) {
            load_par<E>(par.w, (int64_t)g * par.stride + (t + v * team) * E, par.bf16,
                        1.f - par.off, wv);
#pragma unroll
            for (int i = 0; i < E; ++i) wv[i] += par.off;
          } else {
#pragma unroll
            for (int i = 0; i < E; ++i) wv[i] = 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
          h[k][v][i] = in ? (h[k][v][i] - mean) * rs[k] : 0.f;
          const float dv = d[k][v][i];
          ab[v][i] += dv;
          aw[v][i] = fmaf(dv, h[k][v][i], aw[v][i]);
          const float tt = dv * wv[i];
          d[k][v][i] = tt;
          s1 += tt;
          s2 = fmaf(tt, h[k][v][i], s2);
        }
      }
      s[2 * k] = s1;
      s[2 * k + 1] = s2;
    }
    warp_sums<2 * R>(s);
    if constexpr (!WARP) {
      // double-buffered, so one barrier per R rows suffices
      const int wid = threadIdx.x >> 5, nw = blockDim.x >> 5, lane = threadIdx.x & 31;
      if (lane == 0) {
#pragma unroll
        for (int k = 0; k < 2 * R; ++k) red[flip][wid][k] = s[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 2 * R; ++k) s[k] = 0.f;
      for (int i = 0; i < nw; ++i) {
#pragma unroll
        for (int k = 0; k < 2 * R; ++k) s[k] += red[flip][i][k];
      }
      flip ^= 1;
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (rb + k >= r1) continue;
      const float c1 = s[2 * k] * inv, c2 = s[2 * k + 1] * inv;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = (t + v * team) * E;
        if (c < dim) {
          float o[E];
#pragma unroll
          for (int i = 0; i < E; ++i)
            o[i] = rs[k] * (d[k][v][i] - c1 - h[k][v][i] * c2);
          store_e<T, E>(dxg + (int64_t)(rb + k) * dx.sr + c, o);
        }
      }
    }
  }
  float* dst = part + (int64_t)blockIdx.x * 2 * dim;
  if constexpr (WARP) {
    // (teams, 2, dim): joined in warp order
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (t + v * team) * E;
      if (c < dim) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          sm[(me * 2 + 0) * dim + c + i] = aw[v][i];
          sm[(me * 2 + 1) * dim + c + i] = ab[v][i];
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * dim; i += blockDim.x) {
      float a = 0.f;
      for (int k = 0; k < nteam; ++k) a += sm[(k * 2) * dim + i];
      dst[i] = a;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (t + v * team) * E;
      if (c < dim) {
        // part rows start at multiples of dim floats: scalar unless dim % 4 == 0
#pragma unroll
        for (int i = 0; i < E; ++i) {
          dst[c + i] = aw[v][i];
          dst[dim + c + i] = ab[v][i];
        }
      }
    }
  }
}

// out[j][i] = sum over p < parts of part[(j * parts + p)][i], i < 2 dim: one
// column per thread of x, eight threads of y share the parts, joined in order.
__global__ void __launch_bounds__(256)
join_kernel(const float* part, int parts, int dim, float* dw, float* db) {
  __shared__ float s[8][33];
  const int tiles = (2 * dim + 31) / 32, j = blockIdx.x / tiles;
  const int col = (blockIdx.x - j * tiles) * 32 + threadIdx.x;
  float a = 0.f;
  if (col < 2 * dim) {
    const float* p = part + (int64_t)j * parts * 2 * dim + col;
    for (int i = threadIdx.y; i < parts; i += 8) a += p[(int64_t)i * 2 * dim];
  }
  s[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y == 0 && col < 2 * dim) {
    a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a += s[i][threadIdx.x];
    float* dst = col < dim ? dw : db;
    const int c = col < dim ? col : col - dim;
    if (dst != nullptr) dst[(int64_t)j * dim + c] = a;
  }
}

constexpr int kSms = 148;

static bool vec16(const void* p, int64_t a, int64_t b, int es) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (a * es) % 16 == 0 && (b * es) % 16 == 0;
}

// 16-byte accesses everywhere, or one element at a time
static bool can_vector(int es, int dim, const Mat* m, int nm, const Par& par) {
  const int e = 16 / es;
  if (dim % e != 0) return false;
  for (int i = 0; i < nm; ++i)
    if (!vec16(m[i].p, m[i].sg, m[i].sr, es)) return false;
  const int ps = par.bf16 ? 2 : 4;
  const int need = std::min(16, e * ps);  // load_par's widest access
  for (const void* p : {par.w, par.b})
    if (p != nullptr &&
        (reinterpret_cast<uintptr_t>(p) % need != 0 || (par.stride * ps) % need != 0))
      return false;
  return true;
}

template <typename T, int E, int V, bool WARP>
static int fwd_go(const Mat& x, const Mat& y, const Par& par, int64_t n, int rows, int dim,
                  float eps, float* stats, int threads, cudaStream_t st) {
  const int64_t blocks = WARP ? (n + threads / 32 - 1) / (threads / 32) : n;
  fwd_kernel<T, E, V, WARP><<<(unsigned)blocks, threads, 0, st>>>(x, y, par, n, rows, dim, eps,
                                                                  stats);
  return launch_status();
}

template <typename T, int E>
static int fwd_pick(const Mat& x, const Mat& y, const Par& par, int64_t n, int rows, int dim,
                    float eps, float* stats, cudaStream_t st) {
  const int nv = (dim + E - 1) / E;
  // a warp per row while a lane's share stays at 64 values or below
  constexpr int kMost = 64 / E;
  const int need = (nv + 31) / 32;
  if (need <= kMost) {
    // few rows: small blocks, so that they spread over the SMs
    const int th = n >= 8 * kSms ? 256 : (n >= 2 * kSms ? 128 : 32);
    if (need <= kMost / 8) return fwd_go<T, E, kMost / 8, true>(x, y, par, n, rows, dim, eps, stats, th, st);
    if (need <= kMost / 4) return fwd_go<T, E, kMost / 4, true>(x, y, par, n, rows, dim, eps, stats, th, st);
    if (need <= kMost / 2) return fwd_go<T, E, kMost / 2, true>(x, y, par, n, rows, dim, eps, stats, th, st);
    return fwd_go<T, E, kMost, true>(x, y, par, n, rows, dim, eps, stats, th, st);
  }
  constexpr int kV = 32 / E;  // dim <= 16384: 512 threads at most
  const int th = (((nv + kV - 1) / kV) + 31) / 32 * 32;
  return fwd_go<T, E, kV, false>(x, y, par, n, rows, dim, eps, stats, th, st);
}

struct BwdPlan {
  int chunks, per, threads;
  bool warp;
};

// blocks per group: two per SM over all groups, at least eight rows each
static BwdPlan bwd_plan(int groups, int rows) {
  BwdPlan p{};
  const int want = std::max(1, 2 * kSms / std::max(1, groups));
  p.per = std::max(8, (rows + want - 1) / want);
  p.chunks = std::max(1, (rows + p.per - 1) / p.per);
  return p;
}

template <typename T, int E, int V, int R, bool WARP>
static int bwd_go(const Mat& x, const Mat& dy, const Mat& dx, const Par& par, const float* stats,
                  int groups, int rows, int dim, const BwdPlan& pl, int threads, float* part,
                  cudaStream_t st) {
  const int smem = WARP ? threads / 32 * 2 * dim * 4 : 0;
  bwd_kernel<T, E, V, R, WARP><<<(unsigned)((int64_t)groups * pl.chunks), threads, smem, st>>>(
      x, dy, dx, par, stats, (int64_t)groups * rows, rows, dim, pl.per, pl.chunks, part);
  return launch_status();
}

template <typename T, int E>
static int bwd_pick(const Mat& x, const Mat& dy, const Mat& dx, const Par& par,
                    const float* stats, int groups, int rows, int dim, const BwdPlan& pl,
                    float* part, cudaStream_t st) {
  const int nv = (dim + E - 1) / E;
  if (nv <= 32)  // a warp holds the row (dim <= 256): 8 teams, 16 KB of shared memory at most
    return bwd_go<T, E, 1, 4, true>(x, dy, dx, par, stats, groups, rows, dim, pl, 256, part, st);
  auto th = [&](int v) { return ((nv + v - 1) / v + 31) / 32 * 32; };
  if constexpr (E == 1) {
    if (nv <= 4 * 512)
      return bwd_go<T, E, 4, 2, false>(x, dy, dx, par, stats, groups, rows, dim, pl, th(4), part, st);
    return bwd_go<T, E, 32, 1, false>(x, dy, dx, par, stats, groups, rows, dim, pl, th(32), part, st);
  } else {
    if (nv <= 512)
      return bwd_go<T, E, 1, 4, false>(x, dy, dx, par, stats, groups, rows, dim, pl, th(1), part, st);
    if (nv <= 2 * 512)
      return bwd_go<T, E, 2, 2, false>(x, dy, dx, par, stats, groups, rows, dim, pl, th(2), part, st);
    return bwd_go<T, E, 32 / E, 1, false>(x, dy, dx, par, stats, groups, rows, dim, pl, th(32 / E), part, st);
  }
}

}  // namespace ln

static ln::Mat ln_mat(const fa_tensor_t* t) { return ln::Mat{t->data, t->stride_b, t->stride_s}; }

int launch_layer_norm_fwd(int dtype, int groups, int rows, int dim, const fa_tensor_t* x,
                          const void* w, const void* b, int par_dtype, int64_t par_stride,
                          int unit_offset, float eps, const fa_tensor_t* y, float* stats,
                          cudaStream_t st) {
  const int64_t n = (int64_t)groups * rows;
  if (n == 0) return FA_OK;
  const ln::Mat m[2] = {ln_mat(x), ln_mat(y)};
  const ln::Par par{w, b, par_stride, par_dtype == FA_DTYPE_BF16, unit_offset ? 1.f : 0.f};
  if (dtype == FA_DTYPE_BF16) {
    return ln::can_vector(2, dim, m, 2, par)
               ? ln::fwd_pick<__nv_bfloat16, 8>(m[0], m[1], par, n, rows, dim, eps, stats, st)
               : ln::fwd_pick<__nv_bfloat16, 1>(m[0], m[1], par, n, rows, dim, eps, stats, st);
  }
  return ln::can_vector(4, dim, m, 2, par)
             ? ln::fwd_pick<float, 4>(m[0], m[1], par, n, rows, dim, eps, stats, st)
             : ln::fwd_pick<float, 1>(m[0], m[1], par, n, rows, dim, eps, stats, st);
}

size_t layer_norm_bwd_workspace(int groups, int rows, int dim) {
  const ln::BwdPlan pl = ln::bwd_plan(groups, rows);
  return (size_t)groups * pl.chunks * 2 * dim * sizeof(float);
}

int launch_layer_norm_bwd(int dtype, int groups, int rows, int dim, const fa_tensor_t* x,
                          const void* w, int par_dtype, int64_t par_stride, int unit_offset,
                          const fa_tensor_t* dy, const float* stats, const fa_tensor_t* dx,
                          float* dw, float* db, int shared, void* ws, cudaStream_t st) {
  if (groups == 0 && !shared) return FA_OK;
  const ln::BwdPlan pl = ln::bwd_plan(groups, rows);
  float* part = reinterpret_cast<float*>(ws);
  if (groups > 0) {
    const ln::Mat m[3] = {ln_mat(x), ln_mat(dy), ln_mat(dx)};
    const ln::Par par{w, nullptr, par_stride, par_dtype == FA_DTYPE_BF16, unit_offset ? 1.f : 0.f};
    int rc;
    if (dtype == FA_DTYPE_BF16)
      rc = ln::can_vector(2, dim, m, 3, par)
               ? ln::bwd_pick<__nv_bfloat16, 8>(m[0], m[1], m[2], par, stats, groups, rows, dim, pl, part, st)
               : ln::bwd_pick<__nv_bfloat16, 1>(m[0], m[1], m[2], par, stats, groups, rows, dim, pl, part, st);
    else
      rc = ln::can_vector(4, dim, m, 3, par)
               ? ln::bwd_pick<float, 4>(m[0], m[1], m[2], par, stats, groups, rows, dim, pl, part, st)
               : ln::bwd_pick<float, 1>(m[0], m[1], m[2], par, stats, groups, rows, dim, pl, part, st);
    if (rc != FA_OK) return rc;
  }
  if (dw == nullptr && db == nullptr) return FA_OK;
  const int outs = shared ? 1 : groups, parts = shared ? groups * pl.chunks : pl.chunks;
  ln::join_kernel<<<(unsigned)((int64_t)(2 * dim + 31) / 32 * outs), dim3(32, 8), 0, st>>>(part, parts, dim, dw, db);
  return launch_status();
}

}  // namespace fa
