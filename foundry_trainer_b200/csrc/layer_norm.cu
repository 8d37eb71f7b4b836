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
//
// Two forms of each. The ring form (rows of at least 1 KB whose starts are
// 16-byte aligned) keeps the next rows on their way while a block reduces the
// present ones: one thread copies whole rows into a ring in shared memory
// (cp.async.bulk), every thread takes its columns of R rows from there, and
// the block barrier of the rows' sums also tells that thread that the slot is
// free. Loads straight into registers were latency-bound: at 4608 x 2048 bf16
// forward 18.5 us, backward 24 us. The direct form serves every other width,
// stride and alignment (16-byte accesses, pairs or single elements), and the
// forward's smallest calls; its backward of long rows keeps the column sums in
// shared memory.
//
// At 36864 x 4096 bf16: forward 101 us, 5.96 TB/s of the copy's 6.55; backward
// 153 us, 5.92 TB/s. At 4608 x 2048: 10.8 and 14.4 us (5.8 and 8.6 at the
// copy's rate), one wave's ramp and tail. One row of 2048: 2.5 us.
#include <cuda_bf16.h>

#include <algorithm>

#include "attn_common.h"
#include "gemm_ptx.cuh"

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

// E consecutive elements at p: one access (16 bytes, or 2 elements, or 1)
template <typename T, int E>
__device__ __forceinline__ void load_e(const T* p, float* e) {
  if constexpr (E == 1) {
    e[0] = to_f<T>(*p);
  } else if constexpr (E == 2 && sizeof(T) == 4) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    e[0] = v.x; e[1] = v.y;
  } else if constexpr (E == 2) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(p);
    e[0] = bf16_lo(v); e[1] = bf16_hi(v);
  } else if constexpr (sizeof(T) == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    e[0] = v.x; e[1] = v.y; e[2] = v.z; e[3] = v.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    e[0] = bf16_lo(v.x); e[1] = bf16_hi(v.x); e[2] = bf16_lo(v.y); e[3] = bf16_hi(v.y);
    e[4] = bf16_lo(v.z); e[5] = bf16_hi(v.z); e[6] = bf16_lo(v.w); e[7] = bf16_hi(v.w);
  }
}

// The same from column c of a row, zeros past its end. One-element accesses load
// some element in any case: with a branch for each the many loads of a long row
// went out one by one (2000 x 12001 bf16: forward 130 -> 77 us, backward 220 ->
// 97; with pairs the branch is the faster: 6 x 646 x 5426 fp32 42 and 61 us
// against 46 and 79).
template <typename T, int E>
__device__ __forceinline__ void load_in(const T* row, int c, int dim, float* e) {
  if constexpr (E == 1) {
    load_e<T, E>(row + (c < dim ? c : 0), e);
    e[0] = c < dim ? e[0] : 0.f;
  } else if (c < dim) {
    load_e<T, E>(row + c, e);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = 0.f;
  }
}

template <typename T, int E>
__device__ __forceinline__ void store_e(T* p, const float* e) {
  if constexpr (E == 1) {
    if constexpr (sizeof(T) == 4) *p = e[0];
    else *p = __float2bfloat16_rn(e[0]);
  } else if constexpr (E == 2 && sizeof(T) == 4) {
    *reinterpret_cast<float2*>(p) = make_float2(e[0], e[1]);
  } else if constexpr (E == 2) {
    *reinterpret_cast<uint32_t*>(p) = pack_bf16(e[0], e[1]);
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
      load_e<__nv_bfloat16, E>(p, e);
    }
  } else {
    const float* p = reinterpret_cast<const float*>(base) + at;
    if constexpr (E <= 2) {
      load_e<float, E>(p, e);
    } else {
#pragma unroll
      for (int i = 0; i < E; i += 4) load_e<float, 4>(p + i, e + i);
    }
  }
}

// V vectors of E parameters from column c on, `step` columns apart. One branch
// on the type around all the loads, so that they are in flight together.
template <int E, int V>
__device__ __forceinline__ void load_pars(const void* base, int64_t at, int bf16, float none, int c,
                                          int step, int dim, float (*e)[E]) {
  if (base != nullptr && bf16) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (E == 1 || c + v * step < dim)
        load_par<E>(base, at + (c + v * step < dim ? c + v * step : 0), 1, none, e[v]);
  } else if (base != nullptr) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (E == 1 || c + v * step < dim)
        load_par<E>(base, at + (c + v * step < dim ? c + v * step : 0), 0, none, e[v]);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < E; ++i) e[v][i] = none;
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
__global__ void __launch_bounds__(WARP ? 256 : 512, WARP && E == 1 && V == 32 ? 3 : 0)
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
    load_in<T, E>(xr, c, dim, e[v]);
  }
  // the parameters are under way with the row; at 32 values a thread they would
  // spill or leave half the warps (3001 x 1001 bf16 10.8 -> 8.3 us), and come
  // in turns after the statistics
  constexpr int kTurns = V * E < 32 ? 1 : !WARP ? 2 : E == 1 ? 4 : 1, VT = V / kTurns;
  float w[VT][E], b[VT][E];
  auto parameters = [&](int first) {
    const int c = (t + first * team) * E;
    load_pars<E, VT>(par.w, g * par.stride, par.bf16, 1.f - par.off, c, team * E, dim, w);
    load_pars<E, VT>(par.b, g * par.stride, par.bf16, 0.f, c, team * E, dim, b);
  };
  if constexpr (kTurns == 1) parameters(0);
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
  for (int k = 0; k < kTurns; ++k) {
    if constexpr (kTurns > 1) parameters(k * VT);
#pragma unroll
    for (int v = 0; v < VT; ++v) {
      const int c = (t + (k * VT + v) * team) * E;
      if (c < dim) {
        float o[E];
#pragma unroll
        for (int i = 0; i < E; ++i)
          o[i] = fmaf(e[k * VT + v][i] * rstd, par.off + w[v][i], b[v][i]);
        store_e<T, E>(yr + c, o);
      }
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
  float w[V][E], aw[V][E], ab[V][E];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (t + v * team) * E;
#pragma unroll
    for (int i = 0; i < E; ++i) aw[v][i] = ab[v][i] = w[v][i] = 0.f;
    if (c < dim) {
      load_par<E>(par.w, (int64_t)g * par.stride + c, par.bf16, 1.f - par.off, w[v]);
#pragma unroll
      for (int i = 0; i < E; ++i) w[v][i] += par.off;
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
#pragma unroll
        for (int i = 0; i < E; ++i) {
          h[k][v][i] = in ? (h[k][v][i] - mean) * rs[k] : 0.f;
          const float dv = d[k][v][i];
          ab[v][i] += dv;
          aw[v][i] = fmaf(dv, h[k][v][i], aw[v][i]);
          const float tt = dv * w[v][i];
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

// The same for rows of 16 to 32 values a thread: off + w and the columns' sums
// are in shared memory, (3, dim) fp32 that each thread reads and writes at its
// own columns only; registers hold the row alone. (All of it in registers left
// one block an SM and the weight's loads in the row's way: 6 x 646 x 5426 fp32
// 190 -> 61 us, its bytes 39.)
template <typename T, int E, int V>
__global__ void __launch_bounds__(512)
bwd_long_kernel(Mat x, Mat dy, Mat dx, Par par, const float* stats, int64_t n_rows, int rows,
                int dim, int per, int chunks, float* part) {
  extern __shared__ __align__(16) float lsm[];
  __shared__ float red[2][32][2];
  float *sw = lsm, *saw = lsm + dim, *sab = lsm + 2 * dim;
  const int t = threadIdx.x, team = blockDim.x;
  const int g = blockIdx.x / chunks, chunk = blockIdx.x - g * chunks;
  const int r0 = chunk * per, r1 = min(rows, r0 + per);
  const int wid = t >> 5, nw = team >> 5, lane = t & 31;
#pragma unroll 4
  for (int c = t * E; c < dim; c += team * E) {
    float w[E], zero[E] = {};
    load_par<E>(par.w, (int64_t)g * par.stride + c, par.bf16, 1.f - par.off, w);
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] += par.off;
    store_e<float, E>(sw + c, w);
    store_e<float, E>(saw + c, zero);
    store_e<float, E>(sab + c, zero);
  }
  const float inv = 1.f / (float)dim;
  int flip = 0;
  for (int r = r0; r < r1; ++r) {
    const T* xr = reinterpret_cast<const T*>(x.p) + (int64_t)g * x.sg + (int64_t)r * x.sr;
    const T* dyr = reinterpret_cast<const T*>(dy.p) + (int64_t)g * dy.sg + (int64_t)r * dy.sr;
    T* dxr = reinterpret_cast<T*>(dx.p) + (int64_t)g * dx.sg + (int64_t)r * dx.sr;
    const int64_t row = (int64_t)g * rows + r;
    float h[V][E], d[V][E];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (t + v * team) * E;
      load_in<T, E>(xr, c, dim, h[v]);
      load_in<T, E>(dyr, c, dim, d[v]);
    }
    const float mean = stats[row], rs = stats[n_rows + row];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (t + v * team) * E;
      if (c < dim) {
        float w[E], aw[E], ab[E];
        load_e<float, E>(sw + c, w);
        load_e<float, E>(saw + c, aw);
        load_e<float, E>(sab + c, ab);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          h[v][i] = (h[v][i] - mean) * rs;
          ab[i] += d[v][i];
          aw[i] = fmaf(d[v][i], h[v][i], aw[i]);
          d[v][i] *= w[i];
          s[0] += d[v][i];
          s[1] = fmaf(d[v][i], h[v][i], s[1]);
        }
        store_e<float, E>(saw + c, aw);
        store_e<float, E>(sab + c, ab);
      }
    }
    warp_sums<2>(s);
    if (lane == 0) red[flip][wid][0] = s[0], red[flip][wid][1] = s[1];
    __syncthreads();
    s[0] = s[1] = 0.f;
    for (int i = 0; i < nw; ++i) s[0] += red[flip][i][0], s[1] += red[flip][i][1];
    flip ^= 1;  // double-buffered, so one barrier a row suffices
    const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (t + v * team) * E;
      if (c < dim) {
        float o[E];
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = rs * (d[v][i] - c1 - h[v][i] * c2);
        store_e<T, E>(dxr + c, o);
      }
    }
  }
  float* dst = part + (int64_t)blockIdx.x * 2 * dim;
  for (int c = t * E; c < dim; c += team * E) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      dst[c + i] = saw[c + i];
      dst[dim + c + i] = sab[c + i];
    }
  }
}

// ------------------------------------------------------------- ring form

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// The 16 bytes of a row as E / 2 pairs of fp32, for the two-lane arithmetic:
// the kernels' instructions, not memory, set the pace of scalar code here
// (0.6 instructions issued a cycle at 4.0 TB/s; forward 162 us and backward
// 211 us at 36864 x 4096 bf16).
template <int E>
__device__ __forceinline__ void pairs_of(const uint4& v, uint64_t* e) {
  if constexpr (E == 4) {
    e[0] = f2_pack(__uint_as_float(v.x), __uint_as_float(v.y));
    e[1] = f2_pack(__uint_as_float(v.z), __uint_as_float(v.w));
  } else {
    e[0] = f2_pack(bf16_lo(v.x), bf16_hi(v.x));
    e[1] = f2_pack(bf16_lo(v.y), bf16_hi(v.y));
    e[2] = f2_pack(bf16_lo(v.z), bf16_hi(v.z));
    e[3] = f2_pack(bf16_lo(v.w), bf16_hi(v.w));
  }
}
__device__ __forceinline__ uint64_t twice(float v) { return f2_pack(v, v); }
__device__ __forceinline__ float f2_sum(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}
template <typename T, int E>
__device__ __forceinline__ void store_pairs(T* p, const uint64_t* e) {
  float f[E];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) f2_unpack(e[i], f[2 * i], f[2 * i + 1]);
  store_e<T, E>(p, f);
}

constexpr int kMaxStages = 4;

// A ring of `stages` slots of R rows of each of NT tensors; row bytes `rb`.
template <int R, int NT>
struct Ring {
  uint8_t* base;
  uint64_t* full;
  int stages, rb, nb, r0, r1;
  const uint8_t* src[NT];
  int64_t step[NT];  // bytes from row to row

  __device__ __forceinline__ int rows(int it) const { return min(R, r1 - r0 - it * R); }
  __device__ __forceinline__ const uint8_t* slot(int s) const { return base + s * NT * R * rb; }
  // one thread: turn `it` into slot s
  __device__ __forceinline__ void issue(int it, int s) const {
    const int n = rows(it);
    mbar_arrive_expect_tx(&full[s], (uint32_t)(NT * n * rb));
#pragma unroll
    for (int t = 0; t < NT; ++t)
      for (int k = 0; k < n; ++k)
        bulk_load(base + ((s * NT + t) * R + k) * rb, src[t] + (int64_t)(r0 + it * R + k) * step[t],
                  (uint32_t)rb, &full[s]);
  }
  __device__ __forceinline__ void start() const {
    if (threadIdx.x == 0) {
      for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
      fence_mbar_init();
      for (int it = 0; it < min(stages, nb); ++it) issue(it, it);
    }
    __syncthreads();
  }
};

// K block-wide sums (K = 1, 2, 4, 8). Within a warp the lanes halve the set
// they carry with every exchange; across warps a lane takes every 32nd of the
// (warp, value) partials. `red` is one of two buffers used in turn, so one
// barrier a call suffices.
template <int K>
__device__ __forceinline__ void block_sums(float* s, float* red) {
  const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  float v[K];
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = s[k];
  int which = 0;
#pragma unroll
  for (int off = 16, n = K; off > 0; off >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool up = (lane & off) != 0;
      which = 2 * which + (up ? 1 : 0);
#pragma unroll
      for (int k = 0; k < K / 2; ++k) {
        if (k < n) {
          const float send = up ? v[k] : v[k + n], keep = up ? v[k + n] : v[k];
          v[k] = keep + __shfl_xor_sync(0xffffffffu, send, off);
        }
      }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
    }
  }
  if ((lane & (32 / K - 1)) == 0) red[(threadIdx.x >> 5) * K + which] = v[0];
  __syncthreads();
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < K / 2 + (K == 1); ++i)  // at most 16 warps: 16 K partials
    if (lane + 32 * i < nw * K) a += red[lane + 32 * i];
#pragma unroll
  for (int off = 16; off >= K; off >>= 1) a += __shfl_xor_sync(0xffffffffu, a, off);
#pragma unroll
  for (int k = 0; k < K; ++k) s[k] = __shfl_sync(0xffffffffu, a, k);
}

template <typename T, int E, int V, int R>
__global__ void __launch_bounds__(V == 1 ? 256 : 512, V == 1 ? 3 : 1)
fwd_ring_kernel(Mat x, Mat y, Par par, int64_t n_rows, int rows, int dim, float eps, float* stats,
                int per, int chunks, int stages) {
  extern __shared__ __align__(128) uint8_t ring_mem[];
  __shared__ float red[2][16 * R];
  constexpr int P = E / 2;
  const int g = blockIdx.x / chunks, chunk = blockIdx.x - g * chunks;
  Ring<R, 1> q;
  q.rb = dim * (int)sizeof(T);
  q.stages = stages;
  q.r0 = chunk * per;
  q.r1 = min(rows, q.r0 + per);
  q.nb = (q.r1 - q.r0 + R - 1) / R;
  q.base = ring_mem;
  q.full = reinterpret_cast<uint64_t*>(ring_mem + stages * R * q.rb);
  q.src[0] = reinterpret_cast<const uint8_t*>(reinterpret_cast<const T*>(x.p) + (int64_t)g * x.sg);
  q.step[0] = x.sr * (int64_t)sizeof(T);
  q.start();
  const int t = threadIdx.x, team = blockDim.x;
  uint64_t w[V][P], b[V][P];
  {
    float wf[V][E], bf[V][E];
    load_pars<E, V>(par.w, (int64_t)g * par.stride, par.bf16, 1.f - par.off, t * E, team * E, dim, wf);
    load_pars<E, V>(par.b, (int64_t)g * par.stride, par.bf16, 0.f, t * E, team * E, dim, bf);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < P; ++i) {
        w[v][i] = f2_pack(wf[v][2 * i] + par.off, wf[v][2 * i + 1] + par.off);
        b[v][i] = f2_pack(bf[v][2 * i], bf[v][2 * i + 1]);
      }
  }
  bool in[V];
#pragma unroll
  for (int v = 0; v < V; ++v) in[v] = (t + v * team) * E < dim;
  T* yr = reinterpret_cast<T*>(y.p) + (int64_t)g * y.sg + (int64_t)q.r0 * y.sr + t * E;
  const float inv = 1.f / (float)dim;
  bool alive = true;  // false once a wait has run out: the block goes on
                      // without waiting, its barriers stay matched
  int s = 0;
  uint32_t ph = 0;
  for (int it = 0; it < q.nb; ++it) {
    const int n = q.rows(it);
    if (alive) alive = mbar_wait(&q.full[s], ph);
    const uint8_t* slot = q.slot(s) + t * 16;
    uint4 raw[R][V];
    float sum[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      uint64_t a = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        raw[k][v] = make_uint4(0, 0, 0, 0);
        if (k < n && in[v]) raw[k][v] = *reinterpret_cast<const uint4*>(slot + k * q.rb + v * team * 16);
        uint64_t e[P];
        pairs_of<E>(raw[k][v], e);
#pragma unroll
        for (int i = 0; i < P; ++i) a = fadd2(a, e[i]);
      }
      sum[k] = f2_sum(a);
    }
    block_sums<R>(sum, red[0]);
    if (t == 0 && it + stages < q.nb) q.issue(it + stages, s);
    if (++s == stages) s = 0, ph ^= 1;
    float mean[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      mean[k] = sum[k] * inv;
      const uint64_t m = twice(-mean[k]);
      uint64_t a = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (in[v]) {
          uint64_t e[P];
          pairs_of<E>(raw[k][v], e);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const uint64_t d = fadd2(e[i], m);
            a = ffma2(d, d, a);
          }
        }
      }
      sum[k] = f2_sum(a);
    }
    block_sums<R>(sum, red[1]);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (k < n) {
        const float rstd = rsqrtf(sum[k] * inv + eps);
        if (t == 0 && stats != nullptr) {
          const int64_t row = (int64_t)g * rows + q.r0 + it * R + k;
          stats[row] = mean[k];
          stats[n_rows + row] = rstd;
        }
        const uint64_t m = twice(-mean[k]), r = twice(rstd);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (in[v]) {
            uint64_t e[P];
            pairs_of<E>(raw[k][v], e);
#pragma unroll
            for (int i = 0; i < P; ++i) e[i] = ffma2(fmul2(fadd2(e[i], m), r), w[v][i], b[v][i]);
            store_pairs<T, E>(yr + v * team * E, e);
          }
        }
        yr += y.sr;
      }
    }
  }
  if (!alive) drain_delay();
}

template <typename T, int E, int V, int R>
__global__ void __launch_bounds__(V == 1 ? 256 : 512, V == 1 ? 2 : 1)
bwd_ring_kernel(Mat x, Mat dy, Mat dx, Par par, const float* stats, int64_t n_rows, int rows,
                int dim, int per, int chunks, int stages, float* part) {
  extern __shared__ __align__(128) uint8_t ring_mem[];
  __shared__ float red[2][16 * 2 * R];
  constexpr int P = E / 2;
  pdl_launch_next();
  const int g = blockIdx.x / chunks, chunk = blockIdx.x - g * chunks;
  Ring<R, 2> q;
  q.rb = dim * (int)sizeof(T);
  q.stages = stages;
  q.r0 = chunk * per;
  q.r1 = min(rows, q.r0 + per);
  q.nb = (q.r1 - q.r0 + R - 1) / R;
  q.base = ring_mem;
  q.full = reinterpret_cast<uint64_t*>(ring_mem + stages * 2 * R * q.rb);
  q.src[0] = reinterpret_cast<const uint8_t*>(reinterpret_cast<const T*>(x.p) + (int64_t)g * x.sg);
  q.src[1] = reinterpret_cast<const uint8_t*>(reinterpret_cast<const T*>(dy.p) + (int64_t)g * dy.sg);
  q.step[0] = x.sr * (int64_t)sizeof(T);
  q.step[1] = dy.sr * (int64_t)sizeof(T);
  q.start();
  const int t = threadIdx.x, team = blockDim.x;
  uint64_t w[V][P], aw[V][P], ab[V][P];
  bool in[V];
  {
    float wf[V][E];
    load_pars<E, V>(par.w, (int64_t)g * par.stride, par.bf16, 1.f - par.off, t * E, team * E, dim, wf);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      in[v] = (t + v * team) * E < dim;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        w[v][i] = f2_pack(wf[v][2 * i] + par.off, wf[v][2 * i + 1] + par.off);
        aw[v][i] = ab[v][i] = 0;
      }
    }
  }
  T* dxr = reinterpret_cast<T*>(dx.p) + (int64_t)g * dx.sg + (int64_t)q.r0 * dx.sr + t * E;
  const float inv = 1.f / (float)dim;
  const float* st = stats + (int64_t)g * rows + q.r0;
  // a row's statistics are read one turn ahead
  float mean[R], rs[R];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const bool live = k < q.r1 - q.r0;
    mean[k] = live ? st[k] : 0.f;
    rs[k] = live ? st[n_rows + k] : 0.f;
  }
  bool alive = true;
  int s = 0;
  uint32_t ph = 0;
  for (int it = 0; it < q.nb; ++it) {
    const int n = q.rows(it);
    float mean_n[R], rs_n[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const bool live = q.r0 + (it + 1) * R + k < q.r1;
      mean_n[k] = live ? st[(it + 1) * R + k] : 0.f;
      rs_n[k] = live ? st[n_rows + (it + 1) * R + k] : 0.f;
    }
    if (alive) alive = mbar_wait(&q.full[s], ph);
    const uint8_t* slot = q.slot(s) + t * 16;
    uint4 rx[R][V], rd[R][V];
    float sum[2 * R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      uint64_t s1 = 0, s2 = 0;
      const uint64_t r = twice(rs[k]), m = twice(-mean[k]);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        rx[k][v] = rd[k][v] = make_uint4(0, 0, 0, 0);
        if (k < n && in[v]) {
          rx[k][v] = *reinterpret_cast<const uint4*>(slot + k * q.rb + v * team * 16);
          rd[k][v] = *reinterpret_cast<const uint4*>(slot + (R + k) * q.rb + v * team * 16);
          uint64_t e[P], d[P];
          pairs_of<E>(rx[k][v], e);
          pairs_of<E>(rd[k][v], d);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const uint64_t h = fmul2(fadd2(e[i], m), r), tt = fmul2(d[i], w[v][i]);
            ab[v][i] = fadd2(ab[v][i], d[i]);
            aw[v][i] = ffma2(d[i], h, aw[v][i]);
            s1 = fadd2(s1, tt);
            s2 = ffma2(tt, h, s2);
          }
        }
      }
      sum[2 * k] = f2_sum(s1);
      sum[2 * k + 1] = f2_sum(s2);
    }
    block_sums<2 * R>(sum, red[it & 1]);
    if (t == 0 && it + stages < q.nb) q.issue(it + stages, s);
    if (++s == stages) s = 0, ph ^= 1;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (k < n) {
        const float c1 = sum[2 * k] * inv, c2 = sum[2 * k + 1] * inv * rs[k];
        // dx = rs (dy w - c1 - (x - mean) c2)
        const uint64_t r = twice(rs[k]), m = twice(-mean[k]), k1 = twice(-c1 * rs[k]),
                       k2 = twice(-c2 * rs[k]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (in[v]) {
            uint64_t e[P], d[P];
            pairs_of<E>(rx[k][v], e);
            pairs_of<E>(rd[k][v], d);
#pragma unroll
            for (int i = 0; i < P; ++i)
              e[i] = ffma2(d[i], fmul2(w[v][i], r), ffma2(fadd2(e[i], m), k2, k1));
            store_pairs<T, E>(dxr + v * team * E, e);
          }
        }
        dxr += dx.sr;
      }
      mean[k] = mean_n[k];
      rs[k] = rs_n[k];
    }
  }
  float* dst = part + (int64_t)blockIdx.x * 2 * dim;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (t + v * team) * E;
    if (in[v]) {
#pragma unroll
      for (int i = 0; i < P; i += 2) {
        *reinterpret_cast<ulonglong2*>(dst + c + 2 * i) = make_ulonglong2(aw[v][i], aw[v][i + 1]);
        *reinterpret_cast<ulonglong2*>(dst + dim + c + 2 * i) =
            make_ulonglong2(ab[v][i], ab[v][i + 1]);
      }
    }
  }
  if (!alive) drain_delay();
}

// out[j][i] = sum over p < parts of part[(j * parts + p)][i], i < 2 dim: one
// column per thread of x, sixteen threads of y share the parts, joined in order.
__global__ void __launch_bounds__(512)
join_kernel(const float* part, int parts, int dim, float* dw, float* db) {
  __shared__ float s[16][33];
  const int tiles = (2 * dim + 31) / 32, j = blockIdx.x / tiles;
  const int col = (blockIdx.x - j * tiles) * 32 + threadIdx.x;
  float a = 0.f;
  pdl_wait_previous();
  if (col < 2 * dim) {
    const float* p = part + (int64_t)j * parts * 2 * dim + col;
#pragma unroll 8
    for (int i = threadIdx.y; i < parts; i += 16) a += p[(int64_t)i * 2 * dim];
  }
  s[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y == 0 && col < 2 * dim) {
    a = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) a += s[i][threadIdx.x];
    float* dst = col < dim ? dw : db;
    const int c = col < dim ? col : col - dim;
    if (dst != nullptr) dst[(int64_t)j * dim + c] = a;
  }
}

constexpr int kSms = 148;
constexpr int kMaxDim = 16384;

// Elements per access: 16 bytes' worth, 2, or 1, whichever every row start, the
// width and the parameters allow.
static int access_width(int es, int dim, const Mat* m, int nm, const Par& par) {
  const int ps = par.bf16 ? 2 : 4;
  for (int e : {16 / es, 2}) {
    bool ok = dim % e == 0;
    for (int i = 0; i < nm; ++i)
      ok = ok && reinterpret_cast<uintptr_t>(m[i].p) % (e * es) == 0 && m[i].sg % e == 0 &&
           m[i].sr % e == 0;
    const int need = std::min(16, e * ps);  // load_par's widest access
    for (const void* p : {par.w, par.b})
      ok = ok && (p == nullptr || (reinterpret_cast<uintptr_t>(p) % need == 0 &&
                                   (par.stride * ps) % need == 0));
    if (ok) return e;
  }
  return 1;
}

// Rows of a ring kernel's turn, threads and ring depth for a row of nv
// vectors: R V = 4 vectors of every tensor in registers a turn. The forward
// takes two vectors a thread as soon as two warps remain (its two block-wide
// sums a turn cost the same for either: 16384 x 2048 bf16 30 -> 25 us), the
// backward, which has one, from 256 threads on (40 us at one, 41 at two).
struct RingPlan {
  int V, R, threads, stages, smem, per_sm;
};

static RingPlan ring_plan(int nv, int tensors) {
  RingPlan p{};
  p.V = nv <= (tensors == 1 ? 64 : 256) ? 1 : (nv <= 1024 ? 2 : 4);
  p.R = 4 / p.V;
  p.threads = ((nv + p.V - 1) / p.V + 31) / 32 * 32;
  const int stage = tensors * p.R * nv * 16;
  // resident blocks by registers (forward at most 85 a thread at V = 1, the
  // others up to 128), all within the SM's 227 KB
  p.per_sm = std::max(1, std::min(8, (tensors == 1 && p.V == 1 ? 768 : 512) / p.threads));
  p.stages = std::max(2, std::min(kMaxStages, 220 * 1024 / p.per_sm / stage));
  p.smem = p.stages * stage + kMaxStages * 8;
  return p;
}

// A ring needs rows of a kilobyte for its copies to pay, and holds 32 KB ones
static bool use_ring(int nv) { return nv >= 64 && nv <= 2048; }

struct Split {
  int chunks, per;
};

// blocks per group: `slots` over all groups, at least `least` rows each
static Split split_of(int groups, int rows, int slots, int least) {
  Split s{};
  const int want = std::max(1, slots / std::max(1, groups));
  s.per = std::max(least, (rows + want - 1) / want);
  s.chunks = std::max(1, (rows + s.per - 1) / s.per);
  return s;
}

template <typename T, int E, int V, bool WARP>
static int fwd_go(const Mat& x, const Mat& y, const Par& par, int64_t n, int rows, int dim,
                  float eps, float* stats, int threads, cudaStream_t st) {
  const int64_t blocks = WARP ? (n + threads / 32 - 1) / (threads / 32) : n;
  fwd_kernel<T, E, V, WARP><<<(unsigned)blocks, threads, 0, st>>>(x, y, par, n, rows, dim, eps,
                                                                  stats);
  return launch_status();
}

template <typename T, int E, int V>
static int fwd_ring_go(const Mat& x, const Mat& y, const Par& par, int groups, int rows, int dim,
                       float eps, float* stats, const RingPlan& p, int kid, cudaStream_t st) {
  auto* fn = fwd_ring_kernel<T, E, V, 4 / V>;
  const int rc = ensure_smem_attr((const void*)fn, 225 * 1024, kid);
  if (rc) return rc;
  const Split s = split_of(groups, rows, p.per_sm * kSms, 4 / V);
  fn<<<(unsigned)((int64_t)groups * s.chunks), p.threads, p.smem, st>>>(
      x, y, par, (int64_t)groups * rows, rows, dim, eps, stats, s.per, s.chunks, p.stages);
  return launch_status();
}

template <typename T, int E>
static int fwd_pick(const Mat& x, const Mat& y, const Par& par, int groups, int rows, int dim,
                    float eps, float* stats, cudaStream_t st) {
  const int nv = (dim + E - 1) / E;
  const int64_t n = (int64_t)groups * rows;
  if constexpr (E > 2) {
    // a few rows a block, or the ring's set-up is all there is. (It goes by the
    // rows of all groups: many groups of one or two rows take the ring too,
    // whose blocks then turn once.)
    if (use_ring(nv) && n >= 8 * kSms) {
      const RingPlan p = ring_plan(nv, 1);
      const int kid = kKernelNorm + (sizeof(T) == 2 ? 0 : 3);
      if (p.V == 1) return fwd_ring_go<T, E, 1>(x, y, par, groups, rows, dim, eps, stats, p, kid, st);
      if (p.V == 2)
        return fwd_ring_go<T, E, 2>(x, y, par, groups, rows, dim, eps, stats, p, kid + 1, st);
      return fwd_ring_go<T, E, 4>(x, y, par, groups, rows, dim, eps, stats, p, kid + 2, st);
    }
  }
  // a warp per row while the rows are many and a lane's share is at most 32
  // values (with pairs 8: 4000 x 514 bf16 6.9 us as blocks, 9.9 as warps of 16
  // pairs; single elements stay with warps: 1000 x 1001 fp32 4.4 against 4.8);
  // else a block per row, of up to 512 threads and 32 values each
  const int need = (nv + 31) / 32;
  constexpr int kLane = E == 2 ? 4 : 32 / E;
  if (need <= 1 || (need <= kLane && n >= 2 * kSms)) {
    const int th = n >= 8 * kSms ? 256 : (n >= 2 * kSms ? 128 : 32);
    if (need <= 1) return fwd_go<T, E, 1, true>(x, y, par, n, rows, dim, eps, stats, th, st);
    if constexpr (kLane >= 8)
      if (need <= kLane / 4)
        return fwd_go<T, E, kLane / 4, true>(x, y, par, n, rows, dim, eps, stats, th, st);
    if constexpr (E == 1)
      if (need <= 16) return fwd_go<T, E, 16, true>(x, y, par, n, rows, dim, eps, stats, th, st);
    return fwd_go<T, E, kLane, true>(x, y, par, n, rows, dim, eps, stats, th, st);
  }
  auto th = [&](int v) { return ((nv + v - 1) / v + 31) / 32 * 32; };
  if constexpr (E > 2) {
    if (nv <= 512) return fwd_go<T, E, 1, false>(x, y, par, n, rows, dim, eps, stats, th(1), st);
    return fwd_go<T, E, 32 / E, false>(x, y, par, n, rows, dim, eps, stats, th(32 / E), st);
  } else {
    if (nv <= 4 * 512) return fwd_go<T, E, 4, false>(x, y, par, n, rows, dim, eps, stats, th(4), st);
    if (nv <= 16 / E * 512)
      return fwd_go<T, E, 16 / E, false>(x, y, par, n, rows, dim, eps, stats, th(16 / E), st);
    return fwd_go<T, E, 32 / E, false>(x, y, par, n, rows, dim, eps, stats, th(32 / E), st);
  }
}

struct BwdPlan {
  Split s;
  bool ring, lng;
};

// The backward's blocks, each of which leaves one partial sum of dw and db:
// with the ring, or sums in shared memory (beyond 8 values a thread of 512), as
// many as are resident, else four an SM.
static BwdPlan bwd_plan(int es, bool vec, int groups, int rows, int dim) {
  const int nv = dim / (16 / es);
  BwdPlan p{};
  p.ring = vec && use_ring(nv);
  p.lng = !p.ring && dim > 8 * 512;
  const int slots = p.ring ? ring_plan(nv, 2).per_sm : p.lng ? (dim > 16 * 512 ? 1 : 2) : 4;
  p.s = split_of(groups, rows, slots * kSms, p.lng ? 1 : 4);
  return p;
}

template <typename T, int E, int V, int R, bool WARP>
static int bwd_go(const Mat& x, const Mat& dy, const Mat& dx, const Par& par, const float* stats,
                  int groups, int rows, int dim, const Split& s, int threads, float* part,
                  cudaStream_t st) {
  const int smem = WARP ? threads / 32 * 2 * dim * 4 : 0;
  bwd_kernel<T, E, V, R, WARP><<<(unsigned)((int64_t)groups * s.chunks), threads, smem, st>>>(
      x, dy, dx, par, stats, (int64_t)groups * rows, rows, dim, s.per, s.chunks, part);
  return launch_status();
}

template <typename T, int E, int V>
static int bwd_long_go(const Mat& x, const Mat& dy, const Mat& dx, const Par& par,
                       const float* stats, int groups, int rows, int dim, const Split& s, int kid,
                       float* part, cudaStream_t st) {
  auto* fn = bwd_long_kernel<T, E, V>;
  const int rc = ensure_smem_attr((const void*)fn, 3 * kMaxDim * 4, kid);
  if (rc) return rc;
  const int nv = (dim + E - 1) / E, threads = ((nv + V - 1) / V + 31) / 32 * 32;
  fn<<<(unsigned)((int64_t)groups * s.chunks), threads, 3 * dim * 4, st>>>(
      x, dy, dx, par, stats, (int64_t)groups * rows, rows, dim, s.per, s.chunks, part);
  return launch_status();
}

template <typename T, int E, int V>
static int bwd_ring_go(const Mat& x, const Mat& dy, const Mat& dx, const Par& par,
                       const float* stats, int groups, int rows, int dim, const Split& s,
                       const RingPlan& p, int kid, float* part, cudaStream_t st) {
  auto* fn = bwd_ring_kernel<T, E, V, 4 / V>;
  const int rc = ensure_smem_attr((const void*)fn, 225 * 1024, kid);
  if (rc) return rc;
  fn<<<(unsigned)((int64_t)groups * s.chunks), p.threads, p.smem, st>>>(
      x, dy, dx, par, stats, (int64_t)groups * rows, rows, dim, s.per, s.chunks, p.stages, part);
  return launch_status();
}

template <typename T, int E>
static int bwd_pick(const Mat& x, const Mat& dy, const Mat& dx, const Par& par,
                    const float* stats, int groups, int rows, int dim, const BwdPlan& pl,
                    float* part, cudaStream_t st) {
  const int nv = (dim + E - 1) / E;
  const Split& s = pl.s;
  if constexpr (E > 2) {
    if (pl.ring) {
      const RingPlan p = ring_plan(nv, 2);
      const int kid = kKernelNorm + 6 + (sizeof(T) == 2 ? 0 : 3);
      if (p.V == 1) return bwd_ring_go<T, E, 1>(x, dy, dx, par, stats, groups, rows, dim, s, p, kid, part, st);
      if (p.V == 2) return bwd_ring_go<T, E, 2>(x, dy, dx, par, stats, groups, rows, dim, s, p, kid + 1, part, st);
      return bwd_ring_go<T, E, 4>(x, dy, dx, par, stats, groups, rows, dim, s, p, kid + 2, part, st);
    }
  }
  if (nv <= 32)  // a warp holds the row (dim <= 256): 8 teams, 16 KB of shared memory at most
    return bwd_go<T, E, 1, 4, true>(x, dy, dx, par, stats, groups, rows, dim, s, 256, part, st);
  auto th = [&](int v) { return ((nv + v - 1) / v + 31) / 32 * 32; };
  constexpr int kLong = kKernelNormLong + (sizeof(T) == 2 ? 0 : 5);
  if constexpr (E > 2) {
    // 33 to 63 vectors, or fp32 rows of more than 32 KB
    if constexpr (E == 4)
      if (pl.lng)
        return bwd_long_go<T, E, 8>(x, dy, dx, par, stats, groups, rows, dim, s, kLong + 4, part, st);
    return bwd_go<T, E, 1, 4, false>(x, dy, dx, par, stats, groups, rows, dim, s, th(1), part, st);
  } else {
    constexpr int kid = kLong + 2 * (E - 1);
    if (!pl.lng) {
      if (nv <= 4 / E * 512)
        return bwd_go<T, E, 4 / E, 2, false>(x, dy, dx, par, stats, groups, rows, dim, s, th(4 / E), part, st);
      return bwd_go<T, E, 8 / E, 1, false>(x, dy, dx, par, stats, groups, rows, dim, s, th(8 / E), part, st);
    }
    if (nv <= 16 / E * 512)
      return bwd_long_go<T, E, 16 / E>(x, dy, dx, par, stats, groups, rows, dim, s, kid, part, st);
    return bwd_long_go<T, E, 32 / E>(x, dy, dx, par, stats, groups, rows, dim, s, kid + 1, part, st);
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
  const int es = dtype == FA_DTYPE_BF16 ? 2 : 4;
  const int e = ln::access_width(es, dim, m, 2, par);
#define FA_LN(T, E) ln::fwd_pick<T, E>(m[0], m[1], par, groups, rows, dim, eps, stats, st)
  if (es == 2)
    return e == 8   ? FA_LN(__nv_bfloat16, 8)
           : e == 2 ? FA_LN(__nv_bfloat16, 2)
                    : FA_LN(__nv_bfloat16, 1);
  return e == 4 ? FA_LN(float, 4) : e == 2 ? FA_LN(float, 2) : FA_LN(float, 1);
#undef FA_LN
}

size_t layer_norm_bwd_workspace(int groups, int rows, int dim) {
  // the most that any type and alignment takes
  int64_t parts = 0;
  for (int es : {2, 4})
    for (bool vec : {false, true})
      parts = std::max<int64_t>(parts, ln::bwd_plan(es, vec, groups, rows, dim).s.chunks);
  return (size_t)groups * parts * 2 * dim * sizeof(float);
}

int launch_layer_norm_bwd(int dtype, int groups, int rows, int dim, const fa_tensor_t* x,
                          const void* w, int par_dtype, int64_t par_stride, int unit_offset,
                          const fa_tensor_t* dy, const float* stats, const fa_tensor_t* dx,
                          float* dw, float* db, int shared, void* ws, cudaStream_t st) {
  if (groups == 0 && !shared) return FA_OK;
  float* part = reinterpret_cast<float*>(ws);
  const int es = dtype == FA_DTYPE_BF16 ? 2 : 4;
  const ln::Mat m[3] = {ln_mat(x), ln_mat(dy), ln_mat(dx)};
  const ln::Par par{w, nullptr, par_stride, par_dtype == FA_DTYPE_BF16, unit_offset ? 1.f : 0.f};
  const int e = ln::access_width(es, dim, m, 3, par);
  const ln::BwdPlan pl = ln::bwd_plan(es, e == 16 / es, groups, rows, dim);
  if (groups > 0) {
    int rc;
#define FA_LN(T, E) \
  ln::bwd_pick<T, E>(m[0], m[1], m[2], par, stats, groups, rows, dim, pl, part, st)
    if (es == 2)
      rc = e == 8   ? FA_LN(__nv_bfloat16, 8)
           : e == 2 ? FA_LN(__nv_bfloat16, 2)
                    : FA_LN(__nv_bfloat16, 1);
    else
      rc = e == 4 ? FA_LN(float, 4) : e == 2 ? FA_LN(float, 2) : FA_LN(float, 1);
#undef FA_LN
    if (rc != FA_OK) return rc;
  }
  if (dw == nullptr && db == nullptr) return FA_OK;
  const int outs = shared ? 1 : groups, parts = shared ? groups * pl.s.chunks : pl.s.chunks;
  // may start while the backward's last blocks run, and waits for them
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((int64_t)(2 * dim + 31) / 32 * outs));
  cfg.blockDim = dim3(32, 16);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = groups > 0 ? 1 : 0;
  const cudaError_t err =
      cudaLaunchKernelEx(&cfg, ln::join_kernel, (const float*)part, parts, dim, dw, db);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return record_cuda_error(err);
  }
  return launch_status();
}

int norm_device_status() { return tu_device_status(); }

}  // namespace fa
