// orthogonalize.cu — Newton-Schulz orthogonalisation of an update matrix.
//
//   X_0 = G / (|G|_F + eps),   X_{k+1} = a X_k + (b Q + c Q^2) X_k,  Q = X_k X_k^T
//
// pushes every singular value of G towards one: the result approximates the
// orthogonal factor of G's polar decomposition, the step direction of an
// optimiser that treats a weight as a linear map. Two forms, by the short
// side r of the matrix:
//
// r <= 64 (the factors of adapters), thin_kernel. All X_k are X_k = P_k X_0
// with P_k a polynomial in the r x r Gram matrix Q_0 of X_0, and everything
// commutes: with M = a + b Q + c Q^2, P <- M P and Q <- M Q M. So the long
// side is read for Q_0 and once more (from L2) for P X_0, and all steps stay
// on chip. Forming Q_0 squares the singular values, so it, and the steps, are
// in fp64: a direction of relative strength 1e-3 is 1e-6 in Q_0, of which fp32
// sums would leave a digit, while P amplifies it 485-fold. One cluster per
// matrix: its CTAs sum their parts of Q_0, exchange them through distributed
// shared memory in CTA order, run the same steps, and each applies P to its
// own part of the long side.
//
// r > 64: three tensor-core products a step (gemm_wide_sm100.cu; both Gram
// products compute the tiles on and below the diagonal and mirror them).
// Operands are fp16, not bf16: after the normalisation every quantity is
// bounded by about one, so eleven bits are worth more than range (a factor
// 256 on X and 64 on Q keep small entries clear of fp16's subnormals). What
// must not be rounded to 11 bits is X itself, since a rounding of X is noise
// in all directions and the following steps amplify it up to 485-fold where
// G has no strength. X is therefore kept as the sum of two fp16 matrices, hi
// and lo (22 bits); the products read hi, and the epilogue adds a (hi + lo)
// in fp32. Errors of the products stay within G's own directions, where the
// steps contract. Against 64 bits: 2.4e-3 of the result's norm on Gaussian
// noise, 1.7e-3 to 1.9e-3 on a few strong directions over noise; the final
// rounding to bf16 alone is 1.7e-3. Coefficients whose steps would take singular
// values out of fp16's range are refused (in_range).
//
// Measured: 16 x (16 x 4096) bf16 13 us, 8 x (64 x 4096) 78 us (fp64 tensor
// instructions, about half their rate); 4096 x 8192 fp32 2.1 to 2.2 ms under
// the power cap, its products 102 (Gram), 60 (Q^2) and 190 us (update); 1024 x
// 1024 148 us, 512 x 512 89 us, 16 products of 5 to 9 us in a chain.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "attn_common.h"
#include "gemm.h"
#include "gemm_ptx.cuh"

namespace fa {
namespace ns {

constexpr int kThinThreads = 512;

template <typename T>
__device__ __forceinline__ float ld_f(const T* p);
template <>
__device__ __forceinline__ float ld_f<float>(const float* p) { return __ldg(p); }
template <>
__device__ __forceinline__ float ld_f<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}

__device__ __forceinline__ double ld_cluster_f64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}

// Tile t of the upper triangle of an n x n tile grid, row-major: (i, j), i <= j
__device__ __forceinline__ void upper_tile(int t, int n, int& i, int& j) {
  i = 0;
  while (t >= n - i) t -= n - i++;
  j = i + t;
}

// D (8 x 8) += A (8 x 4) B (4 x 8) in fp64. Lane (g, q) = (lane / 4, lane % 4)
// holds A[g][q], B[q][g], and D[g][2 q], D[g][2 q + 1]: a lane's value of a
// symmetric matrix's 8 x 4 block is the same as A and as B.
__device__ __forceinline__ void dmma(double* d, double a, double b) {
  asm volatile(
      "mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
      : "+d"(d[0]), "+d"(d[1])
      : "d"(a), "d"(b));
}

template <int R>
struct Thin {
  static constexpr int kLd = R + 4;  // doubles: an 8 x 4 block has no bank conflicts
  static constexpr int kMat = R * kLd;
  static constexpr int kN = R / 8;
  static constexpr int kTiles = kN * (kN + 1) / 2;
  // Gram sums: warps that split the positions, and per set of 8 x 8 tiles
  static constexpr int kSplit = R >= 48 ? 4 : 16;
  static constexpr int kPart = kSplit * kTiles * 64;
  static constexpr int kRest = 5 * kMat > kPart ? 5 * kMat : kPart;
  static constexpr int kSmem = (kMat + kTiles * 64 + kRest) * 8;
};
static_assert(Thin<64>::kSmem <= 232448, "shared memory");

// The values of 8 rows (8 * tile + g) at the positions of one turn: lane q
// takes the EB positions l + EB q .. (wide) or l + q, l + 4 + q, .. (tall);
// the sum over positions does not ask for their order.
template <typename T, bool TALL>
struct Turn {
  static constexpr int EB = 16 / sizeof(T);
  T e[EB];

  __device__ __forceinline__ void load(const T* g, int64_t row, int r, int j, int l, int l1, bool vec,
                                       int q) {
    if constexpr (TALL) {
#pragma unroll
      for (int u = 0; u < EB; ++u) {
        const int p = l + 4 * u + q;
        e[u] = j < r && p < l1 ? g[(int64_t)p * row + j] : T(0.f);
      }
    } else {
      const int p = l + EB * q;
      if (vec && j < r && p + EB <= l1) {
        *reinterpret_cast<uint4*>(e) = __ldg(reinterpret_cast<const uint4*>(g + (int64_t)j * row + p));
      } else {
#pragma unroll
        for (int u = 0; u < EB; ++u)
          e[u] = j < r && p + u < l1 ? g[(int64_t)j * row + p + u] : T(0.f);
      }
    }
  }
  __device__ __forceinline__ double at(int u) const { return (double)(float)e[u]; }
};

// One cluster per matrix (blockIdx.x / parts). TALL: the long side is the rows.
template <typename T, int R, bool TALL>
__global__ void __launch_bounds__(kThinThreads, R >= 48 ? 1 : 2)
thin_kernel(const T* g, int64_t g_batch, int64_t g_row, __nv_bfloat16* o, int64_t o_batch,
            int64_t o_row, int r, int len, int parts, int steps, int vec, int ovec, double ca,
            double cb, double cc, double eps) {
  using C = Thin<R>;
  constexpr int LD = C::kLd, NT = C::kTiles;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  double* A = reinterpret_cast<double*>(smem_raw);
  double* mine = A + C::kMat;  // this CTA's Gram sums, (tile, 8, 8)
  double* rest = mine + NT * 64;
  const int mat = blockIdx.x / parts, part = blockIdx.x - mat * parts;
  const T* gm = g + (int64_t)mat * g_batch;
  // this CTA's share of the long side, in whole turns
  const int turns = (len + 31) / 32;
  const int l0 = (int)((int64_t)turns * part / parts) * 32;
  const int l1 = min(len, (int)((int64_t)turns * (part + 1) / parts) * 32);
  const int tid = threadIdx.x, warp = warp_id(), lane = lane_id(), gg = lane >> 2, qq = lane & 3;

  // ---- Gram matrix of the share
  {
    constexpr int EB = Turn<T, TALL>::EB, kTurn = 4 * EB;
    // tiles of a warp: all, or from R = 48 on a quarter of the triangle: its
    // first or second half of rows against themselves (10 tiles at R = 64), or
    // the first half's rows with two of the other columns (8)
    constexpr bool kRoles = R >= 48;
    constexpr int NF = kRoles ? C::kN / 2 : C::kN;
    constexpr int ND = NF * (NF + 1) / 2;
    constexpr int NR = kRoles ? NF : 0;  // rows of the rectangles
    const int role = kRoles ? warp & 3 : 0, set = kRoles ? warp >> 2 : warp;
    const int base = role == 1 ? NF : 0;
    const int cols = role == 2 ? NF : NF + 2;  // (R = 48: the second has one column)
    double acc[ND][2];
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i][0] = acc[i][1] = 0.0;
    if (!kRoles || role < 2) {
      for (int l = l0 + set * kTurn; l < l1; l += C::kSplit * kTurn) {
        Turn<T, TALL> f[NF];
#pragma unroll
        for (int i = 0; i < NF; ++i)
          f[i].load(gm, g_row, r, (base + i) * 8 + gg, l, l1, vec, qq);
#pragma unroll
        for (int u = 0; u < EB; ++u) {
          double x[NF];
#pragma unroll
          for (int i = 0; i < NF; ++i) x[i] = f[i].at(u);
          int k = 0;
#pragma unroll
          for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int j = i; j < NF; ++j) dmma(acc[k++], x[i], x[j]);
        }
      }
    } else if constexpr (kRoles) {
      for (int l = l0 + set * kTurn; l < l1; l += C::kSplit * kTurn) {
        Turn<T, TALL> f[NR], h[2];
#pragma unroll
        for (int i = 0; i < NR; ++i) f[i].load(gm, g_row, r, i * 8 + gg, l, l1, vec, qq);
#pragma unroll
        for (int i = 0; i < 2; ++i) h[i].load(gm, g_row, r, (cols + i) * 8 + gg, l, l1, vec, qq);
#pragma unroll
        for (int u = 0; u < EB; ++u) {
          const double y0 = h[0].at(u), y1 = h[1].at(u);
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            const double x = f[i].at(u);
            dmma(acc[2 * i], x, y0);
            dmma(acc[2 * i + 1], x, y1);
          }
        }
      }
    }
    // the sets' sums join in order
    double* p = rest + (int64_t)set * NT * 64;
    auto put = [&](int ti, int tj, const double* d) {
      int at = 0;  // place of (ti, tj) in the upper triangle
      for (int i = 0; i < ti; ++i) at += C::kN - i;
      double* w = p + (at + tj - ti) * 64 + gg * 8 + 2 * qq;
      w[0] = d[0];
      w[1] = d[1];
    };
    if (!kRoles || role < 2) {
      int k = 0;
#pragma unroll
      for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = i; j < NF; ++j) put(base + i, base + j, acc[k++]);
    } else if constexpr (kRoles) {
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (cols + j < C::kN) put(i, cols + j, acc[2 * i + j]);
    }
  }
  __syncthreads();
  for (int i = tid; i < NT * 64; i += kThinThreads) {
    double s = 0.0;
    for (int k = 0; k < C::kSplit; ++k) s += rest[k * NT * 64 + i];
    mine[i] = s;
  }
  // and the CTAs' in CTA order: each CTA sums its share of the entries over
  // the cluster, then takes the other shares from their owners (all reading
  // all took 14 us of a 38 us call at 64 x 4096)
  double* sums = rest;  // (the sets' sums are done with)
  constexpr int kAll = NT * 64;
  const int share = (kAll + parts - 1) / parts;
  if (parts > 1) {
    cluster_sync();
    const int i1 = min(kAll, (part + 1) * share);
    for (int i = part * share + tid; i < i1; i += kThinThreads) {
      const uint32_t at = smem_u32(mine + i);
      double v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = k < parts ? ld_cluster_f64(mapa(at, k)) : 0.0;
      double s = 0.0;
#pragma unroll
      for (int k = 0; k < 16; ++k) s += v[k];
      sums[i] = s;
    }
    cluster_sync();
  } else {
    __syncthreads();
  }
#pragma unroll 5
  for (int i = tid; i < kAll; i += kThinThreads) {
    const double s = parts > 1 ? ld_cluster_f64(mapa(smem_u32(sums + i), i / share)) : mine[i];
    int ti, tj;
    upper_tile(i >> 6, C::kN, ti, tj);
    const int p = ti * 8 + ((i >> 3) & 7), c = tj * 8 + (i & 7);
    A[p * LD + c] = s;
    if (ti != tj) A[c * LD + p] = s;
  }
  if (parts > 1) cluster_sync();  // nobody reads another CTA's memory after this
  else __syncthreads();
  double tr = 0.0;
#pragma unroll 8
  for (int i = 0; i < R; ++i) tr += A[i * LD + i];
  double inv = 1.0 / (sqrt(tr) + eps);
  __syncthreads();
  for (int i = tid; i < R * R; i += kThinThreads) A[(i / R) * LD + i % R] *= inv * inv;
  __syncthreads();

  // ---- the steps. With S = A^2: M = a + b A + c S, P <- M P, and A <- A M^2 =
  // a^2 A + S U, U = c^2 A S + 2 b c S + (b^2 + 2 a c) A + 2 a b; the products
  // of one line below are independent and share the warps.
  double *S = rest, *M = S + C::kMat, *U = M + C::kMat, *P = U + C::kMat, *P2 = P + C::kMat;
  // tile (ti, tj) of X Y for symmetric commuting X, Y; f(row, column, value)
  auto product = [&](int tile, const double* X, const double* Y, auto&& f) {
    int ti, tj;
    upper_tile(tile, C::kN, ti, tj);
    const double* x = X + (ti * 8 + gg) * LD + qq;
    const double* y = Y + (tj * 8 + gg) * LD + qq;
    double d[2][2] = {};
#pragma unroll
    for (int k = 0; k < R; k += 8) {
      dmma(d[0], x[k], y[k]);
      dmma(d[1], x[k + 4], y[k + 4]);
    }
    const int p = ti * 8 + gg, c = tj * 8 + 2 * qq;
    f(p, c, d[0][0] + d[1][0], ti != tj);
    f(p, c + 1, d[0][1] + d[1][1], ti != tj);
  };
  constexpr int kWarps = kThinThreads / 32;
  for (int s = 0; s < steps; ++s) {
    const bool last = s + 1 == steps;
    double* M0 = s == 0 ? P : M;  // the first step's M is P
    for (int t = warp; t < NT; t += kWarps)
      product(t, A, A, [&](int p, int c, double v, bool mirror) {
        const double m = cc * v + cb * A[p * LD + c] + (p == c ? ca : 0.0);
        S[p * LD + c] = v;
        M0[p * LD + c] = m;
        if (mirror) S[c * LD + p] = v, M0[c * LD + p] = m;
      });
    __syncthreads();
    const int n_u = last ? 0 : NT, n_p = s == 0 ? 0 : NT;
    for (int t = warp; t < n_u + n_p; t += kWarps) {
      if (t < n_u)
        product(t, A, S, [&](int p, int c, double v, bool mirror) {
          const double u = cc * cc * v + 2.0 * cb * cc * S[p * LD + c] +
                           (cb * cb + 2.0 * ca * cc) * A[p * LD + c] + (p == c ? 2.0 * ca * cb : 0.0);
          U[p * LD + c] = u;
          if (mirror) U[c * LD + p] = u;
        });
      else
        product(t - n_u, M, P, [&](int p, int c, double v, bool mirror) {
          P2[p * LD + c] = v;
          if (mirror) P2[c * LD + p] = v;
        });
    }
    __syncthreads();
    if (s > 0) {
      double* w = P;
      P = P2;
      P2 = w;
    }
    if (last) break;
    for (int t = warp; t < NT; t += kWarps)
      product(t, S, U, [&](int p, int c, double v, bool mirror) {
        const double n = v + ca * ca * A[p * LD + c];
        A[p * LD + c] = n;
        if (mirror) A[c * LD + p] = n;
      });
    __syncthreads();
  }
  // P / |G| in fp32 (its largest entries are a few hundred times the
  // result's: 24 bits leave the bf16 result its own rounding), in A's place.
  // Where |G| is so small or large that fp32 would lose the quotient, a power
  // of two goes to G's entries instead.
  float* pf = reinterpret_cast<float*>(A);
  int up = isfinite(inv) && inv > 0.0 ? ilogb(inv) : 0;
  up = up > 60 || up < -60 ? max(-126, min(126, up)) : 0;
  const float gain = (float)scalbn(1.0, up);
  inv = scalbn(inv, -up);
  for (int i = tid; i < R * R; i += kThinThreads) pf[i] = (float)(P[(i / R) * LD + i % R] * inv);
  __syncthreads();

  // ---- O = P G over the share, a long position per thread
  __nv_bfloat16* om = o + (int64_t)mat * o_batch;
  for (int l = l0 + tid; l < l1; l += kThinThreads) {
    uint64_t sum[R / 2];
#pragma unroll
    for (int i = 0; i < R / 2; ++i) sum[i] = 0;
    auto add = [&](int j, float x) {
      x *= gain;
      const uint64_t xx = f2_pack(x, x);
      const ulonglong2* pr = reinterpret_cast<const ulonglong2*>(pf + j * R);
#pragma unroll
      for (int i = 0; i < R / 4; ++i) {
        const ulonglong2 w = pr[i];
        sum[2 * i] = ffma2(w.x, xx, sum[2 * i]);
        sum[2 * i + 1] = ffma2(w.y, xx, sum[2 * i + 1]);
      }
    };
    constexpr int EB = 16 / sizeof(T);
    const T* row = gm + (int64_t)l * g_row;
    if (TALL && vec == 1) {  // a row of r values, 8 bytes at a time
#pragma unroll 1
      for (int j = 0; j < r; j += EB / 2) {
        const uint2 raw = __ldg(reinterpret_cast<const uint2*>(row + j));
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int u = 0; u < EB / 2; ++u) add(j + u, (float)e[u]);
      }
    } else if (TALL && vec) {  // 16 bytes
#pragma unroll 1
      for (int j = 0; j < r; j += EB) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row + j));
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int u = 0; u < EB; ++u) add(j + u, (float)e[u]);
      }
    } else {
#pragma unroll 8
      for (int j = 0; j < r; ++j)
        add(j, ld_f<T>(TALL ? gm + (int64_t)l * g_row + j : gm + (int64_t)j * g_row + l));
    }
    if (TALL && ovec == 1) {
#pragma unroll
      for (int i = 0; i < R / 4; ++i) {
        if (4 * i < r) {
          float f[4];
          f2_unpack(sum[2 * i], f[0], f[1]);
          f2_unpack(sum[2 * i + 1], f[2], f[3]);
          *reinterpret_cast<uint2*>(om + (int64_t)l * o_row + 4 * i) =
              make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
        }
      }
    } else if (TALL && ovec) {
#pragma unroll
      for (int i = 0; i < R / 8; ++i) {
        if (8 * i < r) {
          float f[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) f2_unpack(sum[4 * i + k], f[2 * k], f[2 * k + 1]);
          *reinterpret_cast<uint4*>(om + (int64_t)l * o_row + 8 * i) =
              make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]),
                         pack_bf16(f[6], f[7]));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < R / 2; ++i) {
        float u, v;
        f2_unpack(sum[i], u, v);
        __nv_bfloat16* w = TALL ? om + (int64_t)l * o_row + 2 * i : om + (int64_t)(2 * i) * o_row + l;
        if (2 * i < r) w[0] = __float2bfloat16_rn(u);
        if (2 * i + 1 < r) w[TALL ? 1 : o_row] = __float2bfloat16_rn(v);
      }
    }
  }
}

// ------------------------------------------------------------ the wide form

constexpr int kNormBlocks = 592;  // partial sums of squares per matrix: four an SM

// part[mat][block] = sum of squares over every kNormBlocks-th row, in fp64 (the
// squares of fp32 values may leave fp32's range). `vec`: 16-byte loads.
template <typename T>
__global__ void __launch_bounds__(256)
norm_kernel(const T* g, int64_t g_batch, int64_t g_row, int m, int n, int vec, double* part) {
  __shared__ double red[8];
  constexpr int E = 16 / sizeof(T);
  const int mat = blockIdx.y;
  const T* gm = g + (int64_t)mat * g_batch;
  double s = 0.0;
  for (int i = blockIdx.x; i < m; i += kNormBlocks) {
    const T* row = gm + (int64_t)i * g_row;
    int done = 0;
    if (vec) {
      done = n / E * E;
#pragma unroll 4
      for (int j = threadIdx.x * E; j < done; j += 256 * E) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(row + j));
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const double v = (double)(float)e[k];
          s = fma(v, v, s);
        }
      }
    }
    for (int j = done + threadIdx.x; j < n; j += 256) {
      const double v = (double)ld_f<T>(row + j);
      s = fma(v, v, s);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane_id() == 0) red[warp_id()] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) s += red[i];
    part[(int64_t)mat * kNormBlocks + blockIdx.x] = s;
  }
}

// |G| + eps = nu 2^e, 1 <= nu < 2, from the partial sums (256 threads)
__device__ __forceinline__ double norm_of(const double* part, double eps, int* e) {
  __shared__ double red[8];
  double s = 0.0;
  for (int i = threadIdx.x; i < kNormBlocks; i += 256) s += part[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane_id() == 0) red[warp_id()] = s;
  __syncthreads();
  s = red[0];
  for (int i = 1; i < 8; ++i) s += red[i];
  const double v = sqrt(s) + eps;
  *e = isfinite(v) && v > 0.0 ? ilogb(v) : 0;
  return scalbn(v, -*e);
}

// X_0 nu 256 = G 2^(8 - e) as fp16 hi + lo / 2048 (a power of two: exact for
// bf16 inputs in range), transposed when the input is tall. 64 x 64 tiles.
// Block (0, 0) of a matrix also writes its coefficients: the division by nu is
// folded into the first step's. coef: (steps, 2 (Q then X), batch, 2).
template <typename T, bool TALL>
__global__ void __launch_bounds__(256)
split_kernel(const T* g, int64_t g_batch, int64_t g_row, int m, int n, const double* part,
             double eps, __half* hi, __half* lo, int ld, int64_t x_batch, float* coef, int batch,
             int steps, double ca, double cb, double cc) {
  __shared__ float tile[64][65];
  const int mat = blockIdx.z;
  int e;
  const double nu = norm_of(part + (int64_t)mat * kNormBlocks, eps, &e);
  // 2^(8 - e) in two factors: it may lie outside fp32's range
  const float scale = (float)scalbn(1.0, (8 - e) / 2), scale2 = (float)scalbn(1.0, 8 - e - (8 - e) / 2);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < steps) {
    const int s = threadIdx.x;
    const double v = s == 0 ? nu : 1.0;
    float* q = coef + ((int64_t)(2 * s) * batch + mat) * 2;
    q[0] = (float)(cb / (v * v * v));
    q[1] = (float)(cc / (v * v * v * v * v) / 64.0);
    float* x = coef + ((int64_t)(2 * s + 1) * batch + mat) * 2;
    x[0] = (float)(ca / v);
    x[1] = 1.f / 64.f;
  }
  const T* gm = g + (int64_t)mat * g_batch;
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
  const int c = threadIdx.x & 63;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int r = (threadIdx.x >> 6) + 4 * k;
    float v = 0.f;
    if (i0 + r < m && j0 + c < n) v = ld_f<T>(gm + (int64_t)(i0 + r) * g_row + j0 + c);
    tile[r][c] = v * scale * scale2;
  }
  __syncthreads();
  // two columns a thread
  const int rows = TALL ? n : m, cols = TALL ? m : n;  // of X
  const int r0 = TALL ? j0 : i0, c0 = TALL ? i0 : j0;
  const int cp = (threadIdx.x & 31) * 2;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int r = (threadIdx.x >> 5) + 8 * k;
    if (r0 + r < rows && c0 + cp < cols) {
      const float u = TALL ? tile[cp][r] : tile[r][cp], v = TALL ? tile[cp + 1][r] : tile[r][cp + 1];
      const uint32_t h = pack_f16(u, v);
      const float2 hf = unpack_f16(h);
      const int64_t at = (int64_t)mat * x_batch + (int64_t)(r0 + r) * ld + c0 + cp;
      *reinterpret_cast<uint32_t*>(hi + at) = h;  // ld is even: a last odd column has its pad
      *reinterpret_cast<uint32_t*>(lo + at) = pack_f16((u - hf.x) * 2048.f, (v - hf.y) * 2048.f);
    }
  }
}

static size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
static int ld8(int n) { return (n + 7) / 8 * 8; }

struct Space {  // workspace of the wide form
  size_t part, coef, x, q, total;
};

static Space space_of(int batch, int m, int n, int steps) {
  Space s{};
  s.part = align256((size_t)batch * kNormBlocks * 8);
  s.coef = align256((size_t)batch * steps * 4 * 4);
  s.x = align256((size_t)batch * m * ld8(n) * 2);
  s.q = align256((size_t)batch * m * ld8(m) * 2);
  s.total = s.part + s.coef + 3 * s.x + 2 * s.q;
  return s;
}

template <typename T, int R, bool TALL>
static int thin_go(const void* g, int64_t gb, int64_t gr, void* o, int64_t ob, int64_t orow,
                   int batch, int r, int len, int steps, const float* c, float eps, int kid,
                   cudaStream_t st) {
  auto* fn = thin_kernel<T, R, TALL>;
  const int rc = ensure_smem_attr((const void*)fn, Thin<R>::kSmem, kid);
  if (rc) return rc;
  // CTAs per matrix: of 1 .. 16, what is soonest done by the clusters of that
  // size that are resident at once (a cluster stays within a GPC, so large ones
  // leave SMs idle). A matrix costs about as much apart from its positions as
  // 1500 positions do.
  int parts = 1;
  int64_t best = INT64_MAX;
  for (int c = 1; c <= 16; c *= 2) {
    if (c > 1 && c * 128 > len) break;
    int fit = 0;
    const int rf = clusters_that_fit((const void*)fn, kThinThreads, Thin<R>::kSmem, c, kid, &fit);
    if (rf) return rf;
    if (fit <= 0) break;
    const int64_t cost = (int64_t)((batch + fit - 1) / fit) * (1500 + (len + c - 1) / c);
    if (cost < best) best = cost, parts = c;
  }
  const int es = (int)sizeof(T);
  // 16-byte reads of rows (2): wide rows start anywhere in a share of whole
  // turns; tall ones hold a multiple of a vector, or of 8 bytes (1: 16 x 4096 x
  // 12 bf16 12.3 us against 18.9 by elements; the Gram sums read tall rows so)
  auto starts = [&](int bytes) {
    return reinterpret_cast<uintptr_t>(g) % bytes == 0 && gb * es % bytes == 0 &&
           gr * es % bytes == 0 && (!TALL || r * es % bytes == 0);
  };
  const int vec = starts(16) ? 2 : TALL && starts(8) ? 1 : 0;
  const int ovec = r % 8 == 0 ? 2 : r % 4 == 0 ? 1 : 0;  // o's rows start on 16 bytes
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(batch * parts));
  cfg.blockDim = dim3(kThinThreads);
  cfg.dynamicSmemBytes = Thin<R>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(
      &cfg, fn, reinterpret_cast<const T*>(g), gb, gr, reinterpret_cast<__nv_bfloat16*>(o), ob,
      orow, r, len, parts, steps, vec, ovec, (double)c[0], (double)c[1], (double)c[2], (double)eps);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return record_cuda_error(e);
  }
  return launch_status();
}

template <typename T, bool TALL>
static int thin_pick(const void* g, int64_t gb, int64_t gr, void* o, int64_t ob, int64_t orow,
                     int batch, int r, int len, int steps, const float* c, float eps, int kid,
                     cudaStream_t st) {
  if (r <= 16)
    return thin_go<T, 16, TALL>(g, gb, gr, o, ob, orow, batch, r, len, steps, c, eps, kid, st);
  if (r <= 32)
    return thin_go<T, 32, TALL>(g, gb, gr, o, ob, orow, batch, r, len, steps, c, eps, kid + 1, st);
  if (r <= 48)
    return thin_go<T, 48, TALL>(g, gb, gr, o, ob, orow, batch, r, len, steps, c, eps, kid + 2, st);
  return thin_go<T, 64, TALL>(g, gb, gr, o, ob, orow, batch, r, len, steps, c, eps, kid + 3, st);
}

template <typename T>
static int wide_go(const void* g, int64_t gb, int64_t gr, void* o, int64_t ob, int64_t orow,
                   int batch, int rows, int cols, int steps, const float* c, float eps, void* ws,
                   cudaStream_t st) {
  const bool tall = rows > cols;
  const int m = std::min(rows, cols), n = std::max(rows, cols);
  const Space sp = space_of(batch, m, n, steps);
  uint8_t* w = reinterpret_cast<uint8_t*>(ws);
  double* part = reinterpret_cast<double*>(w);
  w += sp.part;
  float* coef = reinterpret_cast<float*>(w);
  w += sp.coef;
  __half* hi[2];
  hi[0] = reinterpret_cast<__half*>(w);
  w += sp.x;
  hi[1] = reinterpret_cast<__half*>(w);
  w += sp.x;
  __half* lo = reinterpret_cast<__half*>(w);
  w += sp.x;
  __half* q = reinterpret_cast<__half*>(w);
  w += sp.q;
  __half* pq = reinterpret_cast<__half*>(w);
  const int ldx = ld8(n), ldq = ld8(m);
  const int64_t xb = (int64_t)m * ldx, qb = (int64_t)m * ldq;
  const T* gp = reinterpret_cast<const T*>(g);
  const int vec = reinterpret_cast<uintptr_t>(g) % 16 == 0 && gb * (int)sizeof(T) % 16 == 0 &&
                  gr * (int)sizeof(T) % 16 == 0;
  norm_kernel<T><<<dim3(kNormBlocks, batch), 256, 0, st>>>(gp, gb, gr, rows, cols, vec, part);
  int rc = launch_status();
  if (rc) return rc;
  const dim3 tiles((cols + 63) / 64, (rows + 63) / 64, batch);
  if (tall)
    split_kernel<T, true><<<tiles, 256, 0, st>>>(gp, gb, gr, rows, cols, part, eps, hi[0], lo, ldx,
                                                 xb, coef, batch, steps, c[0], c[1], c[2]);
  else
    split_kernel<T, false><<<tiles, 256, 0, st>>>(gp, gb, gr, rows, cols, part, eps, hi[0], lo, ldx,
                                                  xb, coef, batch, steps, c[0], c[1], c[2]);
  rc = launch_status();
  if (rc) return rc;
  auto x_mat = [&](const __half* p) { return Mat3{p, batch, m, n, xb, ldx, 0}; };
  auto q_mat = [&](const __half* p) { return Mat3{p, batch, m, m, qb, ldq, 0}; };
  TmapMemo maps;
  for (int s = 0; s < steps; ++s) {
    const __half* h = hi[s & 1];
    {  // Q 64 = (256 X)(256 X)^T / 1024
      WideOperands op;
      op.a = op.b = x_mat(h);
      op.d = q_mat(q);
      WideParams p;
      p.M = p.N = m;
      p.K = n;
      p.batch = batch;
      p.fmt = 0;
      p.early = 2;
      p.symmetric = 1;
      p.alpha = 1.f / 1024.f;
      if ((rc = launch_gemm_wide(op, p, kEpiGram, st, &maps))) return rc;
    }
    {  // (b Q + c Q^2) 64
      WideOperands op;
      op.a = op.b = q_mat(q);
      op.d = q_mat(pq);
      WideParams p;
      p.M = p.N = p.K = m;
      p.batch = batch;
      p.fmt = 0;
      p.early = 2;
      p.symmetric = 1;
      p.coef = coef + (int64_t)(2 * s) * batch * 2;
      p.in_hi = q;
      p.in_batch = qb;
      p.in_ld = ldq;
      if ((rc = launch_gemm_wide(op, p, kEpiPoly, st, &maps))) return rc;
    }
    const bool last = s + 1 == steps;
    WideOperands op;
    op.b_mn = true;
    op.a = q_mat(pq);
    op.b = x_mat(h);
    WideParams p;
    p.M = p.K = m;
    p.N = n;
    p.batch = batch;
    p.fmt = 0;
    p.early = 2;
    p.coef = coef + (int64_t)(2 * s + 1) * batch * 2;
    p.in_hi = h;
    p.in_lo = lo;
    p.in_batch = xb;
    p.in_ld = ldx;
    op.e = x_mat(h);
    op.d2 = x_mat(lo);
    if (!last) {
      op.d = x_mat(hi[(s + 1) & 1]);
    } else {
      p.alpha = 1.f / 256.f;
      if (tall) {
        p.out_t = reinterpret_cast<uint16_t*>(o);
        p.out_t_batch = ob;
        p.out_t_ld = orow;
      } else {
        op.d = Mat3{o, batch, m, n, ob, orow, 1};
      }
    }
    if ((rc = launch_gemm_wide(op, p, last ? kEpiLast : kEpiUpdate, st, &maps))) return rc;
  }
  return FA_OK;
}

constexpr int kThinMost = 64;

// Whether the wide form's fp16 operands hold every step's: singular values start
// in [0, 1]; s, their bound, becomes the largest |p| on [0, s] with each step, p(x) =
// a x + b x^3 + c x^5, which lies at s or where p' = 0 (a quadratic in x^2). No entry of
// X, Q or b Q + c Q^2 exceeds its largest singular value; stored are 256 X, 64 Q and
// 64 (b Q + c Q^2), and fp16 ends at 65504 (64000 leaves room for the roundings
// of the steps before).
static bool in_range(int steps, const float* coef) {
  const double a = coef[0], b = coef[1], c = coef[2], most = 64000.0;
  double s = 1.0;
  for (int k = 0; k < steps; ++k) {
    const double u = s * s;
    double poly = std::abs(u * (b + c * u));  // the largest |b v + c v^2|, v <= u
    if (c != 0.0) {
      const double v = -b / (2.0 * c);
      if (v > 0.0 && v < u) poly = std::max(poly, std::abs(v * (b + c * v)));
    }
    if (!(256.0 * s <= most && 64.0 * u <= most && 64.0 * poly <= most)) return false;
    auto p = [&](double v) { return std::sqrt(v) * std::abs(a + v * (b + c * v)); };  // at x^2 = v
    double top = p(u);
    auto look = [&](double v) {
      if (v > 0.0 && v < u) top = std::max(top, p(v));
    };
    const double disc = 9.0 * b * b - 20.0 * a * c;
    if (c != 0.0 && disc >= 0.0) {
      look((-3.0 * b + std::sqrt(disc)) / (10.0 * c));
      look((-3.0 * b - std::sqrt(disc)) / (10.0 * c));
    } else if (c == 0.0 && b != 0.0) {
      look(-a / (3.0 * b));
    }
    s = top;
  }
  return true;
}

}  // namespace ns

bool orthogonalize_in_range(int rows, int cols, int steps, const float* coef) {
  return std::min(rows, cols) <= ns::kThinMost || ns::in_range(steps, coef);
}

size_t orthogonalize_workspace(int batch, int rows, int cols, int steps) {
  const int m = std::min(rows, cols), n = std::max(rows, cols);
  return m <= ns::kThinMost ? 0 : ns::space_of(batch, m, n, steps).total;
}

int launch_orthogonalize(int dtype, int batch, int rows, int cols, const void* g, int64_t gb,
                         int64_t gr, void* o, int64_t ob, int64_t orow, int steps, const float* c,
                         float eps, void* ws, cudaStream_t st) {
  const bool bf = dtype == FA_DTYPE_BF16, tall = rows > cols;
  const int m = std::min(rows, cols), n = std::max(rows, cols);
  if (m > ns::kThinMost)
    return bf ? ns::wide_go<__nv_bfloat16>(g, gb, gr, o, ob, orow, batch, rows, cols, steps, c, eps, ws, st)
              : ns::wide_go<float>(g, gb, gr, o, ob, orow, batch, rows, cols, steps, c, eps, ws, st);
  const int kid = kKernelThin + (bf ? 0 : 8) + (tall ? 4 : 0);
#define FA_THIN(T, TALL) \
  ns::thin_pick<T, TALL>(g, gb, gr, o, ob, orow, batch, m, n, steps, c, eps, kid, st)
  if (bf) return tall ? FA_THIN(__nv_bfloat16, true) : FA_THIN(__nv_bfloat16, false);
  return tall ? FA_THIN(float, true) : FA_THIN(float, false);
#undef FA_THIN
}

}  // namespace fa
