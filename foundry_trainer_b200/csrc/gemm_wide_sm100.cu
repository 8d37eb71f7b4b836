// gemm_wide_sm100.cu — D = A B^T (+ epilogue) on the tensor cores, for the
// linears with adapters and the orthogonalisation's products.
//
//   D[m, n] = sum_k A[m, k] B[n, k]  (+ sum_j low[m, j] E_slot(m)[n, j])
//
// A is stored K-contiguous; B is K-contiguous (a weight in the forward, a
// symmetric matrix) or N-contiguous (B_MN: a weight in the backward, the
// iterate of the orthogonalisation). fp32 accumulation, 16-bit operands.
//
// Bound by the tensor cores. A pair of CTAs (cta_group::2) owns a 256 x BN
// tile: each stages its 128 rows of A and half of B's BN columns per 64-wide
// K block, so every staged byte of B feeds both SMs: per K block 32 KB land
// and 16 KB + 16 KB are read per SM for 512 cycles of tensor work (BN = 256), below the
// 128 bytes a cycle of shared memory that a single-CTA 128 x 256 tile exceeds.
// The pair is persistent over tiles; the accumulator is double-buffered in
// tensor memory (2 BN columns), so a tile's epilogue runs under the next
// tile's products.
//   warps 0-3  epilogue: one row per thread
//   warp 4     producer: TMA loads (one lane); builds the adapters' A operand
//   warp 5     tcgen05 issue (leader CTA only), tensor memory
//
// Adapters: a row's low-rank term is one more K block per adapter present in
// the tile's 256 rows. Its A operand holds low[m, :] in the rows that use the
// adapter and zeros elsewhere (written by the producer warp in the swizzled
// layout TMA would have written); its B operand is the adapter's own matrix,
// loaded by TMA with zero fill past the rank. So the low-rank product costs
// ceil(r / 16) tensor instructions a tile and no pass over D.
#include <algorithm>

#include "attn_common.h"
#include "gemm.h"
#include "gemm_ptx.cuh"

namespace fa {
namespace wide {

constexpr int kThreads = 192;
constexpr int kStageA = 16384;    // 128 rows x 64 elements
constexpr int kStaging = 16384;   // epilogue tile: 128 rows x 64 elements
constexpr int kBarBytes = 512;

template <int BN>
struct Cfg {
  static constexpr int kStageB = BN / 2 * 128;
  static constexpr int kStage = kStageA + kStageB;
  static constexpr int kStages = BN == 256 ? 6 : 8;
  static constexpr int kOffStaging = kStages * kStage;
  static constexpr int kOffBar = kOffStaging + 2 * kStaging;
  static constexpr int kSmem = kOffBar + kBarBytes + 1024;  // + alignment slack
  static constexpr uint32_t kTmemCols = 2 * BN;
};
static_assert(Cfg<256>::kSmem <= 232448 && Cfg<128>::kSmem <= 232448, "shared memory");

struct Tile {
  int m, n, b;  // 256-row block, BN-column block, batch
};

// Tile t of the walk: eight row blocks high columns first, so that the pairs
// at work at one time share their A rows and B columns in L2. Products with a
// symmetric result visit only the tiles on or below the diagonal.
__device__ __forceinline__ Tile tile_of(int64_t t, const WideParams& p, int BN) {
  Tile o;
  o.b = (int)(t / p.tiles_per_batch);
  int i = (int)(t - (int64_t)o.b * p.tiles_per_batch);
  if (p.symmetric) {
    // row block m has (m + 1) * (256 / BN) column blocks (cut at tiles_n)
    const int per = 256 / BN;
    int m = (int)((sqrtf(8.f * (float)(i / per) + 1.f) - 1.f) * 0.5f);
    while ((int64_t)per * (m + 1) * (m + 2) / 2 <= i) ++m;
    while ((int64_t)per * m * (m + 1) / 2 > i) --m;
    o.m = m;
    o.n = i - per * (m * (m + 1) / 2);
    return o;
  }
  constexpr int kHigh = 8;
  const int band = i / (kHigh * p.tiles_n);
  const int high = min(kHigh, p.tiles_m - band * kHigh);
  i -= band * kHigh * p.tiles_n;
  o.n = i / high;
  o.m = band * kHigh + (i - o.n * high);
  return o;
}

// Adapters' part of a tile: slots used by row block m (0 without adapters)
__device__ __forceinline__ int slots_of(const WideParams& p, int m) {
  if (p.low == nullptr) return 0;
  return p.list_cnt != nullptr ? p.list_cnt[m] : 1;
}

template <int BN, bool B_MN, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
wide_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
            const __grid_constant__ CUtensorMap te, const __grid_constant__ CUtensorMap td,
            const __grid_constant__ CUtensorMap td2, const __grid_constant__ WideParams p) {
  using C = Cfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* full = bars;                      // leader's is used
  uint64_t* empty = bars + C::kStages;        // both
  uint64_t* accfull = bars + 2 * C::kStages;  // both
  uint64_t* accempty = accfull + 2;           // leader's is used
  uint32_t* slot = reinterpret_cast<uint32_t*>(accempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(slot + 1);
  const int warp = warp_id(), lane = lane_id();
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 2);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&accfull[i], 1);
      mbar_init(&accempty[i], 8);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&ta);
    tma_prefetch_desc(&tb);
    tma_prefetch_desc(&td);
  }
  if (warp == 5) {
    tmem_alloc_pair(slot, C::kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *slot;

  const int64_t tiles = (int64_t)p.tiles_per_batch * p.batch;
  const int pairs = gridDim.x >> 1;
  const int kb_main = (p.K + 63) >> 6;
  const int kb_ext = (p.rank + 63) >> 6;  // per slot
  constexpr int kHalfN = BN / 2;

  if (warp == 4) {
    // ------------------------------------------------------------- producer
    bool ok = true;
    int s = 0;
    uint32_t ph = 0;
    for (int64_t t = blockIdx.x >> 1; t < tiles && ok; t += pairs) {
      const Tile tl = tile_of(t, p, BN);
      const int row0 = tl.m * 256 + (int)rank * 128;
      const int col0 = tl.n * BN + (int)rank * kHalfN;
      for (int kb = 0; kb < kb_main; ++kb) {
        if (!(ok = mbar_wait_cluster_w(&empty[s], ph ^ 1))) break;
        uint8_t* sa = smem + s * C::kStage;
        uint8_t* sb = sa + kStageA;
        if (lane == 0) {
          const uint32_t fb = mapa(smem_u32(&full[s]), 0);
          if (leader) {
            mbar_arrive_expect_tx(&full[s], 2 * C::kStage);
            mbar_arrive(&full[s]);  // the second arrival is the other CTA's in adapter blocks
          }
          tma_load_3d_pair(sa, &ta, fb, kb * 64, row0, tl.b);
          if constexpr (B_MN) {
#pragma unroll
            for (int j = 0; j < kHalfN / 64; ++j)
              tma_load_3d_pair(sb + j * 8192, &tb, fb, col0 + j * 64, kb * 64, tl.b);
          } else {
            tma_load_3d_pair(sb, &tb, fb, kb * 64, col0, tl.b);
          }
        }
        if (++s == C::kStages) { s = 0; ph ^= 1; }
      }
      if (!ok || p.low == nullptr) continue;
      const int ns = slots_of(p, tl.m);
      for (int q = 0; q < ns && ok; ++q) {
        const int e = p.list_ids != nullptr ? p.list_ids[(int64_t)tl.m * 256 + q] : 0;
        for (int j = 0; j < kb_ext; ++j) {
          if (!(ok = mbar_wait_cluster_w(&empty[s], ph ^ 1))) break;
          uint8_t* sa = smem + s * C::kStage;
          uint8_t* sb = sa + kStageA;
          // rows that use adapter e: their low values; the others: zeros
          const int cols = min(64, p.low_ld - j * 64);
#pragma unroll 4
          for (int i = lane; i < 1024; i += 32) {
            const int r = i >> 3, c = i & 7, row = row0 + r;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row < p.M && c * 8 < cols && (p.slot == nullptr || p.slot[row] == q))
              v = __ldcg(reinterpret_cast<const uint4*>(p.low + (int64_t)row * p.low_ld + j * 64 +
                                                        c * 8));
            *reinterpret_cast<uint4*>(sa + sw128_offset(r, c)) = v;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            const uint32_t fb = mapa(smem_u32(&full[s]), 0);
            if (leader) mbar_arrive_expect_tx(&full[s], 2 * C::kStageB);
            else mbar_arrive_cluster(fb);
            if constexpr (B_MN) {
#pragma unroll
              for (int i = 0; i < kHalfN / 64; ++i)
                tma_load_3d_pair(sb + i * 8192, &te, fb, col0 + i * 64, j * 64, e);
            } else {
              tma_load_3d_pair(sb, &te, fb, j * 64, col0, e);
            }
          }
          if (++s == C::kStages) { s = 0; ph ^= 1; }
        }
      }
    }
    if (!ok) *abort_flag = 1;
  } else if (warp == 5) {
    // ------------------------------------------------------------ tcgen05
    if (leader) {
      const uint32_t idesc = idesc_f16(p.fmt, 256, BN, false, B_MN);
      bool ok = true;
      int s = 0, it = 0;
      uint32_t ph = 0;
      for (int64_t t = blockIdx.x >> 1; t < tiles && ok; t += pairs, ++it) {
        const Tile tl = tile_of(t, p, BN);
        const int buf = it & 1;
        const uint32_t d = tmem + buf * BN;
        if (!(ok = mbar_wait_cluster_w(&accempty[buf], ((it >> 1) & 1) ^ 1))) break;
        tc_fence_after();
        const int nkb = kb_main + slots_of(p, tl.m) * kb_ext;
        for (int kb = 0; kb < nkb; ++kb) {
          if (!(ok = mbar_wait_cluster_w(&full[s], ph))) break;
          tc_fence_after();
          const uint32_t a = smem_u32(smem + s * C::kStage), b = a + kStageA;
          int steps = 4;
          if (kb >= kb_main) steps = min(4, (p.rank - ((kb - kb_main) % kb_ext) * 64 + 15) >> 4);
          if (elect_one()) {
            for (int kk = 0; kk < steps; ++kk)
              umma_ss_pair(d, kmajor_desc(a, kk, 0),
                           B_MN ? mnmajor_desc(b, kk, 8192) : kmajor_desc(b, kk, 0), idesc,
                           kb > 0 || kk > 0);
            umma_commit_pair(&empty[s]);
            if (kb == nkb - 1) umma_commit_pair(&accfull[buf]);
          }
          __syncwarp();
          if (++s == C::kStages) { s = 0; ph ^= 1; }
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    // ------------------------------------------------------------ epilogue
    bool ok = true;
    int it = 0;
    const int r = threadIdx.x;  // 0..127: the tile row and tensor-memory lane
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    uint8_t* stg = smem + C::kOffStaging;
    float ca = 0.f, cb = 0.f;
    for (int64_t t = blockIdx.x >> 1; t < tiles; t += pairs, ++it) {
      const Tile tl = tile_of(t, p, BN);
      const int buf = it & 1;
      const int row0 = tl.m * 256 + (int)rank * 128, row = row0 + r;
      const bool live = row < p.M;
      if constexpr (EPI == kEpiPoly || EPI == kEpiUpdate || EPI == kEpiLast) {
        // the step's coefficients of this matrix: p.coef (batch, 2)
        ca = p.coef[2 * tl.b];
        cb = p.coef[2 * tl.b + 1];
      }
      ok = mbar_wait_w(&accfull[buf], (it >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      const bool mirror = p.symmetric && tl.n * BN + BN <= tl.m * 256;
#pragma unroll 1
      for (int c = 0; c < BN / 64; ++c) {
        const int col0 = tl.n * BN + c * 64;
        uint32_t acc[64];
        tmem_ld32(tmem + lane_off + buf * BN + c * 64, acc);
        tmem_ld32(tmem + lane_off + buf * BN + c * 64 + 32, acc + 32);
        float* v = reinterpret_cast<float*>(acc);
        uint32_t lo[EPI == kEpiUpdate ? 32 : 1];
        if constexpr (EPI == kEpiLinear) {
          tmem_wait_ld();
          if (p.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (col0 + i < p.N) v[i] += __bfloat162float(p.bias[col0 + i]);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
        } else if constexpr (EPI == kEpiGram) {
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i)
            acc[i] = pack_f16(v[2 * i] * p.alpha, v[2 * i + 1] * p.alpha);
        } else if constexpr (EPI == kEpiPoly) {
          // b Q + c Q^2, Q read back at this tile
          uint4 q[8];
          const uint4* src = reinterpret_cast<const uint4*>(
              p.in_hi + (int64_t)tl.b * p.in_batch + (int64_t)row * p.in_ld + col0);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            q[i] = live && col0 + 8 * i < p.in_ld ? src[i] : make_uint4(0, 0, 0, 0);
          tmem_wait_ld();
          const uint32_t* qw = reinterpret_cast<const uint32_t*>(q);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float2 x = unpack_f16(qw[i]);
            acc[i] = pack_f16(fmaf(cb, v[2 * i], ca * x.x), fmaf(cb, v[2 * i + 1], ca * x.y));
          }
        } else {
          // a X + P X: X read back as hi + lo / 2048
          uint4 q[8], l[8];
          const int64_t at = (int64_t)tl.b * p.in_batch + (int64_t)row * p.in_ld + col0;
          const uint4* sh = reinterpret_cast<const uint4*>(p.in_hi + at);
          const uint4* sl = reinterpret_cast<const uint4*>(p.in_lo + at);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool in = live && col0 + 8 * i < p.in_ld;
            q[i] = in ? sh[i] : make_uint4(0, 0, 0, 0);
            l[i] = in ? sl[i] : make_uint4(0, 0, 0, 0);
          }
          tmem_wait_ld();
          const uint32_t* qw = reinterpret_cast<const uint32_t*>(q);
          const uint32_t* lw = reinterpret_cast<const uint32_t*>(l);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float2 h = unpack_f16(qw[i]), w = unpack_f16(lw[i]);
            const float x0 = fmaf(ca, fmaf(w.x, 1.f / 2048.f, h.x), v[2 * i] * cb);
            const float x1 = fmaf(ca, fmaf(w.y, 1.f / 2048.f, h.y), v[2 * i + 1] * cb);
            if constexpr (EPI == kEpiUpdate) {
              acc[i] = pack_f16(x0, x1);
              const float2 n = unpack_f16(acc[i]);
              lo[i] = pack_f16((x0 - n.x) * 2048.f, (x1 - n.y) * 2048.f);
            } else {
              acc[i] = pack_bf16(x0 * p.alpha, x1 * p.alpha);
            }
          }
        }
        if constexpr (EPI == kEpiLast) {
          if (p.out_t != nullptr) {
            // tall input: the result is stored transposed, a column of 32
            // consecutive rows per warp store
            if (live) {
              const uint16_t* h = reinterpret_cast<const uint16_t*>(acc);
#pragma unroll
              for (int i = 0; i < 64; ++i)
                if (col0 + i < p.N)
                  p.out_t[(int64_t)tl.b * p.out_t_batch + (int64_t)(col0 + i) * p.out_t_ld + row] =
                      h[i];
            }
            continue;
          }
        }
        if constexpr (EPI == kEpiGram || EPI == kEpiPoly) {
          if (mirror && live) {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(acc);
            uint16_t* o = reinterpret_cast<uint16_t*>(p.sym_out) + (int64_t)tl.b * p.sym_batch + row;
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (col0 + i < p.N) o[(int64_t)(col0 + i) * p.sym_ld] = h[i];
          }
        }
        // stage the 128 x 64 tile and store it with TMA (two buffers in turn,
        // or one each for hi and lo)
        constexpr bool kTwo = EPI == kEpiUpdate;
        uint8_t* b0 = kTwo ? stg : stg + (c & 1) * kStaging;
        if (threadIdx.x == 0) {
          if constexpr (kTwo) bulk_wait_group_read0();
          else bulk_wait_group_read1();
        }
        named_bar_sync(1, 128);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<uint4*>(b0 + sw128_offset(r, i)) =
              make_uint4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
        if constexpr (kTwo) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(stg + kStaging + sw128_offset(r, i)) =
                make_uint4(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
        }
        fence_proxy_async_smem();
        named_bar_sync(1, 128);
        if (threadIdx.x == 0) {
          if (row0 < p.M && col0 < p.N) {
            tma_store_3d(&td, b0, col0, row0, tl.b);
            if constexpr (kTwo) tma_store_3d(&td2, stg + kStaging, col0, row0, tl.b);
          }
          bulk_commit_group();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa(smem_u32(&accempty[buf]), 0));
    }
    if (threadIdx.x == 0) bulk_wait_group0();
    if (!ok) *abort_flag = 1;
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) drain_delay();
  cluster_sync();
  if (warp == 5) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem, C::kTmemCols);
  }
}

template <int BN, bool B_MN, int EPI>
static int go(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& te,
              const CUtensorMap& td, const CUtensorMap& td2, const WideParams& p, int kernel_id,
              cudaStream_t st) {
  auto* fn = wide_kernel<BN, B_MN, EPI>;
  const int rc = ensure_smem_attr((const void*)fn, Cfg<BN>::kSmem, kernel_id);
  if (rc) return rc;
  const int64_t tiles = (int64_t)p.tiles_per_batch * p.batch;
  const int pairs = (int)std::min<int64_t>(tiles, 74);
  fn<<<2 * pairs, kThreads, Cfg<BN>::kSmem, st>>>(ta, tb, te, td, td2, p);
  return launch_status();
}

}  // namespace wide

int launch_gemm_wide(const WideOperands& o, WideParams p, int epi, cudaStream_t st) {
  if (p.M == 0 || p.N == 0 || p.batch == 0) return FA_OK;
  // 256-wide tiles, unless 128-wide ones fill the 74 SM pairs better: the
  // cost of a walk is its rounds over the pairs times the tile's width
  auto count = [&](int bn) -> int64_t {
    const int tm = (p.M + 255) / 256, tn = (p.N + bn - 1) / bn;
    if (!p.symmetric) return (int64_t)tm * tn;
    const int per = 256 / bn;
    int64_t n = 0;
    for (int m = 0; m < tm; ++m) n += std::min((m + 1) * per, tn);
    return n;
  };
  const int64_t r256 = (count(256) * p.batch + 73) / 74, r128 = (count(128) * p.batch + 73) / 74;
  const int bn = r128 < 2 * r256 ? 128 : 256;
  p.tiles_m = (p.M + 255) / 256;
  p.tiles_n = (p.N + bn - 1) / bn;
  p.tiles_per_batch = (int)count(bn);
  CUtensorMap ta, tb, te, td, td2;
  int rc = make_tmap_3d(&ta, o.a, 64, 128);
  if (!rc) rc = o.b_mn ? make_tmap_3d(&tb, o.b, 64, 64) : make_tmap_3d(&tb, o.b, 64, bn / 2);
  te = tb;
  if (!rc && p.low != nullptr)
    rc = o.b_mn ? make_tmap_3d(&te, o.e, 64, 64) : make_tmap_3d(&te, o.e, 64, bn / 2);
  td = ta;
  if (!rc && o.d.p != nullptr) rc = make_tmap_3d(&td, o.d, 64, 128);
  td2 = td;
  if (!rc && o.d2.p != nullptr) rc = make_tmap_3d(&td2, o.d2, 64, 128);
  if (rc) return rc;
#define FA_WIDE(EPI, MN, ID)                                                                  \
  if (epi == EPI && o.b_mn == MN)                                                             \
    return bn == 256 ? wide::go<256, MN, EPI>(ta, tb, te, td, td2, p, ID, st)                 \
                     : wide::go<128, MN, EPI>(ta, tb, te, td, td2, p, ID + 1, st);
  FA_WIDE(kEpiLinear, false, kKernelWide)
  FA_WIDE(kEpiLinear, true, kKernelWide + 2)
  FA_WIDE(kEpiGram, false, kKernelWide + 4)
  FA_WIDE(kEpiPoly, false, kKernelWide + 6)
  FA_WIDE(kEpiUpdate, true, kKernelWide + 8)
  FA_WIDE(kEpiLast, true, kKernelWide + 10)
#undef FA_WIDE
  return FA_ERR_UNSUPPORTED;
}

int wide_device_status() { return tu_device_status(); }

}  // namespace fa
