// gemm_ptx.cuh — inline-PTX wrappers the matrix-product kernels add to
// sm100_ptx.cuh: thread-block clusters, distributed shared memory, the
// two-SM (cta_group::2) forms of TMA loads and tcgen05, and 3-D tile copies.
#pragma once

#include <cuda_fp16.h>

#include "sm100_ptx.cuh"

namespace fa {

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::
          : "memory");
}
// The two halves of cluster_sync.
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of this CTA's shared-memory location `addr` in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                              uint32_t d) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}
// Arrives on a barrier of any CTA of the cluster (address from mapa); earlier
// writes of this thread are visible to who waits with cluster scope.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr)
               : "memory");
}

// mbar_wait for a barrier that other CTAs of the cluster arrive on.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity) {
  const uint32_t a = smem_u32(bar);
  const long long t0 = clock64();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(a), "r"(parity)
        : "memory");
    if (ok) return true;
    if (clock64() - t0 > kWaitBudgetCycles) {
      report_status(5 /* FA_ERR_DEVICE_TIMEOUT */);
      return false;
    }
  }
}
__device__ __forceinline__ bool mbar_wait_cluster_w(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait_cluster(bar, parity));
}

// 3-D tile load into this CTA's shared memory, completing on `bar`.
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// The same for a CTA pair: the destination is this CTA's shared memory, the
// barrier (shared::cluster address) may be the other CTA's.
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar,
                                                 int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
      "bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// Tile store (elements outside the tensor are not written).
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int c0,
                                             int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void bulk_wait_group_read1() {
  asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
}

// ------------------------------------------------- tcgen05 over a CTA pair
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_u32(dst_smem)),
               "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
               : "memory");
}
// D (256 rows over the pair's tensor memories) (+)= A (128 rows from each
// CTA's shared memory) * B (half of the columns from each).
__device__ __forceinline__ void umma_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives once on `bar` in both CTAs of the pair when every tcgen05 operation
// this thread issued so far is done.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

// Warp-wide forms (sm100_ptx.cuh says why): one elected lane issues.
__device__ __forceinline__ void umma_ss_pair_w(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                               uint32_t idesc, uint32_t accumulate) {
  if (elect_one()) umma_ss_pair(d_tmem, a_desc, b_desc, idesc, accumulate);
}
__device__ __forceinline__ void umma_commit_pair_w(uint64_t* bar) {
  if (elect_one()) umma_commit_pair(bar);
}

// Instruction descriptor, kind::f16, fp32 D: idesc_bf16's bits with the
// element format of A and B (0 fp16, 1 bf16).
__host__ __device__ constexpr uint32_t idesc_f16(int fmt, int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((a_mn ? 1u : 0u) << 15) |
         ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Last bounded delay (~2 ms) of a CTA whose waits ran out: the copies and
// matrix instructions it issued finish well within it, so its shared and
// tensor memory are not given up under them.
__device__ __forceinline__ void drain_delay() {
  const long long t0 = clock64();
  while (clock64() - t0 < 4000000LL) {
  }
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}

// Programmatic dependent launch: lets the next kernel of the stream start
// before this one has finished, and waits for the one before (completion and
// memory) where this kernel first needs its results.
__device__ __forceinline__ void pdl_launch_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// K-major operand tiles of rows of 32 or 64 bytes (16 or 32 K), swizzled over
// their own width: descriptor (layout 6 or 4, eight rows apart) and the offset
// of 16-byte chunk c of row r.
__device__ __forceinline__ uint64_t kmajor_narrow_desc(uint32_t base, uint32_t row_bytes) {
  return (uint64_t)((base >> 4) & 0x3FFFu) | (1ull << 16) |
         ((uint64_t)((row_bytes * 8) >> 4) << 32) | (1ull << 46) |
         ((row_bytes == 32 ? 6ull : 4ull) << 61);
}
__device__ __forceinline__ uint32_t narrow_offset(uint32_t r, uint32_t c, uint32_t row_bytes) {
  return r * row_bytes + ((row_bytes == 32 ? c ^ ((r >> 2) & 1u) : c ^ ((r >> 1) & 3u)) << 4);
}

// Whether `n` bf16 values from p (16-byte aligned) on hold a NaN or an infinity.
__device__ __forceinline__ bool any_non_finite(const __nv_bfloat16* p, int n) {
  uint32_t bad = 0;
  auto word = [&](uint32_t w) {  // a half whose exponent is all ones
    bad |= (uint32_t)((w & 0x7f80u) == 0x7f80u) | (uint32_t)((w & 0x7f800000u) == 0x7f800000u);
  };
  int k = 0;
  for (; k + 8 <= n; k += 8) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + k));
    word(v.x), word(v.y), word(v.z), word(v.w);
  }
  for (; k < n; ++k) word((uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p) + k));
  return bad != 0;
}

// A block's adapters whose factors' row holds a NaN or an infinity: how many of
// the `cnt` in `list`, as kNoneBad, the slot of the only one, or kSeveralBad. Such a
// factor is what may have reached the rows of other adapters (as zero times
// it); where there is none, a non-finite sum is a row's own.
enum : int { kNoneBad = -1, kSeveralBad = -2 };
static __device__ __noinline__ int bad_factors(const __nv_bfloat16* f, int64_t f_adapter, int rank,
                                        const int* list, int cnt) {
  int bad = kNoneBad;
  for (int q = 0; q < cnt; ++q)
    if (any_non_finite(f + (int64_t)list[q] * f_adapter, rank))
      bad = bad == kNoneBad ? q : kSeveralBad;
  return bad;
}

// D (16 x 8) += A (16 x 16) B (16 x 8), bf16 with fp32 sums: lane (g, q) = (lane / 4,
// lane % 4) holds the k pairs q and q + 4 of A's rows g and g + 8 and of B's
// column g, and D's columns 2 q, 2 q + 1 in those rows.
__device__ __forceinline__ void mma_bf16(float* d, uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// k .. k + 8 of a row of K values (16-byte aligned), zeros past its end
__device__ __forceinline__ uint4 row_piece(const __nv_bfloat16* row, int64_t k, int K) {
  if (k + 8 <= K) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < K)
      w[i >> 1] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(row + k + i)) << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// out[c] = sum over k < K of A[lane, k] B[c, k], c < 32, from memory: the base
// product of 32 rows and 32 columns again, without any adapter. `a_rows` and
// `b_rows` rows exist (rows past them repeat the last one; their results mean
// nothing). For the whole warp. Only for values that another request's broken
// factor reached (0 x inf = NaN). With one of three adapters NaN throughout, 600
// rows x 4096 x 1024 take 0.21 ms (44 us with sound ones; a scalar sum a value, each
// lane at a row of its own: 8.4 ms), 6000 x 4096 x 4096 5.3 ms (0.19; bound by L2).
// The order of the terms does not matter as long as A and B agree: lane q
// takes the eight values from 8 q on of every 32, as two products of 16.
static __device__ __noinline__ void base_products(const __nv_bfloat16* a, int64_t lda, int a_rows,
                                                  const __nv_bfloat16* b, int64_t ldb, int b_rows,
                                                  int K, float* out) {
  const int lane = lane_id(), g = lane >> 2, q = lane & 3;
  const __nv_bfloat16 *ar[4], *br[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ar[i] = a + (int64_t)min(8 * i + g, a_rows - 1) * lda;
    br[i] = b + (int64_t)min(8 * i + g, b_rows - 1) * ldb;
  }
  float d[2][4][4] = {};
#pragma unroll 1
  for (int64_t k = 8 * q; k < (int64_t)(K + 31) / 32 * 32; k += 32) {
    uint4 u[4], w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = row_piece(ar[i], k, K), w[i] = row_piece(br[i], k, K);
    __syncwarp();
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint4 &lo = u[2 * m], &hi = u[2 * m + 1];
        mma_bf16(d[m][n], lo.x, hi.x, lo.y, hi.y, w[n].x, w[n].y);
        mma_bf16(d[m][n], lo.z, hi.z, lo.w, hi.w, w[n].z, w[n].w);
      }
  }
  // row `lane`'s values are with lanes 4 (lane % 8) .. + 3, as rows lane / 16, lane / 8 % 2
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    const int from = 4 * (lane & 7) + ((c & 7) >> 1);
    float v = 0.f;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const float o = __shfl_sync(0xffffffffu, d[h >> 1][c >> 3][2 * (h & 1) + (c & 1)], from);
      if (h == lane >> 3) v = o;
    }
    out[c] = v;
  }
}

// sum over k < rank of low[k] f[k] (both 16-byte aligned): a row's own adapter
static __device__ __noinline__ float own_term(const __nv_bfloat16* low, const __nv_bfloat16* f,
                                              int rank) {
  float acc = 0.f;
  int k = 0;
  for (; k + 8 <= rank; k += 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(low + k);
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(f + k));
    const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc = fmaf(bf16_lo(uw[i]), bf16_lo(vw[i]), acc);
      acc = fmaf(bf16_hi(uw[i]), bf16_hi(vw[i]), acc);
    }
  }
  for (; k < rank; ++k) acc = fmaf(__bfloat162float(low[k]), __bfloat162float(f[k]), acc);
  return acc;
}

}  // namespace fa
