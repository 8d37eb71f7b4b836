// gemm_wide_sm100.cu — D = A B^T (+ epilogue) on the tensor cores, for the
// linears with adapters and the orthogonalisation's products.
//
//   D[m, n] = sum_k A[m, k] B[n, k]  (+ sum_j low[m, j] E_slot(m)[n, j])
//
// A is stored K-contiguous; B is K-contiguous (a weight in the forward, a
// symmetric matrix) or N-contiguous (B_MN: a weight in the backward, the
// iterate of the orthogonalisation). fp32 accumulation, 16-bit operands.
//
// Bound by the tensor cores. A pair of CTAs (cta_group::2) owns a 256 x kBN
// tile: each stages its 128 rows of A and half of B's kBN columns per 64-wide
// K block, so every staged byte of B feeds both SMs: per K block 32 KB land
// and 32 KB are read per SM for 512 cycles of tensor work, within the 128
// bytes a cycle of shared memory that a single-CTA 128 x 256 tile exceeds. A
// 256 x 128 tile was measured to take as long as the 256 x 256 one, so there
// is no narrower form. At 9216 x 4096 x 16384 with an adapter of rank 32: 793
// us forward, 803 us for dx, 1.56 PFLOP/s with the tensor cores 91 to 93
// percent busy and the clock at 1.4 GHz under the power cap (the library
// product's sustained rate there is 1.40).
// The pair is persistent over tiles; the accumulator is double-buffered in
// tensor memory (2 kBN columns), so a tile's epilogue runs under the next
// tile's products.
//   warps 0-3  epilogue: one row per thread
//   warp 4     producer: TMA loads (one lane); builds the adapters' A operand
//   warp 5     tcgen05 issue (leader CTA only), tensor memory
//
// Adapters: a row's low-rank term is one more K block per adapter present in
// the tile's 256 rows. Its A operand holds low[m, :] in the rows that use the
// adapter and zeros elsewhere (written by the producer warp in the swizzled
// layout TMA would have written; by TMA itself where the block has one
// adapter); its B operand is the adapter's own matrix,
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

constexpr int kBN = 256;                     // columns of a tile
constexpr int kStageB = kBN / 2 * 128;
constexpr int kStage = kStageA + kStageB;
// Ring slots and 16 KB epilogue buffers: the orthogonalisation's epilogues read
// and write two matrices, twice buffered.
constexpr int stages_of(int epi) { return epi == kEpiLinear ? 6 : 5; }
constexpr int buffers_of(int epi) { return epi == kEpiLinear ? 2 : 4; }
constexpr int bar_off_of(int epi) { return stages_of(epi) * kStage + buffers_of(epi) * kStaging; }
constexpr int smem_of(int epi) { return bar_off_of(epi) + kBarBytes + 1024; }  // + alignment slack
constexpr uint32_t kTmemCols = 2 * kBN;
static_assert(smem_of(kEpiLinear) <= 232448 && smem_of(kEpiUpdate) <= 232448, "shared memory");

struct Tile {
  int m, n, b;  // 256-row block, kBN-column block, batch
};

// What an orthogonalisation product reads back for 32 columns of its result:
// Q, or X as hi and lo; from memory, or from the row's staged tiles.
template <int EPI>
struct Back {
  static constexpr bool kX = EPI == kEpiUpdate || EPI == kEpiLast;
  static constexpr bool kNone = EPI == kEpiGram || EPI == kEpiLinear;
  uint4 q[kNone ? 1 : 4], l[kX ? 4 : 1];

  __device__ __forceinline__ void load(const WideParams& p, int b, int row, bool live, int col) {
    if constexpr (!kNone) {
      const int64_t at = (int64_t)b * p.in_batch + (int64_t)row * p.in_ld + col;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = live && col + 8 * i < p.in_ld;
        q[i] = in ? *reinterpret_cast<const uint4*>(p.in_hi + at + 8 * i) : make_uint4(0, 0, 0, 0);
        if constexpr (kX)
          l[i] = in ? *reinterpret_cast<const uint4*>(p.in_lo + at + 8 * i) : make_uint4(0, 0, 0, 0);
      }
    }
  }
  __device__ __forceinline__ void take(const uint8_t* hi, const uint8_t* lo, int r, int half) {
    if constexpr (!kNone) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        q[i] = *reinterpret_cast<const uint4*>(hi + sw128_offset(r, 4 * half + i));
        if constexpr (kX) l[i] = *reinterpret_cast<const uint4*>(lo + sw128_offset(r, 4 * half + i));
      }
    }
  }
};

// These 32 columns as they are stored: out (16-bit pairs) and, for X, the
// remainders lo.
template <int EPI>
__device__ __forceinline__ void ns_values(const WideParams& p, const Back<EPI>& back, float ca,
                                          float cb, const uint32_t* acc, uint32_t* out,
                                          uint32_t* lo) {
  const float* v = reinterpret_cast<const float*>(acc);
  const uint32_t* qw = reinterpret_cast<const uint32_t*>(back.q);
  const uint32_t* lw = reinterpret_cast<const uint32_t*>(back.l);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if constexpr (EPI == kEpiGram) {
      out[i] = pack_f16(v[2 * i] * p.alpha, v[2 * i + 1] * p.alpha);
    } else if constexpr (EPI == kEpiPoly) {  // b Q + c Q^2
      const float2 x = unpack_f16(qw[i]);
      out[i] = pack_f16(fmaf(cb, v[2 * i], ca * x.x), fmaf(cb, v[2 * i + 1], ca * x.y));
    } else {  // a X + P X, X = hi + lo / 2048
      const float2 h = unpack_f16(qw[i]), w = unpack_f16(lw[i]);
      const float x0 = fmaf(ca, fmaf(w.x, 1.f / 2048.f, h.x), v[2 * i] * cb);
      const float x1 = fmaf(ca, fmaf(w.y, 1.f / 2048.f, h.y), v[2 * i + 1] * cb);
      if constexpr (EPI == kEpiUpdate) {
        out[i] = pack_f16(x0, x1);
        const float2 n = unpack_f16(out[i]);
        lo[i] = pack_f16((x0 - n.x) * 2048.f, (x1 - n.y) * 2048.f);
      } else {
        out[i] = pack_bf16(x0 * p.alpha, x1 * p.alpha);
      }
    }
  }
}

// The same 32 values of the last product of a tall input to their place in the
// transpose (any alignment): a column of 32 consecutive rows per warp store.
__device__ __forceinline__ void store_columns(uint16_t* o, int64_t ld, int col, int n,
                                              const uint32_t* out) {
  const uint16_t* h = reinterpret_cast<const uint16_t*>(out);
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (col + i < n) o[(int64_t)(col + i) * ld] = h[i];
}

// The staged tiles of 128 rows x 64 columns: columns [32 half, 32 half + 32) of
// this thread's row.
__device__ __forceinline__ void stage_half(uint8_t* buf, int r, int half, const uint32_t* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<uint4*>(buf + sw128_offset(r, 4 * half + i)) =
        make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}

// The same tile transposed, for the mirrored place of a symmetric result: two
// blocks of 64 rows (the tile's columns) x 64 columns.
__device__ __forceinline__ void stage_mirror(uint8_t* buf, int r, int half, const uint32_t* v) {
  const uint16_t* h = reinterpret_cast<const uint16_t*>(v);
  uint8_t* b = buf + (r >> 6) * 8192 + (r & 7) * 2;
#pragma unroll
  for (int i = 0; i < 32; ++i)
    *reinterpret_cast<uint16_t*>(b + sw128_offset(32 * half + i, (r & 63) >> 3)) = h[i];
}

// and its store by one thread: rows col0 .., columns row0 .. of the result
__device__ __forceinline__ void store_mirror(const CUtensorMap* map, const uint8_t* buf, int row0,
                                             int col0, int b, const WideParams& p) {
  tma_store_3d(map, buf, row0, col0, b);
  if (row0 + 64 < p.M) tma_store_3d(map, buf + 8192, row0 + 64, col0, b);
}

// Row block m of a symmetric walk, tiles_of(m) = per (m + 1) column tiles:
// the place of walk position i.
__device__ __forceinline__ void triangle(int i, int per, int& m, int& n) {
  m = (int)((sqrtf(8.f * (float)(i / per) + 1.f) - 1.f) * 0.5f);
  while ((int64_t)per * (m + 1) * (m + 2) / 2 <= i) ++m;
  while ((int64_t)per * m * (m + 1) / 2 > i) --m;
  n = i - per * (m * (m + 1) / 2);
}

// Tile t of the walk: eight row blocks high columns first, so that the pairs
// at work at one time share their A rows and B columns in L2. Products with a
// symmetric result visit only the tiles on or below the diagonal.
__device__ __forceinline__ Tile tile_of(int64_t t, const WideParams& p) {
  Tile o;
  o.b = (int)(t / p.tiles_per_batch);
  int i = (int)(t - (int64_t)o.b * p.tiles_per_batch);
  if (p.symmetric) {
    triangle(i, 1, o.m, o.n);
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

// 32 columns from col0 on of this lane's row (32 rows from row0 on a warp) from
// the rows' own operands alone, where `want` has the column's bit. Only for values
// that a block with adapters left non-finite: there a row's zeros in another
// adapter's K block met a NaN or infinity of that adapter (0 x inf = NaN).
__device__ __noinline__ void own_values(const WideParams& p, int row0, int col0, int m,
                                        uint32_t want, float* v) {
  float base[32];
  base_products(p.raw_x + (int64_t)row0 * p.raw_ldx, p.raw_ldx, min(32, p.M - row0),
                p.raw_w + (int64_t)col0 * p.raw_ldw, p.raw_ldw, min(32, p.N - col0), p.K, base);
  const int row = row0 + lane_id();
  const int s = want != 0 ? p.slot[row] : -1;
  const __nv_bfloat16* l = p.low + (int64_t)row * p.low_stride;
  const __nv_bfloat16* f =
      s >= 0 ? p.raw_f + (int64_t)p.list_ids[(int64_t)m * 256 + s] * p.raw_fe : nullptr;
  for (int c = 0; c < 32; ++c)
    if (want >> c & 1)
      v[c] = base[c] + (s >= 0 ? own_term(l, f + (int64_t)(col0 + c) * p.raw_ldf, p.rank) : 0.f);
}

template <bool B_MN, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
wide_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
            const __grid_constant__ CUtensorMap te, const __grid_constant__ CUtensorMap tl_low,
            const __grid_constant__ CUtensorMap td,
            const __grid_constant__ CUtensorMap td2, const __grid_constant__ WideParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kStages = stages_of(EPI), kOffStaging = kStages * kStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + bar_off_of(EPI));
  uint64_t* full = bars;                      // leader's is used
  uint64_t* empty = bars + kStages;        // both
  uint64_t* accfull = bars + 2 * kStages;  // both
  uint64_t* accempty = accfull + 2;           // leader's is used
  uint64_t* back = accempty + 2;              // what the epilogue reads back landed
  uint32_t* slot = reinterpret_cast<uint32_t*>(back + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(slot + 1);
  const int warp = warp_id(), lane = lane_id();
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 2);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&accfull[i], 1);
      mbar_init(&accempty[i], 8);
      mbar_init(&back[i], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&ta);
    tma_prefetch_desc(&tb);
    tma_prefetch_desc(&td);
  }
  if (warp == 5) {
    tmem_alloc_pair(slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *slot;

  pdl_launch_next();
  if (p.early == 2) pdl_wait_previous();
  const int64_t tiles = (int64_t)p.tiles_per_batch * p.batch;
  const int pairs = gridDim.x >> 1;
  const int kb_main = (p.K + 63) >> 6;
  const int kb_ext = (p.rank + 63) >> 6;  // per slot
  constexpr int kHalfN = kBN / 2;

  if (warp == 4) {
    // ------------------------------------------------------------- producer
    uint8_t* rows_s = reinterpret_cast<uint8_t*>(bars) + 256;  // 128: rows of an adapter
    bool ok = true;
    int s = 0;
    uint32_t ph = 0;
    for (int64_t t = blockIdx.x >> 1; t < tiles && ok; t += pairs) {
      const Tile tl = tile_of(t, p);
      const int row0 = tl.m * 256 + (int)rank * 128;
      const int col0 = tl.n * kBN + (int)rank * kHalfN;
      // A tile of several adapters: this CTA's rows of low and their slots are
      // fetched now, under the main blocks, and kept while the rank is at most
      // 32 (16 registers of 16 bytes a lane); each adapter's operand is then
      // stores alone. Fetched per adapter instead they cost 14 us a tile.
      const int ns = EPI == kEpiLinear ? slots_of(p, tl.m) : 0;
      constexpr int kHold = EPI == kEpiLinear ? 16 : 1;
      uint4 hold[kHold];
      int hold_slot[kHold];
      const int chunks = p.low_ld >> 3, lg = chunks == 4 ? 2 : 1;
      const bool held = EPI == kEpiLinear && (chunks == 2 || chunks == 4);
      // (its lists are older; low itself may be the previous kernel's)
      if (ns > 1 && held && p.early == 1) pdl_wait_previous();
      if (ns > 1 && held) {
#pragma unroll
        for (int i = 0; i < kHold; ++i) {
          const int r = (i * 32 + lane) >> lg, c = lane & (chunks - 1), row = row0 + r;
          const bool in = r < 128 && row < p.M;
          hold_slot[i] = in ? p.slot[row] : -1;
          hold[i] = in ? __ldcg(reinterpret_cast<const uint4*>(p.low + (int64_t)row * p.low_stride + c * 8))
                       : make_uint4(0, 0, 0, 0);
        }
      }
      int row_slot[4];  // of rows lane, lane + 32, ..: where low is not kept
      if (ns > 1 && !held) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int row = row0 + 32 * g + lane;
          row_slot[g] = row < p.M ? p.slot[row] : -1;
        }
      }
      for (int kb = 0; kb < kb_main; ++kb) {
        if (!(ok = mbar_wait_w(&empty[s], ph ^ 1))) break;
        uint8_t* sa = smem + s * kStage;
        uint8_t* sb = sa + kStageA;
        if (lane == 0) {
          const uint32_t fb = mapa(smem_u32(&full[s]), 0);
          if (leader) {
            mbar_arrive_expect_tx(&full[s], 2 * kStage);
            mbar_arrive(&full[s]);  // the second arrival: the other CTA's where it builds A
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
        if (++s == kStages) { s = 0; ph ^= 1; }
      }
      if (!ok || ns == 0) continue;
      if (p.early == 1) pdl_wait_previous();
      for (int q = 0; q < ns && ok; ++q) {
        const int e = p.list_ids != nullptr ? p.list_ids[(int64_t)tl.m * 256 + q] : 0;
        for (int j = 0; j < kb_ext; ++j) {
          if (!(ok = mbar_wait_w(&empty[s], ph ^ 1))) break;
          uint8_t* sa = smem + s * kStage;
          uint8_t* sb = sa + kStageA;
          if (ns > 1) {
            // rows that use adapter e: their low values; the others: zeros
            if (held) {
#pragma unroll
              for (int i = 0; i < kHold; ++i) {
                const int r = (i * 32 + lane) >> lg, c = lane & (chunks - 1);
                if (r < 128)
                  *reinterpret_cast<uint4*>(sa + sw128_offset(r, c)) =
                      hold_slot[i] == q ? hold[i] : make_uint4(0, 0, 0, 0);
              }
            } else {
// zeros, then only the rows that use the adapter, their places by
              // ballots: looking at all 128 took 6.5 us a block (1000 rows of 14
              // adapters of rank 64 at 408 x 920: the call 119 -> 58 us)
              int cnt = 0;
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const uint32_t m = __ballot_sync(0xffffffffu, row_slot[g] == q);
                if (row_slot[g] == q) rows_s[cnt + __popc(m & ((1u << lane) - 1u))] = 32 * g + lane;
                cnt += __popc(m);
              }
#pragma unroll 8
              for (int i = lane; i < kStageA / 16; i += 32)
                *reinterpret_cast<uint4*>(sa + i * 16) = make_uint4(0, 0, 0, 0);
              __syncwarp();
              const int c = lane & 7, col = j * 64 + c * 8;
#pragma unroll 4
              for (int i = lane >> 3; i < cnt; i += 4) {
                const int r = rows_s[i];
                if (col < p.low_ld)
                  *reinterpret_cast<uint4*>(sa + sw128_offset(r, c)) = __ldcg(
                      reinterpret_cast<const uint4*>(p.low + (int64_t)(row0 + r) * p.low_stride + col));
              }
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (lane == 0) {
            const uint32_t fb = mapa(smem_u32(&full[s]), 0);
            if (ns > 1) {
              if (leader) mbar_arrive_expect_tx(&full[s], 2 * kStageB);
              else mbar_arrive_cluster(fb);
            } else {
              // one adapter: rows without it hold zeros in low already
              if (leader) {
                mbar_arrive_expect_tx(&full[s], 2 * kStage);
                mbar_arrive(&full[s]);
              }
              tma_load_3d_pair(sa, &tl_low, fb, j * 64, row0, 0);
            }
            if constexpr (B_MN) {
#pragma unroll
              for (int i = 0; i < kHalfN / 64; ++i)
                tma_load_3d_pair(sb + i * 8192, &te, fb, col0 + i * 64, j * 64, e);
            } else {
              tma_load_3d_pair(sb, &te, fb, j * 64, col0, e);
            }
          }
          if (++s == kStages) { s = 0; ph ^= 1; }
        }
      }
    }
    // (also where no tile had an adapter: this kernel's end stands for the
    // previous one's)
    if (p.early == 1) pdl_wait_previous();
    if (!ok) *abort_flag = 1;
  } else if (warp == 5) {
    // ------------------------------------------------------------ tcgen05
    if (leader) {
      const uint32_t idesc = idesc_f16(p.fmt, 256, kBN, false, B_MN);
      const uint64_t a0 = kmajor_desc(smem_u32(smem), 0, 0);
      const uint64_t b0 = B_MN ? mnmajor_desc(smem_u32(smem) + kStageA, 0, 8192)
                               : kmajor_desc(smem_u32(smem) + kStageA, 0, 0);
      constexpr uint32_t kStepB = B_MN ? 128 : 2;  // 16 K rows of 128 bytes, or 32 bytes
      bool ok = true;
      int s = 0, it = 0;
      uint32_t ph = 0;
      for (int64_t t = blockIdx.x >> 1; t < tiles && ok; t += pairs, ++it) {
        const Tile tl = tile_of(t, p);
        const int buf = it & 1;
        const uint32_t d = tmem + buf * kBN;
        if (!(ok = mbar_wait_w(&accempty[buf], ((it >> 1) & 1) ^ 1))) break;
        tc_fence_after();
        const int nkb = kb_main + slots_of(p, tl.m) * kb_ext;
        for (int kb = 0; kb < nkb; ++kb) {
          // cluster scope where the other CTA may have built its operand
          if (!(ok = kb < kb_main ? mbar_wait_w(&full[s], ph) : mbar_wait_cluster_w(&full[s], ph)))
            break;
          tc_fence_after();
          // the whole warp runs the loop with uniform descriptors: stage and
          // K slice are additions to their 16-byte address fields
          const uint64_t a = a0 + (uint32_t)(s * (kStage >> 4));
          const uint64_t b = b0 + (uint32_t)(s * (kStage >> 4));
          if (kb < kb_main) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_ss_pair_w(d, a + 2 * kk, b + kStepB * kk, idesc, kb > 0 || kk > 0);
          } else {
            const int steps = min(4, (p.rank - ((kb - kb_main) % kb_ext) * 64 + 15) >> 4);
            for (int kk = 0; kk < steps; ++kk)
              umma_ss_pair_w(d, a + 2 * kk, b + kStepB * kk, idesc, 1);
          }
          umma_commit_pair_w(&empty[s]);
          if (kb == nkb - 1) umma_commit_pair_w(&accfull[buf]);
          if (++s == kStages) { s = 0; ph ^= 1; }
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
    uint8_t* stg = smem + kOffStaging;
    float ca = 0.f, cb = 0.f;
    const bool bias_vec = (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0;
    for (int64_t t = blockIdx.x >> 1; t < tiles; t += pairs, ++it) {
      const Tile tl = tile_of(t, p);
      const int buf = it & 1;
      const int row0 = tl.m * 256 + (int)rank * 128, row = row0 + r;
      const bool live = row < p.M;
      if constexpr (EPI == kEpiPoly || EPI == kEpiUpdate || EPI == kEpiLast) {
        // the step's coefficients of this matrix: p.coef (batch, 2)
        ca = p.coef[2 * tl.b];
        cb = p.coef[2 * tl.b + 1];
      }
      constexpr bool kReads = EPI == kEpiPoly || EPI == kEpiUpdate || EPI == kEpiLast;
      constexpr bool kX = EPI == kEpiUpdate || EPI == kEpiLast;
      // chunk g of this CTA's walk uses buffer pair g & 1; thread 0 requests the
      // pair of the next one, whose last store has been read
      auto request = [&](const Tile& o, int c, int g) {
        uint8_t* b = stg + (g & 1) * 2 * kStaging;
        const int row = o.m * 256 + (int)rank * 128, col = o.n * kBN + c * 64;
        mbar_arrive_expect_tx(&back[g & 1], (kX ? 2 : 1) * kStaging);
        tma_load_3d(b, kX ? &te : &ta, &back[g & 1], col, row, o.b);
        if constexpr (kX) tma_load_3d(b + kStaging, &td2, &back[g & 1], col, row, o.b);
      };
      if (kReads && it == 0 && threadIdx.x == 0) request(tl, 0, 0);
      ok = mbar_wait_w(&accfull[buf], (it >> 1) & 1);
      if (named_bar_any(1, 128, !ok)) { ok = false; break; }
      tc_fence_after();
      // a block with adapters of requests: a row must not see those of others
      const bool mixed = EPI == kEpiLinear && p.raw_x != nullptr && slots_of(p, tl.m) > 0;
      const bool mirror = p.symmetric && tl.n < tl.m;
#pragma unroll 1
      for (int c = 0; c < kBN / 64; ++c) {
        const int col0 = tl.n * kBN + c * 64;
        const uint32_t taddr = tmem + lane_off + buf * kBN + c * 64;
        if constexpr (EPI == kEpiLinear) {
          // stage the 128 x 64 tile and store it with TMA, two buffers in turn
          uint8_t* b0 = stg + (c & 1) * kStaging;
          uint32_t acc[64];
          tmem_ld32(taddr, acc);
          tmem_ld32(taddr + 32, acc + 32);
          float* v = reinterpret_cast<float*>(acc);
          tmem_wait_ld();
          if (mixed) {
            // zero times a non-finite entry of another row's adapter: only where
            // the column's factors hold one (a row that is NaN itself is left)
            float z = 0.f;
#pragma unroll
            for (int i = 0; i < 64; ++i) z = fmaf(v[i], 0.f, z);
            const bool odd = z != 0.f && live;
            if (__any_sync(0xffffffffu, odd)) {
              int bad[2];  // of columns lane and lane + 32
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int col = col0 + lane + 32 * h;
                bad[h] = col < p.N ? bad_factors(p.raw_f + (int64_t)col * p.raw_ldf, p.raw_fe, p.rank,
                                                 p.list_ids + (int64_t)tl.m * 256, slots_of(p, tl.m))
                                   : (int)kNoneBad;
              }
              const int own = live ? p.slot[row] : -1;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t want = 0;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                  const int b = __shfl_sync(0xffffffffu, bad[h], i);
                  if (odd && !isfinite(v[32 * h + i]) && b != kNoneBad && b != own) want |= 1u << i;
                }
                if (__any_sync(0xffffffffu, want != 0)) {
                  float mine[32];
                  own_values(p, row0 + 32 * warp, col0 + 32 * h, tl.m, want, mine);
#pragma unroll
                  for (int i = 0; i < 32; ++i)
                    if (want >> i & 1) v[32 * h + i] = mine[i];
                }
              }
            }
          }
          if (p.bias != nullptr) {
            if (bias_vec && col0 + 64 <= p.N) {
              const uint4* b4 = reinterpret_cast<const uint4*>(p.bias + col0);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint4 w = __ldg(b4 + i);
                const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                  v[8 * i + 2 * u] += bf16_lo(ww[u]);
                  v[8 * i + 2 * u + 1] += bf16_hi(ww[u]);
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 64; ++i)
                if (col0 + i < p.N) v[i] += __bfloat162float(p.bias[col0 + i]);
            }
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
          if (threadIdx.x == 0) bulk_wait_group_read1();
          named_bar_sync(1, 128);
          stage_half(b0, r, 0, acc);
          stage_half(b0, r, 1, acc + 16);
          fence_proxy_async_smem();
          named_bar_sync(1, 128);
          if (threadIdx.x == 0) {
            if (row0 < p.M && col0 < p.N) tma_store_3d(&td, b0, col0, row0, tl.b);
            bulk_commit_group();
          }
        } else {
          const int g = it * (kBN / 64) + c;
          const bool direct = EPI == kEpiLast && p.out_t != nullptr;
          uint8_t* b0 = stg + (g & 1) * 2 * kStaging;  // in: Q or hi; out: the tile
          uint8_t* b1 = b0 + kStaging;                 // in and out: lo; out: the mirrored tile
          if (threadIdx.x == 0) {
            if constexpr (kReads) {
              bulk_wait_group_read0();
              const int64_t tn = t + pairs;
              if (c + 1 < kBN / 64) request(tl, c + 1, g + 1);
              else if (tn < tiles) request(tile_of(tn, p), 0, g + 1);
            } else {
              bulk_wait_group_read1();
            }
          }
          if constexpr (kReads) ok = mbar_wait_w(&back[g & 1], (g >> 1) & 1);
          if (named_bar_any(1, 128, !ok)) { ok = false; break; }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t acc[32], out[16], lo[16];
            Back<EPI> bk;
            tmem_ld32(taddr + 32 * h, acc);
            bk.take(b0, b1, r, h);
            tmem_wait_ld();
            ns_values<EPI>(p, bk, ca, cb, acc, out, lo);
            if (direct) {
              if (live)
                store_columns(p.out_t + (int64_t)tl.b * p.out_t_batch + row, p.out_t_ld,
                              col0 + 32 * h, p.N, out);
              continue;
            }
            stage_half(b0, r, h, out);
            if constexpr (EPI == kEpiUpdate) stage_half(b1, r, h, lo);
            if constexpr (!kX)
              if (mirror) stage_mirror(b1, r, h, out);
          }
          fence_proxy_async_smem();
          named_bar_sync(1, 128);
          if (threadIdx.x == 0 && !direct) {
            if (row0 < p.M && col0 < p.N) {
              tma_store_3d(&td, b0, col0, row0, tl.b);
              if constexpr (EPI == kEpiUpdate) tma_store_3d(&td2, b1, col0, row0, tl.b);
              if constexpr (!kX)
                if (mirror) store_mirror(&tl_low, b1, row0, col0, tl.b, p);
            }
            bulk_commit_group();
          }
        }
      }
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa(smem_u32(&accempty[buf]), 0));
    }
    if (threadIdx.x == 0) bulk_wait_group_read0();  // (the grid's end completes the stores)
    if (!ok) *abort_flag = 1;
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) drain_delay();
  cluster_sync();
  if (warp == 5) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem, kTmemCols);
  }
}

template <bool B_MN, int EPI>
static int go(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& te,
              const CUtensorMap& tlow, const CUtensorMap& td, const CUtensorMap& td2, const WideParams& p, int kernel_id,
              cudaStream_t st) {
  auto* fn = wide_kernel<B_MN, EPI>;
  const int rc = ensure_smem_attr((const void*)fn, smem_of(EPI), kernel_id);
  if (rc) return rc;
  const int64_t tiles = (int64_t)p.tiles_per_batch * p.batch;
  const int pairs = (int)std::min<int64_t>(tiles, 74);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_of(EPI);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.early ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, ta, tb, te, tlow, td, td2, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return record_cuda_error(e);
  }
  return launch_status();
}

// ------------------------------------------------------------ narrow form
// The orthogonalisation's products of matrices too small to fill the SM pairs:
// one 128 x 64 tile per CTA (cta_group::1), two CTAs an SM, so that a 1024 x
// 1024 product has 72 to 128 CTAs instead of 10 to 16 pairs. Its time is start,
// latency and epilogue; the next product's CTAs are set up meanwhile
// (programmatic dependent launch). The staging tiles lie over the ring.
constexpr int kNarrowBN = 64;
constexpr int kNarrowStage = kStageA + kNarrowBN * 128;
constexpr int kNarrowStages = 4;
constexpr int kNarrowBar = kNarrowStages * kNarrowStage;
constexpr int kNarrowSums = 128 * kNarrowBN * 4;
constexpr int kNarrowSplit = 4;  // most CTAs a tile
static_assert((kNarrowSplit - 1) * kNarrowSums <= kNarrowBar, "the sums lie over the ring");
constexpr int kNarrowSmem = kNarrowBar + 256 + 1024;

// (bounds of 256 threads: registers are given to four warps at a time)
template <bool B_MN, int EPI, bool SPLIT>
__global__ void __launch_bounds__(256, 2)
narrow_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
              const __grid_constant__ CUtensorMap tmir, const __grid_constant__ CUtensorMap td, const __grid_constant__ CUtensorMap td2,
              const __grid_constant__ WideParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kNarrowBar);
  uint64_t* empty = full + kNarrowStages;
  uint64_t* done = empty + kNarrowStages;
  uint32_t* slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(slot + 1);
  const int warp = warp_id(), lane = lane_id();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kNarrowStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&ta);
    tma_prefetch_desc(&tb);
    tma_prefetch_desc(&td);
  }
  if (warp == 5) {
    tmem_alloc(slot, kNarrowBN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  pdl_launch_next();
  pdl_wait_previous();

  // a tile's contraction may be shared by the CTAs of a cluster (p.split)
  const int split = SPLIT ? p.split : 1;
  const int tile = blockIdx.x / split, part = blockIdx.x - tile * split;
  const int b = tile / p.tiles_per_batch;
  const int i = tile - b * p.tiles_per_batch;
  int tm, tn;
  if (p.symmetric) {
    triangle(i, 2, tm, tn);  // 128-row block m: column tiles 0 .. 2 m + 1
  } else {
    tn = i / p.tiles_m;
    tm = i - tn * p.tiles_m;
  }
  const int row0 = tm * 128, col0 = tn * kNarrowBN;
  const int kbs = (p.K + 63) >> 6;
  const int kb0 = (int)((int64_t)kbs * part / split), kb1 = (int)((int64_t)kbs * (part + 1) / split);
  bool ok = true;
  if (warp == 4) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = mbar_wait(&empty[s], ph ^ 1))) break;
        uint8_t* sa = smem + s * kNarrowStage;
        mbar_arrive_expect_tx(&full[s], kNarrowStage);
        tma_load_3d(sa, &ta, &full[s], kb * 64, row0, b);
        if constexpr (B_MN) tma_load_3d(sa + kStageA, &tb, &full[s], col0, kb * 64, b);
        else tma_load_3d(sa + kStageA, &tb, &full[s], kb * 64, col0, b);
        if (++s == kNarrowStages) { s = 0; ph ^= 1; }
      }
      if (!ok) *abort_flag = 1;
    }
    __syncwarp();
    if (SPLIT) cluster_sync(), cluster_sync();  // (with the epilogue's)
  } else if (warp == 5) {
    const uint32_t idesc = idesc_f16(p.fmt, 128, kNarrowBN, false, B_MN);
    const uint32_t base = smem_u32(smem);
    const uint64_t a0 = kmajor_desc(base, 0, 0);
    const uint64_t b0 = B_MN ? mnmajor_desc(base + kStageA, 0, 8192) : kmajor_desc(base + kStageA, 0, 0);
    int s = 0;
    uint32_t ph = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!(ok = mbar_wait_w(&full[s], ph))) break;
      tc_fence_after();
      const uint64_t a = a0 + (uint32_t)(s * (kNarrowStage >> 4));
      const uint64_t bb = b0 + (uint32_t)(s * (kNarrowStage >> 4));
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        umma_ss_w(tmem, a + 2 * kk, bb + (B_MN ? 128 : 2) * kk, idesc, kb > kb0 || kk > 0);
      umma_commit_w(&empty[s]);
      if (kb == kb1 - 1) umma_commit_w(done);
      if (++s == kNarrowStages) { s = 0; ph ^= 1; }
    }
    if (!ok) *abort_flag = 1;
    __syncwarp();
    if (SPLIT) cluster_sync(), cluster_sync();
  } else {
    const int r = threadIdx.x, row = row0 + r;
    const bool live = row < p.M;
    float ca = 0.f, cb = 0.f;
    if constexpr (EPI != kEpiGram) {
      ca = p.coef[2 * b];
      cb = p.coef[2 * b + 1];
    }
    Back<EPI> back[2];  // on its way under the products
    back[0].load(p, b, row, live, col0);
    back[1].load(p, b, row, live, col0 + 32);
    ok = mbar_wait_w(done, 0);
    const bool bad = named_bar_any(1, 128, !ok);
    tc_fence_after();
    const uint32_t taddr = tmem + ((uint32_t)(warp * 32) << 16);
    if constexpr (SPLIT) {
      // the other CTAs' sums go to the first one's ring, which is idle when all
      // have waited for their products: (split - 1, 64 / 4, 128, 4) fp32
      cluster_sync();
      if (part > 0 && !bad) {
        const uint32_t dst = mapa(smem_u32(smem) + (uint32_t)((part - 1) * kNarrowSums + r * 16), 0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t acc[32];
          tmem_ld32(taddr + 32 * h, acc);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; c += 4)
            st_cluster_v4(dst + (uint32_t)((32 * h + c) * 512), acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
        }
      }
      cluster_sync();
    }
    if (!bad && part == 0) {
      const bool mirror = p.symmetric && tn < 2 * tm;
      const bool direct = EPI == kEpiLast && p.out_t != nullptr;
      uint32_t first[SPLIT ? 32 : 1];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t acc[32], out[16], lo[16];
        tmem_ld32(taddr + 32 * h, acc);
        tmem_wait_ld();
        if constexpr (SPLIT) {  // in CTA order
          float* v = reinterpret_cast<float*>(acc);
          for (int q = 0; q < split - 1; ++q) {
            const float4* s = reinterpret_cast<const float4*>(smem + q * kNarrowSums) + r;
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 w = s[(32 * h + c) * 32];
              v[c] += w.x; v[c + 1] += w.y; v[c + 2] += w.z; v[c + 3] += w.w;
            }
          }
          // the staged tiles lie over the sums
          if (h == 0) {
#pragma unroll
            for (int c = 0; c < 32; ++c) first[c] = acc[c];
            continue;
          }
          named_bar_sync(1, 128);
          uint32_t o0[16];
          ns_values<EPI>(p, back[0], ca, cb, first, o0, lo);
          if (mirror) stage_mirror(smem + kStaging, r, 0, o0);
          stage_half(smem, r, 0, o0);
        }
        ns_values<EPI>(p, back[h], ca, cb, acc, out, lo);
        if (direct) {
          if (live)
            store_columns(p.out_t + (int64_t)b * p.out_t_batch + row, p.out_t_ld, col0 + 32 * h, p.N,
                          out);
          continue;
        }
        if (mirror) stage_mirror(smem + kStaging, r, h, out);
        stage_half(smem, r, h, out);
        if constexpr (EPI == kEpiUpdate) stage_half(smem + kStaging, r, h, lo);
      }
      if (!direct) {
        fence_proxy_async_smem();
        named_bar_sync(1, 128);
        if (threadIdx.x == 0) {
          if (row0 < p.M && col0 < p.N) {
            tma_store_3d(&td, smem, col0, row0, b);
            if constexpr (EPI == kEpiUpdate) tma_store_3d(&td2, smem + kStaging, col0, row0, b);
            if (mirror) store_mirror(&tmir, smem + kStaging, row0, col0, b, p);
          }
          bulk_commit_group();
          bulk_wait_group_read0();
        }
      }
    } else if (bad) {
      *abort_flag = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) drain_delay();
  if (warp == 5) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, kNarrowBN);
  }
}

template <bool B_MN, int EPI, bool SPLIT = false>
static int narrow_go(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tmir,
                     const CUtensorMap& td, const CUtensorMap& td2, const WideParams& p, int kernel_id, cudaStream_t st) {
  auto* fn = narrow_kernel<B_MN, EPI, SPLIT>;
  const int rc = ensure_smem_attr((const void*)fn, kNarrowSmem, kernel_id);
  if (rc) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((int64_t)p.tiles_per_batch * p.batch * p.split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kNarrowSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = p.early != 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = p.split;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = SPLIT ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, ta, tb, tmir, td, td2, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return record_cuda_error(e);
  }
  return launch_status();
}

// Which form is sooner done: rounds of 296 resident tiles of 128 x 64, 0.4 us a
// K block while an SM holds two (0.2 us one), or of 74 pairs' tiles of 256 x
// 256, 0.29 us a K block. A Gram product of few tiles and a long contraction
// splits it over up to four CTAs a tile, for some 2 us (2 x
// 272 x 2792: 195 -> 145 us a call, 100 x 8192 207 -> 123).
static bool use_narrow(WideParams& p, int epi) {
  const int64_t m1 = (p.M + 127) / 128, n1 = (p.N + 63) / 64;
  const int64_t m2 = (p.M + 255) / 256, n2 = (p.N + 255) / 256;
  const int64_t t1 = (p.symmetric ? m1 * (m1 + 1) : m1 * n1) * p.batch;
  const int64_t t2 = (p.symmetric ? m2 * (m2 + 1) / 2 : m2 * n2) * p.batch;
  const int64_t kbs = (p.K + 63) / 64;
  float narrow = 4.f + (t1 <= 148 ? 0.2f * kbs : (t1 + 295) / 296 * kbs * 0.4f);
  p.split = 1;
  for (int c = 2; epi == kEpiGram && c <= kNarrowSplit && t1 * c <= 148 && c <= kbs; ++c) {
    const float time = 6.f + 0.2f * ((kbs + c - 1) / c);
    if (time < narrow) narrow = time, p.split = c;
  }
  const float pairs = 9.f + (t2 + 73) / 74 * kbs * 0.29f;
  return narrow < pairs;
}

}  // namespace wide

int TmapMemo::get(CUtensorMap* map, const Mat3& m, int rows) {
  for (int i = 0; i < n; ++i)
    if (p[i] == m.p && box[i] == rows) {
      *map = maps[i];
      return FA_OK;
    }
  const int rc = make_tmap_3d(map, m, 64, rows);
  if (rc == FA_OK && n < kMost) {
    p[n] = m.p;
    box[n] = rows;
    maps[n++] = *map;
  }
  return rc;
}

int launch_gemm_wide(const WideOperands& o, WideParams p, int epi, cudaStream_t st,
                     TmapMemo* maps) {
  const bool narrow = epi != kEpiLinear && wide::use_narrow(p, epi);
  const int tile_n = narrow ? wide::kNarrowBN : wide::kBN, tile_m = narrow ? 128 : 256;
  p.tiles_m = (p.M + tile_m - 1) / tile_m;
  p.tiles_n = (p.N + tile_n - 1) / tile_n;
  p.tiles_per_batch = !p.symmetric ? p.tiles_m * p.tiles_n
                      : narrow     ? p.tiles_m * (p.tiles_m + 1)
                                   : p.tiles_m * (p.tiles_m + 1) / 2;
  // a pair's CTA loads half of the tile's columns
  const int load_n = narrow ? tile_n : tile_n / 2;
  CUtensorMap ta, tb, te, tlow, td, td2;
  auto encode = [&](CUtensorMap* m, const Mat3& x, int rows) {
    return maps != nullptr ? maps->get(m, x, rows) : make_tmap_3d(m, x, 64, rows);
  };
  int rc = encode(&ta, o.a, 128);
  if (!rc) rc = encode(&tb, o.b, o.b_mn ? 64 : load_n);
  te = tb;
  if (!rc && p.low != nullptr)
    rc = o.b_mn ? make_tmap_3d(&te, o.e, 64, 64) : make_tmap_3d(&te, o.e, 64, load_n);
  tlow = ta;
  if (!rc && p.low != nullptr)
    rc = make_tmap_3d(&tlow, Mat3{p.low, 1, p.M, p.low_ld, 0, p.low_stride, 1}, 64, 128);
  // the orthogonalisation's: X read back, and the mirrored store's 64 x 64 boxes
  if (!rc && o.e.p != nullptr && p.low == nullptr) rc = encode(&te, o.e, 128);
  if (!rc && p.symmetric) rc = encode(&tlow, o.d, 64);
  td = ta;
  if (!rc && o.d.p != nullptr) rc = encode(&td, o.d, 128);
  td2 = td;
  if (!rc && o.d2.p != nullptr) rc = encode(&td2, o.d2, 128);
  if (rc) return rc;
#define FA_WIDE(EPI, MN, ID) \
  if (epi == EPI && o.b_mn == MN) return wide::go<MN, EPI>(ta, tb, te, tlow, td, td2, p, ID, st);
#define FA_NARROW(EPI, MN, ID)                    \
  if (narrow && epi == EPI && o.b_mn == MN)       \
    return wide::narrow_go<MN, EPI>(ta, tb, tlow, td, td2, p, ID, st);
  if (narrow && epi == kEpiGram && p.split > 1)
    return wide::narrow_go<false, kEpiGram, true>(ta, tb, tlow, td, td2, p, kKernelNarrow + 4, st);
  FA_NARROW(kEpiGram, false, kKernelNarrow)
  FA_NARROW(kEpiPoly, false, kKernelNarrow + 1)
  FA_NARROW(kEpiUpdate, true, kKernelNarrow + 2)
  FA_NARROW(kEpiLast, true, kKernelNarrow + 3)
  FA_WIDE(kEpiLinear, false, kKernelWide)
  FA_WIDE(kEpiLinear, true, kKernelWide + 1)
  FA_WIDE(kEpiGram, false, kKernelWide + 2)
  FA_WIDE(kEpiPoly, false, kKernelWide + 3)
  FA_WIDE(kEpiUpdate, true, kKernelWide + 4)
  FA_WIDE(kEpiLast, true, kKernelWide + 5)
#undef FA_WIDE
#undef FA_NARROW
  return FA_ERR_UNSUPPORTED;
}

int wide_device_status() { return tu_device_status(); }

}  // namespace fa
