// gemm_skinny_sm100.cu — products with one short side, on the tensor cores:
//
//   out[i, j] = sum_k Big[i, k] Small[j, k],   j < 256
//
// Uses: a linear for few tokens (Big = the weight, Small = the tokens), the
// adapters' inner products low = s x A^T and s dy B (Big = the tokens), and
// the factors' gradients (Big = x or dy with the tokens as contraction).
//
// Bound by reading Big once from memory. A cluster of C CTAs shares a 128-row
// tile of Big and splits the contraction, so that even few tiles occupy all
// SMs; each CTA streams its K blocks through a TMA ring (two CTAs an SM while
// the short side is at most 128, about 96 KB in flight each) into tcgen05.mma
// with Big as the 128-row operand and the short side as its columns. The partial
// sums stay on chip: every CTA sends the columns it does not own to their
// owner through distributed shared memory, and the owner adds them in CTA
// order (fp32, the same bits every time), then applies the epilogue.
// At 9216 x 4096, rank 32: x A^T 20 us (3.7 TB/s); dy B of 9216 x 16384 60 us
// (5.1 TB/s); both factors' gradients 75 us (5.1 TB/s). 64 tokens x 4096 x
// 16384 with 48 adapters of rank 16: 39 us (4.1 TB/s); one token at 4096 x 4096
// about 7 us.
#include <algorithm>

#include "attn_common.h"
#include "gemm.h"
#include "gemm_ptx.cuh"

namespace fa {
namespace skinny {

constexpr int kThreads = 192;
constexpr int kBig = 16384;  // 128 x 64 elements
constexpr int kMaxStages = 8;
constexpr int kBarBytes = 256;
constexpr int kTwoSmem = 109 * 1024;  // two CTAs an SM, beside their static 3.6 KB
constexpr int kOneSmem = 220 * 1024;
constexpr int kMaxTokens = kMaxColumns;

struct Layout {
  int stage, stages, smem, cols;  // stage bytes, ring depth, launch bytes, TMEM columns
  int exchange;                   // offset of the partial sums: behind the ring, or 0: over it
};

// n: columns of the product (multiple of 16), small_mn: Small stored with its
// short side contiguous (64-wide blocks)
static Layout layout_of(int n, bool small_mn, bool two) {
  Layout l{};
  const int small = small_mn ? (n + 63) / 64 * 8192 * (two ? 2 : 1) : (n * 128 + 1023) / 1024 * 1024;
  l.stage = kBig + small;
  const int budget = (n <= 128 ? kTwoSmem : kOneSmem) - kBarBytes - 1024;
  // the columns' owner's partial sums, owners' shares rounded up to 4 columns.
  // While they are small they get memory of their own, so that a CTA need not
  // wait for the others' rings before it sends.
  const int sums = (n + 32) * 512;
  const bool own = n <= 16;
  l.stages = std::min(kMaxStages, (budget - (own ? sums : 0)) / l.stage);
  l.exchange = own ? l.stage * l.stages : 0;
  l.smem = (own ? l.exchange + sums : std::max(l.stage * l.stages, sums)) + kBarBytes + 1024;
  l.cols = 32;
  while (l.cols < n) l.cols *= 2;
  return l;
}

// The adapters in use by up to 256 tokens, in order of first use, and every
// token's place among them (-1: none).
struct alignas(16) TokenPlan {
  int id[kMaxTokens];
  int list[kMaxTokens];
  int16_t slot[kMaxTokens];
  int heads[8];
  int cnt;
};

// 128 threads (named barrier 1)
__device__ __forceinline__ void plan_tokens(TokenPlan& pl, const int* ids, int cols, int E) {
  const int t = threadIdx.x;
  if (ids == nullptr) {
    for (int j = t; j < kMaxTokens; j += 128) pl.slot[j] = j < cols ? 0 : -1;
    if (t == 0) pl.cnt = 1, pl.list[0] = 0;
    named_bar_sync(1, 128);
    return;
  }
  for (int j = t; j < kMaxTokens; j += 128) {
    const int e = j < cols ? ids[j] : -1;
    pl.id[j] = e >= 0 && e < E ? e : -1;
  }
  named_bar_sync(1, 128);
  int first[2], before[2];
  bool head[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int j = t + 128 * h, e = pl.id[j];
    int f = j;
    if (e >= 0) {  // four at a time; ends at j at the latest
      for (int b = 0;; b += 4) {
        const int4 v = *reinterpret_cast<const int4*>(&pl.id[b]);
        if (v.x == e) { f = b; break; }
        if (v.y == e) { f = b + 1; break; }
        if (v.z == e) { f = b + 2; break; }
        if (v.w == e) { f = b + 3; break; }
      }
    }
    first[h] = f;
    head[h] = e >= 0 && f == j;
    const uint32_t m = __ballot_sync(0xffffffffu, head[h]);
    before[h] = __popc(m & ((1u << lane_id()) - 1u));
    if (lane_id() == 0) pl.heads[4 * h + warp_id()] = __popc(m);
  }
  named_bar_sync(1, 128);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int at = before[h];
    for (int w = 0; w < 4 * h + warp_id(); ++w) at += pl.heads[w];
    if (head[h]) {
      pl.list[at] = pl.id[t + 128 * h];
      pl.slot[t + 128 * h] = (int16_t)at;
    }
  }
  if (t == 0) {
    int n = 0;
    for (int w = 0; w < 8; ++w) n += pl.heads[w];
    pl.cnt = n;
  }
  named_bar_sync(1, 128);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int j = t + 128 * h;
    if (!head[h]) pl.slot[j] = pl.id[j] >= 0 ? pl.slot[first[h]] : (int16_t)-1;
  }
  named_bar_sync(1, 128);
}

// The four columns from j on of tile row r, summed in CTA order: recv (split, own
// / 4, 128, 4), columns j0 on.
__device__ __forceinline__ void sum_columns(const float* recv, int split, int own, int j, int r,
                                            float* acc) {
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int q = 0; q < split; ++q) {
    const float4 v = *reinterpret_cast<const float4*>(recv + (q * own + j) * 128 + r * 4);
    a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
  }
  acc[0] = a.x; acc[1] = a.y; acc[2] = a.z; acc[3] = a.w;
}

// A warp's 32 rows and the tokens [j0, j1) of its CTA, of which some value is not
// finite: those that another token's broken factor reached (zero times a NaN or
// an infinity) are stored again, from their own operands alone, 32 tokens at a
// time. Apart from the kernel's own code, which it costs no registers.
__device__ __noinline__ void repair_tokens(const SkinnyParams& p, const TokenPlan& plan,
                                           const float* recv, int split, int own, int j0, int j1,
                                           int j_base, int i0) {
  const int first = i0 + 32 * warp_id(), i = first + lane_id();
  const bool in = i < p.rows;
  const int bad = in ? bad_factors(p.raw_f + (int64_t)i * p.raw_ldf, p.raw_fe, p.rank, plan.list,
                                   plan.cnt)
                     : (int)kNoneBad;
  if (!__any_sync(0xffffffffu, bad != kNoneBad)) return;
  const float bias = in && p.bias != nullptr ? __bfloat162float(p.bias[i]) : 0.f;
  for (int jb = j0; jb < j1; jb += 32) {
    const int n = min(32, j1 - jb);
    uint32_t want = 0;
    for (int k = 0; k < n; k += 4) {
      float acc[4];
      sum_columns(recv, split, own, jb + k - j0, threadIdx.x, acc);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (bad != kNoneBad && k + u < n && !isfinite(acc[u]) && bad != plan.slot[jb + k + u])
          want |= 1u << (k + u);
    }
    if (!__any_sync(0xffffffffu, want != 0)) continue;
    float base[32];
    base_products(p.raw_w + (int64_t)first * p.raw_ldw, p.raw_ldw, min(32, p.rows - first),
                  p.raw_x + (int64_t)(j_base + jb) * p.raw_ldx, p.raw_ldx, n, p.K, base);
    for (int k = 0; k < n; ++k) {
      if (!(want >> k & 1)) continue;
      const int64_t j = j_base + jb + k;
      const int s = plan.slot[jb + k];
      float v = base[k];
      if (s >= 0)
        v += own_term(p.low + j * p.low_stride,
                      p.raw_f + (int64_t)plan.list[s] * p.raw_fe + (int64_t)i * p.raw_ldf, p.rank);
      p.out[j * p.out_ld + i] = __float2bfloat16_rn(v + bias);
    }
  }
}

// What rounding v to `rounded` dropped; nothing where that is an infinity
__device__ __forceinline__ float remainder(float v, float rounded) {
  return isfinite(rounded) ? v - rounded : 0.f;
}

// Descriptors of Big, Small and `fac`; of the gradients' two products (da and db
// in one launch, as grid rows: each alone leaves SMs idle and costs a launch).
template <int OUT>
struct Maps {
  static constexpr int kProducts = OUT == kSkinnyGrad ? 2 : 1;
  CUtensorMap big[kProducts], small[kProducts], fac[kProducts];
};

// (Bounds of 256 threads: registers are given to four warps at a time, so that
// two blocks of six warps fit an SM as two of eight would, up to 128 a thread.)
template <bool BIG_MN, bool SMALL_MN, int OUT, int PACK, int HOLD>
__global__ void __launch_bounds__(256, 2)
skinny_kernel(const __grid_constant__ Maps<OUT> maps, const __grid_constant__ SkinnyParams p,
              int split, int stage_bytes, int stages, int bar_off, int exchange, int tmem_cols) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + bar_off);
  uint64_t* full = bars;
  uint64_t* empty = bars + kMaxStages;
  uint64_t* done = bars + 2 * kMaxStages;
  uint64_t* planned = done + 1;
  uint64_t* grant = planned + 1;
  uint32_t* slot = reinterpret_cast<uint32_t*>(grant + kMaxStages);
  __shared__ TokenPlan plan;
  __shared__ uint8_t tokens_s[OUT == kSkinnyCols ? 4 : 1][kMaxTokens];  // of an adapter, per warp
  volatile int* abort_flag = reinterpret_cast<volatile int*>(slot + 1);
  const int warp = warp_id(), lane = lane_id();
  const int tile = blockIdx.x / split, part = blockIdx.x - tile * split;
  const int i0 = tile * 128;
  const int which = OUT == kSkinnyGrad ? blockIdx.y : 0;
  const CUtensorMap *tbig = &maps.big[which], *tsmall = &maps.small[which], *tfac = &maps.fac[which];
  const int rows = which ? p.rows2 : p.rows;
  if (OUT == kSkinnyGrad && i0 >= rows) return;  // the same for the whole cluster

  // columns of this pass: adapters [s0, s0 + ns) of the tile's list, or all;
  // of a linear the tokens j_base .. j_base + cols
  int n = p.n, s0 = 0, ns = 1;
  const int j_base = OUT == kSkinnyCols ? blockIdx.y * p.n : 0;
  const int cols = min(p.n, p.cols - j_base);
  const __nv_bfloat16* low = p.low != nullptr ? p.low + (int64_t)j_base * p.low_stride : nullptr;
  if constexpr (OUT == kSkinnyLow) {
    if (p.list_cnt != nullptr) {
      s0 = blockIdx.y * p.slots_per_pass;
      ns = min(p.slots_per_pass, p.list_cnt[i0 >> 8] - s0);
      if (ns <= 0) return;  // the same for the whole cluster
      n = ns * p.low_ld;
    }
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], OUT == kSkinnyCols ? 2 : 1);
      mbar_init(&empty[i], 1);
      mbar_init(&grant[i], 1);
    }
    mbar_init(done, 1);
    mbar_init(planned, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(tbig);
    tma_prefetch_desc(tsmall);
  }
  if (warp == 5) {
    tmem_alloc(slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (split > 1) cluster_arrive();  // this CTA has started: its memory may be written
  const uint32_t tmem = *slot;
  const int kbs = (p.K + 63) >> 6;
  const int kb0 = (int)((int64_t)kbs * part / split), kb1 = (int)((int64_t)kbs * (part + 1) / split);
  bool ok = true;
  // adapters (token columns): after its share of K, the CTA's share of the
  // K blocks that hold (adapter, 64 ranks)
  const bool adapters = OUT == kSkinnyCols && p.low != nullptr;
  const int kbe = (p.rank + 63) >> 6;
  // With requests' adapters of at most 32 ranks a block holds two or four of
  // them, each with tiles of its own width (64 x 4096 x 16384 with 48 adapters
  // of rank 16: 47 us, 53 as blocks of one)
  constexpr int pack = PACK;

  pdl_launch_next();
  if (warp == 4) {
    if (lane == 0) {
      if constexpr (OUT != kSkinnyCols) pdl_wait_previous();
      const int small_blocks = (n + 63) >> 6;
      constexpr bool two = OUT == kSkinnyGrad;
      const uint32_t bytes = kBig + (SMALL_MN ? (two ? 2 : 1) * small_blocks * 8192
                                              : (OUT == kSkinnyCols ? p.n * 128 : n * 128));
      int s = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = mbar_wait(&empty[s], ph ^ 1))) break;
        uint8_t* sa = smem + s * stage_bytes;
        uint8_t* sb = sa + kBig;
        mbar_arrive_expect_tx(&full[s], bytes);
        if constexpr (OUT == kSkinnyCols) mbar_arrive(&full[s]);  // else: the builders' arrival
        if constexpr (BIG_MN) {
          tma_load_3d(sa, tbig, &full[s], i0, kb * 64, 0);
          tma_load_3d(sa + 8192, tbig, &full[s], i0 + 64, kb * 64, 0);
        } else {
          tma_load_3d(sa, tbig, &full[s], kb * 64, i0, 0);
        }
        if constexpr (SMALL_MN) {
          for (int j = 0; j < small_blocks; ++j)
            tma_load_3d(sb + j * 8192, tsmall, &full[s], j * 64, kb * 64, 0);
          if (two)
            for (int j = 0; j < small_blocks; ++j)
              tma_load_3d(sb + (small_blocks + j) * 8192, tfac, &full[s], j * 64, kb * 64, 0);
        } else if constexpr (OUT == kSkinnyLow) {
          for (int q = 0; q < ns; ++q) {
            const int e = p.list_ids != nullptr ? p.list_ids[(int64_t)(i0 >> 8) * 256 + s0 + q] : 0;
            tma_load_3d(sb + q * p.low_ld * 128, tsmall, &full[s], kb * 64, 0, e);
          }
        } else {
          tma_load_3d(sb, tsmall, &full[s], kb * 64, j_base, 0);
        }
        if (++s == stages) { s = 0; ph ^= 1; }
      }
      if (ok && adapters && (ok = mbar_wait(planned, 0))) {
        const int blocks = pack > 1 ? (plan.cnt + pack - 1) / pack : plan.cnt * kbe;
        for (int x = part; x < blocks; x += split) {
          if (!(ok = mbar_wait(&empty[s], ph ^ 1))) break;
          uint8_t* sa = smem + s * stage_bytes;
          mbar_arrive(&grant[s]);
          if constexpr (pack > 1) {
            const int some = min(pack, plan.cnt - x * pack), each = kBig / pack;
            mbar_arrive_expect_tx(&full[s], some * each);
            for (int u = 0; u < some; ++u)
              tma_load_3d(sa + u * each, tfac, &full[s], 0, i0, plan.list[x * pack + u]);
          } else {
            const int e = plan.list[x / kbe], j = x % kbe;
            mbar_arrive_expect_tx(&full[s], kBig);
            if constexpr (BIG_MN) {
              tma_load_3d(sa, tfac, &full[s], i0, j * 64, e);
              tma_load_3d(sa + 8192, tfac, &full[s], i0 + 64, j * 64, e);
            } else {
              tma_load_3d(sa, tfac, &full[s], j * 64, i0, e);
            }
          }
          if (++s == stages) { s = 0; ph ^= 1; }
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == 5) {
    const uint32_t idesc = idesc_f16(1, 128, n, BIG_MN, SMALL_MN);
    const uint32_t base = smem_u32(smem);
    const uint64_t a0 = BIG_MN ? mnmajor_desc(base, 0, 8192) : kmajor_desc(base, 0, 0);
    const uint64_t b0 = SMALL_MN ? mnmajor_desc(base + kBig, 0, 8192)
                                 : kmajor_desc(base + kBig, 0, 0);
    int s = 0;
    uint32_t ph = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!(ok = mbar_wait_w(&full[s], ph))) break;
      tc_fence_after();
      const uint64_t a = a0 + (uint32_t)(s * (stage_bytes >> 4));
      const uint64_t b = b0 + (uint32_t)(s * (stage_bytes >> 4));
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        umma_ss_w(tmem, a + (BIG_MN ? 128 : 2) * kk, b + (SMALL_MN ? 128 : 2) * kk, idesc,
                  kb > kb0 || kk > 0);
      if (OUT == kSkinnyGrad) {
        const uint64_t b2 = b + (uint32_t)(((n + 63) >> 6) * (8192 >> 4));
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_ss_w(tmem, a + (BIG_MN ? 128 : 2) * kk, b2 + 128 * kk, idesc, 1);
      }
      umma_commit_w(&empty[s]);
      if (!adapters && kb == kb1 - 1) umma_commit_w(done);
      if (++s == stages) { s = 0; ph ^= 1; }
    }
    if (ok && adapters && (ok = mbar_wait_w(planned, 0))) {
      const int blocks = pack > 1 ? (plan.cnt + pack - 1) / pack : plan.cnt * kbe;
      for (int x = part; x < blocks; x += split) {
        if (!(ok = mbar_wait_w(&full[s], ph))) break;
        tc_fence_after();
        if constexpr (pack > 1) {
          const int some = min(pack, plan.cnt - x * pack), steps = (p.rank + 15) >> 4;
          uint64_t a = kmajor_narrow_desc(base + s * stage_bytes, 128 / pack);
          uint64_t b = kmajor_narrow_desc(base + s * stage_bytes + kBig, 128 / pack);
          for (int u = 0; u < some; ++u) {
            for (int kk = 0; kk < steps; ++kk) umma_ss_w(tmem, a + 2 * kk, b + 2 * kk, idesc, 1);
            a += (uint32_t)(kBig / pack >> 4);
            b += (uint32_t)(n * 128 / pack >> 4);
          }
        } else {
          const uint64_t a = a0 + (uint32_t)(s * (stage_bytes >> 4));
          const uint64_t b = b0 + (uint32_t)(s * (stage_bytes >> 4));
          const int steps = min(4, (p.rank - (x % kbe) * 64 + 15) >> 4);
          for (int kk = 0; kk < steps; ++kk)
            umma_ss_w(tmem, a + (BIG_MN ? 128 : 2) * kk, b + 2 * kk, idesc, 1);
        }
        umma_commit_w(&empty[s]);
        if (++s == stages) { s = 0; ph ^= 1; }
      }
      if (ok) umma_commit_w(done);
    }
    if (!ok) *abort_flag = 1;
  } else {
    if (adapters) {
      // the tokens' operand of each adapter block: low[j, :] in the tokens that
      // use the adapter, zeros in the others, in the layout TMA writes
      const int t = threadIdx.x;
      plan_tokens(plan, p.ids != nullptr ? p.ids + j_base : nullptr, cols, p.E);
      if (t == 0) mbar_arrive(planned);
      pdl_wait_previous();
      // A warp builds for every fourth slot of the ring. A slot is its when the
      // producer, which has waited for every earlier use of it, grants it: a
      // parity wait on `empty` from here would skip phases and could return
      // for an earlier one.
      const int blocks = pack > 1 ? (plan.cnt + pack - 1) / pack : plan.cnt * kbe;
      int s = (kb1 - kb0) % stages;
      uint32_t turns = 0;  // bit s: parity of the slot's next grant
      // A lane's 16-byte pieces of the operand are the same in every block
      // while one block holds the rank: up to HOLD are kept in registers (with
      // their place, and the adapter's slot above it) and a block is stores
      // alone.
      constexpr int kHold = HOLD;
      const int chunks0 = min(8, p.low_ld >> 3);
      const bool held = kbe == 1 && n * chunks0 <= kHold * 32;
      uint4 hold[kHold];
      int at[kHold];
      if (held) {
#pragma unroll
        for (int k = 0; k < kHold; ++k) {
          const int i = lane + 32 * k, j = i / chunks0, c = i - j * chunks0;
          at[k] = -1;
          hold[k] = make_uint4(0, 0, 0, 0);
          if (i < n * chunks0) {
            const int place = (int)(pack > 1 ? narrow_offset(j, c, 128 / pack) : sw128_offset(j, c));
            at[k] = place | 511 << 16;
            if (j < cols && plan.slot[j] >= 0) {
              at[k] = place | plan.slot[j] << 16;
              hold[k] = *reinterpret_cast<const uint4*>(low + (int64_t)j * p.low_stride + c * 8);
            }
          }
        }
      }
      for (int x = part; x < blocks; x += split, s = s + 1 == stages ? 0 : s + 1) {
        if ((s & 3) != warp) continue;
        if (!(ok = mbar_wait_w(&grant[s], (turns >> s) & 1))) break;
        turns ^= 1u << s;
        const int q = pack > 1 ? x * pack : x / kbe;
        const int some = pack > 1 ? min(pack, plan.cnt - q) : 1;
        uint8_t* sb = smem + s * stage_bytes + kBig;
        if (held) {
          for (int u = 0; u < some; ++u) {
#pragma unroll
            for (int k = 0; k < kHold; ++k)
              if (at[k] >= 0)
                *reinterpret_cast<uint4*>(sb + u * (n * 128 / pack) + (at[k] & 0xffff)) =
                    (at[k] >> 16) == q + u ? hold[k] : make_uint4(0, 0, 0, 0);
          }
        } else {
          // zeros, then only the tokens that use the adapter, their places by
          // ballots (256 tokens of 200 adapters of rank 32, 4096 x 4096: 95 us
          // when every block looked at every token, 63 now)
          const int k0 = pack > 1 ? 0 : (x - q * kbe) * 64;
          const int chunks = pack > 1 ? 8 / pack : min(8, (p.low_ld - k0) >> 3);
          uint8_t* mine = tokens_s[warp];
          for (int u = 0; u < some; ++u) {
            uint8_t* to = sb + u * (n * 128 / pack);
            int cnt = 0;
            for (int g = 0; g < n; g += 32) {
              const bool use = g + lane < cols && plan.slot[g + lane] == q + u;
              const uint32_t m = __ballot_sync(0xffffffffu, use);
              if (use) mine[cnt + __popc(m & ((1u << lane) - 1u))] = (uint8_t)(g + lane);
              cnt += __popc(m);
            }
#pragma unroll 4
            for (int i = lane; i < n * 8 / pack; i += 32)
              *reinterpret_cast<uint4*>(to + i * 16) = make_uint4(0, 0, 0, 0);
            __syncwarp();
            const int lg = chunks <= 2 ? 1 : chunks <= 4 ? 2 : 3;  // lanes a row, 16 bytes each
            const int c = lane & ((1 << lg) - 1);
#pragma unroll 8
            for (int i = lane >> lg; i < cnt; i += 32 >> lg) {
              const int j = mine[i];
              if (c < chunks)
                *reinterpret_cast<uint4*>(
                    to + (pack > 1 ? narrow_offset(j, c, 128 / pack) : sw128_offset(j, c))) =
                    *reinterpret_cast<const uint4*>(low + (int64_t)j * p.low_stride + k0 + c * 8);
            }
            __syncwarp();
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[s]);
      }
    }
    if (ok) ok = mbar_wait_w(done, 0);
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) drain_delay();
  if (split > 1) {
    cluster_wait();  // all have started
    if (exchange == 0) cluster_sync();  // and every ring is idle: its memory takes the sums
  }
  tc_fence_after();

  // columns of owner q: [q * own, (q + 1) * own); sums (split, own / 4, 128, 4)
  const int own = ((n + split - 1) / split + 3) & ~3;
  const int j0 = part * own, j1 = min(n, j0 + own);
  const int r = threadIdx.x;
  float* recv = reinterpret_cast<float*>(smem + exchange);
  const bool good = *abort_flag == 0;
  if (warp < 4 && good) {
    const uint32_t taddr = tmem + ((uint32_t)(warp * 32) << 16);
    const uint32_t mine = smem_u32(recv) + (uint32_t)(part * own * 512 + r * 16);
    int q = 0, at = 0;  // owner of the column, its place there
    uint32_t dst = split > 1 ? mapa(mine, 0) : mine;
    for (int c = 0; c < n; c += 16) {
      uint32_t v[16];
      tmem_ld16(taddr + c, v);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const uint32_t a = dst + (uint32_t)at * 512u;
        if (split > 1) st_cluster_v4(a, v[i], v[i + 1], v[i + 2], v[i + 3]);
        else
          *reinterpret_cast<uint4*>(recv + (c + i) * 128 + r * 4) =
              make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        at += 4;
        if (at == own && q + 1 < split) {
          at = 0;
          dst = mapa(mine, ++q);
        }
      }
    }
  }
  tc_fence_before();
  if (split > 1) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  if (warp == 5) {
    __syncwarp();
    tmem_dealloc(tmem, tmem_cols);
  }
  const int i = i0 + r;
  auto sum4 = [&](int j, float* acc) { sum_columns(recv, split, own, j - j0, r, acc); };
  if constexpr (OUT == kSkinnyCols) {
    // out[j, i], a column a token
    bool odd = false;  // a value of this row is not finite
    if (warp < 4 && good && i < rows) {
      const float bias = p.bias != nullptr ? __bfloat162float(p.bias[i]) : 0.f;
#pragma unroll 2
      for (int j = j0; j < min(j1, cols); j += 4) {
        float acc[4];
        sum4(j, acc);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (j + k >= cols) break;
          odd = odd || !isfinite(acc[k]);
          p.out[(int64_t)(j_base + j + k) * p.out_ld + i] = __float2bfloat16_rn(acc[k] + bias);
        }
      }
    }
    if (adapters && p.ids != nullptr && plan.cnt > 0 && warp < 4 && __any_sync(0xffffffffu, odd))
      repair_tokens(p, plan, recv, split, own, j0, min(j1, cols), j_base, i0);
  }
  if (warp < 4 && good && i < rows) {
    if constexpr (OUT == kSkinnyLow) {
      // out[i, j]: the columns of the row's own adapter, scaled, in bf16, the
      // operand type of the products that follow: one rounding of a term that
      // is added to the output's fp32 sum. The factors' gradients have no
      // other term, so they also multiply the remainders (16 bits in all; with
      // bf16 alone they were 2.4e-3 off, now 1.7e-3, their own rounding).
      const int sl = p.slot != nullptr ? p.slot[i] - s0 : 0;
      float sc = p.scale;
      if (p.scales != nullptr && sl >= 0 && sl < ns)
        sc = p.scales[p.list_ids[(int64_t)(i0 >> 8) * 256 + s0 + sl]];
      const int lo = max(j0, sl * p.low_ld), hi = min(j1, (sl + 1) * p.low_ld);
      if (sl >= 0 && sl < ns) {
        for (int j = lo; j < hi; j += 4) {  // (all bounds are multiples of 4)
          float acc[4];
          sum4(j, acc);
          const int jj = j - sl * p.low_ld;
          __nv_bfloat16* o = p.out + (int64_t)i * p.out_ld + jj;
          // behind the rank zeros, whatever the row holds (a zero factor times
          // an infinity is none)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[k] = jj + k < p.rank ? acc[k] * sc : 0.f;
          const uint2 v = make_uint2(pack_bf16(acc[0], acc[1]), pack_bf16(acc[2], acc[3]));
          *reinterpret_cast<uint2*>(o) = v;
          if (p.lo_at != 0) {
            const float d[4] = {remainder(acc[0], bf16_lo(v.x)), remainder(acc[1], bf16_hi(v.x)),
                                remainder(acc[2], bf16_lo(v.y)), remainder(acc[3], bf16_hi(v.y))};
            *reinterpret_cast<uint2*>(o + p.lo_at) =
                make_uint2(pack_bf16(d[0], d[1]), pack_bf16(d[2], d[3]));
          }
        }
      } else if (p.slot != nullptr && p.slot[i] < 0 && s0 == 0 && part == 0) {
        // a row without an adapter: zeros (a block whose other rows share one
        // adapter is multiplied whole)
        for (int j = 0; j < p.low_ld; ++j) p.out[(int64_t)i * p.out_ld + j] = __float2bfloat16_rn(0.f);
      }
    } else if constexpr (OUT == kSkinnyGrad) {
      __nv_bfloat16* out = which ? p.out2 : p.out;
      const int64_t ld = which ? p.out_ld2 : p.out_ld, lj = which ? p.out_j2 : p.out_j;
      for (int j = j0; j < min(j1, p.cols); j += 4) {
        float acc[4];
        sum4(j, acc);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (j + k < p.cols) out[(int64_t)(j + k) * lj + (int64_t)i * ld] = __float2bfloat16_rn(acc[k]);
      }
    }
  }
}

// Inner products of few rows with their own adapters: low[n, j] = s x[n] A_e[j].
// Four warps share one (a single token's 16 products of 4096 terms would keep
// one SM's warps alone at work for 4 us); columns [rank, low_ld) are zero.
__global__ void __launch_bounds__(256)
low_rows_kernel(const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* a, int64_t a_e,
                int64_t a_r, const int* ids, int E, const float* scales, float scale, int K,
                int rank, int low_ld, __nv_bfloat16* low, int64_t low_stride, int lo_at) {
  __shared__ float red[8];
  pdl_launch_next();
  const int groups = low_ld / 2;
  const int row = blockIdx.x / groups, j = (blockIdx.x - row * groups) * 2 + (warp_id() >> 2);
  const int t = threadIdx.x & 127;
  const int e = ids != nullptr ? ids[row] : 0;
  const bool has = e >= 0 && e < E && j < rank;
  float acc = 0.f;
  if (has) {
    const uint4* xr = reinterpret_cast<const uint4*>(x + (int64_t)row * ldx);
    const uint4* ar = reinterpret_cast<const uint4*>(a + (int64_t)e * a_e + (int64_t)j * a_r);
    const int nv = K >> 3;
#pragma unroll 4
    for (int i = t; i < nv; i += 128) {
      const uint4 u = __ldg(xr + i), v = __ldg(ar + i);
      const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        acc = fmaf(bf16_lo(uw[k]), bf16_lo(vw[k]), acc);
        acc = fmaf(bf16_hi(uw[k]), bf16_hi(vw[k]), acc);
      }
    }
    const int k = (nv << 3) + t;
    if (k < K)
      acc = fmaf(__bfloat162float(x[(int64_t)row * ldx + k]),
                 __bfloat162float(a[(int64_t)e * a_e + (int64_t)j * a_r + k]), acc);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane_id() == 0) red[warp_id()] = acc;
  __syncthreads();
  if (t == 0) {
    const float* s = red + (warp_id() & 4);
    acc = (s[0] + s[1]) + (s[2] + s[3]);
    acc = has ? acc * (scales != nullptr ? scales[e] : scale) : 0.f;
    const __nv_bfloat16 hi = __float2bfloat16_rn(acc);
    low[row * low_stride + j] = hi;
    if (lo_at != 0)
      low[row * low_stride + lo_at + j] = __float2bfloat16_rn(remainder(acc, __bfloat162float(hi)));
  }
}

__global__ void __launch_bounds__(256)
pad_rows_kernel(int64_t n, int cols, const uint16_t* src, int64_t ss, uint16_t* dst, int64_t ds) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t r = i / cols;
  const int c = (int)(i - r * cols);
  dst[r * ds + c] = src[r * ss + c];
}

// Per block of 256 rows: the distinct adapters in order of first use, and
// every row's place among them (-1: none).
__global__ void __launch_bounds__(256)
plan_kernel(const int* ids, int rows, int E, int* cnt, int* list, int* slot) {
  __shared__ int id_s[256], rank_s[256], warp_s[8];
  const int t = threadIdx.x, row = blockIdx.x * 256 + t;
  int id = row < rows ? ids[row] : -1;
  if (id < 0 || id >= E) id = -1;
  id_s[t] = id;
  __syncthreads();
  int first = 0;
  while (id_s[first] != id) ++first;  // ends at t
  const bool head = id >= 0 && first == t;
  const uint32_t m = __ballot_sync(0xffffffffu, head);
  if (lane_id() == 0) warp_s[warp_id()] = __popc(m);
  __syncthreads();
  int before = __popc(m & ((1u << lane_id()) - 1u)), total = 0;
  for (int w = 0; w < 8; ++w) {
    if (w < warp_id()) before += warp_s[w];
    total += warp_s[w];
  }
  rank_s[t] = before;
  __syncthreads();
  if (head) list[(int64_t)blockIdx.x * 256 + before] = id;
  if (row < rows) slot[row] = id < 0 ? -1 : rank_s[first];
  if (t == 0) cnt[blockIdx.x] = total;
}

template <bool BIG_MN, bool SMALL_MN, int OUT, int PACK = 1, int HOLD = 16>
static int go(const Maps<OUT>& maps, const SkinnyParams& p, int passes, int kernel_id, bool early,
              cudaStream_t st) {
  auto* fn = skinny_kernel<BIG_MN, SMALL_MN, OUT, PACK, HOLD>;
  const Layout l = layout_of(p.n, SMALL_MN, OUT == kSkinnyGrad);
  // the largest layout's request, once per kernel
  const int rc = ensure_smem_attr((const void*)fn, kOneSmem, kernel_id);
  if (rc) return rc;
  const int tiles = (std::max(p.rows, p.rows2) + 127) / 128;
  const int64_t work = OUT == kSkinnyGrad ? (p.rows + 127) / 128 + (p.rows2 + 127) / 128
                                          : (int64_t)tiles * passes;
  // K blocks, the requests' adapters' among them (as many as there may be)
  int kbs = (p.K + 63) / 64, most = kbs;
  if (OUT == kSkinnyCols && p.ids != nullptr)
    most += (std::min(p.E, p.n) + PACK - 1) / PACK * ((p.rank + 63) / 64);
  // contraction split: the one whose rounds of resident clusters times blocks
  // per CTA, longer ones where two CTAs share an SM, and some blocks' time for
  // start and exchange, is smallest (factors fitted to some 20 shapes). A wave
  // that spills over costs a whole round: with 72 clusters of 4 where 66 fit, 302
  // MB took 74 us; 64 x 4096 x 16384 with 48 adapters takes 46 us unsplit on 128
  // SMs, 38 as two per tile; the gradients at 4608 x 2560 x 2560 11 us split by
  // 6 over shared SMs, 15 by 3.
  // (The occupancy calculator takes a kernel with tensor memory to fill it, one
  // block an SM; two of at most 128 columns do run together.)
  const bool two = l.smem <= kTwoSmem;
  int split = 1;
  float best = 1e30f;
  for (int c = 1; c <= 8 && c <= kbs; ++c) {
    int fit = 0;
    const int rf = clusters_that_fit((const void*)fn, kThreads, two ? kTwoSmem : kOneSmem, c,
                                     kernel_id + (two ? 0 : kKernelSkinnyBig - kKernelSkinny), &fit);
    if (rf) return rf;
    if (fit <= 0) continue;
    if (two) fit *= 2;
    const int64_t rounds = (work + fit - 1) / fit;
    const bool sharing = two && std::min<int64_t>(work, fit) * c > 148;
    const float block = !sharing ? 1.f : OUT == kSkinnyCols ? 1.25f : 1.6f;
    const float cost = rounds * ((most + c - 1) / c * block + 2.f + (OUT == kSkinnyCols ? 1.f : 0.5f) * c);
    if (cost < best) best = cost, split = c;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * split), passes, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = l.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = early ? 2 : 1;
  const int bar_off = l.smem - kBarBytes - 1024;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, maps, p, split, l.stage, l.stages,
                                           bar_off, l.exchange, l.cols);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return record_cuda_error(e);
  }
  return launch_status();
}

}  // namespace skinny

template <bool BIG_MN, bool SMALL_MN, int OUT, int PACK = 1, int HOLD = 16>
static int launch(const Mat3& big, const Mat3& small, const Mat3& fac, const SkinnyParams& p,
                  int passes, int kernel_id, bool early, cudaStream_t st) {
  skinny::Maps<OUT> m;
  int rc = make_tmap_3d(&m.big[0], big, 64, BIG_MN ? 64 : 128);
  const int box = OUT == kSkinnyLow ? p.low_ld : p.n;
  if (!rc) rc = make_tmap_3d(&m.small[0], small, 64, SMALL_MN ? 64 : box);
  m.fac[0] = m.big[0];
  if (!rc && OUT == kSkinnyCols && p.low != nullptr)
    rc = make_tmap_3d(&m.fac[0], fac, 64 / PACK, BIG_MN ? 64 : 128);
  return rc ? rc : skinny::go<BIG_MN, SMALL_MN, OUT, PACK, HOLD>(m, p, passes, kernel_id, early, st);
}

int launch_gemm_skinny(const Mat3& big, bool big_mn, const Mat3& small, bool small_mn,
                       SkinnyParams p, int out, bool early, cudaStream_t st, const Mat3& fac) {
  if (p.rows == 0) return FA_OK;
  int passes = 1;
  if (out == kSkinnyCols) {  // even blocks of up to 256 tokens
    passes = (p.cols + kMaxColumns - 1) / kMaxColumns;
    p.n = ((p.cols + passes - 1) / passes + 15) / 16 * 16;
    passes = (p.cols + p.n - 1) / p.n;
  }
  if (out == kSkinnyLow && p.list_cnt != nullptr) {
    p.slots_per_pass = std::max(1, 128 / p.low_ld);
    const int most = std::min(p.E, 256);
    p.slots_per_pass = std::min(p.slots_per_pass, most);
    p.n = p.slots_per_pass * p.low_ld;
    passes = (most + p.slots_per_pass - 1) / p.slots_per_pass;
  }
  // requests' adapters of at most 32 ranks: packed; the builders' registers by
  // what they hold (64 x 4096 x 4096, rank 12: 16.2 us with 8, 17.2 with 16)
#define FA_PACK(PACK, HOLD, ID)                                                               \
  return launch<false, false, kSkinnyCols, PACK, HOLD>(big, small, fac, p, passes,            \
                                                       kKernelSkinnyPack + ID, early, st)
  if (out == kSkinnyCols && !big_mn && !small_mn && p.ids != nullptr && p.low_ld == 16) {
    if (p.n <= 128) FA_PACK(4, 8, 0);
    FA_PACK(4, 16, 1);
  }
  if (out == kSkinnyCols && !big_mn && !small_mn && p.ids != nullptr && p.low_ld == 32) {
    if (p.n <= 64) FA_PACK(2, 8, 2);
    FA_PACK(2, 16, 3);
  }
#undef FA_PACK
  if (out == kSkinnyCols && !big_mn && !small_mn)
    return launch<false, false, kSkinnyCols>(big, small, fac, p, passes, kKernelSkinny, early, st);
  if (out == kSkinnyCols && big_mn && !small_mn)
    return launch<true, false, kSkinnyCols>(big, small, fac, p, passes, kKernelSkinny + 1, early, st);
  if (out == kSkinnyLow && !big_mn && !small_mn)
    return launch<false, false, kSkinnyLow>(big, small, fac, p, passes, kKernelSkinny + 2, early, st);
  if (out == kSkinnyLow && !big_mn && small_mn)
    return launch<false, true, kSkinnyLow>(big, small, fac, p, passes, kKernelSkinny + 3, early, st);
  return FA_ERR_UNSUPPORTED;
}

int launch_skinny_grads(const Mat3* big, const Mat3* small, const Mat3* small_lo, SkinnyParams p,
                        cudaStream_t st) {
  skinny::Maps<kSkinnyGrad> m;
  for (int i = 0; i < 2; ++i) {
    int rc = make_tmap_3d(&m.big[i], big[i], 64, 64);
    if (!rc) rc = make_tmap_3d(&m.small[i], small[i], 64, 64);
    if (!rc) rc = make_tmap_3d(&m.fac[i], small_lo[i], 64, 64);
    if (rc) return rc;
  }
  return skinny::go<true, true, kSkinnyGrad>(m, p, 2, kKernelSkinny + 4, true, st);
}

// Estimated microseconds of a linear as token columns: rounds of resident CTAs
// times K blocks of tensor work (0.45 us at 256 columns, shared by the CTAs of
// an SM, 0.19 us at least), no less than the weight's way from memory; and
// what does not depend on K: start, exchange, output. Within 20 percent of
// 88 measured shapes (65 to 2048 rows, 1024 to 16384 wide).
static float cols_time(int64_t out, int64_t K, int rows) {
  const int blocks = (rows + kMaxColumns - 1) / kMaxColumns;
  const int n = ((rows + blocks - 1) / blocks + 15) / 16 * 16;
  const int64_t tiles = (out + 127) / 128 * blocks, kbs = (K + 63) / 64;
  const int per_sm = n <= 128 ? 2 : 1;
  const float kb = std::max(0.45f * n / 256.f, 0.19f) * per_sm;
  float best = 1e30f;
  for (int c = 1; c <= 8 && c <= kbs; ++c) {
    const int fit = per_sm * (c <= 2 ? 148 : (c <= 4 ? 132 : 120)) / c;
    const int64_t rounds = (tiles + fit - 1) / fit;
    best = std::min(best, rounds * (((kbs + c - 1) / c) * kb + 7.5f * n / 256.f));
  }
  return std::max(best, (float)(out * K * 2) / 6e6f) + 7.f;
}

// The same as 256 x 256 tiles of the pair form: 0.29 us a K block, 7 us apart.
static float wide_time(int64_t out, int64_t K, int rows) {
  const int64_t tiles = (int64_t)((rows + 255) / 256) * ((out + 255) / 256), kbs = (K + 63) / 64;
  return 7.f + (tiles + 73) / 74 * kbs * 0.29f;
}

// Few 256 x 256 tiles leave SM pairs idle, where token columns split the
// contraction over clusters (256 rows, 16384 -> 4096: 42 us against 82); many
// fill them at half the staged bytes (512 rows, 4096 -> 16384: 97 against 52).
// Up to 256 rows of requests may use as many adapters as there are, each a K
// block that one warp of a pair builds (1 us, 2.5 beyond rank 32) and that
// columns split over a cluster's CTAs and their four warps (128 rows of 14
// adapters of rank 64 at 408 x 920: 50 us as pairs, 25 as columns).
bool linear_as_columns(int64_t out, int64_t K, int rows, int adapters, int rank) {
  if (rows > kMaxColumns * 65535) return false;  // a block of tokens a grid row
  float wide = wide_time(out, K, rows), cols = cols_time(out, K, rows);
  if (rows <= kMaxColumns) {
    const int blocks = std::min(adapters, rows) * ((rank + 63) / 64);
    wide += blocks * (rank <= 32 ? 1.f : 2.5f);
    cols += blocks * 0.3f;
  }
  return rows <= 64 || cols < wide;
}

int launch_low_rows(const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* a, int64_t a_e,
                    int64_t a_r, const int* ids, int E, const float* scales, float scale, int rows,
                    int K, int rank, int low_ld, __nv_bfloat16* low, int64_t low_stride, int lo_at,
                    cudaStream_t st) {
  skinny::low_rows_kernel<<<(unsigned)(rows * (low_ld / 2)), 256, 0, st>>>(
      x, ldx, a, a_e, a_r, ids, E, scales, scale, K, rank, low_ld, low, low_stride, lo_at);
  return launch_status();
}

int launch_pad_rows(int64_t rows, int cols, const void* src, int64_t src_stride, void* dst,
                    int64_t dst_stride, cudaStream_t st) {
  const int64_t n = rows * cols;
  skinny::pad_rows_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
      n, cols, reinterpret_cast<const uint16_t*>(src), src_stride,
      reinterpret_cast<uint16_t*>(dst), dst_stride);
  return launch_status();
}

int launch_adapter_plan(const int* ids, int rows, int E, int* cnt, int* list, int* slot,
                        cudaStream_t st) {
  skinny::plan_kernel<<<(unsigned)((rows + 255) / 256), 256, 0, st>>>(ids, rows, E, cnt, list, slot);
  return launch_status();
}

int skinny_device_status() { return tu_device_status(); }

}  // namespace fa
