// Gradient of the packed (cu_seqlens-confined) attention, head dim 64, on the sm_100a tensor cores.
//
// With s_ij = q_i k_j / 8 and p_ij = exp(s_ij - lse_i) for the keys j that query i attends, and
// delta_i = sum_d dout_id out_id (which equals sum_j p_ij dP_ij):
//   dP_ij = dout_i v_j      dS_ij = p_ij (dP_ij - delta_i)
//   dv_j = sum_i p_ij dout_i      dk_j = sum_i dS_ij q_i / 8      dq_i = sum_j dS_ij k_j / 8
// The probabilities are recomputed from lse, so nothing of size T x T is ever stored.
//
// Two passes, both with one accumulating owner per output row and therefore without atomics:
// repeated calls give the same bits.
//   key pass   : a tile of 128 keys (rows) walks the queries (columns): S^T = K Q^T and
//                dP^T = V dO^T, then dV += P^T dO and dK += dS^T Q
//   query pass : a tile of 128 queries (rows) walks the keys (columns): S = Q K^T and dP = dO V^T,
//                then dQ += dS K
// Either way a thread owns one row of the score tile, the second products read P and dS straight
// from tensor memory (the A operand of tcgen05.mma), and no score ever passes through shared
// memory.  The price against one pass that would add dQ tiles into global memory is a second S, dP
// and exponential (seven products instead of five); what it buys is a fixed summation order and
// no fp32 dQ buffer: that one pass moves 32 KB of fp32 additions through L2 per tile of 1,280
// tensor clocks, 25 B per clock and SM, more than L2 takes.
//
// Rows are tiled over the packed tokens, not per sequence: a tile of 128 consecutive tokens may
// hold many sequences.  Row i attends the columns [lo_i, hi_i) - its sequence, cut to the window -
// and the relation is symmetric, so the same two numbers serve both passes.  A batch of 30-token
// queries then costs one 128-column tile per four queries instead of one each.  A tile walks the
// columns [min lo, max hi) of its rows; its last column tile ends exactly at max hi (it overlaps the
// one before, whose columns are masked out there), so rows behind the last sequence are never
// fetched as columns and whatever they hold cannot reach a gradient.
#include <algorithm>

#include "attn_tmem.cuh"
#include "pe_host.h"
#include "pe_ptx.cuh"
#include "pe_vec.cuh"

namespace pe {

constexpr int BW_COMPUTE_WARPS = 8;
constexpr int BW_THREADS = 32 * (BW_COMPUTE_WARPS + 2);
constexpr int BW_TILE = 128;
constexpr int BW_TILE_BYTES = BW_TILE * 64 * 2;  // one 128 x 64 bf16 tile
constexpr int BW_STAGES = 4;                     // column tiles in flight: (Q, dO) or (K, V)
constexpr int BW_STATS_BYTES = 2 * BW_TILE * 4;  // lse and delta of 128 columns
constexpr uint32_t BW_TMEM_COLS = 512;
constexpr uint32_t BW_S_COL = 0;      // S: two buffers of 128 columns; P in place (bf16 pairs)
constexpr uint32_t BW_DP_COL = 256;   // dP: 128 columns; dS in place
constexpr uint32_t BW_ACC1_COL = 384; // dK or dQ
constexpr uint32_t BW_ACC2_COL = 448; // dV

// Barriers of one pass; each pass has its own set.
enum {
  WB_FULL = 0,        // BW_STAGES
  WB_EMPTY = 4,       // BW_STAGES
  WB_A_FULL = 8,      // 2
  WB_A_EMPTY = 10,    // 2
  WB_S_FULL = 12,     // 2
  // 2 (tile parity), one arrival per compute warp: P written (key pass) / S read (query pass).  Two,
  // because a warp may be done with the scores of tile g + 1 before another is with those of tile g.
  WB_P_FULL = 14,
  WB_DP_FULL = 16,
  WB_DS_FULL = 17,    // one arrival per compute warp
  WB_DV_DONE = 18,
  WB_DK_DONE = 19,    // dK (or dQ) of a tile has retired
  WB_ACC_EMPTY = 20,  // one arrival per compute warp: the item's accumulators have been read
  WB_COUNT = 21
};
constexpr int BW_BAR_OFFSET = (4 + 2 * BW_STAGES) * BW_TILE_BYTES + BW_STAGES * BW_STATS_BYTES;
constexpr int BW_SMEM = BW_BAR_OFFSET + 2 * WB_COUNT * 8 + 16;

struct BwArgs {
  const int2* row_range;    // [T]: columns [x, y) that row t attends
  const int2* tile_range;   // [tiles]: their union over a tile of 128 rows
  const float* lse2;        // [nh, T]: lse * log2(e)
  const float* delta;       // [nh, T]
  __nv_bfloat16* dqkv;      // [T, 3 nh 64]
  const int64_t* pos;       // [T] or NULL: rotation of q and k undone on dq and dk
  const __nv_bfloat16* table;
  int max_positions;
  int T, nh, n_items;
  int* status;
};

// ---- preparation ------------------------------------------------------------------
// Grid (tiles, heads), 256 threads.  Every block: delta of its 128 rows and head, eight lanes per
// row, and lse in the exponent's base.  Blocks of head 0 also find each row's sequence and window.
// Boundaries are not trusted: a row whose sequence does not come out as begin <= t < end within
// [0, T] attends nothing, and an entry outside [0, T] or below its predecessor is reported.
__global__ void __launch_bounds__(256)
attn_bwd_prepare_kernel(const __nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ dout,
                        const float* __restrict__ lse, const int32_t* __restrict__ cu_seqlens, int n_seqs,
                        int T, int nh, int half_window, int2* __restrict__ row_range,
                        int2* __restrict__ tile_range, float* __restrict__ lse2, float* __restrict__ delta,
                        int* status) {
  const int tile = blockIdx.x, head = blockIdx.y;
  const int H = nh * 64;
  const int sub = threadIdx.x & 7;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = tile * BW_TILE + i * 32 + (threadIdx.x >> 3);
    float acc = 0.f;
    if (t < T) {
      const int64_t at = int64_t(t) * H + head * 64 + sub * 8;
      float a[8], b[8];
      unpack8(*reinterpret_cast<const uint4*>(out + at), a);
      unpack8(*reinterpret_cast<const uint4*>(dout + at), b);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc = fmaf(a[e], b[e], acc);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (t < T && sub == 0) {
      const int64_t at = int64_t(head) * T + t;
      delta[at] = acc;
      lse2[at] = lse[at] * 1.4426950408889634f;
    }
  }
  if (head != 0) return;
  for (int n = blockIdx.x * blockDim.x + threadIdx.x; n < n_seqs; n += gridDim.x * blockDim.x) {
    const int b = cu_seqlens[n], e = cu_seqlens[n + 1];
    if (b < 0 || e < b || e > T) set_status(status, ST_BAD_CU_SEQLENS);
  }
  __shared__ int s_lo[4], s_hi[4];
  if (threadIdx.x < BW_TILE) {
    const int t = tile * BW_TILE + threadIdx.x;
    int lo = INT_MAX, hi = 0;
    if (t < T) {
      int a = 0, b = n_seqs;  // the last n in [0, n_seqs) with cu_seqlens[n] <= t, if any
      while (b - a > 1) {
        const int mid = (a + b) >> 1;
        if (__ldg(cu_seqlens + mid) <= t) a = mid;
        else b = mid;
      }
      const int begin = max(__ldg(cu_seqlens + a), 0), end = min(__ldg(cu_seqlens + a + 1), T);
      int2 r = make_int2(t, t);
      if (begin <= t && t < end) {
        r.x = half_window >= 0 && half_window < t - begin ? t - half_window : begin;
        r.y = half_window >= 0 && half_window < end - 1 - t ? t + half_window + 1 : end;
        lo = r.x;
        hi = r.y;
      }
      row_range[t] = r;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if ((threadIdx.x & 31) == 0) {
      s_lo[threadIdx.x >> 5] = lo;
      s_hi[threadIdx.x >> 5] = hi;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int lo = min(min(s_lo[0], s_lo[1]), min(s_lo[2], s_lo[3]));
    const int hi = max(max(s_hi[0], s_hi[1]), max(s_hi[2], s_hi[3]));
    tile_range[tile] = lo < hi ? make_int2(lo, hi) : make_int2(0, 0);
  }
}

// ---- the two passes -----------------------------------------------------------------

// A cursor over the column tiles of this CTA's items.  Item = (row tile, head), head fastest.
struct BwCursor {
  int item, ord;  // item and how many items this CTA began before it
  int j, n;       // column tile and how many the item has (at least one: an empty item runs one, masked)
  int lo, hi;     // columns of the row tile
  __device__ __forceinline__ void open(const BwArgs& a) {
    if (item >= a.n_items) return;
    const int2 r = __ldg(a.tile_range + item / a.nh);
    lo = r.x;
    hi = r.y;
    j = 0;
    n = max((hi - lo + BW_TILE - 1) / BW_TILE, 1);
  }
  __device__ __forceinline__ void start(const BwArgs& a, int first) {
    item = first;
    ord = 0;
    open(a);
  }
  __device__ __forceinline__ bool valid(const BwArgs& a) const { return item < a.n_items; }
  __device__ __forceinline__ void advance(const BwArgs& a) {
    if (++j == n) {
      item += gridDim.x;
      ++ord;
      open(a);
    }
  }
  // first column of tile j: the last tile ends at hi (it may start below zero: filled, then masked)
  __device__ __forceinline__ int col0() const { return j + 1 == n ? hi - BW_TILE : lo + j * BW_TILE; }
};

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float4 lds128(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}

// Stores 64 gradient values of one row as bf16, after undoing the rotation of its position if a
// table is given (the transpose of the rotation applied to q and k).
__device__ __forceinline__ void bw_store_row(const BwArgs& a, int t, bool empty, bool rotated, float scale,
                                             const uint32_t (&lo)[32], const uint32_t (&hi)[32],
                                             __nv_bfloat16* dst) {
  const uint4* trow = nullptr;
  if (rotated) {
    int64_t p = a.pos[t];
    if (p < 0 || p >= a.max_positions) {
      set_status(a.status, ST_BAD_POSITION);
      p = 0;
    }
    trow = reinterpret_cast<const uint4*>(a.table + p * 64);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = __uint_as_float(lo[c * 8 + e]) * scale;
      y[e] = __uint_as_float(hi[c * 8 + e]) * scale;
    }
    if (rotated) {
      float cs[8], sn[8];
      unpack8(__ldg(trow + c), cs);
      unpack8(__ldg(trow + 4 + c), sn);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float u = x[e], w = y[e];
        x[e] = fmaf(u, cs[e], w * sn[e]);
        y[e] = fmaf(w, cs[e], -(u * sn[e]));
      }
    }
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(dst + c * 8) = empty ? zero : pack8(x);
    *reinterpret_cast<uint4*>(dst + 32 + c * 8) = empty ? zero : pack8(y);
  }
}

// KEYS: the key pass (rows are keys, columns are queries), else the query pass.  `first` is this
// CTA's first item.  Returns false if a bounded wait gave up.
template <bool KEYS>
__device__ __forceinline__ bool bw_pass(const CUtensorMap& tm_qkv, const CUtensorMap& tm_dout, const BwArgs& a,
                                        int first, uint32_t base, uint32_t bar_base, uint32_t tmem_base) {
  auto bar = [&](int i) { return bar_base + 8u * i; };
  const uint32_t sA = base;                                // A[buffer]: (K, V) or (Q, dO)
  const uint32_t sB = base + 4 * BW_TILE_BYTES;            // B[stage]: (Q, dO) or (K, V)
  const uint32_t sStats = sB + 2 * BW_STAGES * BW_TILE_BYTES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = a.nh * 64;
  int* status = a.status;
  bool ok = true;

  if (warp == BW_COMPUTE_WARPS) {
    // ---------------------------------------------------------------- producer
    BwCursor c;
    c.start(a, first);
    uint32_t g = 0;
    while (c.valid(a)) {
      const int row0 = (c.item / a.nh) * BW_TILE, head = c.item % a.nh;
      if (c.j == 0) {
        const uint32_t ab = c.ord & 1;
        if (!mbar_wait(bar(WB_A_EMPTY + ab), ((c.ord >> 1) & 1) ^ 1u, status, ST_ATTN_TIMEOUT)) { ok = false; break; }
        if (lane == 0) {
          const uint32_t dst = sA + ab * 2 * BW_TILE_BYTES;
          mbar_expect_tx(bar(WB_A_FULL + ab), 2 * BW_TILE_BYTES);
          tma_load_2d(dst, &tm_qkv, bar(WB_A_FULL + ab), (KEYS ? H : 0) + head * 64, row0);
          if (KEYS) tma_load_2d(dst + BW_TILE_BYTES, &tm_qkv, bar(WB_A_FULL + ab), 2 * H + head * 64, row0);
          else tma_load_2d(dst + BW_TILE_BYTES, &tm_dout, bar(WB_A_FULL + ab), head * 64, row0);
        }
        __syncwarp();
      }
      const uint32_t st = g % BW_STAGES;
      if (!mbar_wait(bar(WB_EMPTY + st), ((g / BW_STAGES) & 1) ^ 1u, status, ST_ATTN_TIMEOUT)) { ok = false; break; }
      const int col0 = c.col0();
      if (KEYS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int q = min(max(col0 + i * 32 + lane, 0), a.T - 1);
          const int64_t at = int64_t(head) * a.T + q;
          const uint32_t dst = sStats + st * BW_STATS_BYTES + (i * 32 + lane) * 4;
          cp_async4(dst, a.lse2 + at);
          cp_async4(dst + BW_TILE * 4, a.delta + at);
        }
        cp_async_arrive(bar(WB_FULL + st));
      }
      if (lane == 0) {
        const uint32_t dst = sB + st * 2 * BW_TILE_BYTES;
        mbar_expect_tx(bar(WB_FULL + st), 2 * BW_TILE_BYTES);
        tma_load_2d(dst, &tm_qkv, bar(WB_FULL + st), (KEYS ? 0 : H) + head * 64, col0);
        if (KEYS) tma_load_2d(dst + BW_TILE_BYTES, &tm_dout, bar(WB_FULL + st), head * 64, col0);
        else tma_load_2d(dst + BW_TILE_BYTES, &tm_qkv, bar(WB_FULL + st), 2 * H + head * 64, col0);
      }
      __syncwarp();
      ++g;
      c.advance(a);
    }
    if (!ok) {  // gave up: this CTA's copies must have landed before it can leave
      for (uint32_t u = g > BW_STAGES ? g - BW_STAGES : 0; u < g; ++u)
        mbar_wait(bar(WB_FULL + u % BW_STAGES), (u / BW_STAGES) & 1, status, ST_ATTN_TIMEOUT);
      if (c.ord > 0) mbar_wait(bar(WB_A_FULL + ((c.ord - 1) & 1)), ((c.ord - 1) >> 1) & 1, status, ST_ATTN_TIMEOUT);
    }
  } else if (warp == BW_COMPUTE_WARPS + 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, 128, 0);
      constexpr uint32_t idesc_acc = umma_idesc_bf16(128, 64, 1);  // B is MN-major: its rows are the contraction
      BwCursor sc, dc, mc;  // scores, dP, accumulation
      sc.start(a, first);
      dc = sc;
      mc = sc;
      uint32_t gs = 0, gd = 0, g = 0;
      auto wait = [&](int b, uint32_t parity) {
        if (ok && !mbar_wait(bar(b), parity, status, ST_ATTN_MMA_TIMEOUT)) ok = false;
        return ok;
      };
      auto scores = [&](uint32_t d_col, uint32_t a_tile, uint32_t b_tile) {
        const uint64_t ad = umma_smem_desc_sw128(a_tile, 1024), bd = umma_smem_desc_sw128(b_tile, 1024);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_ss(tmem_base + d_col, ad + 2u * kk, bd + 2u * kk, idesc_s, kk != 0 ? 1u : 0u);
      };
      // acc += X B, X (bf16 pairs of 128 columns) in tensor memory: the two halves of a tile were
      // written by different warps, each in place over its own 64 fp32 columns
      auto accumulate = [&](uint32_t acc_col, uint32_t x_col, uint32_t b_tile, bool first_tile) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          g_umma_ts(tmem_base + acc_col, tmem_base + x_col + (kk >> 2) * 64 + (kk & 3) * 8,
                    umma_smem_desc_sw128(b_tile + kk * 2048, 1024), idesc_acc, (!first_tile || kk != 0) ? 1u : 0u);
      };
      auto issue_s = [&]() {
        const uint32_t st = gs % BW_STAGES;
        if (sc.j == 0 && !wait(WB_A_FULL + (sc.ord & 1), (sc.ord >> 1) & 1)) return;
        if (!wait(WB_FULL + st, (gs / BW_STAGES) & 1)) return;
        tc_fence_after();
        scores(BW_S_COL + (gs & 1) * 128, sA + (sc.ord & 1) * 2 * BW_TILE_BYTES, sB + st * 2 * BW_TILE_BYTES);
        umma_commit(bar(WB_S_FULL + (gs & 1)));
        ++gs;
        sc.advance(a);
      };
      auto issue_dp = [&]() {  // its operands arrived with those of the scores of the same tile
        const uint32_t st = gd % BW_STAGES;
        scores(BW_DP_COL, sA + ((dc.ord & 1) * 2 + 1) * BW_TILE_BYTES, sB + (st * 2 + 1) * BW_TILE_BYTES);
        umma_commit(bar(WB_DP_FULL));
        if (dc.j + 1 == dc.n) umma_commit(bar(WB_A_EMPTY + (dc.ord & 1)));
        ++gd;
        dc.advance(a);
      };
      if (sc.valid(a)) {
        issue_s();
        if (ok) issue_dp();
        if (ok && sc.valid(a)) issue_s();
      }
      while (ok && mc.valid(a)) {
        const uint32_t st = g % BW_STAGES;
        const uint32_t b1 = sB + st * 2 * BW_TILE_BYTES, b2 = b1 + BW_TILE_BYTES;
        if (!wait(WB_P_FULL + (g & 1), (g >> 1) & 1)) break;
        // the previous item's accumulators must have been read before they are overwritten
        if (mc.j == 0 && mc.ord > 0 && !wait(WB_ACC_EMPTY, (mc.ord - 1) & 1)) break;
        tc_fence_after();
        if (KEYS) {
          accumulate(BW_ACC2_COL, BW_S_COL + (g & 1) * 128, b2, mc.j == 0);  // dV += P^T dO
          umma_commit(bar(WB_DV_DONE));
        } else if (sc.valid(a)) {
          issue_s();  // the scores of tile g are in registers: its buffer takes those of tile g + 2
        }
        if (!wait(WB_DS_FULL, g & 1)) break;
        tc_fence_after();
        accumulate(BW_ACC1_COL, BW_DP_COL, b1, mc.j == 0);  // dK += dS^T Q, dQ += dS K
        umma_commit(bar(WB_EMPTY + st));
        umma_commit(bar(WB_DK_DONE));
        if (KEYS && sc.valid(a)) {
          if (!wait(WB_DV_DONE, g & 1)) break;  // P of tile g has been read: its buffer is free
          issue_s();
        }
        if (ok && dc.valid(a)) {
          if (!wait(WB_DK_DONE, g & 1)) break;  // dS of tile g has been read
          issue_dp();
        }
        ++g;
        mc.advance(a);
      }
    }
    __syncwarp();
    ok = __all_sync(0xffffffffu, ok);
  } else {
    // ---------------------------------------------------------------- compute warps
    const int half = warp >> 2;                      // which 64 columns of a tile
    const int row = (warp & 3) * 32 + lane;          // row of the tile = tensor-memory lane
    const uint32_t lane_addr = tmem_base + (uint32_t((warp & 3) * 32) << 16);
    const float scale_log2 = 0.125f * 1.4426950408889634f;  // 1/sqrt(64) * log2(e)
    // After a bounded wait has given up the loops still run to their end, without waiting, so that
    // every thread reaches the common exit.
    auto wait = [&](int b, uint32_t parity) {
      if (ok && !mbar_wait(bar(b), parity, status, ST_ATTN_SOFTMAX_TIMEOUT)) ok = false;
    };
    BwCursor c;
    c.start(a, first);
    uint32_t g = 0;
    while (c.valid(a)) {
      const int head = c.item % a.nh;
      const int t = (c.item / a.nh) * BW_TILE + row;
      int2 range = make_int2(0, 0);
      float lse_row = 0.f, delta_row = 0.f;
      if (t < a.T) {
        range = __ldg(a.row_range + t);
        if (!KEYS) {
          lse_row = __ldg(a.lse2 + int64_t(head) * a.T + t);
          delta_row = __ldg(a.delta + int64_t(head) * a.T + t);
        }
      }
      const int n = c.n;
      for (int j = 0; j < n; ++j, ++g) {
        const uint32_t st = g % BW_STAGES;
        const uint32_t s_addr = lane_addr + BW_S_COL + (g & 1) * 128 + half * 64;
        const uint32_t dp_addr = lane_addr + BW_DP_COL + half * 64;
        const uint32_t stats = sStats + st * BW_STATS_BYTES + half * 256;
        // valid columns of this row within its 64: [c_lo, c_hi)
        const int x0 = c.col0() + half * 64;
        const int c_lo = max(range.x, c.lo + j * BW_TILE) - x0, c_hi = range.y - x0;
        const bool full = __all_sync(0xffffffffu, c_lo <= 0 && c_hi >= 64);
        if (KEYS) wait(WB_FULL + st, (g / BW_STAGES) & 1);  // lse and delta of the columns
        wait(WB_S_FULL + (g & 1), (g >> 1) & 1);
        tc_fence_after();
        uint32_t p[64];
        g_tmem_ld32(s_addr, p);
        g_tmem_ld32(s_addr + 32, p + 32);
        tmem_ld_wait();
        if (!KEYS) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(WB_P_FULL + (g & 1)));
        }
        const float2 scale2 = make_float2(scale_log2, scale_log2);
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          float4 l;
          if (KEYS) l = lds128(stats + e * 4);
          else l = make_float4(lse_row, lse_row, lse_row, lse_row);
          const float2 u = __ffma2_rn(make_float2(__uint_as_float(p[e]), __uint_as_float(p[e + 1])), scale2,
                                      make_float2(-l.x, -l.y));
          const float2 w = __ffma2_rn(make_float2(__uint_as_float(p[e + 2]), __uint_as_float(p[e + 3])), scale2,
                                      make_float2(-l.z, -l.w));
          p[e] = __float_as_uint(g_ex2(u.x));
          p[e + 1] = __float_as_uint(g_ex2(u.y));
          p[e + 2] = __float_as_uint(g_ex2(w.x));
          p[e + 3] = __float_as_uint(g_ex2(w.y));
        }
        if (!full) {
#pragma unroll
          for (int e = 0; e < 64; ++e) p[e] = (e >= c_lo && e < c_hi) ? p[e] : 0u;
        }
        if (KEYS) {  // P^T back in place, as the A operand of dV += P^T dO
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              pk[e] = pack_bf16(__uint_as_float(p[h * 32 + 2 * e]), __uint_as_float(p[h * 32 + 2 * e + 1]));
            g_tmem_st16(s_addr + h * 16, pk);
          }
          g_tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(WB_P_FULL + (g & 1)));
        }
        wait(WB_DP_FULL, g & 1);
        tc_fence_after();
        uint32_t dp[64];
        g_tmem_ld32(dp_addr, dp);
        g_tmem_ld32(dp_addr + 32, dp + 32);
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            float4 dl;
            if (KEYS) dl = lds128(stats + BW_TILE * 4 + (h * 32 + e) * 4);
            else dl = make_float4(delta_row, delta_row, delta_row, delta_row);
            const uint32_t* d = dp + h * 32 + e;
            const uint32_t* q = p + h * 32 + e;
            const float2 u = __fmul2_rn(__fadd2_rn(make_float2(__uint_as_float(d[0]), __uint_as_float(d[1])),
                                                   make_float2(-dl.x, -dl.y)),
                                        make_float2(__uint_as_float(q[0]), __uint_as_float(q[1])));
            const float2 w = __fmul2_rn(__fadd2_rn(make_float2(__uint_as_float(d[2]), __uint_as_float(d[3])),
                                                   make_float2(-dl.z, -dl.w)),
                                        make_float2(__uint_as_float(q[2]), __uint_as_float(q[3])));
            pk[e / 2] = pack_bf16(u.x, u.y);
            pk[e / 2 + 1] = pack_bf16(w.x, w.y);
          }
          g_tmem_st16(dp_addr + h * 16, pk);
        }
        g_tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(WB_DS_FULL));
        c.advance(a);
      }
      // The item's accumulators.  Key pass: warps 0..3 store dV, warps 4..7 dK.  Query pass: warps
      // 0..3 store dQ.  Rows that attend nothing are exact zeros.
      wait(WB_DK_DONE, (g - 1) & 1);
      tc_fence_after();
      uint32_t lo[32], hi[32];
      const bool mine = KEYS || half == 0;
      const bool is_v = KEYS && half == 0;
      if (mine) {
        const uint32_t acc = lane_addr + (is_v ? BW_ACC2_COL : BW_ACC1_COL);
        g_tmem_ld32(acc, lo);
        g_tmem_ld32(acc + 32, hi);
        tmem_ld_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(WB_ACC_EMPTY));
      if (mine && ok && t < a.T)
        bw_store_row(a, t, range.x >= range.y, a.pos != nullptr && !is_v, is_v ? 1.0f : 0.125f, lo, hi,
                     a.dqkv + int64_t(t) * 3 * H + (KEYS ? (is_v ? 2 * H : H) : 0) + head * 64);
    }
  }
  return ok;
}

__global__ void __launch_bounds__(BW_THREADS, 1)
attn_bwd_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_dout,
                const BwArgs a) {
  extern __shared__ __align__(1024) uint8_t bw_smem[];
  const uint32_t base = smem_u32(bw_smem);
  if (base & 1023u) {  // the swizzled tiles need it; nothing has been allocated yet
    if (threadIdx.x == 0) set_status(a.status, ST_ATTN_SMEM_MISALIGNED);
    return;
  }
  const uint32_t bar_base = base + BW_BAR_OFFSET;
  const uint32_t tmem_slot = bar_base + 2 * WB_COUNT * 8;
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int pass = 0; pass < 2; ++pass) {
      const uint32_t bb = bar_base + pass * WB_COUNT * 8;
      for (int i = 0; i < WB_COUNT; ++i) {
        uint32_t count = 1;
        // stages of the key pass: the TMA issue and 32 lanes' copies of lse and delta
        if (pass == 0 && i >= WB_FULL && i < WB_FULL + BW_STAGES) count = 33;
        if (i == WB_P_FULL || i == WB_P_FULL + 1 || i == WB_DS_FULL || i == WB_ACC_EMPTY) count = BW_COMPUTE_WARPS;
        mbar_init(bb + 8u * i, count);
      }
    }
    mbar_fence_init();
    tma_prefetch_desc(&tm_qkv);
    tma_prefetch_desc(&tm_dout);
  }
  if (warp == BW_COMPUTE_WARPS + 1) {
    tmem_alloc(tmem_slot, BW_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem_base;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));

  // Items of both passes form one list, the key pass first; a CTA takes every gridDim-th of it, so
  // the passes need no launch boundary and a small batch runs both at the same time.
  const bool ok = bw_pass<true>(tm_qkv, tm_dout, a, blockIdx.x, base, bar_base, tmem_base);
  tc_fence_before();
  const int failed = __syncthreads_or(!ok);
  tc_fence_after();
  if (!failed) {
    int first = int(blockIdx.x) - a.n_items % int(gridDim.x);
    if (first < 0) first += gridDim.x;
    bw_pass<false>(tm_qkv, tm_dout, a, first, base, bar_base + WB_COUNT * 8, tmem_base);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == BW_COMPUTE_WARPS + 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, BW_TMEM_COLS);
  }
}

// Workspace: row_range int2[T], tile_range int2[tiles], lse2 and delta float[nh, T], each part
// rounded up to 256 bytes.
struct BwWorkspace {
  size_t row_range, tile_range, lse2, delta, total;
};
static BwWorkspace bw_workspace(int64_t T, int nh) {
  BwWorkspace w;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off += (bytes + 255) & ~size_t(255);
    return o;
  };
  w.row_range = take(size_t(T) * sizeof(int2));
  w.tile_range = take(size_t((T + BW_TILE - 1) / BW_TILE) * sizeof(int2));
  w.lse2 = take(size_t(T) * nh * sizeof(float));
  w.delta = take(size_t(T) * nh * sizeof(float));
  w.total = off;
  return w;
}

}  // namespace pe

extern "C" size_t pe_attn_backward_workspace_bytes(int64_t T, int nh) {
  if (T < 0 || nh <= 0) return 0;
  return pe::bw_workspace(T, nh).total;
}

extern "C" int pe_attn_varlen_backward(const void* dout, const void* qkv, const void* out, const float* lse,
                                       const int32_t* cu_seqlens, int n_seqs, int64_t T, int nh,
                                       int half_window, const int64_t* position_ids, const void* table,
                                       int max_positions, void* dqkv, void* workspace,
                                       size_t workspace_bytes, int32_t* status, void* stream) {
  using namespace pe;
  PE_REQUIRE(dout && qkv && out && lse && cu_seqlens && dqkv && workspace, "pe_attn_varlen_backward: null pointer");
  PE_REQUIRE(n_seqs > 0 && nh > 0 && nh <= 65535 && T >= 0 && T < (1ll << 31) - 256,
             "pe_attn_varlen_backward: %lld tokens / %d sequences / %d heads out of range", (long long)T, n_seqs, nh);
  PE_REQUIRE((table == nullptr) == (position_ids == nullptr) && (table == nullptr || max_positions > 0),
             "pe_attn_varlen_backward: position_ids and table come together");
  PE_REQUIRE(((uintptr_t)workspace & 15) == 0 && ((uintptr_t)dqkv & 15) == 0 && ((uintptr_t)out & 15) == 0 &&
                 ((uintptr_t)table & 15) == 0,
             "pe_attn_varlen_backward: pointers must be 16-byte aligned");
  const int64_t tiles = (T + BW_TILE - 1) / BW_TILE;
  PE_REQUIRE(tiles * nh < (1ll << 31) - 65536, "pe_attn_varlen_backward: %lld tokens x %d heads are too many tiles",
             (long long)T, nh);
  const BwWorkspace w = bw_workspace(T, nh);
  if (workspace_bytes < w.total) {
    set_last_error("pe_attn_varlen_backward: workspace %zu < %zu bytes", workspace_bytes, w.total);
    return PE_ERR_WORKSPACE;
  }
  if (T == 0) return PE_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  CUtensorMap tm_qkv, tm_dout;
  int rc = make_tmap_bf16_2d(&tm_qkv, qkv, (uint64_t)T, (uint64_t)nh * 192, (uint64_t)nh * 192, BW_TILE);
  if (rc != PE_OK) return rc;
  rc = make_tmap_bf16_2d(&tm_dout, dout, (uint64_t)T, (uint64_t)nh * 64, (uint64_t)nh * 64, BW_TILE);
  if (rc != PE_OK) return rc;
  rc = set_max_dynamic_smem(reinterpret_cast<const void*>(attn_bwd_kernel), BW_SMEM, true);
  if (rc != PE_OK) return rc;
  BwArgs a;
  a.row_range = reinterpret_cast<const int2*>(ws + w.row_range);
  a.tile_range = reinterpret_cast<const int2*>(ws + w.tile_range);
  a.lse2 = reinterpret_cast<const float*>(ws + w.lse2);
  a.delta = reinterpret_cast<const float*>(ws + w.delta);
  a.dqkv = static_cast<__nv_bfloat16*>(dqkv);
  a.pos = position_ids;
  a.table = static_cast<const __nv_bfloat16*>(table);
  a.max_positions = max_positions;
  a.T = (int)T;
  a.nh = nh;
  a.n_items = (int)(tiles * nh);
  a.status = status;
  attn_bwd_prepare_kernel<<<dim3((unsigned)tiles, (unsigned)nh), 256, 0, st>>>(
      static_cast<const __nv_bfloat16*>(out), static_cast<const __nv_bfloat16*>(dout), lse, cu_seqlens, n_seqs,
      (int)T, nh, half_window, const_cast<int2*>(a.row_range), const_cast<int2*>(a.tile_range),
      const_cast<float*>(a.lse2), const_cast<float*>(a.delta), status);
  PE_LAUNCH_CHECK("attn_bwd_prepare_kernel");
  const int grid = (int)std::min<int64_t>(2 * int64_t(a.n_items), sm_count());
  attn_bwd_kernel<<<grid, BW_THREADS, BW_SMEM, st>>>(tm_qkv, tm_dout, a);
  PE_LAUNCH_CHECK("attn_bwd_kernel");
  return PE_OK;
}
