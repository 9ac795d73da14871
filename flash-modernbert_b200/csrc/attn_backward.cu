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
// no fp32 dQ buffer: that one pass moves 32 KB of fp32 additions through L2 per 128 x 128 scores, 25 B
// per clock and SM at the tensor cores' pace, more than L2 takes.
//
// Rows are tiled over the packed tokens, not per sequence: a tile of 128 consecutive tokens may
// hold many sequences.  Row i attends the columns [lo_i, hi_i) - its sequence, cut to the window -
// and the relation is symmetric, so the same two numbers serve both passes.  A batch of 30-token
// queries then costs one row tile per four queries instead of one each.  A tile walks the
// columns [min lo, max hi) of its rows; its last column tile ends exactly at max hi (it overlaps the
// one before, whose columns are masked out there), so rows behind the last sequence are never
// fetched as columns and whatever they hold cannot reach a gradient.
#include <algorithm>
#include <atomic>

#include "attn_tmem.cuh"
#include "pe_host.h"
#include "pe_ptx.cuh"
#include "pe_vec.cuh"

namespace pe {

// Three groups of four compute warps take a row tile's column tiles in turn; each is a chain of tensor
// memory loads, exponentials, stores and barrier round trips that no group could hide alone, and
// three of them fill each other's gaps.  A column tile is 64 wide so that each group can own the two
// 64-column buffers it needs beside the accumulators.  Four more warps move finished accumulators out: a
// group that did it itself was away from its next tiles for some 4,000 clocks per item (307,164
// tokens x 12 heads, window 64: 2.01 ms against 1.43 ms).
constexpr int BW_GROUPS = 3;
constexpr int BW_COMPUTE_WARPS = 4 * BW_GROUPS;
constexpr int BW_PRODUCER = BW_COMPUTE_WARPS;
constexpr int BW_MMA = BW_COMPUTE_WARPS + 1;
constexpr int BW_STORER = BW_COMPUTE_WARPS + 4;       // first of four (two in between idle: registers move by fours)
constexpr int BW_THREADS = 32 * (BW_COMPUTE_WARPS + 8);
// Registers per thread: what the launch gives (65,536 / 640, in eights) and what each role moves to.
constexpr int BW_REGS = 96, BW_REGS_COMPUTE = 120, BW_REGS_FEED = 48, BW_REGS_STORE = 72;
static_assert(BW_COMPUTE_WARPS * BW_REGS_COMPUTE + 4 * BW_REGS_FEED + 4 * BW_REGS_STORE ==
                  (BW_COMPUTE_WARPS + 8) * BW_REGS, "an increase waits until the others have released as many");
constexpr int BW_TILE = 128;                        // rows of a row tile
constexpr int BW_COLS = 64;                         // columns of a column tile
constexpr int BW_A_BYTES = BW_TILE * 64 * 2;        // one operand of a row tile
constexpr int BW_B_BYTES = BW_COLS * 64 * 2;        // one operand of a column tile
// The g-th column tile of a CTA belongs to group w = g % 3 and uses slot 2 w + g / 3 % 2 of everything: the
// operand ring in shared memory ((Q, dO) or (K, V), lse and delta), tensor memory and the barriers,
// whose phases therefore all count g / 6.
constexpr int BW_SLOTS = 2 * BW_GROUPS;
constexpr int BW_STATS_BYTES = 2 * BW_COLS * 4;     // lse and delta of a column tile
constexpr int BW_OUT_BYTES = 2 * 32 * 128;          // 32 rows of both gradients on their way out
constexpr uint32_t BW_TMEM_COLS = 512;
// Tensor memory: a buffer of 64 columns per slot, at 64 c.  The scores of a tile go to its own slot's buffer,
// dP to the group's other one (c ^ 1).  The scores are replaced in place by P (32 columns of bf16
// pairs) and dS (32 more).  Once dP has been read its buffer takes the group's next scores; once P
// and dS have been multiplied theirs takes the next dP.
constexpr uint32_t BW_ACC1_COL = 384;  // dK; dQ of even items
constexpr uint32_t BW_ACC2_COL = 448;  // dV; dQ of odd items

// Barriers of one pass; each pass has its own set.  [c]: one per slot.
enum {
  WB_IN = 0,                            // [c] the tile's operands are here, dS of the tile three before it is written
  WB_S_FULL = WB_IN + BW_SLOTS,         // [c]
  WB_DP_FULL = WB_S_FULL + BW_SLOTS,    // [c]
  WB_DONE = WB_DP_FULL + BW_SLOTS,      // [c] the tile has been accumulated
  WB_A_FULL = WB_DONE + BW_SLOTS,       // [2]
  WB_A_EMPTY = WB_A_FULL + 2,           // [2]
  WB_ACC_FULL = WB_A_EMPTY + 2,         // [2] one per accumulator
  WB_ACC_EMPTY = WB_ACC_FULL + 2,       // [2] it has been read
  WB_COUNT = WB_ACC_EMPTY + 2
};
constexpr int BW_OUT_OFFSET = 4 * BW_A_BYTES + BW_SLOTS * 2 * BW_B_BYTES;
constexpr int BW_STATS_OFFSET = BW_OUT_OFFSET + 4 * BW_OUT_BYTES;
constexpr int BW_BAR_OFFSET = BW_STATS_OFFSET + BW_SLOTS * BW_STATS_BYTES;
constexpr int BW_SMEM = BW_BAR_OFFSET + 2 * WB_COUNT * 8 + 16;
static_assert(BW_SMEM <= 227 * 1024, "shared memory of one CTA");

struct BwArgs {
  const int2* row_range;    // [T]: columns [x, y) that row t attends
  const int2* tile_range;   // [tiles]: their union over a tile of 128 rows
  const float* neg_lse2;    // [nh, T]: -lse * log2(e)
  const float* neg_delta;   // [nh, T]
  __nv_bfloat16* dqkv;      // [T, 3 nh 64]
  const int64_t* pos;       // [T] or NULL: rotation of q and k undone on dq and dk
  const __nv_bfloat16* table;
  int max_positions;
  int T, nh, n_items;
  int* status;
};

// ---- preparation ------------------------------------------------------------------
// Grid (tiles, heads), 256 threads.  Every block: delta of its 128 rows and head, eight lanes per
// row, and lse in the exponent's base, both negated as the passes use them.  Blocks of head 0 also find
// each row's sequence and window.
// Boundaries are not trusted: a row whose sequence does not come out as begin <= t < end within
// [0, T] attends nothing, and an entry outside [0, T] or below its predecessor is reported.
__global__ void __launch_bounds__(256)
attn_bwd_prepare_kernel(const __nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ dout,
                        const float* __restrict__ lse, const int32_t* __restrict__ cu_seqlens, int n_seqs,
                        int T, int nh, int half_window, int2* __restrict__ row_range,
                        int2* __restrict__ tile_range, float* __restrict__ neg_lse2, float* __restrict__ neg_delta,
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
      neg_delta[at] = -acc;
      neg_lse2[at] = lse[at] * -1.4426950408889634f;
    }
  }
  if (head != 0) return;
  for (int64_t n = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; n < n_seqs; n += int64_t(gridDim.x) * blockDim.x) {
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

// One of this CTA's items: (row tile, head), head fastest, every gridDim-th.  The column range of the
// item after is fetched a whole item ahead, and nothing is divided on the way.
struct BwItem {
  int index, tile, head;
  int lo, hi;  // columns of the row tile
  int n;       // its column tiles (at least one: an empty item runs one, masked)
  int d_tile, d_head;
  int2 ahead;
  __device__ __forceinline__ void fetch(const BwArgs& a) {
    int t = tile + d_tile, h = head + d_head;
    if (h >= a.nh) ++t;
    ahead = index + int(gridDim.x) < a.n_items ? __ldg(a.tile_range + t) : make_int2(0, 0);
  }
  __device__ __forceinline__ void open(const BwArgs& a, int2 range) {
    lo = range.x;
    hi = range.y;
    n = max((hi - lo + BW_COLS - 1) / BW_COLS, 1);
    fetch(a);
  }
  __device__ __forceinline__ void start(const BwArgs& a, int first) {
    index = first;
    tile = first / a.nh;
    head = first % a.nh;
    d_tile = int(gridDim.x) / a.nh;
    d_head = int(gridDim.x) % a.nh;
    open(a, index < a.n_items ? __ldg(a.tile_range + tile) : make_int2(0, 0));
  }
  __device__ __forceinline__ bool valid(const BwArgs& a) const { return index < a.n_items; }
  __device__ __forceinline__ void next(const BwArgs& a) {
    index += gridDim.x;
    tile += d_tile;
    head += d_head;
    if (head >= a.nh) {
      head -= a.nh;
      ++tile;
    }
    open(a, ahead);
  }
  // first column of tile j: the last tile ends at hi (it may start below zero: filled, then masked)
  __device__ __forceinline__ int col0(int j) const { return j + 1 == n ? hi - BW_COLS : lo + j * BW_COLS; }
};

// Bounded: the instruction itself waits up to about half a microsecond, so this gives up after seconds at most.
__device__ __forceinline__ bool bw_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred P;\n\t.reg .u32 n;\n\t"
      "mov.u32 n, 0;\n\t"
      "WAIT:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2, %3;\n\t"
      "@P bra DONE;\n\t"
      "add.u32 n, n, 1;\n\t"
      "setp.lt.u32 P, n, 4194304;\n\t"
      "@P bra WAIT;\n\t"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, P;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity), "r"(500u)
      : "memory");
  return done != 0;
}
// Four products over 16 of 64 dimensions each (or columns, below), an arrival on `commit` when all issued so far
// have retired, and the state of another barrier, which is asked for before and read after: the answer
// takes about as long as the products take to be accepted.
__device__ __forceinline__ bool bw_products_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                               uint32_t commit, uint32_t test, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred T, P, Q;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 T, [%7], %8;\n\t"
      "setp.ne.b32 P, %1, %1;\n\t"
      "setp.eq.b32 Q, %1, %1;\n\t"
      "mov.b64 a, {%2, %4};\n\tmov.b64 b, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], a, b, %5, P;\n\t"
      "add.u32 x, %2, 2;\n\tadd.u32 y, %3, 2;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], a, b, %5, Q;\n\t"
      "add.u32 x, %2, 4;\n\tadd.u32 y, %3, 4;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], a, b, %5, Q;\n\t"
      "add.u32 x, %2, 6;\n\tadd.u32 y, %3, 6;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], a, b, %5, Q;\n\t"
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t"
      "selp.u32 %0, 1, 0, T;\n\t}\n"
      : "=r"(done)
      : "r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(commit), "r"(test), "r"(parity)
      : "memory");
  return done != 0;
}
// A in tensor memory (64 columns as pairs), B's rows 2048 bytes (descriptor units of 16) further on each time.
__device__ __forceinline__ bool bw_products_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                               uint32_t add, uint32_t commit, uint32_t test, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred T, P, Q;\n\t.reg .b64 b;\n\t.reg .b32 x, y;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 T, [%8], %9;\n\t"
      "setp.ne.b32 P, %6, 0;\n\t"
      "setp.eq.b32 Q, %1, %1;\n\t"
      "mov.b64 b, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], b, %5, P;\n\t"
      "add.u32 x, %2, 8;\n\tadd.u32 y, %3, 128;\n\tmov.b64 b, {y, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], [x], b, %5, Q;\n\t"
      "add.u32 x, %2, 16;\n\tadd.u32 y, %3, 256;\n\tmov.b64 b, {y, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], [x], b, %5, Q;\n\t"
      "add.u32 x, %2, 24;\n\tadd.u32 y, %3, 384;\n\tmov.b64 b, {y, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%1], [x], b, %5, Q;\n\t"
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%7];\n\t"
      "selp.u32 %0, 1, 0, T;\n\t}\n"
      : "=r"(done)
      : "r"(d), "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(add), "r"(commit), "r"(test), "r"(parity)
      : "memory");
  return done != 0;
}
// Slot of the tile after the one in slot c: 0, 2, 4, 1, 3, 5, 0, ...
__device__ __forceinline__ uint32_t bw_next_slot(uint32_t c) {
  return c + 2 < BW_SLOTS ? c + 2 : BW_SLOTS + 1 - (c + 2);
}
// Bits [lo, hi) of a word.
__device__ __forceinline__ uint32_t bw_bits(int lo, int hi) {
  const uint32_t below_hi = hi >= 32 ? 0xffffffffu : (1u << max(hi, 0)) - 1u;
  return lo >= 32 ? 0u : below_hi & ~((1u << max(lo, 0)) - 1u);
}
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

// 64 accumulated values of a row, scaled, as bf16 to the warp's block of shared memory, a row of 128 bytes per
// thread; zeros if the row attends nothing.  With `trow` (the rotation table's row of the row's position) the
// rotation is undone first: the transpose of what was applied to q and k.
__device__ __forceinline__ void bw_finish_row(uint32_t acc_addr, float scale, const uint4* trow, bool empty,
                                              uint32_t block, int lane) {
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {  // dimensions [16 c, 16 c + 16) and those they are paired with, 32 further on
    uint32_t lo[16], hi[16];
    g_tmem_ld16(acc_addr + c * 16, lo);
    g_tmem_ld16(acc_addr + 32 + c * 16, hi);
    tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[8], y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = __uint_as_float(lo[h * 8 + e]) * scale;
        y[e] = __uint_as_float(hi[h * 8 + e]) * scale;
      }
      if (trow != nullptr) {
        float cs[8], sn[8];
        unpack8(__ldg(trow + c * 2 + h), cs);
        unpack8(__ldg(trow + 4 + c * 2 + h), sn);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float u = x[e], w = y[e];
          x[e] = fmaf(u, cs[e], w * sn[e]);
          y[e] = fmaf(w, cs[e], -(u * sn[e]));
        }
      }
      const int i = c * 2 + h;  // 16-byte chunk of the row
      const uint32_t row = block + lane * 128;
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((i ^ (lane & 7)) << 4)),
                   "r"(pack_bf16(x[0], x[1])), "r"(pack_bf16(x[2], x[3])), "r"(pack_bf16(x[4], x[5])),
                   "r"(pack_bf16(x[6], x[7]))
                   : "memory");
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + (((i + 4) ^ (lane & 7)) << 4)),
                   "r"(pack_bf16(y[0], y[1])), "r"(pack_bf16(y[2], y[3])), "r"(pack_bf16(y[4], y[5])),
                   "r"(pack_bf16(y[6], y[7]))
                   : "memory");
    }
  }
  if (empty) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(block + lane * 128 + (i << 4)), "r"(0) : "memory");
  }
}
// The block's rows to memory, four whole rows per instruction; `dst` is the first row's, `rows` how many of them exist.
__device__ __forceinline__ void bw_store_rows(__nv_bfloat16* dst, int64_t ld, int rows, uint32_t block, int lane) {
#pragma unroll 4
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 3);
    uint4 u;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                 : "r"(block + r * 128 + (((lane & 7) ^ (r & 7)) << 4))
                 : "memory");
    if (r < rows) *reinterpret_cast<uint4*>(dst + r * ld + (lane & 7) * 8) = u;
  }
}

// KEYS: the key pass (rows are keys, columns are queries), else the query pass.  `first` is this
// CTA's first item.  Returns false if a bounded wait gave up.
enum { BW_FEED, BW_COMPUTE, BW_STORE };
template <bool KEYS, int ROLE>
__device__ __forceinline__ bool bw_pass(const CUtensorMap& tm_qkv, const CUtensorMap& tm_qkv_cols,
                                        const CUtensorMap& tm_dout, const CUtensorMap& tm_dout_cols,
                                        const BwArgs& a, int first, uint32_t base, uint32_t bar_base,
                                        uint32_t tmem_base) {
  auto bar = [&](int i) { return bar_base + 8u * i; };
  const uint32_t sA = base;                  // A[buffer]: (K, V) or (Q, dO)
  const uint32_t sB = base + 4 * BW_A_BYTES; // B[slot]: (Q, dO) or (K, V)
  const uint32_t sStats = base + BW_STATS_OFFSET;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = a.nh * 64;
  int* status = a.status;
  bool ok = true;
  BwItem it;
  it.start(a, first);

  if (ROLE == BW_FEED && warp == BW_PRODUCER) {
    // ---------------------------------------------------------------- producer
    uint32_t c = 0, lap = 0, loads = 0, ord = 0;
    for (; it.valid(a) && ok; it.next(a), ++ord) {
      const uint32_t ab = ord & 1;
      const int col = it.head * 64, row0 = it.tile * BW_TILE;
      if (!bw_wait(bar(WB_A_EMPTY + ab), ((ord >> 1) & 1) ^ 1u)) { ok = false; break; }
      if (lane == 0) {
        const uint32_t dst = sA + ab * 2 * BW_A_BYTES;
        mbar_expect_tx(bar(WB_A_FULL + ab), 2 * BW_A_BYTES);
        tma_load_2d(dst, &tm_qkv, bar(WB_A_FULL + ab), (KEYS ? H : 0) + col, row0);
        if (KEYS) tma_load_2d(dst + BW_A_BYTES, &tm_qkv, bar(WB_A_FULL + ab), 2 * H + col, row0);
        else tma_load_2d(dst + BW_A_BYTES, &tm_dout, bar(WB_A_FULL + ab), col, row0);
      }
      __syncwarp();
      const float* lse_head = a.neg_lse2 + int64_t(it.head) * a.T;
      const float* delta_head = a.neg_delta + int64_t(it.head) * a.T;
#pragma unroll 1
      for (int j = 0; j < it.n; ++j) {
        if (!bw_wait(bar(WB_DONE + c), lap ^ 1u)) { ok = false; break; }
        const int col0 = it.col0(j);
        if (KEYS) {
#pragma unroll
          for (int i = 0; i < BW_COLS / 32; ++i) {
            const int q = min(max(col0 + i * 32 + lane, 0), a.T - 1);
            const uint32_t dst = sStats + c * BW_STATS_BYTES + (i * 32 + lane) * 4;
            cp_async4(dst, lse_head + q);
            cp_async4(dst + BW_COLS * 4, delta_head + q);
          }
          cp_async_arrive(bar(WB_IN + c));
        }
        if (lane == 0) {
          const uint32_t dst = sB + c * 2 * BW_B_BYTES;
          mbar_expect_tx(bar(WB_IN + c), 2 * BW_B_BYTES);
          tma_load_2d(dst, &tm_qkv_cols, bar(WB_IN + c), (KEYS ? 0 : H) + col, col0);
          if (KEYS) tma_load_2d(dst + BW_B_BYTES, &tm_dout_cols, bar(WB_IN + c), col, col0);
          else tma_load_2d(dst + BW_B_BYTES, &tm_qkv_cols, bar(WB_IN + c), 2 * H + col, col0);
        }
        __syncwarp();
        ++loads;
        c = bw_next_slot(c);
        lap ^= c == 0;
      }
    }
    // three tiles that are not there arrive empty, so that every tile's dS finds its barrier
#pragma unroll 1
    for (int j = 0; j < BW_GROUPS && ok && loads > 0; ++j) {
      if (!bw_wait(bar(WB_DONE + c), lap ^ 1u)) { ok = false; break; }
      if (KEYS) mbar_arrive(bar(WB_IN + c));
      if (lane == 0) mbar_arrive(bar(WB_IN + c));
      c = bw_next_slot(c);
        lap ^= c == 0;
    }
    if (!ok) {  // gave up: this CTA's copies must have landed before it can leave
      set_status(status, ST_ATTN_TIMEOUT);
#pragma unroll 1
      for (uint32_t u = loads > BW_SLOTS ? loads - BW_SLOTS : 0; u < loads; ++u)
        bw_wait(bar(WB_IN + u % BW_GROUPS * 2 + u / BW_GROUPS % 2), (u / BW_SLOTS) & 1);
#pragma unroll 1
      for (uint32_t u = ord > 1 ? ord - 2 : 0; u <= ord; ++u)  // (one that was never issued runs into its limit)
        bw_wait(bar(WB_A_FULL + (u & 1)), (u >> 1) & 1);
    }
  } else if (ROLE == BW_FEED && warp == BW_MMA) {
    // ---------------------------------------------------------------- MMA issuer
    // The scores run three tiles ahead of the accumulation and dP two, so that by the time something
    // is waited for it has usually happened.  This one thread is what bounds the kernel: an MMA costs it
    // 23 clocks to issue on an idle scheduler and 32 beside busy warps (sixteen per tile), a look at a
    // barrier about a hundred.  So a tile needs two barriers only (WB_IN stands for two events, and
    // P and dS are announced together), and their state is asked for ahead of four MMAs and read after
    // them.  Electing a lane for each group of MMAs inside a loop of the whole warp, which would keep the
    // descriptors in uniform registers, made it 100 clocks per MMA.
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_bf16(BW_TILE, BW_COLS, 0);
      constexpr uint32_t idesc_acc = umma_idesc_bf16(BW_TILE, 64, 1);  // B is MN-major: its rows are the contraction
      const uint64_t a_desc = umma_smem_desc_sw128(sA, 1024), b_desc = umma_smem_desc_sw128(sB, 1024);
      const uint32_t desc_hi = uint32_t(a_desc >> 32);  // the same for both
      auto desc = [&](uint32_t lo) { return (uint64_t(desc_hi) << 32) | lo; };
      auto scores = [&](uint32_t d, uint32_t ad, uint32_t bd) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) umma_ss(d, desc(ad + 2u * kk), desc(bd + 2u * kk), idesc_s, kk != 0 ? 1u : 0u);
      };
      // acc += X B, X (bf16 pairs of 64 columns) in tensor memory
      auto accumulate = [&](uint32_t acc_col, uint32_t x, uint32_t bd, uint32_t add) {
#pragma unroll
        for (int kk = 0; kk < BW_COLS / 16; ++kk)
          g_umma_ts(tmem_base + acc_col, x + kk * 8, desc(bd + uint32_t(kk * 2048 >> 4)), idesc_acc,
                    kk != 0 ? 1u : add);
      };
      // A tile on its way from scores to accumulation: A buffer (1), first (2) and last (4) of its
      // item, present (8)
      int left = it.valid(a) ? it.n : 0;  // tiles of the item whose scores come next
      uint32_t fresh = 2u, ab = 0, a_phase = 0;
      auto next_tile = [&]() {
        if (left == 0) return 0u;
        uint32_t f = 8u | ab | fresh;
        fresh = 0;
        if (--left == 0) {
          f |= 4u;
          fresh = 2u;
          ab ^= 1u;
          it.next(a);
          left = it.valid(a) ? it.n : 0;
        }
        return f;
      };
      const uint32_t a_lo = uint32_t(a_desc), b_lo = uint32_t(b_desc);
      auto issue_s = [&](uint32_t f, uint32_t c) {  // of the tile in slot c, whose columns have arrived
        if (f & 2u) {
          if (!bw_wait(bar(WB_A_FULL) + (f & 1) * 8u, a_phase >> 1)) return false;
          a_phase = (a_phase + 1) & 3u;
          tc_fence_after();
        }
        scores(tmem_base + c * 64, a_lo + (f & 1) * (2 * BW_A_BYTES >> 4), b_lo + c * (2 * BW_B_BYTES >> 4));
        umma_commit(bar(WB_S_FULL) + c * 8u);
        return true;
      };
      auto issue_dp = [&](uint32_t f, uint32_t c) {
        scores(tmem_base + (c ^ 1u) * 64, a_lo + ((f & 1) * 2 + 1) * (BW_A_BYTES >> 4),
               b_lo + (c * 2 + 1) * (BW_B_BYTES >> 4));
        umma_commit(bar(WB_DP_FULL) + c * 8u);
        if (f & 4u) umma_commit(bar(WB_A_EMPTY) + (f & 1) * 8u);
      };
      uint32_t f0 = 0, f1 = 0, f2 = 0;  // tiles g, g + 1, g + 2
#pragma unroll 1
      for (uint32_t g = 0; g < BW_GROUPS && ok; ++g) {
        f0 = f1;
        f1 = f2;
        f2 = next_tile();
        if (!f2) continue;
        ok = bw_wait(bar(WB_IN) + g * 16u, 0);
        tc_fence_after();
        ok = ok && issue_s(f2, g * 2);
        if (ok && g < 2) issue_dp(f2, g * 2);
      }
      // Slots of tiles g and g - 1 and the parities of their laps (before the first tile: of a barrier's
      // state before its first phase).
      uint32_t c = 0, lap = 0, cm = BW_SLOTS - 1, lapm = 1;
      uint32_t acc_phase = KEYS ? 1u : 2u, acc_col = tmem_base + BW_ACC1_COL, acc_bar = 0;
      uint32_t f3 = next_tile();  // tile g + 3
      bool in = false;
#pragma unroll 1
      while (ok && f0) {
        // dS of tile g is written (its dP has been read) and the columns of tile g + 3 are here
        if (!in && !bw_wait(bar(WB_IN) + (c ^ 1u) * 8u, (lap ^ c) & 1u)) { ok = false; break; }
        tc_fence_after();
        bool done;
        if (f3) {
          if (f3 & 2u) {
            if (!bw_wait(bar(WB_A_FULL) + (f3 & 1) * 8u, a_phase >> 1)) { ok = false; break; }
            a_phase = (a_phase + 1) & 3u;
            tc_fence_after();
          }
          done = bw_products_ss(tmem_base + (c ^ 1u) * 64, a_lo + (f3 & 1) * (2 * BW_A_BYTES >> 4),
                                b_lo + (c ^ 1u) * (2 * BW_B_BYTES >> 4), desc_hi, idesc_s,
                                bar(WB_S_FULL) + (c ^ 1u) * 8u, bar(WB_DONE) + cm * 8u, lapm);
        } else {
          done = false;
        }
        const uint32_t x = tmem_base + c * 64, b1 = b_lo + c * (2 * BW_B_BYTES >> 4);
        uint32_t add = 1;
        if (f0 & 2u) {  // the previous item's accumulators must have been read before they are overwritten
          if (KEYS) {
            if (!bw_wait(bar(WB_ACC_EMPTY + 1), acc_phase)) { ok = false; break; }
          } else {  // dQ needs one accumulator only: items take the two in turn
            acc_bar = (f0 & 1) * 8u;
            if (!bw_wait(bar(WB_ACC_EMPTY) + acc_bar, acc_phase >> 1)) { ok = false; break; }
            acc_phase = (acc_phase + 1) & 3u;
            acc_col = tmem_base + BW_ACC1_COL + (f0 & 1) * 64;
          }
          tc_fence_after();
          add = 0;
        }
        if (KEYS) {
          accumulate(BW_ACC2_COL, x, b1 + (BW_B_BYTES >> 4), add);  // dV += P^T dO
          if (f0 & 4u) umma_commit(bar(WB_ACC_FULL + 1));
        }
        const uint32_t f4 = next_tile();
        if (f2) {  // P and dS of tile g - 1 have been multiplied: their buffer takes dP of tile g + 2
          if (!done && !bw_wait(bar(WB_DONE) + cm * 8u, lapm)) { ok = false; break; }
          tc_fence_after();
          issue_dp(f2, cm ^ 1u);
        }
        if (KEYS && !add) {
          if (!bw_wait(bar(WB_ACC_EMPTY), acc_phase)) { ok = false; break; }
          tc_fence_after();
          acc_phase ^= 1u;
        }
        const uint32_t c_next = bw_next_slot(c), lap_next = lap ^ (c_next == 0 ? 1u : 0u);
        // dK += dS^T Q, dQ += dS K
        in = bw_products_ts(acc_col, x + 32, b1, desc_hi, idesc_acc, add, bar(WB_DONE) + c * 8u,
                            bar(WB_IN) + (c_next ^ 1u) * 8u, (lap_next ^ c_next) & 1u);
        if (f0 & 4u) umma_commit(bar(WB_ACC_FULL) + acc_bar);
        f0 = f1;
        f1 = f2;
        f2 = f3;
        f3 = f4;
        cm = c;
        lapm = lap;
        c = c_next;
        lap = lap_next;
      }
      if (!ok) set_status(status, ST_ATTN_MMA_TIMEOUT);
    }
    __syncwarp();
    ok = __all_sync(0xffffffffu, ok);
  } else if (ROLE == BW_STORE) {
    // ---------------------------------------------------------------- gradients out of the accumulators
    const int row = (warp & 3) * 32 + lane;  // row of the tile = tensor-memory lane
    const uint32_t lane_addr = tmem_base + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t block = base + BW_OUT_OFFSET + (warp & 3) * BW_OUT_BYTES;
    uint32_t ord = 0;
#pragma unroll 1
    for (; it.valid(a); it.next(a), ++ord) {
      const int t = it.tile * BW_TILE + row;
      bool empty = true;
      const uint4* trow = nullptr;
      if (t < a.T) {
        const int2 range = __ldg(a.row_range + t);
        empty = range.x >= range.y;  // rows that attend nothing are exact zeros
        if (a.pos != nullptr) {
          int64_t ps = a.pos[t];
          if (ps < 0 || ps >= a.max_positions) {
            set_status(status, ST_BAD_POSITION);
            ps = 0;
          }
          trow = reinterpret_cast<const uint4*>(a.table + ps * 64);
        }
      }
      auto take = [&](uint32_t b, uint32_t phase, float scale, const uint4* turn, uint32_t to) {
        if (ok) ok = bw_wait(bar(WB_ACC_FULL) + b * 8, phase);
        tc_fence_after();
        bw_finish_row(lane_addr + BW_ACC1_COL + b * 64, scale, turn, empty, to, lane);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(WB_ACC_EMPTY) + b * 8);
      };
      if (KEYS) take(1, ord & 1, 1.0f, nullptr, block + 32 * 128);  // dV is complete before dK
      if (KEYS) take(0, ord & 1, 0.125f, trow, block);
      else take(ord & 1, (ord >> 1) & 1, 0.125f, trow, block);
      const int row0 = it.tile * BW_TILE + (warp & 3) * 32;
      const int rows = ok ? a.T - row0 : 0;
      const int64_t ld = 3 * int64_t(H);
      __nv_bfloat16* dst = a.dqkv + row0 * ld + (KEYS ? H : 0) + it.head * 64;
      bw_store_rows(dst, ld, rows, block, lane);
      if (KEYS) bw_store_rows(dst + H, ld, rows, block + 32 * 128, lane);
      __syncwarp();
    }
    if (!ok) set_status(status, ST_ATTN_SOFTMAX_TIMEOUT);
  } else if (ROLE == BW_COMPUTE) {
    // ---------------------------------------------------------------- compute warps
    const int w = warp >> 2;                         // group
    const int row = (warp & 3) * 32 + lane;          // row of the tile = tensor-memory lane
    const uint32_t lane_addr = tmem_base + (uint32_t((warp & 3) * 32) << 16);
    const float scale_log2 = 0.125f * 1.4426950408889634f;  // 1/sqrt(64) * log2(e)
    const float2 scale2 = make_float2(scale_log2, scale_log2);
    // After a bounded wait has given up the loops still run to their end, without waiting, so that
    // every thread reaches the common exit.
    auto wait = [&](int b, uint32_t parity) {
      if (ok) ok = bw_wait(bar(b), parity);
    };
    auto arrive = [&](int b) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(b));
    };
    if (lane == 0) mbar_arrive(bar(WB_IN + 2 * w));  // no tile comes three before the first three
    int j = w;       // this group's next tile, counted from the item's first
    uint32_t i = 0;  // tiles of this group so far
    for (; it.valid(a); it.next(a)) {
      if (j < it.n) {
        // what this thread's row brings along
        const int t = it.tile * BW_TILE + row;
        int2 range = make_int2(0, 0);
        float neg_lse = 0.f, neg_delta = 0.f;
        if (t < a.T) {
          range = __ldg(a.row_range + t);
          if (!KEYS) {
            const int64_t at = int64_t(it.head) * a.T + t;
            neg_lse = __ldg(a.neg_lse2 + at);
            neg_delta = __ldg(a.neg_delta + at);
          }
        }
        for (; j < it.n; j += BW_GROUPS, ++i) {
          const uint32_t c = 2 * w + (i & 1), lap = (i >> 1) & 1;
          const uint32_t s_addr = lane_addr + c * 64;
          const uint32_t dp_addr = s_addr ^ 64u;
          const uint32_t stats = sStats + c * BW_STATS_BYTES;
          if (KEYS) wait(WB_IN + c, lap);  // long complete: makes lse and delta visible
          // valid columns of this row within the tile: [c_lo, c_hi)
          const int x0 = it.col0(j);
          const int c_lo = max(range.x, it.lo + j * BW_COLS) - x0, c_hi = range.y - x0;
          const bool full = __all_sync(0xffffffffu, c_lo <= 0 && c_hi >= BW_COLS);
          const bool none = __all_sync(0xffffffffu, c_lo >= c_hi || c_hi <= 0 || c_lo >= BW_COLS);
          wait(WB_S_FULL + c, lap);
          tc_fence_after();
          if (none) {  // no row of this warp attends any of the columns
            uint32_t zero[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) zero[e] = 0;
            wait(WB_DP_FULL + c, lap);
#pragma unroll 1
            for (int h = KEYS ? 0 : 2; h < 4; ++h) g_tmem_st16(s_addr + h * 16, zero);
          } else {
            uint32_t p[64];
            g_tmem_ld32(s_addr, p);
            tmem_ld_wait();
            g_tmem_ld32(s_addr + 32, p + 32);  // in flight during the first half's exponentials
            auto exponentials = [&](int e0) {
#pragma unroll
              for (int e = e0; e < e0 + 32; e += 4) {
                float4 l;
                if (KEYS) l = lds128(stats + e * 4);
                else l = make_float4(neg_lse, neg_lse, neg_lse, neg_lse);
                const float2 u = __ffma2_rn(make_float2(__uint_as_float(p[e]), __uint_as_float(p[e + 1])), scale2,
                                            make_float2(l.x, l.y));
                const float2 v = __ffma2_rn(make_float2(__uint_as_float(p[e + 2]), __uint_as_float(p[e + 3])), scale2,
                                            make_float2(l.z, l.w));
                p[e] = __float_as_uint(g_ex2(u.x));
                p[e + 1] = __float_as_uint(g_ex2(u.y));
                p[e + 2] = __float_as_uint(g_ex2(v.x));
                p[e + 3] = __float_as_uint(g_ex2(v.y));
              }
            };
            exponentials(0);
            tmem_ld_wait();
            exponentials(32);
            if (!full) {
              // columns [c_lo, c_hi) of the tile as bits
              const uint32_t m0 = bw_bits(c_lo, c_hi), m1 = bw_bits(c_lo - 32, c_hi - 32);
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                p[e] = (m0 >> e & 1u) ? p[e] : 0u;
                p[e + 32] = (m1 >> e & 1u) ? p[e + 32] : 0u;
              }
            }
            if (KEYS) {  // P^T in place of the first half of the scores: the A operand of dV += P^T dO
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  pk[e] = pack_bf16(__uint_as_float(p[h * 32 + 2 * e]), __uint_as_float(p[h * 32 + 2 * e + 1]));
                g_tmem_st16(s_addr + h * 16, pk);
              }
            }
            wait(WB_DP_FULL + c, lap);
            tc_fence_after();
            uint32_t dp[2][16];
            g_tmem_ld16(dp_addr, dp[0]);
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              tmem_ld_wait();
              if (h < 3) g_tmem_ld16(dp_addr + (h + 1) * 16, dp[(h + 1) & 1]);  // in flight during this quarter
              const uint32_t* d = dp[h & 1];
              uint32_t pk[8];
#pragma unroll
              for (int e = 0; e < 16; e += 4) {
                float4 dl;
                if (KEYS) dl = lds128(stats + BW_COLS * 4 + (h * 16 + e) * 4);
                else dl = make_float4(neg_delta, neg_delta, neg_delta, neg_delta);
                const uint32_t* q = p + h * 16 + e;
                const float2 u = __fmul2_rn(__fadd2_rn(make_float2(__uint_as_float(d[e]), __uint_as_float(d[e + 1])),
                                                       make_float2(dl.x, dl.y)),
                                            make_float2(__uint_as_float(q[0]), __uint_as_float(q[1])));
                const float2 v = __fmul2_rn(__fadd2_rn(make_float2(__uint_as_float(d[e + 2]), __uint_as_float(d[e + 3])),
                                                       make_float2(dl.z, dl.w)),
                                            make_float2(__uint_as_float(q[2]), __uint_as_float(q[3])));
                pk[e / 2] = pack_bf16(u.x, u.y);
                pk[e / 2 + 1] = pack_bf16(v.x, v.y);
              }
              g_tmem_st8(s_addr + 32 + h * 8, pk);  // dS in place of the second half
            }
          }
          g_tmem_st_wait();
          arrive(WB_IN + (c ^ 1u));
        }
      }
      j -= it.n;
    }
    if (!ok) set_status(status, ST_ATTN_SOFTMAX_TIMEOUT);
  }
  return ok;
}

template <int ROLE>
__device__ __forceinline__ void bw_both(const CUtensorMap& tm_qkv, const CUtensorMap& tm_qkv_cols,
                                        const CUtensorMap& tm_dout, const CUtensorMap& tm_dout_cols,
                                        const BwArgs& a, int second, uint32_t base, uint32_t bar_base,
                                        uint32_t tmem_base) {
  const bool ok = bw_pass<true, ROLE>(tm_qkv, tm_qkv_cols, tm_dout, tm_dout_cols, a, blockIdx.x, base, bar_base,
                                         tmem_base);
  tc_fence_before();
  uint32_t failed;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 0, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(failed)
      : "r"(ok ? 0u : 1u)
      : "memory");
  tc_fence_after();
  if (!failed)
    bw_pass<false, ROLE>(tm_qkv, tm_qkv_cols, tm_dout, tm_dout_cols, a, second, base, bar_base + WB_COUNT * 8,
                            tmem_base);
}

__global__ void __launch_bounds__(BW_THREADS, 1)
attn_bwd_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_qkv_cols,
                const __grid_constant__ CUtensorMap tm_dout, const __grid_constant__ CUtensorMap tm_dout_cols,
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
        // four compute warps, the TMA issue and in the key pass 32 lanes' copies of lse and delta
        if (i < WB_IN + BW_SLOTS) count = pass == 0 ? 37 : 5;
        if (i >= WB_ACC_EMPTY) count = 4;
        mbar_init(bb + 8u * i, count);
      }
    }
    mbar_fence_init();
    tma_prefetch_desc(&tm_qkv);
    tma_prefetch_desc(&tm_qkv_cols);
    tma_prefetch_desc(&tm_dout);
    tma_prefetch_desc(&tm_dout_cols);
  }
  if (warp == BW_MMA) {
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
  int second = int(blockIdx.x) - a.n_items % int(gridDim.x);
  if (second < 0) second += gridDim.x;
  if (warp < BW_COMPUTE_WARPS) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(BW_REGS_COMPUTE));
    bw_both<BW_COMPUTE>(tm_qkv, tm_qkv_cols, tm_dout, tm_dout_cols, a, second, base, bar_base, tmem_base);
  } else if (warp < BW_STORER) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BW_REGS_FEED));
    bw_both<BW_FEED>(tm_qkv, tm_qkv_cols, tm_dout, tm_dout_cols, a, second, base, bar_base, tmem_base);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BW_REGS_STORE));
    bw_both<BW_STORE>(tm_qkv, tm_qkv_cols, tm_dout, tm_dout_cols, a, second, base, bar_base, tmem_base);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == BW_MMA) {
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
  CUtensorMap tm_qkv, tm_qkv_cols, tm_dout, tm_dout_cols;
  const uint64_t wide = (uint64_t)nh * 192, narrow = (uint64_t)nh * 64;
  int rc = make_tmap_bf16_2d(&tm_qkv, qkv, (uint64_t)T, wide, wide, BW_TILE);
  if (rc == PE_OK) rc = make_tmap_bf16_2d(&tm_qkv_cols, qkv, (uint64_t)T, wide, wide, BW_COLS);
  if (rc == PE_OK) rc = make_tmap_bf16_2d(&tm_dout, dout, (uint64_t)T, narrow, narrow, BW_TILE);
  if (rc == PE_OK) rc = make_tmap_bf16_2d(&tm_dout_cols, dout, (uint64_t)T, narrow, narrow, BW_COLS);
  if (rc != PE_OK) return rc;
  rc = set_max_dynamic_smem(reinterpret_cast<const void*>(attn_bwd_kernel), BW_SMEM, true);
  if (rc != PE_OK) return rc;
  // A build that needed fewer registers at launch would leave the increase above waiting for good.
  static std::atomic<int> launch_regs{0};
  if (launch_regs.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes attr;
    PE_CUDA(cudaFuncGetAttributes(&attr, reinterpret_cast<const void*>(attn_bwd_kernel)));
    launch_regs.store(attr.numRegs, std::memory_order_relaxed);
  }
  PE_REQUIRE(launch_regs.load(std::memory_order_relaxed) == BW_REGS,
             "pe_attn_varlen_backward: built with %d registers per thread instead of %d",
             launch_regs.load(std::memory_order_relaxed), BW_REGS);
  BwArgs a;
  a.row_range = reinterpret_cast<const int2*>(ws + w.row_range);
  a.tile_range = reinterpret_cast<const int2*>(ws + w.tile_range);
  a.neg_lse2 = reinterpret_cast<const float*>(ws + w.lse2);
  a.dqkv = static_cast<__nv_bfloat16*>(dqkv);
  a.neg_delta = reinterpret_cast<const float*>(ws + w.delta);
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
      const_cast<float*>(a.neg_lse2), const_cast<float*>(a.neg_delta), status);
  PE_LAUNCH_CHECK("attn_bwd_prepare_kernel");
  const int grid = (int)std::min<int64_t>(2 * int64_t(a.n_items), sm_count());
  attn_bwd_kernel<<<grid, BW_THREADS, BW_SMEM, st>>>(tm_qkv, tm_qkv_cols, tm_dout, tm_dout_cols, a);
  PE_LAUNCH_CHECK("attn_bwd_kernel");
  return PE_OK;
}
