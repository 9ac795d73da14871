// Log-probabilities of given tokens over a vocabulary, with entropy and the top alternatives, and
// the gradient with respect to the logits.
//
// One pass over a row keeps, per thread, the running maximum m, s = sum e^(x - m) and
// w = sum e^(x - m) (x - m) in fp32; raising m by d scales s by e^-d and turns w into
// (w - s d) e^-d.  Then lse = m + log s, the token's log-probability is x_t - lse and the entropy
// log s - w / s: no difference of large numbers, wherever the logits lie.  lse alone would lose log s
// to rounding where the logits are far from zero (in a row of nothing but the type's lowest value, all
// of it), so what its rounding left is kept beside it and every difference x - lse takes both.  The
// gradient is
//   dx_j = g (1[j = t] - p_j) - h p_j (log p_j + H) + z p_j
// with g, h, z the gradients of the log-probability, the entropy and lse.
//
// Bound by memory: the logits are read once (and in the backward pass read and written once).  A
// row belongs to one CTA, or, when there are too few rows to fill the GPU, to a cluster of up to
// eight CTAs that each take a part of the vocabulary and join through distributed shared memory.
//
// Top k: the pass also leaves, in shared memory, the largest of every sixteen logits (or multiple of
// sixteen) that a thread has read.  A threshold follows from them at once: the k / W-th largest (rounded
// up) of a warp's 32 thread maxima, the least of these over the W warps - at least k logits
// reach it.  Only the sixteens whose largest reaches the threshold are read again, some tens of 3,000 in a
// row of 50,368, and what reaches the threshold in them is pushed into a small list.  Order is total:
// a candidate is the 64-bit number (value's bits made monotone, complement of the index), so
// equal values rank by lowest index.  The list stays bounded whatever the data: when more than 32 threads
// hold something to push at once, the threshold is raised first to the k-th best of the threads'
// own best, which leaves at most k of them, and the list is cut back to k by counting ranks when
// it fills up.
#include <algorithm>
#include <type_traits>

#include "pe_host.h"
#include "pe_vec.cuh"

#include <cuda_fp16.h>

namespace pe {

constexpr int LP_MAX_TOP = 32;
constexpr int LP_MAX_CLUSTER = 8;
constexpr int LP_CROWD = 32;  // threads that may push without raising the threshold first

template <typename E>
struct LogitVec {
  static constexpr int N = 16 / sizeof(E);  // elements per 16-byte load
};

__device__ __forceinline__ float logit_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float logit_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float logit_f32(float v) { return v; }
__device__ __forceinline__ void logit_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void logit_put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void logit_put(float* p, float v) { *p = v; }

__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The larger of two, NaN if either is: a NaN logit makes the row's statistics NaN.
__device__ __forceinline__ float lp_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Order of candidates: by value (a NaN above everything), then by lowest index; 0 is "none".
__device__ __forceinline__ unsigned long long lp_key(float x, uint32_t index) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);  // -0 and +0 are equal
  const uint32_t v = x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(v) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ float lp_key_value(unsigned long long k) {
  const uint32_t v = uint32_t(k >> 32);
  if (v == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float((v & 0x80000000u) ? (v & 0x7fffffffu) : ~v);
}

struct LpStat {
  float m, s, w;
};
__device__ __forceinline__ LpStat lp_join(const LpStat& a, const LpStat& b) {
  const float m = lp_max_nan(a.m, b.m);
  const float ref = m == -INFINITY ? 0.f : m;
  // a part that has seen only -inf has s = w = 0 and any finite reference serves it
  const float da = a.m == -INFINITY ? 0.f : a.m - ref, db = b.m == -INFINITY ? 0.f : b.m - ref;
  const float ea = lp_ex2(da * 1.4426950408889634f), eb = lp_ex2(db * 1.4426950408889634f);
  LpStat r;
  r.m = m;
  r.s = a.s * ea + b.s * eb;
  // a part so far below that nothing of it is left may have s d = -inf (logits masked with the type's
  // lowest value): it adds nothing
  r.w = (ea > 0.f ? (a.w + a.s * da) * ea : 0.f) + (eb > 0.f ? (b.w + b.s * db) * eb : 0.f);
  return r;
}

constexpr int LP_TOPS = 16;  // maxima that a thread leaves behind; beyond, sixteens are joined

template <int NT, bool TOP>
struct LpShared {
  static constexpr int CAP = 16 * LP_CROWD + 4 * NT;  // list of candidates; a round adds at most 16 * LP_CROWD
  LpStat stat[NT / 32];
  LpStat part[LP_MAX_CLUSTER];                       // parts of the cluster's CTAs, in rank 0
  float lse[2];
  unsigned long long part_top[TOP ? LP_MAX_CLUSTER * LP_MAX_TOP : 1];
  union {
    unsigned long long best[TOP ? NT : 1];
    uint32_t again[TOP ? 2 * NT : 1];                // sixteens to read again: round * NT + thread
  };
  unsigned long long list[TOP ? CAP : 1];
  unsigned long long kept[TOP ? LP_MAX_TOP : 1];
  float tops[TOP ? LP_TOPS + 1 : 1][TOP ? NT : 1];   // the last row: the odd logits at a row's ends
  float bound[NT / 32];
  unsigned long long tau;
  int count, n_again;
};

// Writes the k best of list[0 .. n) to out[0 .. k) in descending order (0 beyond n).  All threads.
template <int NT>
__device__ __forceinline__ void lp_select(const unsigned long long* list, int n, int k, unsigned long long* out) {
  for (int i = threadIdx.x; i < k; i += NT)
    if (i >= n) out[i] = 0ull;
  for (int i = threadIdx.x; i < n; i += NT) {
    const unsigned long long mine = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > mine;
    if (rank < k) out[rank] = mine;
  }
}

struct LpArgs {
  const void* logits;
  int64_t ld;             // elements between rows
  const int64_t* targets;
  int64_t ignore_index;
  int vocab, top_k;
  float* logprobs;
  float* entropy;
  float* lse;
  float* lse_rest;        // lse + lse_rest = m + log s to twice fp32's precision
  int64_t* top_ids;
  float* top_logprobs;
  int* status;
};

// Eight or four logits in 16 bytes as fp32.
template <typename E>
__device__ __forceinline__ void lp_unpack(const uint4& u, float (&f)[LogitVec<E>::N]) {
  const E* p = reinterpret_cast<const E*>(&u);
#pragma unroll
  for (int i = 0; i < LogitVec<E>::N; ++i) f[i] = logit_f32(p[i]);
}

// The largest of VECS vectors of logits, NaN if one is: two at a time where the type is packed.
template <typename E, int VECS>
__device__ __forceinline__ float lp_top(const uint4 (&u)[VECS]) {
  if constexpr (sizeof(E) == 4) {
    float t = __uint_as_float(u[0].x);
#pragma unroll
    for (int i = 0; i < VECS; ++i)
      t = lp_max_nan(lp_max_nan(t, lp_max_nan(__uint_as_float(u[i].x), __uint_as_float(u[i].y))),
                     lp_max_nan(__uint_as_float(u[i].z), __uint_as_float(u[i].w)));
    return t;
  } else {
    using E2 = typename std::conditional<std::is_same<E, __half>::value, __half2, __nv_bfloat162>::type;
    E2 t[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const E2* h = reinterpret_cast<const E2*>(&u[i]);
      t[i] = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    }
#pragma unroll
    for (int i = 1; i < VECS; ++i) t[0] = __hmax2_nan(t[0], t[i]);
    return lp_max_nan(logit_f32(t[0].x), logit_f32(t[0].y));
  }
}

// Registers: for 1,280 threads per SM (48 each); fp32 with the top for 1,024 (64), which was faster there
// (515 x 256,001, top five: 97 us against 100; 16-bit types the other way, 8,192 x 50,368: 243 against 221).
template <typename E, int NT, bool TOP>
__global__ void __launch_bounds__(NT, (TOP && sizeof(E) == 4 ? 4 : 5) * (256 / NT))
token_logprobs_kernel(const LpArgs a, int cluster) {
  constexpr int N = LogitVec<E>::N;
  constexpr int VECS = 16 / N;  // 16-byte loads per thread and chunk: 16 logits
  constexpr int CHUNK = NT * VECS;
  constexpr int WARPS = NT / 32;
  __shared__ LpShared<NT, TOP> sh;
  const int tid = threadIdx.x;
  const int rank = cluster > 1 ? int(cluster_ctarank()) : 0;
  const int64_t row = blockIdx.x / cluster;
  const E* x = static_cast<const E*>(a.logits) + row * a.ld;
  const int k = a.top_k;
  // The row in 16-byte vectors from its first 16-byte boundary on; the few logits before that and
  // behind the last whole vector (`odd` in all, fewer than 2 N) are rank 0's, one to a thread.
  const int head = min(a.vocab, int((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(E)));
  const int vecs = (a.vocab - head) / N;
  const int odd = a.vocab - vecs * N;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  const int per_cta = (vecs + cluster - 1) / cluster;
  const int v_begin = min(vecs, rank * per_cta), v_end = min(vecs, v_begin + per_cta);
  const int chunks = (v_end - v_begin + CHUNK - 1) / CHUNK;
  const int join = (chunks + LP_TOPS - 1) / LP_TOPS;  // chunks to a row of sh.tops
  const int odd_id = rank == 0 && tid < odd ? (tid < head ? tid : vecs * N + tid) : -1;

  // the row's target, fetched now so that nothing waits for it at the end
  int64_t target = 0;
  float x_target = 0.f;
  if (rank == 0 && tid == 0) {
    target = a.targets[row];
    if (target >= 0 && target < a.vocab) x_target = logit_f32(x[target]);
  }
  LpStat st{-INFINITY, 0.f, 0.f};
  auto raise = [&](float top) {
    if (!(top <= st.m)) {  // a new maximum (or a NaN): move the sums to it
      const float d = st.m == -INFINITY ? 0.f : st.m - top;
      const float z = lp_ex2(d * 1.4426950408889634f);
      st.w = z > 0.f ? (st.w + st.s * d) * z : 0.f;
      st.s *= z;
      st.m = top;
    }
  };
  const float2 log2e = make_float2(1.4426950408889634f, 1.4426950408889634f);
  float2 s2 = make_float2(0.f, 0.f), w2 = s2;
  // Whole chunks and one partial, absent vectors as -inf; the next chunk's loads are in flight while
  // one is worked on.
  const uint32_t lowest = sizeof(E) == 4 ? 0xff800000u : (std::is_same<E, __half>::value ? 0xfc00fc00u : 0xff80ff80u);
  uint4 next[VECS];
  auto load = [&](int v0) {
    const uint4* at = xv + v0 + tid;
    if (v0 + CHUNK <= v_end) {  // the same for the whole CTA: only the last chunk asks vector by vector
#pragma unroll
      for (int i = 0; i < VECS; ++i) next[i] = ld_stream(at + i * NT);
    } else {
#pragma unroll
      for (int i = 0; i < VECS; ++i)
        next[i] = v0 + i * NT + tid < v_end ? ld_stream(at + i * NT) : make_uint4(lowest, lowest, lowest, lowest);
    }
  };
  if (chunks > 0) load(v_begin);
  float joined = -INFINITY;
  int filled = 0, kept_rows = 0;  // chunks in `joined`, rows of sh.tops written
  for (int c = 0; c < chunks; ++c) {
    const float top = lp_top<E, VECS>(next);
    float f[VECS][N];
#pragma unroll
    for (int i = 0; i < VECS; ++i) lp_unpack<E>(next[i], f[i]);
    if (c + 1 < chunks) load(v_begin + (c + 1) * CHUNK);
    if (TOP) {
      joined = lp_max_nan(joined, top);
      if (++filled == join || c + 1 == chunks) {
        sh.tops[kept_rows++][tid] = joined;
        joined = -INFINITY;
        filled = 0;
      }
    }
    if (!(top <= st.m)) {
      st.s += s2.x + s2.y;
      st.w += w2.x + w2.y;
      s2 = w2 = make_float2(0.f, 0.f);
      raise(top);
    }
    const float ref = st.m == -INFINITY ? 0.f : st.m;
    const float2 neg_ref = make_float2(-ref, -ref);
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        float2 d = __fadd2_rn(make_float2(f[i][e], f[i][e + 1]), neg_ref);
        const float2 y = __fmul2_rn(d, log2e);
        const float2 q = make_float2(lp_ex2(y.x), lp_ex2(y.y));
        d = make_float2(fmaxf(d.x, -3.0e38f), fmaxf(d.y, -3.0e38f));  // 0 * -inf would be NaN
        s2 = __fadd2_rn(s2, q);
        w2 = __ffma2_rn(q, d, w2);
      }
  }
  st.s += s2.x + s2.y;
  st.w += w2.x + w2.y;
  if (odd_id >= 0) {
    const float v = logit_f32(x[odd_id]);
    raise(v);
    const float ref = st.m == -INFINITY ? 0.f : st.m;
    const float d = v - ref, q = lp_ex2(d * 1.4426950408889634f);
    st.s += q;
    st.w = fmaf(q, fmaxf(d, -3.0e38f), st.w);
    if (TOP) sh.tops[LP_TOPS][tid] = v;
  }

  if (TOP) {
    // Threshold: from the warps whose lanes all have logits (or the first, if k of its lanes have some), so that
    // at least k reach it (none: 0).
    const int full_warps = max(min(WARPS, (v_end - v_begin) / 32), v_end - v_begin >= k ? 1 : 0);
    {
      const int lane = tid & 31;
      uint32_t mine = uint32_t(lp_key(st.m, 0) >> 32), level = 0u;
      for (int taken = 0; taken < k; taken += full_warps == 0 ? k : full_warps) {
        level = __reduce_max_sync(0xffffffffu, mine);
        const uint32_t holders = __ballot_sync(0xffffffffu, mine == level);
        if (lane == __ffs(holders) - 1) mine = 0u;
      }
      if (lane == 0) sh.bound[tid >> 5] = __uint_as_float(level);
    }
    if (tid == 0) sh.count = sh.n_again = 0;
    __syncthreads();
    uint32_t level = full_warps == 0 ? 0u : 0xffffffffu;
    for (int i = 0; i < full_warps; ++i) level = min(level, __float_as_uint(sh.bound[i]));
    // what equals the threshold may be pushed too
    unsigned long long tau = level == 0u ? 0ull : (static_cast<unsigned long long>(level) << 32) - 1ull;
    // The usual way: list the sixteens that reach tau, then read them all at once, one to a thread.
    const float reach = level == 0u ? -INFINITY : lp_key_value(static_cast<unsigned long long>(level) << 32);
    for (int q = 0; q < kept_rows; ++q)
      if (!(sh.tops[q][tid] < reach))  // (or a NaN)
        for (int r = q * join; r < min(chunks, (q + 1) * join); ++r)
          if (v_begin + r * CHUNK + tid < v_end) {
            const int at = atomicAdd(&sh.n_again, 1);
            if (at < 2 * NT) sh.again[at] = uint32_t(r) * NT + tid;
          }
    auto push = [&](unsigned long long key) {
      if (key > tau) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < LpShared<NT, TOP>::CAP) sh.list[at] = key;
      }
    };
    if (odd_id >= 0) push(lp_key(logit_f32(x[odd_id]), uint32_t(odd_id)));
    __syncthreads();
    const int n_again = sh.n_again;
    if (n_again <= 2 * NT) {
      for (int i = tid; i < n_again; i += NT) {
        const int r = sh.again[i] / NT, v0 = v_begin + r * CHUNK + int(sh.again[i] % NT);
        uint4 u[VECS];
#pragma unroll
        for (int q = 0; q < VECS; ++q) u[q] = v0 + q * NT < v_end ? __ldg(xv + v0 + q * NT) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int q = 0; q < VECS; ++q) {
          float f[N];
          lp_unpack<E>(u[q], f);
          if (v0 + q * NT < v_end) {
#pragma unroll
            for (int e = 0; e < N; ++e) push(lp_key(f[e], uint32_t(head + (v0 + q * NT) * N + e)));
          }
        }
      }
    }
    __syncthreads();
    const bool crowded = n_again > 2 * NT || sh.count > LpShared<NT, TOP>::CAP;  // the same for every thread
    if (crowded) {
      __syncthreads();
      if (tid == 0) sh.count = 0;
      __syncthreads();
    }
    // Otherwise, whatever the data, in rounds of bounded size.
    // Round r < chunks: sixteen logits of every thread whose maximum is not below tau; the last round:
    // the odd ones.
    for (int r = 0; crowded && r <= chunks; ++r) {
      const bool ends = r == chunks;
      const int v0 = v_begin + r * CHUNK + tid;  // its vectors: v0, v0 + NT, ...
      bool flag = ends ? odd_id >= 0 : v0 < v_end;
      if (flag) flag = lp_key(sh.tops[ends ? LP_TOPS : r / join][tid], 0u) > tau;
      const int flagged = __syncthreads_count(flag);
      if (flagged == 0) continue;
      float f[VECS][N];
      if (flag) {
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
          if (!ends && v0 + i * NT < v_end) lp_unpack<E>(__ldg(xv + v0 + i * NT), f[i]);
        }
        if (ends) f[0][0] = logit_f32(x[odd_id]);
      }
      auto key_of = [&](int i, int e) {  // 0: not there
        if (ends) return i == 0 && e == 0 ? lp_key(f[0][0], uint32_t(odd_id)) : 0ull;
        return v0 + i * NT < v_end ? lp_key(f[i][e], uint32_t(head + (v0 + i * NT) * N + e)) : 0ull;
      };
      if (flagged > LP_CROWD) {
        unsigned long long best = 0ull;
        if (flag) {
#pragma unroll
          for (int i = 0; i < VECS; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const unsigned long long key = key_of(i, e);
              best = key > best ? key : best;
            }
          if (best <= tau) best = 0ull;
        }
        sh.best[tid] = best;
        if (tid == 0) sh.tau = tau;
        __syncthreads();
        if (best != 0ull) {
          int above = 0;
          for (int j = 0; j < NT; ++j) above += sh.best[j] > best;
          if (above == k - 1) sh.tau = best - 1ull;  // everything from the k-th best on may push
        }
        __syncthreads();
        tau = sh.tau;
        flag = flag && best > tau;
      }
      if (flag) {
#pragma unroll
        for (int i = 0; i < VECS; ++i)
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const unsigned long long key = key_of(i, e);
            if (key > tau) sh.list[atomicAdd(&sh.count, 1)] = key;
          }
      }
      __syncthreads();
      const int n = sh.count;
      if (n > LpShared<NT, TOP>::CAP - 16 * LP_CROWD) {  // the next round might not fit: keep the k best
        lp_select<NT>(sh.list, n, k, sh.kept);
        __syncthreads();
        for (int i = tid; i < k; i += NT) sh.list[i] = sh.kept[i];
        if (tid == 0) sh.count = k;
        tau = sh.kept[k - 1];
        __syncthreads();
      }
    }
  }

  // join the threads, then the CTAs of the cluster
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpStat other;
    other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    other.w = __shfl_xor_sync(0xffffffffu, st.w, o);
    st = lp_join(st, other);
  }
  if ((threadIdx.x & 31) == 0) sh.stat[threadIdx.x >> 5] = st;
  __syncthreads();
  if (TOP) lp_select<NT>(sh.list, sh.count, k, sh.kept);
  if (threadIdx.x < 32) {
    st = threadIdx.x < WARPS ? sh.stat[threadIdx.x] : LpStat{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) {
      LpStat other;
      other.m = __shfl_down_sync(0xffffffffu, st.m, o);
      other.s = __shfl_down_sync(0xffffffffu, st.s, o);
      other.w = __shfl_down_sync(0xffffffffu, st.w, o);
      st = lp_join(st, other);
    }
  }
  if (cluster > 1) {
    __syncthreads();
    const uint32_t to = cluster_map(smem_u32(&sh.part[rank]), 0);
    const uint32_t to_top = cluster_map(smem_u32(&sh.part_top[rank * LP_MAX_TOP]), 0);
    if (threadIdx.x == 0) {
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(st.m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(st.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(st.w) : "memory");
    }
    if (TOP && threadIdx.x < k)
      asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(to_top + 8 * threadIdx.x), "l"(sh.kept[threadIdx.x])
                   : "memory");
    cluster_sync_all();
    if (rank != 0) return;
    if (threadIdx.x == 0)
      for (int i = 0; i < cluster; ++i) st = i == 0 ? sh.part[0] : lp_join(st, sh.part[i]);
    if (TOP) {
      for (int i = threadIdx.x; i < cluster * k; i += NT) sh.list[i] = sh.part_top[(i / k) * LP_MAX_TOP + i % k];
      __syncthreads();
      lp_select<NT>(sh.list, cluster * k, k, sh.kept);
    }
  }
  if (threadIdx.x == 0) {
    const float log_s = logf(st.s);
    const float lse = __fadd_rn(st.m, log_s);
    const float back = __fsub_rn(lse, st.m);
    float rest = __fadd_rn(__fsub_rn(st.m, __fsub_rn(lse, back)), __fsub_rn(log_s, back));
    if (!(fabsf(lse) <= 3.4028234e38f)) rest = 0.f;
    a.lse[row] = lse;
    a.lse_rest[row] = rest;
    a.entropy[row] = log_s - st.w / st.s;
    float lp = 0.f;
    if (target >= 0 && target < a.vocab) lp = target == a.ignore_index ? 0.f : (x_target - lse) - rest;
    else if (target != a.ignore_index) set_status(a.status, ST_BAD_TARGET);
    a.logprobs[row] = lp;
    sh.lse[0] = lse;
    sh.lse[1] = rest;
  }
  if (TOP) {
    __syncthreads();
    if (threadIdx.x < k) {
      const unsigned long long key = sh.kept[threadIdx.x];
      a.top_ids[row * k + threadIdx.x] = int64_t(0xffffffffu - uint32_t(key));
      a.top_logprobs[row * k + threadIdx.x] = (lp_key_value(key) - sh.lse[0]) - sh.lse[1];
    }
  }
}

struct LpBackArgs {
  const void* logits;
  int64_t ld;
  const int64_t* targets;
  int64_t ignore_index;
  const float* lse;
  const float* lse_rest;
  const float* entropy;
  const float* d_logprobs;  // each may be NULL: zero
  const float* d_entropy;
  const float* d_lse;
  void* dlogits;
  int64_t ld_out;
  int vocab;
};

// Grid (parts of the vocabulary, rows); a block walks its part, the loads of its next step in flight while it
// works on one.  VECTOR: input and output rows lie alike relative to 16-byte boundaries, so a piece
// is 16 bytes, else one logit.  A row whose three gradients are zero (an ignored target) is not read.
constexpr int LP_BACK = 2;  // pieces per thread and step

__device__ __forceinline__ void lp_pack(uint4& u, const float (&f)[8], __nv_bfloat16) { u = pack8(f); }
__device__ __forceinline__ void lp_pack(uint4& u, const float (&f)[8], __half) {
  __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ void lp_pack(uint4& u, const float (&f)[4], float) {
  u = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

template <typename E, bool VECTOR>
__global__ void __launch_bounds__(256, 5)
token_logprobs_backward_kernel(const LpBackArgs a, int64_t rows) {
  constexpr int N = VECTOR ? LogitVec<E>::N : 1;
  constexpr int LANES = LogitVec<E>::N;  // of a register vector, of which !VECTOR uses the first
  constexpr int STEP = 256 * LP_BACK;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const E* x = static_cast<const E*>(a.logits) + row * a.ld;
    E* dx = static_cast<E*>(a.dlogits) + row * a.ld_out;
    const int lead = VECTOR ? int((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(E)) : 0;
    const int vecs = (a.vocab + lead + N - 1) / N;  // the first and the last may stick out of the row
    const int steps = (vecs + STEP - 1) / STEP, per_part = (steps + int(gridDim.x) - 1) / int(gridDim.x);
    const int s_end = min(steps, (int(blockIdx.x) + 1) * per_part);
    int s = int(blockIdx.x) * per_part;
    if (s >= s_end) continue;
    const int64_t t = a.targets[row];
    const bool kept = t >= 0 && t < a.vocab && t != a.ignore_index;
    const float g = kept && a.d_logprobs != nullptr ? a.d_logprobs[row] : 0.f;
    const float h = a.d_entropy != nullptr ? a.d_entropy[row] : 0.f;
    const float z = a.d_lse != nullptr ? a.d_lse[row] : 0.f;
    const float lse = a.lse[row], rest = a.lse_rest[row], ent = a.entropy[row];
    const bool nothing = g == 0.f && h == 0.f && z == 0.f;
    const float zg = z - g;
    // p (z - g - h (log p + H)) of one logit; log p is kept finite, so a token of probability zero has
    // no part in the entropy's gradient
    auto gradient = [&](float v) {
      const float lp = (v - lse) - rest;
      return lp_ex2(lp * 1.4426950408889634f) * fmaf(-h, fmaxf(lp, -1.0e30f) + ent, zg);
    };
    auto whole = [&](int v) { return VECTOR && v * N >= lead && v * N - lead + N <= a.vocab; };
    uint4 next[LP_BACK];
    auto load = [&](int step) {
#pragma unroll
      for (int i = 0; i < LP_BACK; ++i) {
        next[i] = make_uint4(0u, 0u, 0u, 0u);
        const int v = step * STEP + i * 256 + int(threadIdx.x), e0 = v * N - lead;
        if (nothing || v >= vecs) continue;
        if (whole(v)) {
          next[i] = *reinterpret_cast<const uint4*>(x + e0);
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (e0 + e >= 0 && e0 + e < a.vocab) reinterpret_cast<E*>(&next[i])[e] = x[e0 + e];
        }
      }
    };
    load(s);
    for (; s < s_end; ++s) {
      uint4 u[LP_BACK];
#pragma unroll
      for (int i = 0; i < LP_BACK; ++i) u[i] = next[i];
      if (s + 1 < s_end) load(s + 1);
#pragma unroll
      for (int i = 0; i < LP_BACK; ++i) {
        const int v = s * STEP + i * 256 + int(threadIdx.x), e0 = v * N - lead;
        if (v >= vecs) break;
        const bool mine = !nothing && t >= e0 && t < e0 + N;  // the target is among these
        float at_target = 0.f;
        if (!nothing) {
          float f[LANES];
          lp_unpack<E>(u[i], f);
          if (mine) {
#pragma unroll
            for (int e = 0; e < N; ++e)
              if (e0 + e == t) at_target = gradient(f[e]) + g;
          }
#pragma unroll
          for (int e = 0; e < N; ++e) f[e] = gradient(f[e]);
          lp_pack(u[i], f, E());
        }
        if (whole(v)) {
          *reinterpret_cast<uint4*>(dx + e0) = u[i];
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (e0 + e >= 0 && e0 + e < a.vocab) dx[e0 + e] = reinterpret_cast<const E*>(&u[i])[e];
        }
        if (mine) logit_put(dx + t, at_target);
      }
    }
  }
}

template <typename E, int NT>
static int launch_logprobs(const LpArgs& a, int64_t rows, cudaStream_t st) {
  auto kern = a.top_k > 0 ? token_logprobs_kernel<E, NT, true> : token_logprobs_kernel<E, NT, false>;
  // A row is split over a cluster while the rows alone leave SMs idle and a CTA keeps at least one
  // full chunk (4,096 logits) of work.
  int cluster = 1;
  while (cluster < LP_MAX_CLUSTER && rows * cluster * 2 <= sm_count() && a.vocab >= cluster * 2 * 16 * NT) cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PE_CUDA(cudaLaunchKernelEx(&cfg, kern, a, cluster));
  PE_LAUNCH_CHECK("token_logprobs_kernel");
  return PE_OK;
}

template <typename E>
static int launch_logprobs_backward(const LpBackArgs& a, int64_t rows, cudaStream_t st) {
  const bool alike = ((uintptr_t)a.logits & 15) == ((uintptr_t)a.dlogits & 15) &&
                     (a.ld - a.ld_out) * int64_t(sizeof(E)) % 16 == 0;
  const int per_thread = alike ? LogitVec<E>::N : 1;
  // A row to a block as long as there are enough of them to keep every SM's five blocks busy for a few
  // turns, else parts of a row, down to one step (4,096 logits of 16 bits) each.
  const int64_t per_step = int64_t(256) * LP_BACK * per_thread;
  const int64_t steps = (a.vocab + (per_thread - 1) + per_step - 1) / per_step;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(steps, int64_t(sm_count()) * 20 / rows));
  const dim3 grid((unsigned)parts, (unsigned)std::min<int64_t>(rows, 65535));
  auto kern = alike ? token_logprobs_backward_kernel<E, true> : token_logprobs_backward_kernel<E, false>;
  kern<<<grid, 256, 0, st>>>(a, rows);
  PE_LAUNCH_CHECK("token_logprobs_backward_kernel");
  return PE_OK;
}

static int check_logits(const char* who, const void* logits, int64_t ld, int64_t rows, int64_t vocab, int dtype) {
  PE_REQUIRE(dtype == PE_BF16 || dtype == PE_FP16 || dtype == PE_FP32, "%s: unknown type %d", who, dtype);
  PE_REQUIRE(rows >= 0 && rows < (1ll << 27) && vocab > 0 && vocab < (1ll << 31) - (1 << 20) && ld >= vocab,
             "%s: %lld rows of %lld logits (stride %lld) out of range", who, (long long)rows, (long long)vocab,
             (long long)ld);
  PE_REQUIRE(logits != nullptr || rows == 0, "%s: null pointer", who);
  PE_REQUIRE(((uintptr_t)logits & (dtype == PE_FP32 ? 3 : 1)) == 0, "%s: unaligned pointer", who);
  return PE_OK;
}

}  // namespace pe

extern "C" int pe_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld,
                                 const int64_t* targets, int64_t ignore_index, int top_k, float* logprobs,
                                 float* entropy, float* lse, float* lse_rest, int64_t* top_ids, float* top_logprobs,
                                 int32_t* status, void* stream) {
  using namespace pe;
  int rc = check_logits("pe_token_logprobs", logits, ld, rows, vocab, dtype);
  if (rc != PE_OK) return rc;
  PE_REQUIRE(top_k >= 0 && top_k <= LP_MAX_TOP && top_k <= vocab, "pe_token_logprobs: top_k=%d is not within 0..min(%d, %lld)",
             top_k, LP_MAX_TOP, (long long)vocab);
  if (rows == 0) return PE_OK;
  PE_REQUIRE(targets && logprobs && entropy && lse && lse_rest && (top_k == 0 || (top_ids && top_logprobs)),
             "pe_token_logprobs: null pointer");
  const LpArgs a{logits, ld, targets, ignore_index, (int)vocab, top_k, logprobs, entropy, lse, lse_rest, top_ids,
                 top_logprobs, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // 128 threads to a row where the rows fill the GPU several times over: half as much joining and selecting
  // per row (8,192 x 50,368 bf16: 157 us against 165, with the top five 202 against 221; 16,384 x 8,000
  // 73 against 91, 134 against 181).  With fewer rows, or sixteens joined too often for the top, 256
  // (515 x 256,001 fp32: 88 us against 109, with the top five 94 against 254).
  const bool many = rows >= 6 * int64_t(sm_count()) && (top_k == 0 || vocab <= 65536);
  switch (dtype) {
    case PE_BF16: return many ? launch_logprobs<__nv_bfloat16, 128>(a, rows, st) : launch_logprobs<__nv_bfloat16, 256>(a, rows, st);
    case PE_FP16: return many ? launch_logprobs<__half, 128>(a, rows, st) : launch_logprobs<__half, 256>(a, rows, st);
    default: return many ? launch_logprobs<float, 128>(a, rows, st) : launch_logprobs<float, 256>(a, rows, st);
  }
}

extern "C" int pe_token_logprobs_backward(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld,
                                          const int64_t* targets, int64_t ignore_index, const float* lse,
                                          const float* lse_rest, const float* entropy, const float* d_logprobs,
                                          const float* d_entropy, const float* d_lse, void* dlogits, int64_t ld_out, void* stream) {
  using namespace pe;
  int rc = check_logits("pe_token_logprobs_backward", logits, ld, rows, vocab, dtype);
  if (rc == PE_OK) rc = check_logits("pe_token_logprobs_backward", dlogits, ld_out, rows, vocab, dtype);
  if (rc != PE_OK || rows == 0) return rc;
  PE_REQUIRE(targets && lse && lse_rest && entropy, "pe_token_logprobs_backward: null pointer");
  const LpBackArgs a{logits, ld, targets, ignore_index, lse, lse_rest, entropy, d_logprobs, d_entropy, d_lse, dlogits,
                     ld_out, (int)vocab};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case PE_BF16: return launch_logprobs_backward<__nv_bfloat16>(a, rows, st);
    case PE_FP16: return launch_logprobs_backward<__half>(a, rows, st);
    default: return launch_logprobs_backward<float>(a, rows, st);
  }
}
