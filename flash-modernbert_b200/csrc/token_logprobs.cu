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
// Top k without a second pass: candidates are pushed into a small shared-memory list as they
// stream by, if they beat the threshold tau, the k-th best so far.  Order is total: a candidate is the
// 64-bit number (value's bits made monotone, complement of the index), so equal values
// rank by lowest index.  When more than 32 threads of a chunk hold a value that beats tau - in the
// first chunk all do - tau is raised first to the k-th best of the threads' own best, which leaves
// at most k threads with anything to push; so a chunk adds a bounded number of candidates whatever
// the data, and the list is cut back to k by counting ranks when it fills up.
#include <algorithm>

#include "pe_host.h"
#include "pe_ptx.cuh"

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

template <int NT>
struct LpShared {
  static constexpr int CAP = 1536;  // list of candidates; a chunk adds at most 16 * LP_CROWD = 512
  LpStat stat[NT / 32];
  LpStat part[LP_MAX_CLUSTER];                       // parts of the cluster's CTAs, in rank 0
  unsigned long long part_top[LP_MAX_CLUSTER * LP_MAX_TOP];
  unsigned long long best[NT];
  unsigned long long list[CAP];
  unsigned long long kept[LP_MAX_TOP];
  unsigned long long tau;
  int count;
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

template <typename E, int NT, bool TOP>
__global__ void __launch_bounds__(NT)
token_logprobs_kernel(const LpArgs a, int cluster) {
  constexpr int N = LogitVec<E>::N;
  constexpr int VECS = 16 / N;  // 16-byte loads per thread and chunk: 16 elements
  constexpr int WARPS = NT / 32;
  __shared__ LpShared<NT> sh;
  const int rank = cluster > 1 ? int(cluster_ctarank()) : 0;
  const int64_t row = blockIdx.x / cluster;
  const E* x = static_cast<const E*>(a.logits) + row * a.ld;
  const int k = a.top_k;
  // Vectors are counted from the 16-byte boundary at or below the row's start; those that stick out
  // of the row (the first and the last at most) are read element by element.
  const int lead = int((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(E));
  const int vecs = (a.vocab + lead + N - 1) / N;
  const int per_cta = (vecs + cluster - 1) / cluster;
  const int v_begin = min(vecs, rank * per_cta), v_end = min(vecs, v_begin + per_cta);

  auto load = [&](int v, float (&f)[N]) {
    const int e0 = v * N - lead;
    if (v < v_end && e0 >= 0 && e0 + N <= a.vocab) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(x + e0));
      const E* p = reinterpret_cast<const E*>(&u);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = logit_f32(p[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        f[i] = v < v_end && e0 + i >= 0 && e0 + i < a.vocab ? logit_f32(x[e0 + i]) : -INFINITY;
    }
  };

  if (TOP && threadIdx.x == 0) {
    sh.tau = 0ull;
    sh.count = 0;
  }
  if (TOP) __syncthreads();

  LpStat st{-INFINITY, 0.f, 0.f};
  float tau_value = -INFINITY;  // value of sh.tau
  unsigned long long tau = 0ull;
  for (int c0 = v_begin; c0 < v_end; c0 += NT * VECS) {
    float f[VECS][N];
#pragma unroll
    for (int i = 0; i < VECS; ++i) load(c0 + i * NT + int(threadIdx.x), f[i]);
    float top = f[0][0];
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) top = lp_max_nan(top, f[i][e]);
    if (!(top <= st.m)) {  // a new maximum (or a NaN): move the sums to it
      const float d = st.m == -INFINITY ? 0.f : st.m - top;
      const float z = lp_ex2(d * 1.4426950408889634f);
      st.w = z > 0.f ? (st.w + st.s * d) * z : 0.f;
      st.s *= z;
      st.m = top;
    }
    const float ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = f[i][e] - ref;
        const float p = lp_ex2(d * 1.4426950408889634f);
        st.s += p;
        st.w = fmaf(p, fmaxf(d, -3.0e38f), st.w);  // 0 * -inf would be NaN
      }
    if (TOP) {
      // the best of this thread's sixteen that beats tau
      unsigned long long best = 0ull;
      if (!(top < tau_value)) {
#pragma unroll
        for (int i = 0; i < VECS; ++i)
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const int id = (c0 + i * NT + int(threadIdx.x)) * N - lead + e;
            const bool real = id >= 0 && id < a.vocab && c0 + i * NT + int(threadIdx.x) < v_end;
            const unsigned long long key = real ? lp_key(f[i][e], uint32_t(id)) : 0ull;
            if (key > tau && key > best) best = key;
          }
      }
      const int holders = __syncthreads_count(best != 0ull);
      if (holders > 0) {
        if (holders > LP_CROWD) {
          sh.best[threadIdx.x] = best;
          __syncthreads();
          if (best != 0ull) {
            int above = 0;
            for (int j = 0; j < NT; ++j) above += sh.best[j] > best;
            if (above == k - 1) sh.tau = best - 1;  // everything from the k-th best on may push
          }
          __syncthreads();
          tau = sh.tau;
        }
        if (best > tau) {
#pragma unroll
          for (int i = 0; i < VECS; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const int id = (c0 + i * NT + int(threadIdx.x)) * N - lead + e;
              const bool real = id >= 0 && id < a.vocab && c0 + i * NT + int(threadIdx.x) < v_end;
              const unsigned long long key = real ? lp_key(f[i][e], uint32_t(id)) : 0ull;
              if (key > tau) sh.list[atomicAdd(&sh.count, 1)] = key;
            }
        }
        __syncthreads();
        const int n = sh.count;
        if (n > LpShared<NT>::CAP - 16 * LP_CROWD) {  // the next chunk might not fit: keep the k best
          lp_select<NT>(sh.list, n, k, sh.kept);
          __syncthreads();
          for (int i = threadIdx.x; i < k; i += NT) sh.list[i] = sh.kept[i];
          if (threadIdx.x == 0) {
            sh.count = k;
            sh.tau = sh.kept[k - 1];
          }
          __syncthreads();
          tau = sh.tau;
        }
        tau_value = tau != 0ull ? lp_key_value(tau) : -INFINITY;
        if (tau_value != tau_value) tau_value = INFINITY;  // only NaN can still beat a NaN: none does by value
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
  if (threadIdx.x == 0) {
    st = sh.stat[0];
    for (int i = 1; i < WARPS; ++i) st = lp_join(st, sh.stat[i]);
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
    const int64_t t = a.targets[row];
    float lp = 0.f;
    if (t >= 0 && t < a.vocab) lp = t == a.ignore_index ? 0.f : (logit_f32(x[t]) - lse) - rest;
    else if (t != a.ignore_index) set_status(a.status, ST_BAD_TARGET);
    a.logprobs[row] = lp;
    sh.stat[0].m = lse;
    sh.stat[0].s = rest;
  }
  if (TOP) {
    __syncthreads();
    if (threadIdx.x < k) {
      const unsigned long long key = sh.kept[threadIdx.x];
      a.top_ids[row * k + threadIdx.x] = int64_t(0xffffffffu - uint32_t(key));
      a.top_logprobs[row * k + threadIdx.x] = (lp_key_value(key) - sh.stat[0].m) - sh.stat[0].s;
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

// Grid (chunks of the vocabulary, rows).  VECTOR: input and output rows lie alike relative to
// 16-byte boundaries, so a thread moves 16 bytes at a time.
template <typename E, bool VECTOR>
__global__ void __launch_bounds__(256)
token_logprobs_backward_kernel(const LpBackArgs a, int64_t rows) {
  constexpr int N = VECTOR ? LogitVec<E>::N : 1;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const E* x = static_cast<const E*>(a.logits) + row * a.ld;
    E* dx = static_cast<E*>(a.dlogits) + row * a.ld_out;
    const int64_t t = a.targets[row];
    const bool kept = t >= 0 && t < a.vocab && t != a.ignore_index;
    const float g = kept && a.d_logprobs != nullptr ? a.d_logprobs[row] : 0.f;
    const float h = a.d_entropy != nullptr ? a.d_entropy[row] : 0.f;
    const float z = a.d_lse != nullptr ? a.d_lse[row] : 0.f;
    const bool nothing = g == 0.f && h == 0.f && z == 0.f;  // an ignored row: zeros, nothing read
    const float lse = a.lse[row], rest = a.lse_rest[row], ent = a.entropy[row];
    const int lead = VECTOR ? int((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(E)) : 0;
    const int vecs = (a.vocab + lead + N - 1) / N;
    for (int v = blockIdx.x * blockDim.x + threadIdx.x; v < vecs; v += gridDim.x * blockDim.x) {
      const int e0 = v * N - lead;
      const bool whole = e0 >= 0 && e0 + N <= a.vocab;
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      E* q = reinterpret_cast<E*>(&u);
      if (!nothing) {
        if (VECTOR && whole) {
          u = *reinterpret_cast<const uint4*>(x + e0);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (e0 + i >= 0 && e0 + i < a.vocab) q[i] = x[e0 + i];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float lp = (logit_f32(q[i]) - lse) - rest;
          const float p = lp_ex2(lp * 1.4426950408889634f);
          // p (z - g - h (log p + H)); a token of probability zero has no part in the entropy
          float d = p * (z - g - (p == 0.f ? 0.f : h * (lp + ent)));
          if (e0 + i == t) d += g;
          logit_put(q + i, d);
        }
      }
      if (VECTOR && whole) {
        *reinterpret_cast<uint4*>(dx + e0) = u;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (e0 + i >= 0 && e0 + i < a.vocab) dx[e0 + i] = q[i];
      }
    }
  }
}

template <typename E>
static int launch_logprobs(const LpArgs& a, int64_t rows, cudaStream_t st) {
  constexpr int NT = 256;
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
  const int64_t chunks = (a.vocab + int64_t(256) * per_thread * 4 - 1) / (int64_t(256) * per_thread * 4);
  const dim3 grid((unsigned)chunks, (unsigned)std::min<int64_t>(rows, 65535));
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
  switch (dtype) {
    case PE_BF16: return launch_logprobs<__nv_bfloat16>(a, rows, st);
    case PE_FP16: return launch_logprobs<__half>(a, rows, st);
    default: return launch_logprobs<float>(a, rows, st);
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
