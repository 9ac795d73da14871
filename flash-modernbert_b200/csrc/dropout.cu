// Dropout whose mask is never stored: y = keep ? x / (1 - p) : 0, optionally plus a residual, with
// `keep` a function of (seed, position, element) alone, so the backward pass recomputes it.
//
// Generator: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011).  One call gives 128 bits for EIGHT elements, 16 bits each: element e uses
// field e % 8 (low half of word 0 first) of the block with counter position + e / 8 and key = seed,
// and is kept if the field is at least round(p * 65536).  At 32 bits per element the generator
// alone would take 20 wide multiplies per four elements; at 16 it stays below what memory
// allows, and a drop probability in steps of 2^-16 is finer than anyone sets it.  Survivors
// are scaled by what that rounded probability makes of them, so the expectation is exact.
#include <algorithm>
#include <type_traits>

#include "pe_host.h"
#include "pe_vec.cuh"

#include <cuda_fp16.h>

namespace pe {

struct PhiloxKeys {
  uint32_t k0, k1;
};

__device__ __forceinline__ uint4 philox4x32_10(uint64_t counter, PhiloxKeys k) {
  uint32_t c0 = uint32_t(counter), c1 = uint32_t(counter >> 32), c2 = 0, c3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = uint64_t(c0) * 0xD2511F53u, b = uint64_t(c2) * 0xCD9E8D57u;
    c0 = uint32_t(b >> 32) ^ c1 ^ k.k0;
    c1 = uint32_t(b);
    c2 = uint32_t(a >> 32) ^ c3 ^ k.k1;
    c3 = uint32_t(a);
    k.k0 += 0x9E3779B9u;
    k.k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Eight consecutive elements: as they lie in memory, and as fp32 (back with one rounding to nearest even).
template <typename E>
struct Octet {
  static constexpr int VECS = int(sizeof(E)) / 2;
  uint4 u[VECS];
  __device__ __forceinline__ void load(const E* p) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) u[i] = ld_stream(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void store(E* p) const {
#pragma unroll
    for (int i = 0; i < VECS; ++i) reinterpret_cast<uint4*>(p)[i] = u[i];
  }
  __device__ __forceinline__ void unpack(float (&f)[8]) const {
    if constexpr (std::is_same<E, float>::value) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = reinterpret_cast<const float*>(u)[i];
    } else if constexpr (std::is_same<E, __half>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(reinterpret_cast<const __half2*>(u)[i]);
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
      }
    } else {
      unpack8(u[0], f);
    }
  }
  __device__ __forceinline__ void pack(const float (&f)[8]) {
    if constexpr (std::is_same<E, float>::value) {
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<float*>(u)[i] = f[i];
    } else if constexpr (std::is_same<E, __half>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<__half2*>(u)[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    } else {
      u[0] = pack8(f);
    }
  }
};
__device__ __forceinline__ float element_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float element_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float element_f32(float v) { return v; }
__device__ __forceinline__ void element_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void element_put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void element_put(float* p, float v) { *p = v; }

// y of eight elements, in place of x.  A 16-bit field is compared where it stands: the high half of a word
// is at least t if the word is at least t 2^16, the low half after a shift.  Dropped elements are
// selected away, not multiplied by zero, so a NaN or infinity among them leaves no trace.
template <bool RESIDUAL>
__device__ __forceinline__ void dropout_octet(float (&v)[8], const float (&r)[8], uint4 bits, uint32_t threshold_hi,
                                              bool all, float scale) {
  const uint32_t word[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = __fmul2_rn(make_float2(v[2 * i], v[2 * i + 1]), make_float2(scale, scale));
    v[2 * i] = !all && (word[i] << 16) >= threshold_hi ? u.x : 0.f;
    v[2 * i + 1] = !all && word[i] >= threshold_hi ? u.y : 0.f;
    if (RESIDUAL) {
      v[2 * i] += r[2 * i];
      v[2 * i + 1] += r[2 * i + 1];
    }
  }
}

// VECTOR: every pointer is 16-byte aligned, whole octets move in 16-byte pieces (the last, partial one
// element by element).  threshold_hi: the drop threshold times 2^16; `all`: everything is dropped.
// Eight blocks per SM, all 64 warps, hide the generator's latency; two octets per thread and step, or the next
// octet's loads issued a step ahead, cost the registers that the warps need and were slower
// (306,851 x 768 bf16: 193 us as it is, 196 - 212 us so).
template <typename E, bool RESIDUAL, bool VECTOR>
__global__ void __launch_bounds__(256, 8)
dropout_kernel(const E* x, const E* residual, E* y, int64_t n, uint32_t threshold_hi, bool all, float scale,
               const int64_t* __restrict__ rng, int64_t* __restrict__ rng_used) {
  const uint64_t seed = uint64_t(__ldg(rng)), position = uint64_t(__ldg(rng + 1));
  if (rng_used != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
    rng_used[0] = int64_t(seed);
    rng_used[1] = int64_t(position);
  }
  const PhiloxKeys keys{uint32_t(seed), uint32_t(seed >> 32)};
  const int64_t octets = (n + 7) >> 3;
  for (int64_t o = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; o < octets;
       o += int64_t(gridDim.x) * blockDim.x) {
    const int64_t at = o * 8;
    const int count = int(n - at < 8 ? n - at : 8);
    const bool whole = VECTOR && count == 8;
    float v[8], r[8];
    if (whole) {
      Octet<E> c;
      c.load(x + at);
      c.unpack(v);
      if (RESIDUAL) {
        c.load(residual + at);
        c.unpack(r);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = i < count ? element_f32(x[at + i]) : 0.f;
        r[i] = RESIDUAL && i < count ? element_f32(residual[at + i]) : 0.f;
      }
    }
    dropout_octet<RESIDUAL>(v, r, philox4x32_10(position + uint64_t(o), keys), threshold_hi, all, scale);
    if (whole) {
      Octet<E> c;
      c.pack(v);
      c.store(y + at);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < count) element_put(y + at + i, v[i]);
    }
  }
}

template <typename E>
static int launch_dropout(const void* x, const void* residual, void* y, int64_t n, uint32_t threshold, float scale,
                          const int64_t* rng, int64_t* rng_used, cudaStream_t st) {
  const bool vec = (((uintptr_t)x | (uintptr_t)y | (uintptr_t)residual) & 15) == 0;
  const int64_t octets = (n + 7) / 8;
  // Blocks that come and go balance the SMs better than eight that stay (16-bit: 64 per SM 193 us, 8 per SM
  // 208 us, one octet per thread 237 us), fp32, with half the generator's work per byte, the more the better.
  const int per_sm = sizeof(E) == 4 ? 256 : 64;
  const unsigned blocks = (unsigned)std::min<int64_t>((octets + 255) / 256, int64_t(sm_count()) * per_sm);
  auto kern = residual != nullptr ? (vec ? dropout_kernel<E, true, true> : dropout_kernel<E, true, false>)
                                  : (vec ? dropout_kernel<E, false, true> : dropout_kernel<E, false, false>);
  kern<<<blocks, 256, 0, st>>>(static_cast<const E*>(x), static_cast<const E*>(residual), static_cast<E*>(y), n,
                               threshold << 16, threshold >= 65536u, scale, rng, rng_used);
  PE_LAUNCH_CHECK("dropout_kernel");
  return PE_OK;
}

}  // namespace pe

extern "C" int pe_dropout(const void* x, const void* residual, int dtype, int64_t n, double p,
                          const int64_t* rng, int64_t* rng_used, void* y, void* stream) {
  using namespace pe;
  PE_REQUIRE(n >= 0 && n <= (int64_t(1) << 62), "pe_dropout: %lld elements out of range", (long long)n);
  PE_REQUIRE(p >= 0.0 && p <= 1.0, "pe_dropout: p=%g is not a probability", p);
  PE_REQUIRE(rng != nullptr && ((uintptr_t)rng & 7) == 0, "pe_dropout: rng is NULL or unaligned");
  PE_REQUIRE(dtype == PE_BF16 || dtype == PE_FP16 || dtype == PE_FP32, "pe_dropout: unknown type %d", dtype);
  if (n == 0) {
    if (rng_used != nullptr)
      PE_CUDA(cudaMemcpyAsync(rng_used, rng, 16, cudaMemcpyDeviceToDevice, static_cast<cudaStream_t>(stream)));
    return PE_OK;
  }
  PE_REQUIRE(x && y, "pe_dropout: null pointer");
  const uintptr_t elt = dtype == PE_FP32 ? 4 : 2;
  PE_REQUIRE((((uintptr_t)x | (uintptr_t)y | (uintptr_t)residual) & (elt - 1)) == 0, "pe_dropout: unaligned pointer");
  const uint32_t threshold = (uint32_t)(p * 65536.0 + 0.5);
  const float scale = threshold >= 65536u ? 0.f : (float)(65536.0 / (65536.0 - threshold));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case PE_BF16: return launch_dropout<__nv_bfloat16>(x, residual, y, n, threshold, scale, rng, rng_used, st);
    case PE_FP16: return launch_dropout<__half>(x, residual, y, n, threshold, scale, rng, rng_used, st);
    default: return launch_dropout<float>(x, residual, y, n, threshold, scale, rng, rng_used, st);
  }
}
