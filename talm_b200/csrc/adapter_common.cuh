// Parts that the adapter's kernels share: the dropout's generator and masks, and the splits of fp32
// operands.
#pragma once

#include "common.cuh"

namespace talm {
namespace adapter {

constexpr int MAX_RANK = 64;
constexpr int DROP_ALL = 32768;

struct Dropout {
  const long long* seed;  // device; null: no dropout (drop must be 0)
  uint32_t drop;          // 0..32768
  float factor;           // 32768 / (32768 - drop), 0 when everything is dropped
};

// WIDE: one 64-bit product instead of its two halves. Fewer instructions, which counts where the
// generator runs beside HBM at full rate, but a longer wait for each: dropout of 16384 x 8960 bf16
// (forward and backward) 206.7 -> 200.1 us, of 2048 x 1536 fp16 6.5 -> 6.9, the branch 306 -> 310.
template <bool WIDE>
__device__ __forceinline__ void philox_round(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
  uint32_t h0, l0, h1, l1;
  if (WIDE) {
    const uint64_t p0 = static_cast<uint64_t>(c[0]) * 0xD2511F53u;
    const uint64_t p1 = static_cast<uint64_t>(c[2]) * 0xCD9E8D57u;
    h0 = static_cast<uint32_t>(p0 >> 32), l0 = static_cast<uint32_t>(p0);
    h1 = static_cast<uint32_t>(p1 >> 32), l1 = static_cast<uint32_t>(p1);
  } else {
    h0 = __umulhi(c[0], 0xD2511F53u), l0 = c[0] * 0xD2511F53u;
    h1 = __umulhi(c[2], 0xCD9E8D57u), l1 = c[2] * 0xCD9E8D57u;
  }
  c[0] = h1 ^ c[1] ^ k0;
  c[1] = l1;
  c[2] = h0 ^ c[3] ^ k1;
  c[3] = l0;
}

// The four words of group q (elements 8 q .. 8 q + 7).
template <bool WIDE = false>
__device__ __forceinline__ void philox(uint64_t q, uint64_t key, uint32_t (&c)[4]) {
  uint32_t k0 = static_cast<uint32_t>(key), k1 = static_cast<uint32_t>(key >> 32);
  c[0] = static_cast<uint32_t>(q);
  c[1] = static_cast<uint32_t>(q >> 32);
  c[2] = 0;
  c[3] = 0;
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    philox_round<WIDE>(c, k0, k1);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

__device__ __forceinline__ bool kept(const uint32_t (&c)[4], int i, uint32_t drop) {
  return ((c[i >> 1] >> (16 * (i & 1))) & 0x7FFFu) >= drop;
}

// All ones in each half of the result whose element is kept: the 15-bit draws of a word plus
// 0x8000 - drop carry into bit 15 of their own half exactly when they reach the threshold, and the
// permutation copies that bit over the half.
__device__ __forceinline__ uint32_t keep_mask2(uint32_t word, uint32_t bias2) {
  const uint32_t sum = (word & 0x7FFF7FFFu) + bias2;
  uint32_t mask;
  asm("prmt.b32 %0, %1, 0, 0xBB99;" : "=r"(mask) : "r"(sum));
  return mask;
}
__device__ __forceinline__ uint32_t keep_bias2(uint32_t drop) {
  return (0x8000u - drop) * 0x10001u;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
// The two bf16 parts of a pair.
__device__ __forceinline__ void split_bf16(float v0, float v1, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16(v0, v1);
  lo = pack_bf16(v0 - __uint_as_float(hi << 16), v1 - __uint_as_float(hi & 0xFFFF0000u));
}
// The two fp16 parts of a pair that has been scaled.
__device__ __forceinline__ void split_f16(float v0, float v1, uint32_t& hi, uint32_t& lo) {
  hi = pack_half2(v0, v1);
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  lo = pack_half2(v0 - h.x, v1 - h.y);
}
// The kernels of one branch follow one another closely: each may start its set-up while the one
// before it ends (programmatic stream serialization) and waits in grid_dependency_wait before it
// touches global memory.
template <class... Params, class... Args>
int launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, int smem,
                     cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
  if (e != cudaSuccess) return set_error(TALM_ECUDA, "adapter kernel: %s", cudaGetErrorString(e));
  return TALM_OK;
}

}  // namespace adapter
}  // namespace talm
