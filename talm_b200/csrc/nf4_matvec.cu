// Products of a few rows with NF4 weights (the single-token form of a 4-bit projection), with an
// optional LoRA adapter added in the epilogue.
//
//   y[n, o] = fp16( sum_k L[code[o, k]] S[o, k] x[n, k] + bias[o] + s sum_j t[n, j] B[o, j] )
//   t[n, j] = sum_k x[n, k] A[j, k]
//
// L are the 16 levels, S the scale of the block that the flattened weight element o * K + k is in:
// an fp32 absmax, or fp32(fp32(code2[absmax8] * absmax2) + offset2) as in nf4.cu. Products and
// sums are fp32 and the result is rounded once: the weight itself is not rounded to fp16, which
// the dequantised copy of a weight is.
#include "common.cuh"

namespace talm {
namespace nf4v {

constexpr int MAX_ROWS = 32;   // rows of x in one call
constexpr int MAX_RANK = 64;

struct Weight {
  const uint8_t* packed;
  const uint8_t* absmax8;  // null: `absmax` holds fp32 scales
  const float* absmax;
  const float* code;
  const float* absmax2;
  const float* offset2;
  const float* levels;     // null: kNf4Levels
  int64_t row0;            // group-wide index of this weight's first block
  int64_t blocksize, qblock2;
  int64_t n_out, n_in;
  __device__ __forceinline__ float scale(int64_t block) const {
    if (absmax8 == nullptr) return __ldg(absmax + block);
    const int64_t b2 = (row0 + block) / qblock2;
    return __fadd_rn(__fmul_rn(__ldg(code + __ldg(absmax8 + block)), __ldg(absmax2 + b2)),
                     __ldg(offset2 + b2));
  }
};

struct Epilogue {
  const __half* bias;   // null: none
  const float* t;       // [n_rows, rank] or null
  const float* lora_b;  // [n_out, rank]
  int rank;
  float scaling;
};

// t = x A^T: one warp per (row, adapter row).
__global__ void __launch_bounds__(256) adapter_down_kernel(const __half* __restrict__ x,
                                                           int64_t ld_x,
                                                           const float* __restrict__ a,
                                                           int64_t n_in, int n_rows, int rank,
                                                           float* __restrict__ t) {
  const int lane = threadIdx.x & 31;
  const int pair = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (pair >= n_rows * rank) return;
  const int n = pair / rank, j = pair % rank;
  float acc = 0.0f;
  for (int64_t k = lane; k < n_in; k += 32)
    acc = fmaf(__half2float(x[n * ld_x + k]), a[j * n_in + k], acc);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, d);
  if (lane == 0) t[pair] = acc;
}

// Any even row length and block size: one warp per output, a byte (two weights) per lane and
// step, eight rows of x at a time.
__global__ void __launch_bounds__(256) nf4_matvec_any_kernel(const __half* __restrict__ x,
                                                             int64_t ld_x, int n_rows, Weight w,
                                                             Epilogue ep, __half* __restrict__ y,
                                                             int64_t ld_y) {
  __shared__ float lut[16];
  if (threadIdx.x < 16)
    lut[threadIdx.x] = w.levels ? w.levels[threadIdx.x] : kNf4Levels[threadIdx.x];
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int64_t o = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (o >= w.n_out) return;
  for (int n0 = 0; n0 < n_rows; n0 += 8) {
    float acc[8] = {};
    for (int64_t i = lane; i < w.n_in / 2; i += 32) {
      const int64_t e = o * w.n_in + 2 * i;
      const uint32_t byte = w.packed[e >> 1];
      const float s = w.scale(e / w.blocksize);
      const float w0 = lut[byte >> 4] * s, w1 = lut[byte & 15u] * s;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        if (n0 + n < n_rows) {
          const __half* xr = x + (n0 + n) * ld_x + 2 * i;
          acc[n] = fmaf(w0, __half2float(xr[0]), fmaf(w1, __half2float(xr[1]), acc[n]));
        }
      }
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      if (n0 + n >= n_rows) break;
      float extra = 0.0f;
      if (ep.t != nullptr)
        for (int j = lane; j < ep.rank; j += 32)
          extra = fmaf(ep.t[(n0 + n) * ep.rank + j], ep.lora_b[o * ep.rank + j], extra);
      float v = fmaf(ep.scaling, extra, acc[n]);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
      if (lane == 0) {
        if (ep.bias != nullptr) v += __half2float(ep.bias[o]);
        y[(n0 + n) * ld_y + o] = __float2half_rn(v);
      }
    }
  }
}

}  // namespace nf4v
}  // namespace talm

extern "C" {

int talm_nf4_matvec(const uint16_t* x, int64_t ld_x, int64_t n_rows, const uint8_t* packed,
                    const uint8_t* absmax8, const float* absmax, const float* code,
                    const float* absmax2, const float* offset2, const float* levels,
                    int64_t absmax_row0, int64_t w_rows, int64_t w_cols, int64_t blocksize,
                    int64_t qblock2, const uint16_t* bias, const float* lora_a,
                    const float* lora_b, int64_t rank, float scaling, float* down,
                    uint16_t* y, int64_t ld_y, void* stream_) {
  using namespace talm;
  using namespace talm::nf4v;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (n_rows < 0 || n_rows > MAX_ROWS)
    return set_error(TALM_EINVAL, "the few-row product takes 0 to %d rows (got %lld)", MAX_ROWS,
                     (long long)n_rows);
  if (w_rows < 0 || w_cols < 2 || w_cols % 2 != 0)
    return set_error(TALM_EINVAL, "weight rows must be >= 0 and columns even and >= 2");
  if (blocksize < 2 || blocksize % 2 != 0)
    return set_error(TALM_EINVAL, "blocksize must be even and >= 2 (got %lld)",
                     (long long)blocksize);
  if (absmax8 != nullptr && (qblock2 < 1 || absmax_row0 < 0))
    return set_error(TALM_EINVAL, "bad second-level blocks");
  if (rank < 0 || rank > MAX_RANK)
    return set_error(TALM_EINVAL, "adapter rank %lld is not in 0..%d", (long long)rank, MAX_RANK);
  if (ld_x < w_cols || ld_y < w_rows)
    return set_error(TALM_EINVAL, "row strides must cover the rows");
  if (w_cols >= (int64_t{1} << 31) || w_rows >= (int64_t{1} << 31) ||
      (w_rows > 0 && w_cols > (int64_t{1} << 40) / w_rows))
    return set_error(TALM_ERANGE, "weight of %lld x %lld is beyond the kernel's range",
                     (long long)w_rows, (long long)w_cols);
  if (n_rows == 0 || w_rows == 0) return TALM_OK;
  if (!x || !packed || !y || (!absmax8 && !absmax) ||
      (absmax8 && (!code || !absmax2 || !offset2 || !levels)) ||
      (rank > 0 && (!lora_a || !lora_b || !down)))
    return set_error(TALM_EINVAL, "null pointer");
  const Weight w{packed, absmax8, absmax,      code,      absmax2, offset2,
                 levels, absmax_row0, blocksize, qblock2, w_rows,  w_cols};
  const Epilogue ep{reinterpret_cast<const __half*>(bias), rank > 0 ? down : nullptr, lora_b,
                    static_cast<int>(rank), scaling};
  const __half* xh = reinterpret_cast<const __half*>(x);
  if (rank > 0) {
    LaunchTimer timer(TALM_KERNEL_ADAPTER_DOWN, stream);
    const int warps = static_cast<int>(n_rows * rank);
    adapter_down_kernel<<<(warps + 7) / 8, 256, 0, stream>>>(xh, ld_x, lora_a, w_cols,
                                                            static_cast<int>(n_rows),
                                                            static_cast<int>(rank), down);
    const int st = check_launch("adapter down kernel");
    if (st != TALM_OK) return st;
  }
  LaunchTimer timer(TALM_KERNEL_NF4_MATVEC, stream);
  nf4_matvec_any_kernel<<<static_cast<unsigned>((w_rows + 7) / 8), 256, 0, stream>>>(
      xh, ld_x, static_cast<int>(n_rows), w, ep, reinterpret_cast<__half*>(y), ld_y);
  return check_launch("nf4 matvec kernel");
}

}  // extern "C"
