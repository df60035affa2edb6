// Counter-based dropout and the training form of a LoRA adapter (the branch beside a frozen
// projection), forward and backward.
//
//   dropout: y[e] = keep(e) ? x[e] * f : 0,  f = 32768 / (32768 - d)
//   branch:  xd = dropout(x), t = xd A^T, y = fp16(base + s t B^T)
//            dt = s g B, dB = s g^T t, dA = dt^T xd, dx = fp16(keep f (dt A))
//
// The mask is never stored: keep(e) comes from Philox4x32 (Salmon, Moraes, Dror, Shaw: "Parallel
// random numbers: as easy as 1, 2, 3", 2011) with 7 rounds, the fewest that the paper's
// statistical tests pass. The key is the call's 64-bit seed, read from device memory so that a
// captured graph draws a new mask on every replay; the counter is e / 8 for element e in row-major
// order, and the eight 16-bit halves of the four result words belong to the eight elements. The
// low 15 bits u of its half keep an element when u >= d, d = round(p * 32768): 15 bits let two
// elements be compared in one 32-bit register without a carry between them.
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

__device__ __forceinline__ void philox_round(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
  const uint32_t h0 = __umulhi(c[0], 0xD2511F53u), l0 = c[0] * 0xD2511F53u;
  const uint32_t h1 = __umulhi(c[2], 0xCD9E8D57u), l1 = c[2] * 0xCD9E8D57u;
  c[0] = h1 ^ c[1] ^ k0;
  c[1] = l1;
  c[2] = h0 ^ c[3] ^ k1;
  c[3] = l0;
}

// The four words of group q (elements 8 q .. 8 q + 7).
__device__ __forceinline__ void philox(uint64_t q, uint64_t key, uint32_t (&c)[4]) {
  uint32_t k0 = static_cast<uint32_t>(key), k1 = static_cast<uint32_t>(key >> 32);
  c[0] = static_cast<uint32_t>(q);
  c[1] = static_cast<uint32_t>(q >> 32);
  c[2] = 0;
  c[3] = 0;
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    philox_round(c, k0, k1);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

__device__ __forceinline__ bool kept(const uint32_t (&c)[4], int i, uint32_t drop) {
  return ((c[i >> 1] >> (16 * (i & 1))) & 0x7FFFu) >= drop;
}

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
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

__device__ __forceinline__ uint32_t scale2(uint32_t v, float f, __half) {
  const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&v));
  return pack_half2(p.x * f, p.y * f);
}
__device__ __forceinline__ uint32_t scale2(uint32_t v, float f, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(__uint_as_float(v << 16) * f,
                                                 __uint_as_float(v & 0xFFFF0000u) * f);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// The flattened tensor on 16-byte boundaries: a thread takes UNROLL groups of eight elements, their
// loads first.
template <class T, int UNROLL>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, int64_t n,
                                                      Dropout d, T* __restrict__ y) {
  constexpr int V = sizeof(T) == 4 ? 2 : 1;  // 16-byte pieces of a group
  const uint64_t key = static_cast<uint64_t>(__ldg(d.seed));
  const uint32_t bias2 = keep_bias2(d.drop);
  const int64_t n_groups = n >> 3;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * (256 * UNROLL);
  for (int64_t q0 = static_cast<int64_t>(blockIdx.x) * (256 * UNROLL) + threadIdx.x;
       q0 < n_groups; q0 += stride) {
    uint4 v[UNROLL][V];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (q0 + u * 256 < n_groups)
          v[u][i] = __ldg(reinterpret_cast<const uint4*>(x) + (q0 + u * 256) * V + i);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int64_t q = q0 + u * 256;
      if (q >= n_groups) break;
      uint32_t c[4];
      philox(static_cast<uint64_t>(q), key, c);
      uint4* out = reinterpret_cast<uint4*>(y) + q * V;
      if constexpr (V == 1) {
        const uint4 w = v[u][0];
        out[0] = make_uint4(scale2(w.x, d.factor, T()) & keep_mask2(c[0], bias2),
                            scale2(w.y, d.factor, T()) & keep_mask2(c[1], bias2),
                            scale2(w.z, d.factor, T()) & keep_mask2(c[2], bias2),
                            scale2(w.w, d.factor, T()) & keep_mask2(c[3], bias2));
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const uint32_t w[4] = {v[u][i].x, v[u][i].y, v[u][i].z, v[u][i].w};
          uint32_t r[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            r[k] = kept(c, 4 * i + k, d.drop) ? __float_as_uint(__uint_as_float(w[k]) * d.factor)
                                              : 0u;
          out[i] = make_uint4(r[0], r[1], r[2], r[3]);
        }
      }
    }
  }
  // the elements behind the last whole group
  const int tail = static_cast<int>(n & 7);
  if (tail != 0 && blockIdx.x == 0 && threadIdx.x < tail) {
    uint32_t c[4];
    philox(static_cast<uint64_t>(n_groups), key, c);
    const int64_t e = 8 * n_groups + threadIdx.x;
    y[e] = kept(c, threadIdx.x, d.drop) ? from_f32<T>(to_f32(x[e]) * d.factor) : from_f32<T>(0.0f);
  }
}

// Any strides and alignment: one thread per group of eight elements in row-major order.
template <class T>
__global__ void __launch_bounds__(256) dropout_rows_kernel(const T* __restrict__ x, int64_t ld_x,
                                                           int64_t n_cols, int64_t n, Dropout d,
                                                           T* __restrict__ y) {
  const uint64_t key = static_cast<uint64_t>(*d.seed);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t q = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; 8 * q < n;
       q += stride) {
    uint32_t c[4];
    philox(static_cast<uint64_t>(q), key, c);
    int64_t row = 8 * q / n_cols, col = 8 * q - row * n_cols;
    for (int i = 0; i < 8; ++i) {
      const int64_t e = 8 * q + i;
      if (e >= n) break;
      const float v = to_f32(x[row * ld_x + col]);
      y[e] = kept(c, i, d.drop) ? from_f32<T>(v * d.factor) : from_f32<T>(0.0f);
      if (++col == n_cols) {
        col = 0;
        ++row;
      }
    }
  }
}

template <class T>
int run_dropout(const void* x_, int64_t ld_x, int64_t n_rows, int64_t n_cols, const Dropout& d,
                void* y_, cudaStream_t stream) {
  const T* x = static_cast<const T*>(x_);
  T* y = static_cast<T*>(y_);
  const int64_t n = n_rows * n_cols;
  const int sms = current_sm_count();
  if (sms <= 0) return set_error(TALM_ENODEV, "no CUDA device");
  LaunchTimer timer(TALM_KERNEL_DROPOUT, stream);
  const bool flat = ld_x == n_cols || n_rows == 1;
  const int64_t cap = int64_t{sms} * 8;
  if (flat && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0) {
    constexpr int UNROLL = sizeof(T) == 4 ? 2 : 4;
    const int64_t want = (n / 8 + 256 * UNROLL - 1) / (256 * UNROLL);
    const int64_t grid = want < 1 ? 1 : want < cap ? want : cap;
    dropout_kernel<T, UNROLL><<<static_cast<unsigned>(grid), 256, 0, stream>>>(x, n, d, y);
  } else {
    const int64_t want = (n + 2047) / 2048;
    dropout_rows_kernel<<<static_cast<unsigned>(want < cap ? want : cap), 256, 0, stream>>>(
        x, ld_x, n_cols, n, d, y);
  }
  return check_launch("dropout kernel");
}

// ------------------------------------------------------------------------------------------
// the branch
// ------------------------------------------------------------------------------------------
struct Shape {
  int64_t n_rows, n_in, n_out;
  int rank;
};

// The eight dropped-out inputs of group (row n, columns k .. k + 7), without the factor.
__device__ __forceinline__ void masked8(const __half* x, int64_t ld_x, int64_t n, int64_t k,
                                        int64_t n_in, uint64_t key, const Dropout& d,
                                        float (&v)[8]) {
  const uint4 raw = __ldg(reinterpret_cast<const uint4*>(x + n * ld_x + k));
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
  if (d.drop == 0) return;
  uint32_t c[4];
  philox(static_cast<uint64_t>((n * n_in + k) >> 3), key, c);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (!kept(c, i, d.drop)) v[i] = 0.0f;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// t[n, j] = f sum_k keep x[n, k] A[j, k]: one warp per row, 16 adapter rows per pass
__global__ void __launch_bounds__(256) down_kernel(const __half* __restrict__ x, int64_t ld_x,
                                                   const float* __restrict__ a, Shape s,
                                                   Dropout d, float* __restrict__ t) {
  const int lane = threadIdx.x & 31;
  const int64_t n = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (n >= s.n_rows) return;
  const uint64_t key = d.drop ? static_cast<uint64_t>(*d.seed) : 0;
  for (int j0 = 0; j0 < s.rank; j0 += 16) {
    float acc[16] = {};
    for (int64_t k = 8 * lane; k < s.n_in; k += 256) {
      float v[8];
      masked8(x, ld_x, n, k, s.n_in, key, d, v);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j0 + j < s.rank)
          for (int i = 0; i < 8; ++i) acc[j] = fmaf(v[i], a[(j0 + j) * s.n_in + k + i], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float v = warp_sum(acc[j]);
      if (lane == 0 && j0 + j < s.rank) t[n * s.rank + j0 + j] = v * d.factor;
    }
  }
}

// y = fp16(base + s t B^T): one thread per output
__global__ void __launch_bounds__(256) up_kernel(const __half* __restrict__ base, int64_t ld_base,
                                                 const float* __restrict__ t,
                                                 const float* __restrict__ b, Shape s,
                                                 float scaling, __half* __restrict__ y) {
  const int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (e >= s.n_rows * s.n_out) return;
  const int64_t n = e / s.n_out, o = e % s.n_out;
  float acc = 0.0f;
  for (int j = 0; j < s.rank; ++j) acc = fmaf(t[n * s.rank + j], b[o * s.rank + j], acc);
  y[e] = __float2half_rn(fmaf(scaling, acc, __half2float(base[n * ld_base + o])));
}

// dt[n, j] = s sum_o g[n, o] B[o, j]: one warp per row
__global__ void __launch_bounds__(256) grad_t_kernel(const __half* __restrict__ g, int64_t ld_g,
                                                     const float* __restrict__ b, Shape s,
                                                     float scaling, float* __restrict__ dt) {
  const int lane = threadIdx.x & 31;
  const int64_t n = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (n >= s.n_rows) return;
  for (int j0 = 0; j0 < s.rank; j0 += 16) {
    float acc[16] = {};
    for (int64_t o = lane; o < s.n_out; o += 32) {
      const float v = __half2float(g[n * ld_g + o]);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j0 + j < s.rank) acc[j] = fmaf(v, b[o * s.rank + j0 + j], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float v = warp_sum(acc[j]);
      if (lane == 0 && j0 + j < s.rank) dt[n * s.rank + j0 + j] = v * scaling;
    }
  }
}

// dB[o, j] = s sum_n g[n, o] t[n, j]: one thread per element; the sum over the rows is made of
// sums over 128 rows, so that a long one does not lose its low bits
__global__ void __launch_bounds__(256) grad_b_kernel(const __half* __restrict__ g, int64_t ld_g,
                                                     const float* __restrict__ t, Shape s,
                                                     float scaling, float* __restrict__ db) {
  const int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (e >= s.n_out * s.rank) return;
  const int64_t j = e / s.n_out, o = e % s.n_out;
  float total = 0.0f;
  for (int64_t n0 = 0; n0 < s.n_rows; n0 += 128) {
    float part = 0.0f;
    for (int64_t n = n0; n < n0 + 128 && n < s.n_rows; ++n)
      part = fmaf(__half2float(g[n * ld_g + o]), t[n * s.rank + j], part);
    total += part;
  }
  db[o * s.rank + j] = total * scaling;
}

// dA[j, k] = f sum_n dt[n, j] keep x[n, k]: one thread per adapter row and eight columns
__global__ void __launch_bounds__(256) grad_a_kernel(const __half* __restrict__ x, int64_t ld_x,
                                                     const float* __restrict__ dt, Shape s,
                                                     Dropout d, float* __restrict__ da) {
  const int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t chunks = s.n_in / 8;
  if (e >= chunks * s.rank) return;
  const int64_t j = e / chunks, k = (e % chunks) * 8;
  const uint64_t key = d.drop ? static_cast<uint64_t>(*d.seed) : 0;
  float total[8] = {};
  for (int64_t n0 = 0; n0 < s.n_rows; n0 += 128) {
    float part[8] = {};
    for (int64_t n = n0; n < n0 + 128 && n < s.n_rows; ++n) {
      float v[8];
      masked8(x, ld_x, n, k, s.n_in, key, d, v);
      const float w = dt[n * s.rank + j];
      for (int i = 0; i < 8; ++i) part[i] = fmaf(v[i], w, part[i]);
    }
    for (int i = 0; i < 8; ++i) total[i] += part[i];
  }
  for (int i = 0; i < 8; ++i) da[j * s.n_in + k + i] = total[i] * d.factor;
}

// dx[n, k] = fp16(keep f sum_j dt[n, j] A[j, k]): one thread per eight columns of a row
__global__ void __launch_bounds__(256) grad_x_kernel(const float* __restrict__ dt,
                                                     const float* __restrict__ a, Shape s,
                                                     Dropout d, __half* __restrict__ dx) {
  const int64_t q = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (8 * q >= s.n_rows * s.n_in) return;
  const int64_t n = 8 * q / s.n_in, k = 8 * q % s.n_in;
  float acc[8] = {};
  for (int j = 0; j < s.rank; ++j) {
    const float w = dt[n * s.rank + j];
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, a[j * s.n_in + k + i], acc[i]);
  }
  uint32_t c[4] = {};
  if (d.drop) philox(static_cast<uint64_t>(q), static_cast<uint64_t>(*d.seed), c);
  for (int i = 0; i < 8; ++i)
    dx[8 * q + i] = __float2half_rn(kept(c, i, d.drop) ? acc[i] * d.factor : 0.0f);
}

int check_dropout(int64_t drop, const int64_t* seed, Dropout* d) {
  if (drop < 0 || drop > DROP_ALL)
    return set_error(TALM_EINVAL, "drop threshold %lld is not in 0..%d", (long long)drop,
                     DROP_ALL);
  if (drop > 0 && seed == nullptr) return set_error(TALM_EINVAL, "dropout without a seed");
  d->seed = reinterpret_cast<const long long*>(seed);
  d->drop = static_cast<uint32_t>(drop);
  d->factor = drop < DROP_ALL ? static_cast<float>(32768.0 / static_cast<double>(DROP_ALL - drop))
                              : 0.0f;
  return TALM_OK;
}

int check_shape(int64_t n_rows, int64_t n_in, int64_t n_out, int64_t rank) {
  if (n_rows < 0) return set_error(TALM_EINVAL, "negative row count");
  if (n_in < 8 || n_in % 8 != 0 || n_out < 8 || n_out % 8 != 0)
    return set_error(TALM_EINVAL, "the branch's widths must be multiples of 8 (got %lld, %lld)",
                     (long long)n_in, (long long)n_out);
  if (rank < 1 || rank > MAX_RANK)
    return set_error(TALM_EINVAL, "adapter rank %lld is not in 1..%d", (long long)rank, MAX_RANK);
  if (n_rows >= (int64_t{1} << 31) || n_in >= (int64_t{1} << 24) || n_out >= (int64_t{1} << 24))
    return set_error(TALM_ERANGE, "sizes beyond the branch kernels' range");
  return TALM_OK;
}

bool rows_ok(const void* p, int64_t ld, int64_t cols) {
  return ld >= cols && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

unsigned blocks(int64_t threads) { return static_cast<unsigned>((threads + 255) / 256); }

}  // namespace adapter
}  // namespace talm

extern "C" {

int talm_dropout(const void* x, int64_t ld_x, int64_t n_rows, int64_t n_cols, int dtype,
                 const int64_t* seed, int64_t drop, void* y, void* stream_) {
  using namespace talm;
  using namespace talm::adapter;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  Dropout d;
  const int st = check_dropout(drop, seed, &d);
  if (st != TALM_OK) return st;
  if (n_rows < 0 || n_cols < 0 || ld_x < n_cols)
    return set_error(TALM_EINVAL, "bad sizes or a row stride shorter than the row");
  if (dtype != TALM_DTYPE_F16 && dtype != TALM_DTYPE_BF16 && dtype != TALM_DTYPE_F32)
    return set_error(TALM_EINVAL, "dtype %d is not a TALM_DTYPE_* value", dtype);
  if (n_rows == 0 || n_cols == 0) return TALM_OK;
  if (n_cols > (int64_t{1} << 48) / n_rows) return set_error(TALM_ERANGE, "too many elements");
  if (!x || !y || !seed) return set_error(TALM_EINVAL, "null pointer");
  if (dtype == TALM_DTYPE_F16) return run_dropout<__half>(x, ld_x, n_rows, n_cols, d, y, stream);
  if (dtype == TALM_DTYPE_BF16)
    return run_dropout<__nv_bfloat16>(x, ld_x, n_rows, n_cols, d, y, stream);
  return run_dropout<float>(x, ld_x, n_rows, n_cols, d, y, stream);
}

int talm_lora_sizes(int64_t n_rows, int64_t n_in, int64_t n_out, int64_t rank, size_t* saved,
                    size_t* backward_ws) {
  using namespace talm;
  const int st = adapter::check_shape(n_rows, n_in, n_out, rank);
  if (st != TALM_OK) return st;
  if (!saved || !backward_ws) return set_error(TALM_EINVAL, "null pointer");
  *saved = static_cast<size_t>(n_rows * rank) * 4;
  *backward_ws = static_cast<size_t>(n_rows * rank) * 4;
  return TALM_OK;
}

int talm_lora_forward(const uint16_t* x, int64_t ld_x, const uint16_t* base, int64_t ld_base,
                      const float* lora_a, const float* lora_b, int64_t n_rows, int64_t n_in,
                      int64_t n_out, int64_t rank, float scaling, const int64_t* seed,
                      int64_t drop, uint16_t* y, void* saved, size_t saved_bytes, void* stream_) {
  using namespace talm;
  using namespace talm::adapter;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  Dropout d;
  int st = check_shape(n_rows, n_in, n_out, rank);
  if (st == TALM_OK) st = check_dropout(drop, seed, &d);
  if (st != TALM_OK) return st;
  size_t need = 0, need_ws = 0;
  talm_lora_sizes(n_rows, n_in, n_out, rank, &need, &need_ws);
  if (n_rows == 0) return TALM_OK;
  if (!x || !base || !lora_a || !lora_b || !y || !saved)
    return set_error(TALM_EINVAL, "null pointer");
  if (!rows_ok(x, ld_x, n_in) || !rows_ok(base, ld_base, n_out) || !rows_ok(y, n_out, n_out))
    return set_error(TALM_EINVAL, "rows must be 16-byte aligned with strides of 8 elements");
  if (saved_bytes < need) return set_error(TALM_EINVAL, "saved buffer too small");
  const Shape s{n_rows, n_in, n_out, static_cast<int>(rank)};
  float* t = static_cast<float*>(saved);
  LaunchTimer timer(TALM_KERNEL_LORA_FORWARD, stream);
  down_kernel<<<blocks(32 * n_rows), 256, 0, stream>>>(reinterpret_cast<const __half*>(x), ld_x,
                                                       lora_a, s, d, t);
  up_kernel<<<blocks(n_rows * n_out), 256, 0, stream>>>(reinterpret_cast<const __half*>(base),
                                                        ld_base, t, lora_b, s, scaling,
                                                        reinterpret_cast<__half*>(y));
  return check_launch("adapter forward kernels");
}

int talm_lora_backward(const uint16_t* g, int64_t ld_g, const uint16_t* x, int64_t ld_x,
                       const float* lora_a, const float* lora_b, const void* saved,
                       size_t saved_bytes, int64_t n_rows, int64_t n_in, int64_t n_out,
                       int64_t rank, float scaling, const int64_t* seed, int64_t drop,
                       uint16_t* dx, float* grad_a, float* grad_b, void* workspace,
                       size_t ws_bytes, void* stream_) {
  using namespace talm;
  using namespace talm::adapter;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  Dropout d;
  int st = check_shape(n_rows, n_in, n_out, rank);
  if (st == TALM_OK) st = check_dropout(drop, seed, &d);
  if (st != TALM_OK) return st;
  size_t need = 0, need_ws = 0;
  talm_lora_sizes(n_rows, n_in, n_out, rank, &need, &need_ws);
  if (!dx && !grad_a && !grad_b) return TALM_OK;
  if (n_rows == 0) {  // no rows: the weights' gradients are zero
    cudaError_t e = cudaSuccess;
    if (grad_a) e = cudaMemsetAsync(grad_a, 0, static_cast<size_t>(rank * n_in) * 4, stream);
    if (e == cudaSuccess && grad_b)
      e = cudaMemsetAsync(grad_b, 0, static_cast<size_t>(rank * n_out) * 4, stream);
    return e == cudaSuccess ? TALM_OK : set_error(TALM_ECUDA, "memset: %s", cudaGetErrorString(e));
  }
  if (!g || !x || !lora_a || !lora_b || !saved || !workspace)
    return set_error(TALM_EINVAL, "null pointer");
  if (!rows_ok(g, ld_g, n_out) || !rows_ok(x, ld_x, n_in) || (dx && !rows_ok(dx, n_in, n_in)))
    return set_error(TALM_EINVAL, "rows must be 16-byte aligned with strides of 8 elements");
  if (saved_bytes < need || ws_bytes < need_ws)
    return set_error(TALM_EINVAL, "saved buffer or workspace too small");
  const Shape s{n_rows, n_in, n_out, static_cast<int>(rank)};
  const float* t = static_cast<const float*>(saved);
  float* dt = static_cast<float*>(workspace);
  const __half* gh = reinterpret_cast<const __half*>(g);
  LaunchTimer timer(TALM_KERNEL_LORA_BACKWARD, stream);
  if (dx || grad_a)
    grad_t_kernel<<<blocks(32 * n_rows), 256, 0, stream>>>(gh, ld_g, lora_b, s, scaling, dt);
  if (grad_b)
    grad_b_kernel<<<blocks(n_out * rank), 256, 0, stream>>>(gh, ld_g, t, s, scaling, grad_b);
  if (grad_a)
    grad_a_kernel<<<blocks(n_in / 8 * rank), 256, 0, stream>>>(
        reinterpret_cast<const __half*>(x), ld_x, dt, s, d, grad_a);
  if (dx)
    grad_x_kernel<<<blocks(n_rows * n_in / 8), 256, 0, stream>>>(dt, lora_a, s, d,
                                                                 reinterpret_cast<__half*>(dx));
  return check_launch("adapter backward kernels");
}

}  // extern "C"
