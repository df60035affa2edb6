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
#include "adapter_gemm.cuh"

namespace talm {
namespace adapter {

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
// loads first. Bound by HBM: 16384 x 8960 bf16, forward and backward, 200 us (1.17 GB, 5.9 TB/s,
// 0.90 of the measured copy); a group costs 14 multiplications and about 100 operations in all, 46
// % of the ALU's rate at that speed (10 rounds, or 32 bits per element, would be the bound
// themselves).
template <class T, int UNROLL, bool WIDE>
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
      philox<WIDE>(static_cast<uint64_t>(q), key, c);
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

// Any strides and alignment: one thread per group of eight elements in row-major order, an element
// at a time (a row may start anywhere in a group and off any boundary). Bound by its scalar loads
// and stores: rows of a wider tensor, 16384 x 8960, one pass 410 us in 16 bits (flat 100), 686 in
// fp32 (flat 208); 2048 x 1536 11 us (flat 3.7).
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
    // 16-bit elements and more than six rounds of the grid: the generator of fewer instructions
    // (both forms, forward + backward: fp16 25 M elements 35.8 and 36.7 us, 50 M 67.0 and 67.3,
    // 101 M 139.3 and 130.4; fp32 within 2 % everywhere)
    auto kernel = dropout_kernel<T, UNROLL, false>;
    if constexpr (sizeof(T) == 2)
      if (want > 6 * cap) kernel = dropout_kernel<T, UNROLL, true>;
    kernel<<<static_cast<unsigned>(grid), 256, 0, stream>>>(x, n, d, y);
  } else {
    const int64_t want = (n + 2047) / 2048;
    dropout_rows_kernel<<<static_cast<unsigned>(want < cap ? want : cap), 256, 0, stream>>>(
        x, ld_x, n_cols, n, d, y);
  }
  return check_launch("dropout kernel");
}

// ------------------------------------------------------------------------------------------
// the branch
//
// Six products, each of a wide activation and a rank-wide operand (adapter_gemm.cuh):
//   inner   t = keep x A^T and dt = s g B            sums over the activation's columns
//   outer   dA = dt^T keep x and dB = s g^T t        sums over its rows
//   up      y = base + s t B^T and dx = keep dt A    sums over the rank
// and between them small kernels that turn the rank-wide fp32 operands into 16-bit parts for the
// tensor cores. Where the other operand is an fp16 activation and the result fp32 (inner, outer)
// they are two fp16 parts of the operand scaled by a power of two that brings its largest element
// to [2^14, 2^15), one for every rank and 128 elements of the reduction: 2^-22 of an element that
// is at least 2^-17 of the largest of its 128, 2^-40 of that largest below, at any size of a rank
// beside the others (one scale for all ranks of 128 rows left a rank of 2^-24 of its neighbour
// 2^-16 wrong). Where both operands are fp32 and the result is fp16 (up) they are two bf16 parts
// without scale, and the product of the two small ones is left out: under 2^-16 of each term, a
// sixteenth of the result's own rounding.
//
// Measured on one B200, forward and backward replayed in a graph: q_proj of 2048 rows, rank 16, 39
// us (38 MB; nine launches of about 4 us each are the bound), 16384 x 1536 to 8960, rank 64, 305 us
// (1.04 GB, 3.4 TB/s, 0.52 of the measured copy: g is read twice, once for dt and once for dB, 45
// us that the floor does not have, and the masked passes, 74 us for 23 us of bytes, wait for their
// masks; y runs at 0.9).
// ------------------------------------------------------------------------------------------
struct Shape {
  int64_t n_rows, n_in, n_out;
  int rank;
};

// ---- prepared operands -----------------------------------------------------------------------
// RP: the rank rounded up to 16, 32 or 64, zeros behind it.
//   Rows:  fp16 parts of an adapter matrix with the rank in the rows (A, B^T), 128 columns of a row
//          scaled together: parts [2 RP, n], the small parts behind the large ones; down [ceil(n /
//          128)][RP] undoes the scale.
//   cat:   bf16 parts (hi | lo) of an adapter matrix with the rank in the columns (B, A^T), or of t or
//          dt, in rows of up::chunks(RP) * 64 (what is behind the parts is not read).
//   pair:  fp16 parts (hi | lo) of t or dt in rows of sums::pair_width(RP) (likewise), 128 rows of a rank
//          scaled together; down [ceil(rows / 128)][RP] undoes it.
struct Rows {
  __half* parts;
  float* down;
};
struct TParts {
  uint4 *cat, *pair;
  float* down;
};

__host__ __device__ constexpr int padded_rank(int rank) {
  return rank <= 16 ? 16 : rank <= 32 ? 32 : 64;
}

constexpr int PREP_THREADS = 1024;

// Ranks j .. j + 7 of row r of a cat: both parts of eight values.
__device__ __forceinline__ void put_cat(uint4* cat, int64_t r, int j, int rp, const float (&v)[8]) {
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) split_bf16(v[2 * k], v[2 * k + 1], hi[k], lo[k]);
  uint4* row = cat + r * (up::chunks(rp) * 8);
  row[j / 8] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  row[(rp + j) / 8] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// An adapter matrix: element (rank j, column c) at m[j * dj + c * dc].
struct Matrix {
  const float* m;
  int64_t dj, dc;
  int n;
};

// The operands of one matrix: rows for the sums, cat for the rank-wide product; null where it is
// not wanted.
struct Operands {
  Rows rows;
  uint4* cat;
};

// A CTA takes 128 columns of A or of B^T into shared memory and builds both of its operands.
template <int RP>
__global__ void __launch_bounds__(PREP_THREADS) prepare_kernel(Matrix a, Matrix b, Operands of_a,
                                                               Operands of_b, int rank) {
  constexpr int LD = 128 + 1;
  extern __shared__ float tile[];  // [RP][LD]
  grid_launch_dependents();
  grid_dependency_wait();
  const int a_ctas = (a.n + 127) / 128;
  const bool is_a = static_cast<int>(blockIdx.x) < a_ctas;
  const Matrix& s = is_a ? a : b;
  const Operands& out = is_a ? of_a : of_b;
  const int block = is_a ? blockIdx.x : blockIdx.x - a_ctas;
  const int c0 = block * 128;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // neighbours read neighbours: A's columns, B's ranks
#pragma unroll 8
  for (int i = tid; i < RP * 128; i += PREP_THREADS) {
    const int j = is_a ? i >> 7 : i % RP, c = is_a ? i & 127 : i / RP;
    tile[j * LD + c] =
        j < rank && c0 + c < s.n ? __ldg(s.m + j * s.dj + (c0 + c) * s.dc) : 0.0f;
  }
  __syncthreads();
  if (out.rows.parts != nullptr) {
    uint32_t* parts = reinterpret_cast<uint32_t*>(out.rows.parts);
    const int64_t ld = s.n / 2;  // pairs; n is even
    for (int j = warp; j < RP; j += PREP_THREADS / 32) {
      const float* row = tile + j * LD;
      float v[2][2], most = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          v[h][u] = row[64 * h + 2 * lane + u];
          most = fmaxf(most, fabsf(v[h][u]));
        }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
      float up, down;
      power_scale(most, &up, &down);
      if (lane == 0) out.rows.down[block * RP + j] = down;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t c = c0 / 2 + 32 * h + lane;
        if (c >= ld) continue;
        uint32_t hi, lo;
        split_f16(v[h][0] * up, v[h][1] * up, hi, lo);
        parts[j * ld + c] = hi;
        parts[(RP + j) * ld + c] = lo;
      }
    }
  }
  if (out.cat != nullptr) {
    constexpr int PIECES = RP / 8;
    for (int i = tid; i < 128 * PIECES; i += PREP_THREADS) {
      const int c = i / PIECES, j = (i % PIECES) * 8;
      if (c0 + c >= s.n) break;  // so are the columns behind it
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = tile[(j + k) * LD + c];
      put_cat(out.cat, c0 + c, j, RP, v);
    }
  }
}

// ---- the operands made of t (or dt) ----------------------------------------------------------
// t[n, j] = factor * (sum of the parts): a CTA per 128 rows, of which each rank has its own scale.
// The pair is built where it is wanted (out.pair not null).
constexpr int T_THREADS = 1024;

template <int RP>
__global__ void __launch_bounds__(T_THREADS)
    t_parts_kernel(const float* __restrict__ part, int splits, int64_t n_rows,
                   float factor, TParts out) {
  extern __shared__ float t_smem[];  // [128][RP + 1]
  __shared__ float scale_up[RP];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * 128;
  constexpr int E = 128 * RP / T_THREADS, U = 8 / E;  // elements of a thread; eight loads at a time
  float v[E] = {};
  const int64_t live = (n_rows - row0 < 128 ? n_rows - row0 : 128) * RP;
  const float* p = part + row0 * RP + threadIdx.x;
  for (int k0 = 0; k0 < splits; k0 += U) {
    float x[E][U];
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int u = 0; u < U; ++u)
        x[i][u] = k0 + u < splits && i * T_THREADS + threadIdx.x < live
                      ? __ldcg(p + static_cast<int64_t>(k0 + u) * n_rows * RP + i * T_THREADS)
                      : 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int u = 0; u < U; ++u) v[i] += x[i][u];
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int e = i * T_THREADS + threadIdx.x;
    t_smem[e / RP * (RP + 1) + e % RP] = v[i] * factor;
  }
  __syncthreads();
  if (out.pair != nullptr)
    for (int j = warp; j < RP; j += T_THREADS / 32) {  // a warp per rank
      float most = 0.0f;
#pragma unroll
      for (int r = 0; r < 128; r += 32) most = fmaxf(most, fabsf(t_smem[(r + lane) * (RP + 1) + j]));
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
      float up, back;
      power_scale(most, &up, &back);
      if (lane == 0) {
        scale_up[j] = up;
        out.down[static_cast<int64_t>(blockIdx.x) * RP + j] = back;
      }
    }
  constexpr int PIECES = RP / 8;  // of eight ranks
  for (int i = threadIdx.x; i < 128 * PIECES; i += T_THREADS) {
    const int r = i / PIECES, j = (i % PIECES) * 8;
    if (row0 + r >= n_rows) break;  // so are the rows behind it
    float m[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = t_smem[r * (RP + 1) + j + k];
    put_cat(out.cat, row0 + r, j, RP, m);
  }
  if (out.pair == nullptr) return;
  __syncthreads();
  for (int i = threadIdx.x; i < 128 * PIECES; i += T_THREADS) {
    const int r = i / PIECES, j = (i % PIECES) * 8;
    if (row0 + r >= n_rows) break;
    const float *m = t_smem + r * (RP + 1) + j, *up = scale_up + j;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      split_f16(m[2 * k] * up[2 * k], m[2 * k + 1] * up[2 * k + 1], hi[k], lo[k]);
    uint4* row = out.pair + (row0 + r) * (sums::pair_width(RP) / 8);
    row[j / 8] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    row[PIECES + j / 8] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// The weights' gradients: factor * (sum of the parts) as [rank, n] (A) or [n, rank] (B).
struct PartSum {
  const float* part;  // [splits, RP, n]
  int splits, n;
  float factor;
  float* out;  // null: not wanted
};

// A CTA per 32 columns of one of them, a warp per rank.
constexpr int SUM_THREADS = 1024;

__global__ void __launch_bounds__(SUM_THREADS) sum_parts_kernel(PartSum a, PartSum b, int rank, int rp) {
  __shared__ float turned[32][64 + 1];
  grid_launch_dependents();
  grid_dependency_wait();
  const int a_ctas = a.out ? (a.n + 31) / 32 : 0;
  const bool is_a = static_cast<int>(blockIdx.x) < a_ctas;
  const PartSum& s = is_a ? a : b;
  const int c0 = (is_a ? blockIdx.x : blockIdx.x - a_ctas) * 32;
  const int c = threadIdx.x & 31, live = min(32, s.n - c0);
  const int64_t step = static_cast<int64_t>(rp) * s.n;
  for (int j = threadIdx.x >> 5; j < rank; j += SUM_THREADS / 32) {
    const float* p = s.part + static_cast<int64_t>(j) * s.n + c0 + c;
    float v = 0.0f;
    for (int k0 = 0; k0 < s.splits; k0 += 8) {
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        x[u] = k0 + u < s.splits && c < live ? __ldcg(p + (k0 + u) * step) : 0.0f;
#pragma unroll
      for (int u = 0; u < 8; ++u) v += x[u];
    }
    if (is_a && c < live) s.out[static_cast<int64_t>(j) * s.n + c0 + c] = v * s.factor;
    if (!is_a) turned[c][j] = v * s.factor;
  }
  if (is_a) return;
  __syncthreads();
  for (int i = threadIdx.x; i < live * rank; i += SUM_THREADS)
    s.out[static_cast<int64_t>(c0) * rank + i] = turned[i / rank][i % rank];
}

// ---- host: workspaces and launches ------------------------------------------------------------
struct Carve {  // hands out 256-byte aligned pieces; counts them when there is no base
  char* base;
  size_t used;
  template <class T>
  T* take(size_t n) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += (n * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

// What the forward pass leaves for the backward pass: t's pair and the adapter's other operands.
struct Saved {
  Carve carve;
  TParts t;
  Rows b_rows;
  uint4* a_cat;
  Saved(void* base, const Shape& s, int rp) : carve{static_cast<char*>(base), 0} {
    t.cat = nullptr;
    t.pair = carve.take<uint4>(static_cast<size_t>(s.n_rows) * (sums::pair_width(rp) / 8));
    t.down = carve.take<float>(static_cast<size_t>((s.n_rows + 127) / 128) * rp);
    b_rows.parts = carve.take<__half>(static_cast<size_t>(2 * rp) * s.n_out);
    b_rows.down = carve.take<float>(static_cast<size_t>((s.n_out + 127) / 128) * rp);
    a_cat = carve.take<uint4>(static_cast<size_t>(s.n_in) * up::chunks(rp) * 8);
  }
};

struct ForwardWork {
  Carve carve;
  Rows a_rows;
  uint4 *b_cat, *t_cat;
  float* part;
  ForwardWork(void* base, const Shape& s, int rp) : carve{static_cast<char*>(base), 0} {
    a_rows.parts = carve.take<__half>(static_cast<size_t>(2 * rp) * s.n_in);
    a_rows.down = carve.take<float>(static_cast<size_t>((s.n_in + 127) / 128) * rp);
    b_cat = carve.take<uint4>(static_cast<size_t>(s.n_out) * up::chunks(rp) * 8);
    t_cat = carve.take<uint4>(static_cast<size_t>(s.n_rows) * up::chunks(rp) * 8);
    // without a mask there are at least as many splits
    part = carve.take<float>(
        static_cast<size_t>(sums::Plan(false, false, s.n_rows, s.n_in).splits) * s.n_rows * rp);
  }
};

struct BackwardWork {
  Carve carve;
  TParts dt;
  float *t_part, *b_part, *a_part;
  BackwardWork(void* base, const Shape& s, int rp) : carve{static_cast<char*>(base), 0} {
    dt.cat = carve.take<uint4>(static_cast<size_t>(s.n_rows) * up::chunks(rp) * 8);
    dt.pair = carve.take<uint4>(static_cast<size_t>(s.n_rows) * (sums::pair_width(rp) / 8));
    dt.down = carve.take<float>(static_cast<size_t>((s.n_rows + 127) / 128) * rp);
    t_part = carve.take<float>(static_cast<size_t>(sums::Plan(false, false, s.n_rows, s.n_out).splits) *
                               s.n_rows * rp);
    b_part = carve.take<float>(static_cast<size_t>(sums::Plan(true, true, s.n_rows, s.n_out).splits) *
                               rp * s.n_out);
    a_part = carve.take<float>(static_cast<size_t>(sums::Plan(true, false, s.n_rows, s.n_in).splits) *
                               rp * s.n_in);
  }
};

// The operands made of the inner sums of an activation.
template <int RP>
int make_t_parts(const float* part, int splits, int64_t n_rows, float factor, const TParts& out,
                 cudaStream_t stream) {
  constexpr int smem = 128 * (RP + 1) * 4;
  static_assert(smem <= 48 * 1024, "no opt-in");
  return launch_dependent(t_parts_kernel<RP>, static_cast<unsigned>((n_rows + 127) / 128),
                          T_THREADS, smem, stream, part, splits, n_rows, factor, out);
}

template <int RP>
int run_forward(const __half* x, int64_t ld_x, const __half* base, int64_t ld_base,
                const float* a, const float* b, const Shape& s, float scaling, const Dropout& d,
                __half* y, void* saved, void* work, cudaStream_t stream) {
  const ForwardWork w(work, s, RP);
  const Saved keep(saved, s, RP);
  const Matrix ma{a, s.n_in, 1, static_cast<int>(s.n_in)};
  const Matrix mb{b, 1, s.rank, static_cast<int>(s.n_out)};
  const Operands of_a{w.a_rows, keep.a_cat};
  const Operands of_b{saved ? keep.b_rows : Rows{nullptr, nullptr}, w.b_cat};
  constexpr int smem = RP * 129 * 4;
  static_assert(smem <= 48 * 1024, "no opt-in");
  int st = launch_dependent(prepare_kernel<RP>,
                            static_cast<unsigned>((s.n_in + 127) / 128 + (s.n_out + 127) / 128),
                            PREP_THREADS, smem, stream, ma, mb, of_a, of_b, s.rank);
  const sums::Plan plan(false, d.drop != 0, s.n_rows, s.n_in);
  const TParts t{w.t_cat, saved ? keep.t.pair : nullptr, saved ? keep.t.down : nullptr};
  if (st == TALM_OK)
    st = d.drop ? sums::launch<RP, false, true>(plan, x, ld_x, s.n_rows, s.n_in, w.a_rows.parts,
                                                w.a_rows.down, d, w.part, stream)
                : sums::launch<RP, false, false>(plan, x, ld_x, s.n_rows, s.n_in, w.a_rows.parts,
                                                 w.a_rows.down, d, w.part, stream);
  if (st == TALM_OK)
    st = make_t_parts<RP>(w.part, plan.splits, s.n_rows, d.factor, t, stream);
  if (st != TALM_OK) return st;
  return up::launch<RP, false>(w.t_cat, w.b_cat, base, ld_base, y, s.n_rows, s.n_out,
                                           scaling, d, stream);
}

template <int RP>
int run_backward(const __half* g, int64_t ld_g, const __half* x, int64_t ld_x, const Shape& s,
                 float scaling, const Dropout& d, const void* saved, __half* dx, float* da,
                 float* db, void* work, cudaStream_t stream) {
  const BackwardWork w(work, s, RP);
  const Saved keep(const_cast<void*>(saved), s, RP);
  const Dropout none{nullptr, 0, 1.0f};
  int st = TALM_OK;
  const bool want_dt = da || dx;
  const sums::Plan dt_plan(false, false, s.n_rows, s.n_out), db_plan(true, true, s.n_rows, s.n_out);
  const sums::Plan da_plan(true, d.drop != 0, s.n_rows, s.n_in);
  if (want_dt && db)
    st = sums::launch_pair<RP>(dt_plan, db_plan, g, ld_g, s.n_rows, s.n_out, keep.b_rows.parts,
                               keep.b_rows.down, w.t_part, keep.t.pair, keep.t.down, w.b_part,
                               stream);
  else if (want_dt)
    st = sums::launch<RP, false, false>(dt_plan, g, ld_g, s.n_rows, s.n_out, keep.b_rows.parts,
                                        keep.b_rows.down, none, w.t_part, stream);
  else
    st = sums::launch<RP, true, false>(db_plan, g, ld_g, s.n_rows, s.n_out, keep.t.pair,
                                       keep.t.down, none, w.b_part, stream);
  if (want_dt && st == TALM_OK)
    st = make_t_parts<RP>(w.t_part, dt_plan.splits, s.n_rows, scaling, w.dt, stream);
  if (da && st == TALM_OK)
    st = d.drop ? sums::launch<RP, true, true>(da_plan, x, ld_x, s.n_rows, s.n_in, w.dt.pair,
                                               w.dt.down, d, w.a_part, stream)
                : sums::launch<RP, true, false>(da_plan, x, ld_x, s.n_rows, s.n_in, w.dt.pair,
                                                w.dt.down, d, w.a_part, stream);
  if (dx && st == TALM_OK)
    st = up::launch<RP, true>(w.dt.cat, keep.a_cat, nullptr, 0, dx, s.n_rows, s.n_in,
                                          d.factor, d, stream);
  if ((da || db) && st == TALM_OK) {
    const PartSum sa{w.a_part, da_plan.splits, static_cast<int>(s.n_in), d.factor, da};
    const PartSum sb{w.b_part, db_plan.splits, static_cast<int>(s.n_out), scaling, db};
    const int64_t ctas = (da ? (s.n_in + 31) / 32 : 0) + (db ? (s.n_out + 31) / 32 : 0);
    st = launch_dependent(sum_parts_kernel, static_cast<unsigned>(ctas), SUM_THREADS, 0, stream, sa, sb,
                          s.rank, RP);
  }
  return st;
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
                    size_t* forward_ws, size_t* backward_ws) {
  using namespace talm;
  using namespace talm::adapter;
  const int st = check_shape(n_rows, n_in, n_out, rank);
  if (st != TALM_OK) return st;
  if (!saved || !forward_ws || !backward_ws) return set_error(TALM_EINVAL, "null pointer");
  const Shape s{n_rows, n_in, n_out, static_cast<int>(rank)};
  const int rp = padded_rank(s.rank);
  const bool none = n_rows == 0;
  *saved = none ? 0 : Saved(nullptr, s, rp).carve.used;
  *forward_ws = none ? 0 : ForwardWork(nullptr, s, rp).carve.used;
  *backward_ws = none ? 0 : BackwardWork(nullptr, s, rp).carve.used;
  return TALM_OK;
}

int talm_lora_forward(const uint16_t* x, int64_t ld_x, const uint16_t* base, int64_t ld_base,
                      const float* lora_a, const float* lora_b, int64_t n_rows, int64_t n_in,
                      int64_t n_out, int64_t rank, float scaling, const int64_t* seed,
                      int64_t drop, uint16_t* y, void* saved, size_t saved_bytes,
                      void* workspace, size_t ws_bytes, void* stream_) {
  using namespace talm;
  using namespace talm::adapter;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  Dropout d;
  int st = check_shape(n_rows, n_in, n_out, rank);
  if (st == TALM_OK) st = check_dropout(drop, seed, &d);
  if (st != TALM_OK) return st;
  size_t need = 0, need_forward = 0, need_backward = 0;
  talm_lora_sizes(n_rows, n_in, n_out, rank, &need, &need_forward, &need_backward);
  if (n_rows == 0) return TALM_OK;
  if (!x || !base || !lora_a || !lora_b || !y || !workspace)
    return set_error(TALM_EINVAL, "null pointer");
  if (!rows_ok(x, ld_x, n_in) || !rows_ok(base, ld_base, n_out) || !rows_ok(y, n_out, n_out) ||
      ((reinterpret_cast<uintptr_t>(saved) | reinterpret_cast<uintptr_t>(workspace)) & 15) != 0)
    return set_error(TALM_EINVAL, "rows must be 16-byte aligned with strides of 8 elements");
  if ((saved && saved_bytes < need) || ws_bytes < need_forward)
    return set_error(TALM_EINVAL, "saved buffer or workspace too small");
  const Shape s{n_rows, n_in, n_out, static_cast<int>(rank)};
  LaunchTimer timer(TALM_KERNEL_LORA_FORWARD, stream);
  const int rp = padded_rank(s.rank);
  auto run = rp == 16 ? run_forward<16> : rp == 32 ? run_forward<32> : run_forward<64>;
  return run(reinterpret_cast<const __half*>(x), ld_x, reinterpret_cast<const __half*>(base),
             ld_base, lora_a, lora_b, s, scaling, d, reinterpret_cast<__half*>(y), saved, workspace,
             stream);
}

int talm_lora_backward(const uint16_t* g, int64_t ld_g, const uint16_t* x, int64_t ld_x,
                       const void* saved, size_t saved_bytes, int64_t n_rows, int64_t n_in, int64_t n_out,
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
  size_t need = 0, need_forward = 0, need_backward = 0;
  talm_lora_sizes(n_rows, n_in, n_out, rank, &need, &need_forward, &need_backward);
  if (!dx && !grad_a && !grad_b) return TALM_OK;
  if (n_rows == 0) {  // no rows: the weights' gradients are zero
    cudaError_t e = cudaSuccess;
    if (grad_a) e = cudaMemsetAsync(grad_a, 0, static_cast<size_t>(rank * n_in) * 4, stream);
    if (e == cudaSuccess && grad_b)
      e = cudaMemsetAsync(grad_b, 0, static_cast<size_t>(rank * n_out) * 4, stream);
    return e == cudaSuccess ? TALM_OK : set_error(TALM_ECUDA, "memset: %s", cudaGetErrorString(e));
  }
  if (!g || !x || !saved || !workspace)
    return set_error(TALM_EINVAL, "null pointer");
  if (!rows_ok(g, ld_g, n_out) || !rows_ok(x, ld_x, n_in) || (dx && !rows_ok(dx, n_in, n_in)) ||
      ((reinterpret_cast<uintptr_t>(saved) | reinterpret_cast<uintptr_t>(workspace)) & 15) != 0)
    return set_error(TALM_EINVAL, "rows must be 16-byte aligned with strides of 8 elements");
  if (saved_bytes < need || ws_bytes < need_backward)
    return set_error(TALM_EINVAL, "saved buffer or workspace too small");
  const Shape s{n_rows, n_in, n_out, static_cast<int>(rank)};
  LaunchTimer timer(TALM_KERNEL_LORA_BACKWARD, stream);
  const int rp = padded_rank(s.rank);
  auto run = rp == 16 ? run_backward<16> : rp == 32 ? run_backward<32> : run_backward<64>;
  return run(reinterpret_cast<const __half*>(g), ld_g, reinterpret_cast<const __half*>(x), ld_x,
             s, scaling, d, saved, reinterpret_cast<__half*>(dx), grad_a, grad_b, workspace, stream);
}

}  // extern "C"
