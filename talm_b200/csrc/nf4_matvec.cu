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

// t = x A^T: a CTA takes eight rows of x and two of A, its warps share the reduction.
constexpr int DOWN_WARPS = 8;
constexpr int DOWN_ROWS = 8;
constexpr int DOWN_RANKS = 2;

template <bool VEC>
__global__ void __launch_bounds__(32 * DOWN_WARPS) adapter_down_kernel(
    const __half* __restrict__ x, int64_t ld_x, const float* __restrict__ a, int n_in, int n_rows,
    int rank, float* __restrict__ t) {
  __shared__ float part[DOWN_WARPS][DOWN_ROWS * DOWN_RANKS];
  // the product that follows may start now: it reads t only after it has waited for this grid
  grid_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n0 = blockIdx.x * DOWN_ROWS, j0 = blockIdx.y * DOWN_RANKS;
  const int nt = min(DOWN_ROWS, n_rows - n0);
  const bool two = j0 + 1 < rank;
  const float* a0 = a + int64_t{j0} * n_in;
  const float* a1 = two ? a0 + n_in : a0;
  float acc[DOWN_ROWS * DOWN_RANKS] = {};
  constexpr int STEP = VEC ? 4 : 1;
  for (int k = (warp * 32 + lane) * STEP; k < n_in; k += 32 * DOWN_WARPS * STEP) {
    float v0[STEP], v1[STEP];
    if constexpr (VEC) {
      const float4 f0 = __ldg(reinterpret_cast<const float4*>(a0 + k));
      const float4 f1 = __ldg(reinterpret_cast<const float4*>(a1 + k));
      v0[0] = f0.x; v0[1] = f0.y; v0[2] = f0.z; v0[3] = f0.w;
      v1[0] = f1.x; v1[1] = f1.y; v1[2] = f1.z; v1[3] = f1.w;
    } else {
      v0[0] = __ldg(a0 + k);
      v1[0] = __ldg(a1 + k);
    }
#pragma unroll
    for (int n = 0; n < DOWN_ROWS; ++n) {
      if (n >= nt) break;
      const __half* xr = x + (n0 + n) * ld_x + k;
      float xv[STEP];
      if constexpr (VEC) {
        const uint2 h = __ldg(reinterpret_cast<const uint2*>(xr));
        const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&h.x));
        const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&h.y));
        xv[0] = lo.x; xv[1] = lo.y; xv[2] = hi.x; xv[3] = hi.y;
      } else {
        xv[0] = __half2float(xr[0]);
      }
#pragma unroll
      for (int i = 0; i < STEP; ++i) {
        acc[2 * n] = fmaf(xv[i], v0[i], acc[2 * n]);
        acc[2 * n + 1] = fmaf(xv[i], v1[i], acc[2 * n + 1]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < DOWN_ROWS * DOWN_RANKS; ++i) {
    if (i >= 2 * nt) break;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], d);
    if (lane == 0) part[warp][i] = acc[i];
  }
  __syncthreads();
  const int n = threadIdx.x / DOWN_RANKS, j = threadIdx.x % DOWN_RANKS;
  if (n < nt && j0 + j < rank) {
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < DOWN_WARPS; ++w) sum += part[w][threadIdx.x];
    t[(n0 + n) * rank + j0 + j] = sum;
  }
}

// ------------------------------------------------------------------------------------------
// The main kernel: rows of whole 64-column blocks on the tensor cores (mma.sync m16n8k16, the
// weight as the 16-row operand, up to 8 NT rows of x as the n operand).
//
// A warp takes tiles of 16 weight rows; lane (g, t) = (lane / 4, lane % 4) reads 8 packed bytes of
// rows g and g + 8 per block (a quad reads a row's 32 bytes) and turns each byte into the fp16
// pair of its two levels by one shared-memory read: a table of 256 pairs, one copy per lane, so
// that no two lanes meet in a bank. The reduction index may be permuted as long as both operands
// agree, so a lane's 16 consecutive weights go into four mma's as they are and the matching
// operand is 32 consecutive bytes of x. A block's 64 columns have one scale per row: its four
// mma's start from zero and their result is added to the fp32 sum with one FMA per value, times
// the scale.
//
// The table holds fp16(LEVEL_GAIN * level) and the scale takes 1 / LEVEL_GAIN: the gain is the one
// in [1, 2) whose 16 rounded levels are nearest to the true ones (6.2e-5 in the mean square
// against 1.56e-4 without it and 2.1e-4 for the result's own rounding).
// ------------------------------------------------------------------------------------------
constexpr int WARPS = 16;
constexpr int STEP_BLOCKS = 4;  // blocks of 64 columns that a warp loads ahead
constexpr float LEVEL_GAIN = 1.6776883602142334f;
constexpr int LUT_BYTES = 256 * 32 * 4;
constexpr int STAGES = 4;       // a warp's ring of steps
constexpr int STAGE_BYTES = 16 * 32 * STEP_BLOCKS;

template <int NT>
constexpr int mma_smem() {
  return LUT_BYTES + WARPS * STAGES * STAGE_BYTES + 256 * 4 + WARPS * 16 * 8 * NT * 4;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct Split {
  int warps_per_tile;  // W: warps that share a tile's columns (a power of two up to WARPS)
  int n_tiles;         // 16-row tiles
  int n_blocks;        // 64-column blocks of a row
  int shift;           // log2(blocksize)
  int shift2;          // log2(qblock2)
};

// The scale inputs that a lane has loaded for one step: those of block t of the step for its two
// rows (the quad exchanges the finished scales).
struct ScaleIn {
  float s[2], a2[2], o2[2];
  uint32_t a8[2];
};

template <bool GROUPED>
__device__ __forceinline__ void load_scales(ScaleIn& in, const Weight& w, const Split& sp,
                                            int64_t row0, int64_t row1, int b) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t block = ((h ? row1 : row0) * w.n_in + int64_t{b} * 64) >> sp.shift;
    if constexpr (GROUPED) {
      const int64_t second = (w.row0 + block) >> sp.shift2;
      in.a8[h] = __ldg(w.absmax8 + block);
      in.a2[h] = __ldg(w.absmax2 + second);
      in.o2[h] = __ldg(w.offset2 + second);
    } else {
      in.s[h] = __ldg(w.absmax + block);
    }
  }
}

// x of rows 8 q + g (zeros past n_rows), the 16 columns of lane t in block b
template <int NT>
__device__ __forceinline__ void load_x(uint32_t (&v)[NT][8], const __half* x, int64_t ld_x,
                                       int n_rows, int g, int t, int b) {
#pragma unroll
  for (int q = 0; q < NT; ++q) {
    const int n = q * 8 + g;
    uint4 v0 = make_uint4(0, 0, 0, 0), v1 = v0;
    if (n < n_rows) {
      const uint4* p = reinterpret_cast<const uint4*>(x + n * ld_x + b * 64 + t * 16);
      v0 = __ldg(p);
      v1 = __ldg(p + 1);
    }
    v[q][0] = v0.x; v[q][1] = v0.y; v[q][2] = v0.z; v[q][3] = v0.w;
    v[q][4] = v1.x; v[q][5] = v1.y; v[q][6] = v1.z; v[q][7] = v1.w;
  }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int NT, bool GROUPED>
__global__ void __launch_bounds__(32 * WARPS, 1)
    nf4_mma_kernel(const __half* __restrict__ x, int64_t ld_x, int n_rows, Weight w, Split sp,
                   Epilogue ep, __half* __restrict__ y, int64_t ld_y) {
  extern __shared__ __align__(128) uint32_t mv_smem[];
  uint32_t* lut = mv_smem;                                        // [256][32]
  uint8_t* rings = reinterpret_cast<uint8_t*>(lut + 256 * 32);    // [WARPS][STAGES][16][128]
  float* code_s = reinterpret_cast<float*>(rings + WARPS * STAGES * STAGE_BYTES);  // [256]
  float* part = code_s + 256;                                     // [WARPS][8 NT rows of x][16]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int W = sp.warps_per_tile, groups = WARPS / W;
  const int group = warp / W, share = warp % W;
  const int b_first = static_cast<int>(int64_t{sp.n_blocks} * share / W);
  const int b_last = static_cast<int>(int64_t{sp.n_blocks} * (share + 1) / W);
  const int n_steps = (b_last - b_first + STEP_BLOCKS - 1) / STEP_BLOCKS;  // of one tile
  const int stride = gridDim.x * groups;
  const int first_tile = blockIdx.x * groups + group;

  auto sync_tile = [&] {  // the warps of this tile; W >= 2 leaves at most eight barriers
    if (W == 1)
      __syncwarp();
    else
      named_barrier(1 + group, 32 * W);
  };
  // rows past the end read the last one's bytes
  auto row_of = [&](int tile, int r) {
    const int64_t v = int64_t{tile} * 16 + r;
    return v < w.n_out ? v : w.n_out - 1;
  };

  // This warp's ring of packed bytes: a stage holds four blocks (128 bytes) of the tile's 16 rows,
  // the 16-byte chunk c of row r at chunk c ^ (r & 7) (the reads of eight rows then meet in no
  // bank). The warp fills and reads it alone, STAGES - 1 steps ahead.
  const uint32_t ring = smem_u32(rings) + warp * (STAGES * STAGE_BYTES);
  int f_tile = first_tile, f_b = b_first, f_stage = 0;
  auto fetch = [&] {
    if (f_tile < sp.n_tiles && n_steps > 0) {
      const int chunk = lane & 7;
      if (f_b + (chunk >> 1) < b_last) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * i + (lane >> 3);
          const uint8_t* src = w.packed + row_of(f_tile, r) * (w.n_in >> 1) +
                               static_cast<int64_t>(f_b) * 32 + chunk * 16;
          cp_async16(ring + f_stage * STAGE_BYTES + r * 128 + ((chunk ^ (r & 7)) << 4), src);
        }
      }
      f_b += STEP_BLOCKS;
      if (f_b >= b_last) {
        f_b = b_first;
        f_tile += stride;
      }
      f_stage = f_stage + 1 == STAGES ? 0 : f_stage + 1;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch();

  const bool any = n_steps > 0 && first_tile < sp.n_tiles;
  ScaleIn cur;
  uint32_t xv[NT][8];
  if (any) {
    load_scales<GROUPED>(cur, w, sp, row_of(first_tile, g), row_of(first_tile, g + 8),
                         min(b_first + t, b_last - 1));
    load_x<NT>(xv, x, ld_x, n_rows, g, t, b_first);
  }
  static_assert(32 * WARPS == 512, "two threads fill the 32 copies of a table entry");
  {
    const int i = threadIdx.x & 255, half = threadIdx.x >> 8;
    const float hi = w.levels ? __ldg(w.levels + (i >> 4)) : kNf4Levels[i >> 4];
    const float lo = w.levels ? __ldg(w.levels + (i & 15)) : kNf4Levels[i & 15];
    const uint32_t pair = pack_half2(LEVEL_GAIN * hi, LEVEL_GAIN * lo);
    const uint4 four = make_uint4(pair, pair, pair, pair);
#pragma unroll
    for (int k = 0; k < 4; ++k)  // eight neighbours write eight different bank groups
      reinterpret_cast<uint4*>(lut)[i * 8 + ((4 * half + k + i) & 7)] = four;
    if (GROUPED && half == 0) code_s[i] = __ldg(w.code + i);
  }
  __syncthreads();
  const uint32_t* my_lut = lut + lane;
  const uint8_t* my_ring = rings + warp * (STAGES * STAGE_BYTES) + g * 128 + (t & 1) * 8;

  int stage = 0;
  for (int tile = first_tile; tile < sp.n_tiles; tile += stride) {
    float acc[NT][4] = {};
    for (int b = b_first; b < b_last; b += STEP_BLOCKS) {
      fetch();
      cp_async_wait<STAGES - 1>();
      __syncwarp();  // every lane's copies of this stage have landed
      // the step after this one (of the next tile behind the last): scales now, x block by block
      const bool last = b + STEP_BLOCKS >= b_last;
      const int n_tile = last ? tile + stride : tile;
      const int n_b = last ? b_first : b + STEP_BLOCKS;
      const bool more = n_tile < sp.n_tiles;
      ScaleIn next = cur;
      if (more)
        load_scales<GROUPED>(next, w, sp, row_of(n_tile, g), row_of(n_tile, g + 8),
                             min(n_b + t, b_last - 1));
      float mine[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float s;
        if constexpr (GROUPED)
          s = __fadd_rn(__fmul_rn(code_s[cur.a8[h]], cur.a2[h]), cur.o2[h]);
        else
          s = cur.s[h];
        mine[h] = s * (1.0f / LEVEL_GAIN);
      }
      const uint8_t* st = my_ring + stage * STAGE_BYTES;
#pragma unroll
      for (int i = 0; i < STEP_BLOCKS; ++i) {
        if (b + i >= b_last) break;  // the same for the whole warp
        const float s0 = __shfl_sync(0xffffffffu, mine[0], (lane & 28) | i);
        const float s1 = __shfl_sync(0xffffffffu, mine[1], (lane & 28) | i);
        uint32_t xn[NT][8];
        const bool in_step = i + 1 < STEP_BLOCKS && b + i + 1 < b_last;
        if (in_step || more)
          load_x<NT>(xn, x, ld_x, n_rows, g, t, in_step ? b + i + 1 : n_b);
        const int at = ((2 * i + (t >> 1)) ^ g) << 4;
        const uint2 wa2 = *reinterpret_cast<const uint2*>(st + at);
        const uint2 wb2 = *reinterpret_cast<const uint2*>(st + 8 * 128 + at);
        float c[NT][4] = {};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const uint32_t wa = m < 2 ? wa2.x : wa2.y, wb = m < 2 ? wb2.x : wb2.y;
          const int sh = 16 * (m & 1);
          const uint32_t a[4] = {my_lut[((wa >> sh) & 0xFFu) * 32],
                                 my_lut[((wb >> sh) & 0xFFu) * 32],
                                 my_lut[((wa >> (sh + 8)) & 0xFFu) * 32],
                                 my_lut[((wb >> (sh + 8)) & 0xFFu) * 32]};
#pragma unroll
          for (int q = 0; q < NT; ++q) mma_f16(c[q], a, xv[q][2 * m], xv[q][2 * m + 1]);
        }
#pragma unroll
        for (int q = 0; q < NT; ++q) {
          acc[q][0] = fmaf(s0, c[q][0], acc[q][0]);
          acc[q][1] = fmaf(s0, c[q][1], acc[q][1]);
          acc[q][2] = fmaf(s1, c[q][2], acc[q][2]);
          acc[q][3] = fmaf(s1, c[q][3], acc[q][3]);
#pragma unroll
          for (int k = 0; k < 8; ++k) xv[q][k] = xn[q][k];
        }
      }
      __syncwarp();  // the stage has been read; the next fetch may fill it
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      cur = next;
    }
    // the warps of a tile add their shares in share order
    float* mine = part + warp * (128 * NT);
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      mine[(q * 8 + 2 * t) * 16 + g] = acc[q][0];
      mine[(q * 8 + 2 * t + 1) * 16 + g] = acc[q][1];
      mine[(q * 8 + 2 * t) * 16 + g + 8] = acc[q][2];
      mine[(q * 8 + 2 * t + 1) * 16 + g + 8] = acc[q][3];
    }
    sync_tile();
    if (ep.t != nullptr) grid_dependency_wait();  // t comes from the launch before this one
    for (int i = share * 32 + lane; i < 16 * n_rows; i += 32 * W) {
      const int n = i >> 4;
      const int64_t o = int64_t{tile} * 16 + (i & 15);
      if (o >= w.n_out) continue;
      float v = 0.0f;
      for (int k = 0; k < W; ++k) v += part[(group * W + k) * (128 * NT) + i];
      if (ep.t != nullptr) {
        float extra = 0.0f;
#pragma unroll 8
        for (int j = 0; j < ep.rank; ++j)
          extra = fmaf(__ldcg(ep.t + n * ep.rank + j), __ldg(ep.lora_b + o * ep.rank + j), extra);
        v = fmaf(ep.scaling, extra, v);
      }
      if (ep.bias != nullptr) v += __half2float(ep.bias[o]);
      y[n * ld_y + o] = __float2half_rn(v);
    }
    sync_tile();
  }
  cp_async_wait<0>();
}

// Launches the tensor-core kernel for NT groups of eight rows.
template <int NT, bool GROUPED>
int run_mma(const __half* x, int64_t ld_x, int n_rows, const Weight& w, Split sp,
            const Epilogue& ep, __half* y, int64_t ld_y, cudaStream_t stream) {
  static bool ready[kMaxDevices];
  int dev = 0;
  int st = current_device(&dev);
  if (st != TALM_OK) return st;
  constexpr int smem = mma_smem<NT>();
  if (!ready[dev]) {  // setting it twice from two threads is harmless
    const cudaError_t e = cudaFuncSetAttribute(nf4_mma_kernel<NT, GROUPED>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess)
      return set_error(TALM_ECUDA, "nf4 matvec set-up: %s", cudaGetErrorString(e));
    ready[dev] = true;
  }
  const int sms = current_sm_count();
  if (sms <= 0) return set_error(TALM_ENODEV, "no CUDA device");
  int W = 1;
  while (W < WARPS && int64_t{sp.n_tiles} * W < int64_t{sms} * WARPS && W < sp.n_blocks) W *= 2;
  sp.warps_per_tile = W;
  const int groups = WARPS / W;
  const int ctas = (sp.n_tiles + groups - 1) / groups;
  const int cap = sms;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas < cap ? ctas : cap), 1, 1);
  cfg.blockDim = dim3(32 * WARPS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  // behind the adapter's down kernel only: it starts once everything before it has completed, and
  // this kernel waits for it before it reads t
  cfg.numAttrs = ep.t != nullptr ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, nf4_mma_kernel<NT, GROUPED>, x, ld_x, n_rows, w,
                                           sp, ep, y, ld_y);
  if (e != cudaSuccess) return set_error(TALM_ECUDA, "nf4 matvec: %s", cudaGetErrorString(e));
  return check_launch("nf4 matvec kernel");
}

template <bool GROUPED>
int run_mma_rows(const __half* x, int64_t ld_x, int n_rows, const Weight& w, const Split& sp,
                 const Epilogue& ep, __half* y, int64_t ld_y, cudaStream_t stream) {
  if (n_rows <= 8) return run_mma<1, GROUPED>(x, ld_x, n_rows, w, sp, ep, y, ld_y, stream);
  if (n_rows <= 16) return run_mma<2, GROUPED>(x, ld_x, n_rows, w, sp, ep, y, ld_y, stream);
  return run_mma<4, GROUPED>(x, ld_x, n_rows, w, sp, ep, y, ld_y, stream);
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
    const dim3 grid(static_cast<unsigned>((n_rows + DOWN_ROWS - 1) / DOWN_ROWS),
                    static_cast<unsigned>((rank + DOWN_RANKS - 1) / DOWN_RANKS), 1);
    const bool vec = w_cols % 4 == 0 && ld_x % 4 == 0 &&
                     (reinterpret_cast<uintptr_t>(x) & 7) == 0 &&
                     (reinterpret_cast<uintptr_t>(lora_a) & 15) == 0;
    auto kernel = vec ? adapter_down_kernel<true> : adapter_down_kernel<false>;
    kernel<<<grid, 32 * DOWN_WARPS, 0, stream>>>(xh, ld_x, lora_a, static_cast<int>(w_cols),
                                                 static_cast<int>(n_rows),
                                                 static_cast<int>(rank), down);
    const int st = check_launch("adapter down kernel");
    if (st != TALM_OK) return st;
  }
  LaunchTimer timer(TALM_KERNEL_NF4_MATVEC, stream);
  // The tensor-core kernel takes whole 64-column blocks of one scale each, on the boundaries of its
  // wide loads; anything else the byte-wise kernel.
  const int shift = log2_exact(blocksize), shift2 = absmax8 ? log2_exact(qblock2) : 0;
  if (w_cols % 64 == 0 && shift >= 6 && shift2 >= 0 && ld_x % 8 == 0 &&
      (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(packed) & 7) == 0) {
    const Split sp{1, static_cast<int>((w_rows + 15) / 16), static_cast<int>(w_cols / 64), shift,
                   shift2};
    __half* yh = reinterpret_cast<__half*>(y);
    const int n = static_cast<int>(n_rows);
    return absmax8 ? run_mma_rows<true>(xh, ld_x, n, w, sp, ep, yh, ld_y, stream)
                   : run_mma_rows<false>(xh, ld_x, n, w, sp, ep, yh, ld_y, stream);
  }
  nf4_matvec_any_kernel<<<static_cast<unsigned>((w_rows + 7) / 8), 256, 0, stream>>>(
      xh, ld_x, static_cast<int>(n_rows), w, ep, reinterpret_cast<__half*>(y), ld_y);
  return check_launch("nf4 matvec kernel");
}

}  // extern "C"
