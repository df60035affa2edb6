// Products of a few rows with NF4 weights (the single-token form of a 4-bit projection), with an
// optional LoRA adapter added in the epilogue.
//
//   y[n, o] = fp16( sum_k L[code[o, k]] S[o, k] x[n, k] + bias[o] + s sum_j t[n, j] B[o, j] )
//   t[n, j] = sum_k x[n, k] A[j, k]
//
// L are the 16 levels, S the scale of the block that the flattened weight element o * K + k is in:
// an fp32 absmax, or fp32(fp32(code2[absmax8] * absmax2) + offset2) as in nf4.cu. Products and
// sums are fp32 and the result is rounded once: the weight itself is not rounded to fp16, which
// the dequantised copy of a weight is, and its levels keep 22 bits and more of their fp32 values.
//
// Measured on one B200, calls replayed in a graph over two sets of inputs (29 MB: L2 holds them):
// gate + up of the Qwen2.5-1.5B layer (17920 x 1536) for one row 9.3 us (14.2 MB, 1.5 TB/s; the
// floor at the measured copy bandwidth is 2.2 us), k_proj 3.8 us, down_proj for 13 rows 11.2 us,
// down_proj for 32 rows with an adapter of rank 64 16.7 us; with the weights from HBM (30 copies
// and more) 11.7, 4.2, 14.2 and 18.2. Dequantising the layer and multiplying moves 117 MB for the
// same 23 MB of weights.
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

// fp32 on the tensor cores: an operand is split into a tf32 part (11 significant bits, cut off) and
// the exact rest, whose own tf32 part leaves 2^-21 of the operand. mma.sync m16n8k8.
__device__ __forceinline__ void split_tf32(float v, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(v) & 0xFFFFE000u;
  lo = __float_as_uint(v - __uint_as_float(hi));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// t = x A^T: a cluster takes 16 rows of A, its CTAs (DOWN_PARTS or fewer) a part of the columns
// each, their warps share those; the CTAs add up their sums in rank order through each other's
// shared memory. fp16 x is exact in tf32, A is split in two.
constexpr int DOWN_WARPS = 16;
constexpr int DOWN_PARTS = 8;

template <int NT, bool VEC>
__global__ void __launch_bounds__(32 * DOWN_WARPS) adapter_down_kernel(
    const __half* __restrict__ x, int64_t ld_x, const float* __restrict__ a, int n_in, int n_rows,
    int rank, float* __restrict__ t_out) {
  __shared__ float part[DOWN_WARPS][128 * NT];
  // the product that follows may start now: it reads t only after it has waited for this grid
  grid_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int j0 = blockIdx.x * 16;
  const float* a0 = a + int64_t{min(j0 + g, rank - 1)} * n_in;
  const float* a1 = a + int64_t{min(j0 + g + 8, rank - 1)} * n_in;
  const __half* xp[NT];
#pragma unroll
  for (int q = 0; q < NT; ++q) xp[q] = x + min(q * 8 + g, n_rows - 1) * ld_x;
  float acc[NT][4] = {};
  // steps of 16 columns, four consecutive ones per lane of a quad
  const int steps = (n_in + 15) / 16;
  const int shares = gridDim.y * DOWN_WARPS, share = blockIdx.y * DOWN_WARPS + warp;
#pragma unroll 2
  for (int s = share; s < steps; s += shares) {
    const int k = s * 16 + t * 4;
    float v0[4], v1[4];
    uint32_t xv[NT][4];
    if (VEC && k + 4 <= n_in) {
      const float4 f0 = __ldg(reinterpret_cast<const float4*>(a0 + k));
      const float4 f1 = __ldg(reinterpret_cast<const float4*>(a1 + k));
      v0[0] = f0.x; v0[1] = f0.y; v0[2] = f0.z; v0[3] = f0.w;
      v1[0] = f1.x; v1[1] = f1.y; v1[2] = f1.z; v1[3] = f1.w;
#pragma unroll
      for (int q = 0; q < NT; ++q) {
        const uint2 h = __ldg(reinterpret_cast<const uint2*>(xp[q] + k));
        const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&h.x));
        const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&h.y));
        xv[q][0] = __float_as_uint(lo.x);
        xv[q][1] = __float_as_uint(lo.y);
        xv[q][2] = __float_as_uint(hi.x);
        xv[q][3] = __float_as_uint(hi.y);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = k + i < n_in;
        v0[i] = in ? __ldg(a0 + k + i) : 0.0f;
        v1[i] = in ? __ldg(a1 + k + i) : 0.0f;
#pragma unroll
        for (int q = 0; q < NT; ++q)
          xv[q][i] = in ? __float_as_uint(__half2float(xp[q][k + i])) : 0u;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t hi[4], lo[4];
      split_tf32(v0[2 * h], hi[0], lo[0]);
      split_tf32(v1[2 * h], hi[1], lo[1]);
      split_tf32(v0[2 * h + 1], hi[2], lo[2]);
      split_tf32(v1[2 * h + 1], hi[3], lo[3]);
#pragma unroll
      for (int q = 0; q < NT; ++q) {
        mma_tf32(acc[q], lo, xv[q][2 * h], xv[q][2 * h + 1]);
        mma_tf32(acc[q], hi, xv[q][2 * h], xv[q][2 * h + 1]);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < NT; ++q) {
    part[warp][(q * 8 + 2 * t) * 16 + g] = acc[q][0];
    part[warp][(q * 8 + 2 * t + 1) * 16 + g] = acc[q][1];
    part[warp][(q * 8 + 2 * t) * 16 + g + 8] = acc[q][2];
    part[warp][(q * 8 + 2 * t + 1) * 16 + g + 8] = acc[q][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * n_rows; i += blockDim.x) {
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < DOWN_WARPS; ++v) sum += part[v][i];
    part[0][i] = sum;
  }
  const int parts = gridDim.y, me = static_cast<int>(cluster_ctarank());
  if (parts > 1)
    cluster_sync();
  else
    __syncthreads();
  for (int i = me * blockDim.x + threadIdx.x; i < 16 * n_rows; i += parts * blockDim.x) {
    const int j = j0 + (i & 15);
    const uint32_t at = smem_u32(&part[0][i]);
    float sum = 0.0f;
    for (int c = 0; c < parts; ++c) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(at, c)));
      sum += v;
    }
    if (j < rank) t_out[(i >> 4) * rank + j] = sum;
  }
  if (parts > 1) cluster_sync();  // every CTA has read the others' sums
}

// ------------------------------------------------------------------------------------------
// The main kernel: rows of whole 64-column blocks on the tensor cores (mma.sync m16n8k16, eight
// weight rows in two parts as the 16-row operand, up to 8 NT rows of x as the n operand).
//
// A warp takes tiles of 16 weight rows; lane (g, t) = (lane / 4, lane % 4) reads 8 packed bytes of
// rows g and g + 8 per block (a quad reads a row's 32 bytes, lane t bytes 4 t .. 4 t + 3 of both
// halves) and turns each byte into the fp16 pairs of its two levels by one 64-bit shared-memory
// read: a table of 256 entries, sixteen copies side by side, so that no two lanes of the half warp
// that such a read takes at a time meet in a bank. Entries lie 256 bytes apart (the second 128 are
// not used), so that one byte permutation makes the address: the packed byte above the lane's own
// eight-byte offset. The reduction index may be permuted as long as both operands agree, so a
// lane's two runs of eight consecutive weights go into four steps as they are and the matching
// operand is two 16-byte pieces of x, a quad's pieces side by side. A block's 64 columns have one
// scale per row: its mma's start from zero and their result is added to the fp32 sum with one FMA
// per value, times the scale.
//
// A level has 24 bits and an fp16 operand 11, so a level is two parts (split_levels): an mma takes
// eight weight rows, the large parts as its upper eight operand rows and the small ones as the
// lower eight, and the two halves of its result are added. With one part, under the best common
// gain, outputs were 4 to 7 % farther from the exact ones than their own rounding puts them, and a
// table other than NF4's could be off by 2^-11 of a term or pass fp16's range; the second part
// costs twice the table's bytes and the mma's (17920 x 1536: one row 7.6 -> 9.3 us, 32 rows 14.8 ->
// 17.0). (16 rows and one part per mma, its operands gathered from the reads by moves: 32 rows 13 %
// more.) The levels take a power of two that brings the largest to [2^14, 2^15), undone by the
// scales: parts are exact to 2^-22 of a level that is at least 2^-17 of the largest, and to 2^-40
// of the largest below.
//
// From nine rows on (NT 2 and 4) a warp takes two such tiles, 32 weight rows, against the same x,
// and a CTA has half as many warps with twice the registers: x is read half as often (with one tile
// and 16 warps 17920 x 1536 took a quarter more at 16 rows, 8 % more at 32). The table reads of an
// mma are made before the mma's ahead of it, and each half of x is replaced as soon as the block is
// done with it. A step's blocks are a loop: as four copies of a block the kernel spilled and waited
// for instructions (32 rows 19.1 -> 17.0 us, one row 9.7 -> 9.3). Prefetching the next blocks of x
// into L1 was slower (32 rows 19.1 -> 20.9).
//
// What bounds it: one row, the latency of dependent shared-memory reads at four warps per scheduler
// (by count a block of a warp is 40 cycles of the SM's shared memory, 32 of them the table's: 7.3k
// of gate + up's 17.8k); 32 rows, 64 mma's per 32 x 64 weights (128 cycles of the tensor cores:
// 11.6k of 32k) and the reads of x, at two warps per scheduler. 32 warps of 64 registers were
// slower with half the table reads (9.7 us against 7.9, spills), and so were entries 128 bytes
// apart (two operations per address).
// ------------------------------------------------------------------------------------------
// 16-row tiles of a warp, and the warps of a CTA
__host__ __device__ constexpr int tiles_of(int nt) { return nt >= 2 ? 2 : 1; }
__host__ __device__ constexpr int warps_of(int nt) { return 16 / tiles_of(nt); }
constexpr int STEP_BLOCKS = 4;  // blocks of 64 columns that a warp loads ahead
constexpr int LUT_BYTES = 256 * 256;
constexpr int STAGES = 4;       // a warp's ring of steps
constexpr int TILE_STAGE_BYTES = 16 * 32 * STEP_BLOCKS;

template <int NT>
constexpr int mma_smem() {
  return LUT_BYTES + 16 * STAGES * TILE_STAGE_BYTES + 256 * 4 + 16 * 16 * 8 * NT * 4;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4],
                                              uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// The fp16 parts of two scaled levels: cut towards zero, and the rest (2^-22 of the level and
// better). The rest of a level that fp16 holds exactly is one step instead of zero, so that both
// parts have the level's sign: an infinite input then gives an infinity of the right sign, where a
// rest of zero or of the other sign would make NaN.
__device__ __forceinline__ float below_exact(float v) {
  const uint32_t bits = __float_as_uint(v);
  return __uint_as_float((bits & 0x1FFFu) == 0 && v != 0.0f ? bits - 1 : bits);
}
__device__ __forceinline__ void split_levels(float v0, float v1, uint32_t& hi, uint32_t& lo) {
  v0 = below_exact(v0);
  v1 = below_exact(v1);
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(v1), "f"(v0));
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  lo = pack_half2(v0 - h.x, v1 - h.y);
}

struct Split {
  int log_w;           // log2 of W, the warps of a CTA that share a tile's columns
  int cluster;         // CTAs that share a tile's columns
  int n_tiles;         // a warp's tiles of 16 or 32 rows
  int n_blocks;        // 64-column blocks of a row
  int shift;           // log2(blocksize)
  int shift2;          // log2(qblock2)
};

// The scale inputs that a lane has loaded for one step: those of block t of the step for its H
// rows (the quad exchanges the finished scales).
template <int H>
struct ScaleIn {
  float s[H], a2[H], o2[H];
  uint32_t a8[H];
};

template <bool GROUPED, int H>
__device__ __forceinline__ void load_scales(ScaleIn<H>& in, const Weight& w, const Split& sp,
                                            const int64_t (&first)[H], int b) {
#pragma unroll
  for (int h = 0; h < H; ++h) {  // first[h]: the flattened index of the row's first weight
    const int64_t block = (first[h] + b * 64) >> sp.shift;
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

// x of one row (xp: at lane t's columns), the 8 columns of lane t in a half of block b: 8 t .. 8 t
// + 7
__device__ __forceinline__ uint4 load_x(const __half* xp, int b, int half) {
  return __ldg(reinterpret_cast<const uint4*>(xp + b * 64) + 4 * half);
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
__global__ void __launch_bounds__(32 * warps_of(NT), 1)
    nf4_mma_kernel(const __half* __restrict__ x, int64_t ld_x, int n_rows, Weight w, Split sp,
                   Epilogue ep, __half* __restrict__ y, int64_t ld_y) {
  constexpr int MT = tiles_of(NT), WARPS = warps_of(NT), ROWS = 16 * MT;
  constexpr int STAGE_BYTES = MT * TILE_STAGE_BYTES;
  constexpr int PART = ROWS * 8 * NT;
  extern __shared__ __align__(128) uint32_t mv_smem[];
  uint8_t* lut = reinterpret_cast<uint8_t*>(mv_smem);             // [256][256]
  uint8_t* rings = lut + LUT_BYTES;                               // [WARPS][STAGES][ROWS][128]
  float* part = reinterpret_cast<float*>(rings + WARPS * STAGES * STAGE_BYTES);
  float* code_s = part + WARPS * PART;  // part: [WARPS][8 NT rows of x][ROWS]; code: [256]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  // W warps of each of the cluster's CTAs share a tile's columns; a CTA works on WARPS / W tiles
  const int W = 1 << sp.log_w, groups = WARPS >> sp.log_w;
  const int group = warp >> sp.log_w, share = warp & (W - 1);
  const int rank = NT == 1 ? 0 : static_cast<int>(cluster_ctarank());
  const int shares = NT == 1 ? W : W * sp.cluster;
  const int place = rank * W + share;
  const int b_first = static_cast<int>(static_cast<unsigned>(sp.n_blocks) * place / shares);
  const int b_last = static_cast<int>(static_cast<unsigned>(sp.n_blocks) * (place + 1) / shares);
  const int n_steps = (b_last - b_first + STEP_BLOCKS - 1) / STEP_BLOCKS;  // of one tile
  const int stride = (NT == 1 ? gridDim.x : gridDim.x / sp.cluster) * groups;
  const int base_tile = (NT == 1 ? blockIdx.x : blockIdx.x / sp.cluster) * groups;
  const int first_tile = base_tile + group;
  const int n_out = static_cast<int>(w.n_out);

  auto sync_tile = [&] {  // the warps of this tile; W >= 2 leaves at most eight barriers
    if (W == 1)
      __syncwarp();
    else
      named_barrier(1 + group, 32 * W);
  };
  // rows past the end read the last one's bytes
  auto row_of = [&](int tile, int r) { return static_cast<int64_t>(min(tile * ROWS + r, n_out - 1)); };

  // This warp's ring of packed bytes: a stage holds four blocks (128 bytes) of the tile's rows,
  // the 16-byte chunk c of row r at chunk c ^ (r & 7) (the reads of eight rows then meet in no
  // bank). The warp fills and reads it alone, STAGES - 1 steps ahead.
  const uint32_t ring = smem_u32(rings) + warp * (STAGES * STAGE_BYTES);
  const int chunk = lane & 7, r8 = lane >> 3;  // this lane copies that chunk of rows r8 + 4 i
  const uint32_t dst0 = ring + r8 * 128 + ((chunk ^ r8) << 4);
  const uint32_t dst1 = ring + (r8 + 4) * 128 + ((chunk ^ (r8 + 4)) << 4);
  const uint8_t* src[4 * MT];
  auto aim = [&](int tile) {
#pragma unroll
    for (int i = 0; i < 4 * MT; ++i)
      src[i] = w.packed + row_of(tile, 4 * i + r8) * (w.n_in >> 1) + chunk * 16;
  };
  int f_tile = first_tile, f_b = b_first;
  uint32_t f_at = 0;
  if (n_steps > 0 && f_tile < sp.n_tiles) aim(f_tile);
  auto fetch = [&] {
    if (f_tile < sp.n_tiles && n_steps > 0) {
      if (f_b + (chunk >> 1) < b_last) {
        const int off = f_b * 32;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
          cp_async16(dst0 + f_at + i * 1024, src[2 * i] + off);
          cp_async16(dst1 + f_at + i * 1024, src[2 * i + 1] + off);
        }
      }
      f_b += STEP_BLOCKS;
      if (f_b >= b_last) {
        f_b = b_first;
        f_tile += stride;
        if (f_tile < sp.n_tiles) aim(f_tile);
      }
      f_at = f_at + STAGE_BYTES == STAGES * STAGE_BYTES ? 0 : f_at + STAGE_BYTES;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch();

  const bool any = n_steps > 0 && first_tile < sp.n_tiles;
  const __half* xp[NT];
#pragma unroll
  for (int q = 0; q < NT; ++q)
    // rows past n_rows read the last one: their columns of the result are not stored
    xp[q] = x + min(q * 8 + g, n_rows - 1) * ld_x + t * 8;
  int64_t e[2 * MT];  // of the tile whose scales are loaded: the flattened index of rows g + 8 h
  auto first_of = [&](int tile) {
#pragma unroll
    for (int h = 0; h < 2 * MT; ++h) e[h] = row_of(tile, g + 8 * h) * w.n_in;
  };
  ScaleIn<2 * MT> cur;
  uint4 xv[NT][2];
  if (any) {
    first_of(first_tile);
    load_scales<GROUPED>(cur, w, sp, e, min(b_first + t, b_last - 1));
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      xv[q][0] = load_x(xp[q], b_first, 0);
      xv[q][1] = load_x(xp[q], b_first, 1);
    }
  }
  // the levels' own scale: the largest magnitude to [2^14, 2^15), undone by the blocks' scales
  float most = fabsf(w.levels ? __ldg(w.levels + (lane & 15)) : kNf4Levels[lane & 15]);
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
  float level_up, level_down;
  power_scale(most, &level_up, &level_down);
  static_assert(32 * WARPS == 512 || 32 * WARPS == 256, "threads fill halves of the table's rows");
#pragma unroll
  for (int half = threadIdx.x >> 8; half < 2; half += WARPS / 8) {
    const int i = threadIdx.x & 255;
    const float v0 = w.levels ? __ldg(w.levels + (i >> 4)) : kNf4Levels[i >> 4];
    const float v1 = w.levels ? __ldg(w.levels + (i & 15)) : kNf4Levels[i & 15];
    uint32_t hi, lo;
    split_levels(level_up * v0, level_up * v1, hi, lo);
    const uint4 two = make_uint4(hi, lo, hi, lo);
#pragma unroll
    for (int k = 0; k < 4; ++k)  // eight neighbours write eight different bank groups
      reinterpret_cast<uint4*>(lut)[i * 16 + ((4 * half + k + i) & 7)] = two;
    if (GROUPED && half == 0) code_s[i] = __ldg(w.code + i);
  }
  __syncthreads();
  // the pair of byte i of v: bytes (lane * 4, v.i, 0, 0) are the entry's offset
  const char* const lut_bytes = reinterpret_cast<const char*>(mv_smem);
  const uint32_t lane8 = (lane & 15) * 8;  // a 64-bit read takes half a warp at a time
  auto level_pair = [&](uint32_t v, int i) {
    return *reinterpret_cast<const uint2*>(lut_bytes + __byte_perm(v, lane8, 0x5504 | (i << 4)));
  };
  const uint8_t* my_ring = rings + warp * (STAGES * STAGE_BYTES) + g * 128 + t * 4;

  int stage = 0;
  // every warp of a cluster makes the same rounds, those without a tile in the last one too
  for (int base = base_tile; base < sp.n_tiles; base += stride) {
    const int tile = base + group;
    const bool has = tile < sp.n_tiles;
    float acc[MT][NT][4] = {};
    for (int b = has ? b_first : b_last; b < b_last; b += STEP_BLOCKS) {
      fetch();
      cp_async_wait<STAGES - 1>();
      __syncwarp();  // every lane's copies of this stage have landed
      // the step after this one (of the next tile behind the last): scales now, x block by block
      const bool last = b + STEP_BLOCKS >= b_last;
      const int n_tile = last ? tile + stride : tile;
      const int n_b = last ? b_first : b + STEP_BLOCKS;
      const bool more = n_tile < sp.n_tiles;
      ScaleIn<2 * MT> next = cur;
      if (more) {
        if (last) first_of(n_tile);
        load_scales<GROUPED>(next, w, sp, e, min(n_b + t, b_last - 1));
      }
      float mine[2 * MT];
#pragma unroll
      for (int h = 0; h < 2 * MT; ++h) {
        float s;
        if constexpr (GROUPED)
          s = __fadd_rn(__fmul_rn(code_s[cur.a8[h]], cur.a2[h]), cur.o2[h]);
        else
          s = cur.s[h];
        mine[h] = s * level_down;
      }
      const uint8_t* st = my_ring + stage * STAGE_BYTES;
      // block b + i of this step with its x in xv, which then gets that of block `ahead`
      auto block = [&](int i, int ahead) {
        // One mma takes eight weight rows: the large parts of their levels as the operand's upper
        // eight rows, the small parts as the lower eight, so that a read of the table is two
        // operand registers as it is. Unit u: row tile u / 8, its rows g + 8 (u % 2), step u / 2 %
        // 4.
        float c[2][NT][4];
        uint2 e[2][2];
        auto look = [&](int u) {
          const int step = u / 2 % 4;
          const uint32_t word = *reinterpret_cast<const uint32_t*>(
              st + (u / 8) * TILE_STAGE_BYTES + (u % 2) * (8 * 128) + (((2 * i + step / 2) ^ g) << 4));
          e[u & 1][0] = level_pair(word, 2 * (step & 1));
          e[u & 1][1] = level_pair(word, 2 * (step & 1) + 1);
        };
        look(0);
#pragma unroll
        for (int u = 0; u < 8 * MT; ++u) {
          const int mt = u / 8, step = u / 2 % 4, h = u % 2;
          if (u + 1 < 8 * MT) look(u + 1);
          const uint32_t a[4] = {e[h][0].x, e[h][0].y, e[h][1].x, e[h][1].y};
#pragma unroll
          for (int q = 0; q < NT; ++q) {
            const uint4 v = xv[q][step / 2];
            const uint32_t b0 = step & 1 ? v.z : v.x, b1 = step & 1 ? v.w : v.y;
            if (step == 0)
              mma_f16_first(c[h][q], a, b0, b1);
            else
              mma_f16(c[h][q], a, b0, b1);
          }
          // this half of x is done with: that of the next block, which is needed half a block later
          if (mt == MT - 1 && step % 2 == 1 && h == 1)
#pragma unroll
            for (int q = 0; q < NT; ++q) xv[q][step / 2] = load_x(xp[q], ahead, step / 2);
          if (step == 3) {
            const float s = __shfl_sync(0xffffffffu, mine[2 * mt + h], i, 4);
#pragma unroll
            for (int q = 0; q < NT; ++q)
#pragma unroll
              for (int k = 0; k < 2; ++k)
                acc[mt][q][2 * h + k] =
                    fmaf(s, c[h][q][k] + c[h][q][2 + k], acc[mt][q][2 * h + k]);
          }
        }
      };
      const int behind = more ? n_b : b;  // whose x is loaded behind this step's
      const int n_here = min(STEP_BLOCKS, b_last - b);
#pragma unroll 1
      for (int i = 0; i < n_here; ++i) block(i, i + 1 < n_here ? b + i + 1 : behind);
      __syncwarp();  // the stage has been read; the next fetch may fill it
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      cur = next;
    }
    // the outputs that this thread finishes, bias first: i = (row of x) * ROWS + (row of the tile)
    const int i0 = (rank * W + share) * 32 + lane, i_step = 32 * shares;
    const int o = tile * ROWS + (lane & (ROWS - 1));  // i0 and i_step are multiples of 32 apart
    const float bias = ep.bias != nullptr && has && o < n_out ? __half2float(ep.bias[o]) : 0.0f;
    if (ep.t != nullptr && has) {
      // scaling * t B^T, eight columns of the rank per share, as tf32 products of split operands
      // (without the product of the two rests): lane columns j + 2 t and j + 2 t + 1. The loads of
      // UNROLL such steps go out together, B's before the wait for t: one latency for all of them
      // (17920 x 1536 at rank 64: one row 14.9 -> 10.6 us, eight 21.5 -> 12.1, with t read through
      // L1 as well).
      constexpr int UNROLL = NT == 4 ? 2 : 4;  // (registers)
      for (int j0 = 8 * place; j0 < ep.rank; j0 += UNROLL * 8 * shares) {
        float bv[UNROLL][4 * MT];
#pragma unroll
        for (int v = 0; v < UNROLL; ++v) {
          const int j = j0 + v * 8 * shares + 2 * t;
#pragma unroll
          for (int h = 0; h < 2 * MT; ++h) {
            const float* br = ep.lora_b + row_of(tile, g + 8 * h) * ep.rank;
#pragma unroll
            for (int u = 0; u < 2; ++u)
              bv[v][h / 2 * 4 + h % 2 + 2 * u] = j + u < ep.rank ? __ldg(br + j + u) : 0.0f;
          }
        }
        grid_dependency_wait();  // t comes from the launch before this one
#pragma unroll
        for (int v = 0; v < UNROLL; ++v) {
          const int j = j0 + v * 8 * shares + 2 * t;
          if (j0 + v * 8 * shares >= ep.rank) break;
          uint32_t b_hi[MT][4], b_lo[MT][4];
#pragma unroll
          for (int u = 0; u < 4 * MT; ++u)
            split_tf32(bv[v][u] * ep.scaling, b_hi[u / 4][u % 4], b_lo[u / 4][u % 4]);
#pragma unroll
          for (int q = 0; q < NT; ++q) {
            const float* tp = ep.t + min(q * 8 + g, n_rows - 1) * ep.rank + j;
            uint32_t t_hi[2], t_lo[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
              split_tf32(j + u < ep.rank ? tp[u] : 0.0f, t_hi[u], t_lo[u]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_tf32(acc[mt][q], b_lo[mt], t_hi[0], t_hi[1]);
              mma_tf32(acc[mt][q], b_hi[mt], t_lo[0], t_lo[1]);
              mma_tf32(acc[mt][q], b_hi[mt], t_hi[0], t_hi[1]);
            }
          }
        }
      }
    }
    // the tile's warps add their shares in share order, then the cluster's CTAs in rank order
    float* mine = part + warp * PART;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int q = 0; q < NT; ++q) {
        float* at = mine + (q * 8 + 2 * t) * ROWS + 16 * mt + g;
        at[0] = acc[mt][q][0];
        at[ROWS] = acc[mt][q][1];
        at[8] = acc[mt][q][2];
        at[ROWS + 8] = acc[mt][q][3];
      }
    sync_tile();
    // Several outputs of a lane at a time, so that their reads are under way together (one after
    // another they took 3 of 9.6 us for 32 rows of 4736 x 64).
    float* sums = part + (group << sp.log_w) * PART;
    constexpr int U = NT == 1 ? 1 : 8;
    const int live = has && o < n_out ? ROWS * n_rows : 0;
    if (NT == 1 || sp.cluster == 1) {
      for (int i = i0; i < live; i += U * i_step) {
        float v[U] = {};
        for (int k = 0; k < W; ++k)
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (i + u * i_step < live) v[u] += sums[k * PART + i + u * i_step];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i + u * i_step < live)
            y[(i + u * i_step) / ROWS * ld_y + o] = __float2half_rn(v[u] + bias);
      }
      sync_tile();
    } else {
      if (W > 1) {
        for (int i = share * 32 + lane; i < ROWS * n_rows; i += U * 32 * W) {
          float v[U] = {};
          for (int k = 0; k < W; ++k)
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (i + u * 32 * W < ROWS * n_rows) v[u] += sums[k * PART + i + u * 32 * W];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (i + u * 32 * W < ROWS * n_rows) sums[i + u * 32 * W] = v[u];
        }
      }
      cluster_sync();
      for (int i = i0; i < live; i += U * i_step) {
        float v[U] = {};
        for (int c = 0; c < sp.cluster; ++c) {
          const uint32_t at = mapa_shared(smem_u32(sums + i), c);
          float p[U];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (i + u * i_step < live)
              asm volatile("ld.shared::cluster.f32 %0, [%1];"
                           : "=f"(p[u]) : "r"(at + u * i_step * 4));
            else
              p[u] = 0.0f;
#pragma unroll
          for (int u = 0; u < U; ++u) v[u] += p[u];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i + u * i_step < live)
            y[(i + u * i_step) / ROWS * ld_y + o] = __float2half_rn(v[u] + bias);
      }
      cluster_sync();  // the sums have been read by every CTA
    }
  }
  cp_async_wait<0>();
  if (ep.t != nullptr) grid_dependency_wait();  // no CTA completes before the launch it follows
}

// Launches the tensor-core kernel for NT groups of eight rows.
template <int NT, bool GROUPED>
int run_mma(const __half* x, int64_t ld_x, int n_rows, const Weight& w, Split sp,
            const Epilogue& ep, __half* y, int64_t ld_y, cudaStream_t stream) {
  static bool ready[kMaxDevices];
  int dev = 0;
  int st = current_device(&dev);
  if (st != TALM_OK) return st;
  constexpr int smem = mma_smem<NT>(), WARPS = warps_of(NT), MT = tiles_of(NT);
  sp.n_tiles = (static_cast<int>(w.n_out) + 16 * MT - 1) / (16 * MT);
  if (!ready[dev]) {  // setting it twice from two threads is harmless
    const cudaError_t e = cudaFuncSetAttribute(nf4_mma_kernel<NT, GROUPED>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess)
      return set_error(TALM_ECUDA, "nf4 matvec set-up: %s", cudaGetErrorString(e));
    ready[dev] = true;
  }
  const int sms = current_sm_count();
  if (sms <= 0) return set_error(TALM_ENODEV, "no CUDA device");
  // How many warps (and CTAs) share a tile's columns: the least time by a model in cycles, fitted
  // to ten shapes with every choice forced (with one part per level; with two its choices are
  // within 4 % of the best of 66 shapes but for 4736 x 64 at one and eight rows, 3.5 against 3.1
  // us). In each round of tiles a warp works through its blocks one after another, finishes the
  // tile (its outputs divided over the warps that share it, whose sums each of them reads) and, in
  // a cluster, meets the other CTAs twice. (17920 x 1536, 32 rows: W = 2, one round of 12 blocks,
  // 17.2 us; W = 4, two rounds of 6, 18.6. 1536 x 8960, 32 rows: clusters of 4 15.0 us, none 23.4.
  // 3000 x 4096, 32 rows: none 13.2, clusters of 2 13.7.) Clusters of 4 find 33 places.
  constexpr int BLOCK = NT == 1 ? 640 : NT == 2 ? 910 : 1490, ROUND = NT == 1 ? 1600 : 2800;
  constexpr int OUTPUTS = 200, JOIN = NT == 1 ? 50 : 150, MEET = NT == 2 ? 2300 : 3200;
  int64_t least = -1;
  int groups = 1, clusters = 1;
  for (int c = 1; c <= (NT == 1 ? 1 : 4); c *= 2) {
    for (int lw = 0; (1 << lw) <= WARPS; ++lw) {
      const int64_t places = c == 4 ? sms * 33 / 148 : sms / c;
      const int64_t slots = (places > 0 ? places : 1) * (WARPS >> lw);
      const int64_t rounds = (sp.n_tiles + slots - 1) / slots;
      const int64_t blocks = (sp.n_blocks + (c << lw) - 1) / (c << lw);
      const int64_t cost = rounds * (blocks * BLOCK + ROUND + OUTPUTS * n_rows / (c << lw) +
                                     (JOIN << lw) + (c > 1 ? MEET : 0));
      if (least < 0 || cost < least) {
        least = cost;
        sp.log_w = lw;
        sp.cluster = c;
        groups = WARPS >> lw;
        clusters = static_cast<int>(places);
      }
    }
  }
  const int wanted = (sp.n_tiles + groups - 1) / groups;
  const int grid = (wanted < clusters ? wanted : clusters) * sp.cluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(32 * WARPS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (sp.cluster > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(sp.cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if (ep.t != nullptr) {
    // behind the adapter's down kernel only: that one starts once everything before it has
    // completed, and this kernel waits for it before it reads t
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
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

// Any even row length, block size and alignment: one warp per output, a byte (two weights) per lane
// and step, eight rows of x at a time. For correctness beside the kernel above, not for speed:
// bound by its two 64-bit divisions and its scale per byte (17920 x 1536: one row 97 us, 32 rows
// 416; 256 x 1536: 16 and 78). Checkpoints as bitsandbytes writes them have blocks of powers of two
// from 64 on, rows of whole blocks and aligned buffers, and do not come here.
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
  if (w_cols >= (int64_t{1} << 30) || w_rows >= (int64_t{1} << 30) ||
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
  const __half* xh = reinterpret_cast<const __half*>(x);
  if (rank > 0) {
    LaunchTimer timer(TALM_KERNEL_ADAPTER_DOWN, stream);
    // as many parts as leave each a thousand columns
    int parts = static_cast<int>(w_cols / 1024 < 1 ? 1 : w_cols / 1024);
    parts = parts < DOWN_PARTS ? parts : DOWN_PARTS;
    const bool vec = w_cols % 4 == 0 && ld_x % 4 == 0 &&
                     (reinterpret_cast<uintptr_t>(x) & 7) == 0 &&
                     (reinterpret_cast<uintptr_t>(lora_a) & 15) == 0;
    auto kernel = n_rows <= 8 ? (vec ? adapter_down_kernel<1, true> : adapter_down_kernel<1, false>)
                              : (vec ? adapter_down_kernel<4, true> : adapter_down_kernel<4, false>);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((rank + 15) / 16), static_cast<unsigned>(parts), 1);
    cfg.blockDim = dim3(32 * DOWN_WARPS, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = static_cast<unsigned>(parts);
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e =
        cudaLaunchKernelEx(&cfg, kernel, xh, ld_x, lora_a, static_cast<int>(w_cols),
                           static_cast<int>(n_rows), static_cast<int>(rank), down);
    if (e != cudaSuccess)
      return set_error(TALM_ECUDA, "adapter down kernel: %s", cudaGetErrorString(e));
  }
  const Epilogue ep{reinterpret_cast<const __half*>(bias), rank > 0 ? down : nullptr, lora_b,
                    static_cast<int>(rank), scaling};
  LaunchTimer timer(TALM_KERNEL_NF4_MATVEC, stream);
  // The tensor-core kernel takes whole 64-column blocks of one scale each, on the boundaries of its
  // wide loads; anything else the byte-wise kernel.
  const int shift = log2_exact(blocksize), shift2 = absmax8 ? log2_exact(qblock2) : 0;
  if (w_cols % 64 == 0 && shift >= 6 && shift2 >= 0 && ld_x % 8 == 0 &&
      ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(packed)) & 15) == 0) {
    const Split sp{0, 1, 0, static_cast<int>(w_cols / 64), shift, shift2};
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
