// The adapter's rank-wide product on tcgen05: for an activation of n_rows x n_cols,
//   ADD:   y  = fp16(base + scale * T M^T)       (the branch's output: T = t, M = B)
//   MASK:  dx = fp16(keep(...) * scale * T M^T)  (the input's gradient: T = dt, M = A^T)
// T [n_rows, rank] and M [n_cols, rank] are fp32, each split in two bf16 parts that stand side by
// side in rows (hi | lo); a 16-rank slice is three tcgen05 steps, lo hi + hi lo + hi hi (the fourth
// is under 2^-16 of a term). (The 16 x 8 x 16 mma.sync form of the same product needed 96 mma's and
// 40 16-byte loads per 16 x 64 outputs at rank 64, and took 300 us for 16384 x 8960 outputs.)
//
// Bound by HBM: base is read and y written once (4 bytes per output). A persistent CTA walks 128 x
// 128 tiles down the rows of a column tile, whose M stays in shared memory:
//   warp 0      TMA producer: M when the column tile changes, T (three stages), base in boxes of 64
//               columns (six slots)
//   warp 1      MMA issuer: 3 x tcgen05.mma (128 x 128 x 16) per 16 ranks into one of two TMEM
//               buffers
//   warp 2      TMA stores of finished boxes; frees their slots
//   warps 4-19  epilogue: four groups of 128 threads, half a box each: TMEM -> fp32 -> + base (or
//               mask) -> fp16, in place in the box's slot
// Every wait is bounded; a wait that gives up ends the CTA's roles and records TALM_ETIMEOUT.
//
// Measured: ADD 16384 x 8960 at rank 64 100 us (587 MB, 5.9 TB/s, 0.90 of the measured copy); with
// T loaded three parts wide and two stages it was 118 us, the MMA issuer waiting for T a third of
// the time. MASK 16384 x 1536 25 us: 7.7 us of bytes; the generator and the conversions of 128 x
// 128 outputs per CTA take the rest.
#pragma once

#include "adapter_common.cuh"

namespace talm {
namespace adapter {
namespace up {

constexpr int TILE = 128;
constexpr int CHUNK_BYTES = TILE * 128;  // 128 rows of 64 bf16, 128-byte swizzle
constexpr int BOX_BYTES = TILE * 128;    // 128 rows of 64 fp16
constexpr int SLOTS = 6;
constexpr int T_STAGES = 3;
constexpr int EPI_WARPS = 16;
constexpr int FIRST_EPI_WARP = 4;
constexpr int THREADS = 32 * (FIRST_EPI_WARP + EPI_WARPS);

// 64-column chunks of an operand's row (hi | lo)
__host__ __device__ constexpr int chunks(int rp) { return (2 * rp + 63) / 64; }
__host__ __device__ constexpr int smem_bytes(int rp) {
  return (1 + T_STAGES) * chunks(rp) * CHUNK_BYTES + SLOTS * BOX_BYTES + 1024 + 512;
}
static_assert(smem_bytes(64) <= 232448, "shared memory of one CTA");
// where 16 columns from `col` start in a staged operand (chunks of 128-byte rows)
__host__ __device__ constexpr int slice(int col) {
  return col / 64 * CHUNK_BYTES + col % 64 * 2;
}

struct Ctl {
  uint64_t m_full, m_empty;
  uint64_t t_full[T_STAGES], t_empty[T_STAGES];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t box_full[SLOTS], box_done[SLOTS], box_empty[SLOTS];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

struct Params {
  int64_t n_rows;
  int n_cols, row_tiles;
  int64_t n_tiles;
  float scale;
  Dropout drop;
};

template <int RP, bool MASK>
__global__ void __launch_bounds__(THREADS, 1)
    up_kernel(const __grid_constant__ CUtensorMap tm_t, const __grid_constant__ CUtensorMap tm_m,
              const __grid_constant__ CUtensorMap tm_base,
              const __grid_constant__ CUtensorMap tm_out, Params p) {
  constexpr int CHUNKS = chunks(RP);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* m_s = smem;
  uint8_t* t_s = m_s + CHUNKS * CHUNK_BYTES;
  uint8_t* box_s = t_s + T_STAGES * CHUNKS * CHUNK_BYTES;
  Ctl* ctl = reinterpret_cast<Ctl*>(box_s + SLOTS * BOX_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // this CTA's tiles, numbered down the rows of one column tile after another
  const int64_t first = p.n_tiles * blockIdx.x / gridDim.x;
  const int64_t last = p.n_tiles * (blockIdx.x + 1) / gridDim.x;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_t);
    prefetch_tmap(&tm_m);
    prefetch_tmap(&tm_base);
    prefetch_tmap(&tm_out);
    mbar_init(&ctl->m_full, 1);
    mbar_init(&ctl->m_empty, 1);
    for (int i = 0; i < T_STAGES; ++i) {
      mbar_init(&ctl->t_full[i], 1);
      mbar_init(&ctl->t_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->acc_full[i], 1);
      mbar_init(&ctl->acc_empty[i], EPI_WARPS);
    }
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&ctl->box_full[i], 1);
      mbar_init(&ctl->box_done[i], EPI_WARPS / 2);
      mbar_init(&ctl->box_empty[i], 1);
    }
    mbar_init(&ctl->drain, 1);
    ctl->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem_base, 2 * TILE);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_launch_dependents();
  grid_dependency_wait();
  const uint32_t tmem_base = ctl->tmem_base;
  volatile int* abort = &ctl->abort;

  if (warp == 0) {
    if (lane == 0) {  // producer
      int64_t column = -1;
      uint32_t m_phase = 0, m_n = 0, t_n[T_STAGES] = {}, box_n[SLOTS] = {};  // copies issued
      int i = 0;  // tiles so far
      for (int64_t tile = first; tile < last; ++tile, ++i) {
        const int ct = static_cast<int>(tile / p.row_tiles);
        const int row0 = static_cast<int>(tile % p.row_tiles) * TILE;
        if (ct != column) {
          if (column >= 0) {  // the MMAs of the column tile before are done with M
            if (!mbar_wait(&ctl->m_empty, m_phase, abort)) break;
            m_phase ^= 1;
          }
          column = ct;
          ++m_n;
          mbar_arrive_expect_tx(&ctl->m_full, CHUNKS * CHUNK_BYTES);
          for (int c = 0; c < CHUNKS; ++c)
            tma_load_2d(m_s + c * CHUNK_BYTES, &tm_m, &ctl->m_full, c * 64, ct * TILE);
        }
        const int st = i % T_STAGES;
        if (!mbar_wait(&ctl->t_empty[st], ((i / T_STAGES) & 1) ^ 1, abort)) break;
        ++t_n[st];
        mbar_arrive_expect_tx(&ctl->t_full[st], CHUNKS * CHUNK_BYTES);
        for (int c = 0; c < CHUNKS; ++c)
          tma_load_2d(t_s + (st * CHUNKS + c) * CHUNK_BYTES, &tm_t, &ctl->t_full[st], c * 64, row0);
        if (!MASK) {
          bool ok = true;
          for (int q = 0; q < 2; ++q) {
            const int slot = (2 * i + q) % SLOTS;
            if (!mbar_wait(&ctl->box_empty[slot], ((i / (SLOTS / 2)) & 1) ^ 1, abort)) {
              ok = false;
              break;
            }
            ++box_n[slot];
            // a box past the last column is filled with zeros and not stored
            mbar_arrive_expect_tx(&ctl->box_full[slot], BOX_BYTES);
            tma_load_2d(box_s + slot * BOX_BYTES, &tm_base, &ctl->box_full[slot],
                        ct * TILE + q * 64, row0);
          }
          if (!ok) break;
        }
      }
      // every copy issued lands before the CTA gives up its shared memory
      if (m_n) mbar_drain(&ctl->m_full, (m_n - 1) & 1);
      for (int k = 0; k < T_STAGES; ++k)
        if (t_n[k]) mbar_drain(&ctl->t_full[k], (t_n[k] - 1) & 1);
      for (int k = 0; k < SLOTS; ++k)
        if (box_n[k]) mbar_drain(&ctl->box_full[k], (box_n[k] - 1) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {  // MMA issuer
      constexpr uint32_t idesc = idesc_bf16_f32(TILE, TILE, false, false);
      int64_t column = -1;
      uint32_t m_phase = 0;
      int i = 0;
      for (int64_t tile = first; tile < last; ++tile, ++i) {
        const int64_t ct = tile / p.row_tiles;
        if (ct != column) {
          if (!mbar_wait(&ctl->m_full, m_phase, abort)) break;
          m_phase ^= 1;
          column = ct;
        }
        const int st = i % T_STAGES, acc = i & 1;
        if (!mbar_wait(&ctl->t_full[st], (i / T_STAGES) & 1, abort)) break;
        if (!mbar_wait(&ctl->acc_empty[acc], ((i >> 1) & 1) ^ 1, abort)) break;
        tc_fence_after();
        const uint32_t a0 = smem_u32(t_s + st * CHUNKS * CHUNK_BYTES), b0 = smem_u32(m_s);
        const uint32_t d = tmem_base + acc * TILE;
#pragma unroll
        for (int j = 0; j < RP; j += 16) {
          const uint64_t t_hi = smem_desc_sw128(a0 + slice(j), 16, 1024);
          const uint64_t t_lo = smem_desc_sw128(a0 + slice(RP + j), 16, 1024);
          const uint64_t m_hi = smem_desc_sw128(b0 + slice(j), 16, 1024);
          const uint64_t m_lo = smem_desc_sw128(b0 + slice(RP + j), 16, 1024);
          umma_f16(d, t_lo, m_hi, idesc, j != 0);
          umma_f16(d, t_hi, m_lo, idesc, 1);
          umma_f16(d, t_hi, m_hi, idesc, 1);
        }
        umma_commit(&ctl->t_empty[st]);
        umma_commit(&ctl->acc_full[acc]);
        if (tile + 1 < last && (tile + 1) / p.row_tiles != ct) umma_commit(&ctl->m_empty);
      }
      umma_commit(&ctl->drain);
      mbar_drain(&ctl->drain, 0);
    }
  } else if (warp == 2) {
    if (lane == 0) {  // stores
      int i = 0;
      for (int64_t tile = first; tile < last; ++tile, ++i) {
        const int ct = static_cast<int>(tile / p.row_tiles);
        const int row0 = static_cast<int>(tile % p.row_tiles) * TILE;
        bool ok = true;
        for (int q = 0; q < 2; ++q) {
          const int slot = (2 * i + q) % SLOTS;
          if (!mbar_wait(&ctl->box_done[slot], (i / (SLOTS / 2)) & 1, abort)) {
            ok = false;
            break;
          }
          if (ct * TILE + q * 64 < p.n_cols)
            tma_store_2d(&tm_out, box_s + slot * BOX_BYTES, ct * TILE + q * 64, row0);
          bulk_commit();
          // the store before this one has read its slot: free it
          bulk_wait_read<1>();
          if (i > 0 || q > 0) mbar_arrive(&ctl->box_empty[(2 * i + q - 1) % SLOTS]);
        }
        if (!ok) break;
      }
      bulk_wait_all();
    }
  } else if (warp >= FIRST_EPI_WARP) {
    const int quarter = warp & 3, group = (warp - FIRST_EPI_WARP) >> 2;
    const int q = group >> 1, h = group & 1;  // box, and which 32 columns of it
    const int r = quarter * 32 + lane;
    const uint64_t key = MASK && p.drop.drop ? static_cast<uint64_t>(__ldg(p.drop.seed)) : 0;
    const uint32_t bias2 = keep_bias2(p.drop.drop);
    int i = 0;
    for (int64_t tile = first; tile < last; ++tile, ++i) {
      const int ct = static_cast<int>(tile / p.row_tiles);
      const int64_t row = tile % p.row_tiles * TILE + r;
      const int slot = (2 * i + q) % SLOTS, acc = i & 1;
      const uint32_t phase = (i / (SLOTS / 2)) & 1;
      // the masks of these columns while the product is made
      uint32_t keep[MASK ? 16 : 1];
      if (MASK) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[4] = {};
          if (p.drop.drop)
            philox(static_cast<uint64_t>(
                       (row * p.n_cols + ct * TILE + q * 64 + h * 32 + c * 8) >> 3),
                   key, w);
#pragma unroll
          for (int k = 0; k < 4; ++k) keep[4 * c + k] = keep_mask2(w[k], bias2);
        }
      }
      bool ok;
      if (MASK)
        ok = mbar_wait(&ctl->box_empty[slot], phase ^ 1, abort);
      else
        ok = mbar_wait(&ctl->box_full[slot], phase, abort);
      if (ok) ok = mbar_wait(&ctl->acc_full[acc], (i >> 1) & 1, abort);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      uint8_t* box = box_s + slot * BOX_BYTES + r * 128;
      uint32_t d[32];
      tmem_ld_32x32b_x32(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * TILE +
                             q * 64 + h * 32,
                         d);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 4; ++c) {  // eight columns
        uint4* at = reinterpret_cast<uint4*>(box + (((4 * h + c) ^ (r & 7)) << 4));
        uint32_t o[4];
        if (MASK) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            o[k] = pack_half2(p.scale * __uint_as_float(d[8 * c + 2 * k]),
                              p.scale * __uint_as_float(d[8 * c + 2 * k + 1])) &
                   keep[4 * c + k];
        } else {
          const uint4 b = *at;
          const uint32_t bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&bw[k]));
            o[k] = pack_half2(fmaf(p.scale, __uint_as_float(d[8 * c + 2 * k]), f.x),
                              fmaf(p.scale, __uint_as_float(d[8 * c + 2 * k + 1]), f.y));
          }
        }
        *at = make_uint4(o[0], o[1], o[2], o[3]);
      }
      tc_fence_before();
      fence_proxy_async_smem();  // the box is read by a bulk store
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&ctl->acc_empty[acc]);
        mbar_arrive(&ctl->box_done[slot]);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 2 * TILE);
}

// t_op [n_rows, 64 chunks(RP)], m_op [n_cols, 64 chunks(RP)]: the bf16 parts (hi | lo)
template <int RP, bool MASK>
int launch(const void* t_op, const void* m_op, const void* base, int64_t ld_base, void* out,
           int64_t n_rows, int64_t n_cols, float scale, const Dropout& d, cudaStream_t stream) {
  constexpr int smem = smem_bytes(RP), CHUNKS = chunks(RP);
  auto kernel = up_kernel<RP, MASK>;
  // Set on every call: it only notes the value, and it makes the device's context current in a
  // thread that has made no CUDA call yet (autograd's), which the tensor map encoder asks for.
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return set_error(TALM_ECUDA, "smem: %s", cudaGetErrorString(e));
  CUtensorMap tm_t, tm_m, tm_base, tm_out;
  int st = talm_make_tmap_2d_f16(&tm_t, t_op, CHUNKS * 64, n_rows, CHUNKS * 64, 64, TILE);
  if (st == TALM_OK)
    st = talm_make_tmap_2d_f16(&tm_m, m_op, CHUNKS * 64, n_cols, CHUNKS * 64, 64, TILE);
  if (st == TALM_OK) st = talm_make_tmap_2d_f16(&tm_out, out, n_cols, n_rows, n_cols, 64, TILE);
  if (st == TALM_OK)
    st = MASK ? (tm_base = tm_out, TALM_OK)
              : talm_make_tmap_2d_f16(&tm_base, base, n_cols, n_rows, ld_base, 64, TILE);
  if (st != TALM_OK) return st;
  Params p;
  p.n_rows = n_rows;
  p.n_cols = static_cast<int>(n_cols);
  p.row_tiles = static_cast<int>((n_rows + TILE - 1) / TILE);
  p.n_tiles = static_cast<int64_t>(p.row_tiles) * ((n_cols + TILE - 1) / TILE);
  p.scale = scale;
  p.drop = d;
  const int sms = current_sm_count();
  if (sms <= 0) return set_error(TALM_ENODEV, "no CUDA device");
  const unsigned grid = static_cast<unsigned>(p.n_tiles < sms ? p.n_tiles : sms);
  return launch_dependent(kernel, grid, THREADS, smem, stream, tm_t, tm_m, tm_base, tm_out, p);
}

}  // namespace up

// The adapter's sums over an activation X [n_rows, n_cols] on tcgen05, X optionally dropped out:
//   INNER:  part[split][n][j] = sum over the split's columns of X[n, c] W[j, c]
//   OUTER:  part[split][j][c] = sum over the split's rows of X[n, c] T[n, j]
// W (an adapter matrix) and T (t or dt) are fp32, scaled by powers of two (a scale for every 128 of
// the reduction and each rank) and split in two fp16 parts that stand side by side as the n operand
// (N = 2 RP), so that X passes the tensor core once; the epilogue adds the two halves of the
// result. X is the 128-row m operand as it lies in memory: rows of it, K-major, for INNER, columns
// of it, MN-major, for OUTER.
//
// Bound by HBM: X is read once (2 bytes per element, 4 RP flops). One CTA per 128 rows (INNER) or
// columns (OUTER) and split, stages of 64 of the reduction:
//   warp 0        TMA producer           warp 1      MMA issuer, into one of two TMEM buffers
//   warps 4-11    epilogue: two groups of 128 threads, half the ranks each. The buffer is moved
//                 into fp32 registers every two stages, which share a scale; the tensor core's
//                 sums, which are not rounded to nearest, stay short by that.
//   warps 12-19   (MASK) drop X in shared memory before it is multiplied: a 16-byte piece is one
//                 group of the generator
//
// Measured at rank 64, captures with cold caches: dt and dB of 16384 x 8960 in one launch 98 to 100
// us (g is 294 MB and read for each; 493 MB of the 588 come from HBM), dB by itself, where no dt is
// wanted, 66 us (its splits are those of the pair, so that it has the pair's bits); with the
// dropout of 16384 x 1536 t 25 to 27 us and dA 22 to 23 (7.7 us of bytes): of the 1600 cycles that
// a stage takes a mask warp, 850 go into the generator and 380 into the and, at 45 % of the issue
// slots: latency with eight mask warps per SM, not the generator's own rate (some 9 us in all); 16
// mask warps or its products as whole 64-bit ones changed nothing. The mma.sync form of t, dt, dB
// and dA took 70, 171, 276 and 74 us.
namespace sums {

constexpr int TILE = 128;
constexpr int X_BYTES = 16384;  // 64 x 128 fp16
constexpr int EPI_WARPS = 8, MASK_WARPS = 8;
constexpr int FIRST_EPI_WARP = 4, FIRST_MASK_WARP = FIRST_EPI_WARP + EPI_WARPS;
constexpr int MAX_STAGES = 6;

__host__ __device__ constexpr int pair_width(int rp) { return 2 * rp < 64 ? 64 : 2 * rp; }
template <int RP, bool OUTER>
__host__ __device__ constexpr int other_bytes() {  // of the n operand per stage
  return OUTER ? pair_width(RP) * 64 * 2 : 2 * RP * 128;
}
template <int RP, bool OUTER, bool MASK>
__host__ __device__ constexpr int stages() {  // two CTAs per SM, or one with its mask warps
  return MASK ? MAX_STAGES : 98304 / (X_BYTES + other_bytes<RP, OUTER>());
}
template <int RP, bool OUTER, bool MASK>
__host__ __device__ constexpr int smem_bytes() {
  return stages<RP, OUTER, MASK>() * (X_BYTES + other_bytes<RP, OUTER>()) + 1024 + 512;
}
__host__ __device__ constexpr int threads(bool mask) {
  return 32 * (FIRST_MASK_WARP + (mask ? MASK_WARPS : 0));
}

struct Ctl {
  uint64_t full[MAX_STAGES], masked[MAX_STAGES], empty[MAX_STAGES];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

struct Params {
  int64_t n_rows;
  int n_cols;
  int steps, steps_per_split;  // 64-wide stages of the whole reduction, and of a split
  const float* down;           // what undoes the scales: [blocks of 128][RP]
  float* part;
  Dropout drop;
};

// One CTA: the tile's split `split`.
template <int RP, bool OUTER, bool MASK>
__device__ __forceinline__ void sums_cta(const CUtensorMap& tm_x, const CUtensorMap& tm_o,
                                         const Params& p, int tile, int split) {
  constexpr int STAGES = stages<RP, OUTER, MASK>();
  constexpr int O_BYTES = other_bytes<RP, OUTER>();
  constexpr int N = 2 * RP;
  constexpr int COLS = N < 32 ? 32 : N;  // TMEM columns of a buffer
  constexpr int FLUSH = 2;  // stages of a scale
  extern __shared__ uint8_t smem_raw[];
  uint8_t* x_s = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                            ~uintptr_t(1023));
  uint8_t* o_s = x_s + STAGES * X_BYTES;
  Ctl* ctl = reinterpret_cast<Ctl*>(o_s + STAGES * O_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t origin = static_cast<int64_t>(tile) * TILE;  // first row / column
  const int s0 = split * p.steps_per_split;
  const int n_steps = min(p.steps, s0 + p.steps_per_split) - s0;  // at least one

  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_o);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&ctl->full[i], 1);
      mbar_init(&ctl->masked[i], MASK_WARPS);
      mbar_init(&ctl->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->acc_full[i], 1);
      mbar_init(&ctl->acc_empty[i], EPI_WARPS);
    }
    mbar_init(&ctl->drain, 1);
    ctl->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem_base, 2 * COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_launch_dependents();
  grid_dependency_wait();
  const uint32_t tmem_base = ctl->tmem_base;
  volatile int* abort = &ctl->abort;

  if (warp == 0) {
    if (lane == 0) {  // producer
      int i = 0;
      for (; i < n_steps; ++i) {
        const int st = i % STAGES;
        if (!mbar_wait(&ctl->empty[st], ((i / STAGES) & 1) ^ 1, abort)) break;
        const int at = (s0 + i) * 64, o = static_cast<int>(origin);
        uint8_t* x = x_s + st * X_BYTES;
        uint8_t* w = o_s + st * O_BYTES;
        mbar_arrive_expect_tx(&ctl->full[st], X_BYTES + O_BYTES);
        if (OUTER) {  // 64 rows of 2 x 64 columns; the parts' 64 rows
          tma_load_2d(x, &tm_x, &ctl->full[st], o, at);
          tma_load_2d(x + 8192, &tm_x, &ctl->full[st], o + 64, at);
          for (int b = 0; b < O_BYTES / 8192; ++b)
            tma_load_2d(w + b * 8192, &tm_o, &ctl->full[st], b * 64, at);
        } else {  // 128 rows of 64 columns; the parts' 64 columns
          tma_load_2d(x, &tm_x, &ctl->full[st], at, o);
          tma_load_2d(w, &tm_o, &ctl->full[st], at, 0);
        }
      }
      for (int k = 0; k < STAGES; ++k) {  // every copy issued lands before the CTA ends
        const int n = (i - k + STAGES - 1) / STAGES;
        if (i > k) mbar_drain(&ctl->full[k], (n - 1) & 1);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {  // MMA issuer
      constexpr uint32_t idesc = idesc_f16_f32(TILE, N, OUTER, OUTER);
      for (int i = 0; i < n_steps; ++i) {
        const int st = i % STAGES, f = i / FLUSH;
        if (i % FLUSH == 0 &&
            !mbar_wait(&ctl->acc_empty[f & 1], ((f >> 1) & 1) ^ 1, abort)) break;
        if (!mbar_wait(&ctl->full[st], (i / STAGES) & 1, abort)) break;
        if (MASK && !mbar_wait(&ctl->masked[st], (i / STAGES) & 1, abort)) break;
        tc_fence_after();
        const uint32_t a = smem_u32(x_s + st * X_BYTES), b = smem_u32(o_s + st * O_BYTES);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // MN-major: 16 rows of 128 bytes further, 8 KiB between groups of 64 columns;
          // K-major: 32 bytes further
          const uint64_t ad = OUTER ? smem_desc_sw128(a + k * 2048, 8192, 1024)
                                    : smem_desc_sw128(a + k * 32, 16, 1024);
          const uint64_t bd = OUTER ? smem_desc_sw128(b + k * 2048, 8192, 1024)
                                    : smem_desc_sw128(b + k * 32, 16, 1024);
          umma_f16(tmem_base + (f & 1) * COLS, ad, bd, idesc, i % FLUSH != 0 || k != 0);
        }
        umma_commit(&ctl->empty[st]);
        if (i % FLUSH == FLUSH - 1 || i + 1 == n_steps) umma_commit(&ctl->acc_full[f & 1]);
      }
      umma_commit(&ctl->drain);
      mbar_drain(&ctl->drain, 0);
    }
  } else if (warp >= FIRST_EPI_WARP && warp < FIRST_MASK_WARP) {
    constexpr int HR = RP / 2;  // ranks of a group
    const int quarter = warp & 3, q = (warp - FIRST_EPI_WARP) >> 2;
    const int r = quarter * 32 + lane;
    float acc[HR] = {};
    const int flushes = (n_steps + FLUSH - 1) / FLUSH;
    bool ok = true;
    for (int f = 0; f < flushes; ++f) {
      const float4* down = reinterpret_cast<const float4*>(
          p.down + static_cast<int64_t>(s0 / FLUSH + f) * RP + q * HR);
      ok = mbar_wait(&ctl->acc_full[f & 1], (f >> 1) & 1, abort);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t ta = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                          (f & 1) * COLS + q * HR;
      constexpr int STEP = HR < 16 ? HR : 16;
#pragma unroll
      for (int j = 0; j < HR; j += STEP) {
        uint32_t hi[STEP], lo[STEP];
#pragma unroll
        for (int u = 0; u < STEP; u += 8) {
          tmem_ld_32x32b_x8(ta + j + u, hi + u);
          tmem_ld_32x32b_x8(ta + RP + j + u, lo + u);
        }
        tmem_wait_ld();
#pragma unroll
        for (int u = 0; u < STEP; u += 4) {
          const float4 scale = __ldg(down + (j + u) / 4);
          const float by[4] = {scale.x, scale.y, scale.z, scale.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            acc[j + u + k] = fmaf(by[k], __uint_as_float(hi[u + k]) + __uint_as_float(lo[u + k]),
                                  acc[j + u + k]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->acc_empty[f & 1]);
    }
    const int64_t at = origin + r;
    if (ok && at < (OUTER ? p.n_cols : p.n_rows)) {
      if (OUTER) {
        float* out = p.part + (static_cast<int64_t>(split) * RP + q * HR) * p.n_cols + at;
#pragma unroll
        for (int j = 0; j < HR; ++j) out[static_cast<int64_t>(j) * p.n_cols] = acc[j];
      } else {
        float4* out = reinterpret_cast<float4*>(
            p.part + (static_cast<int64_t>(split) * p.n_rows + at) * RP + q * HR);
#pragma unroll
        for (int j = 0; j < HR; j += 4)
          out[j / 4] = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
      }
    }
  } else if (MASK && warp >= FIRST_MASK_WARP) {
    const int id = threadIdx.x - 32 * FIRST_MASK_WARP;
    const uint64_t key = static_cast<uint64_t>(__ldg(p.drop.seed));
    const uint32_t bias2 = keep_bias2(p.drop.drop);
    constexpr int U = X_BYTES / 16 / (32 * MASK_WARPS);  // pieces of a thread
    constexpr int LINES = 32 * MASK_WARPS / 8;           // between a thread's pieces
    // A piece is a group of eight columns of line id / 8 + u * LINES of the stage; a line is 128
    // bytes: a row of INNER's 64 columns; OUTER: row + 64 * (column group). q[u]: the group's
    // number, which moves on by a constant from stage to stage.
    const int64_t row_groups = p.n_cols / 8;
    int64_t q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int line = id / 8 + u * LINES;
      q[u] = OUTER ? (static_cast<int64_t>(s0) * 64 + (line & 63)) * row_groups + origin / 8 +
                         (line >> 6) * 8 + (id & 7)
                   : (origin + line) * row_groups + s0 * 8 + (id & 7);
    }
    for (int i = 0; i < n_steps; ++i) {
      const int st = i % STAGES;
      uint8_t* x = x_s + st * X_BYTES;
      uint32_t w[U][4];  // the masks while the stage is on its way
#pragma unroll
      for (int u = 0; u < U; ++u) {
        philox(static_cast<uint64_t>(q[u]), key, w[u]);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[u][k] = keep_mask2(w[u][k], bias2);
        q[u] += OUTER ? 64 * row_groups : 8;
      }
      const bool ok = mbar_wait(&ctl->full[st], (i / STAGES) & 1, abort);
      if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = u * (32 * MASK_WARPS) + id, line = e >> 3, c = e & 7;
        uint4* at = reinterpret_cast<uint4*>(x + line * 128 + ((c ^ (line & 7)) << 4));
        uint4 v = *at;
        v.x &= w[u][0];
        v.y &= w[u][1];
        v.z &= w[u][2];
        v.w &= w[u][3];
        *at = v;
      }
      fence_proxy_async_smem();  // the tensor core reads it
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->masked[st]);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 2 * COLS);
}

template <int RP, bool OUTER, bool MASK>
__global__ void __launch_bounds__(threads(MASK), MASK ? 1 : 2)
    sums_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_o,
                const __grid_constant__ Params p) {
  sums_cta<RP, OUTER, MASK>(tm_x, tm_o, p, blockIdx.x, blockIdx.y);
}

// dt and dB, which read the same gradient and do not wait for one another, in one launch. dB's CTAs
// come first, one per SM, and a row tile's splits side by side (16384 x 1536 to 8960, forward and
// backward: rank 16 269 -> 262 us, rank 64 307 -> 304, against dt first and dB with two CTAs per
// SM).
template <int RP>
__global__ void __launch_bounds__(threads(false), 2)
    sums_pair_kernel(const __grid_constant__ CUtensorMap in_x,
                     const __grid_constant__ CUtensorMap in_o, const __grid_constant__ Params in_p,
                     int inner_splits, const __grid_constant__ CUtensorMap out_x,
                     const __grid_constant__ CUtensorMap out_o,
                     const __grid_constant__ Params out_p, int outer_tiles, int outer_ctas) {
  const int id = blockIdx.x, inner = id - outer_ctas;
  if (inner >= 0)
    sums_cta<RP, false, false>(in_x, in_o, in_p, inner / inner_splits, inner % inner_splits);
  else
    sums_cta<RP, true, false>(out_x, out_o, out_p, id % outer_tiles, id / outer_tiles);
}

// How the reduction is divided: as many CTAs as 148 SMs hold at a time (two of them, or `one` per
// SM: with its mask warps, and for dB beside dt), two blocks of 128 (which share a scale) for a CTA
// at least. A B200's 148 are a constant: the sizes of workspaces and the order of sums go by it,
// and neither may depend on which device is current when it is asked.
struct Plan {
  int tiles = 0, steps = 0, steps_per_split = 0, splits = 0;
  Plan() = default;
  Plan(bool outer, bool one, int64_t n_rows, int64_t n_cols) {
    tiles = static_cast<int>(((outer ? n_cols : n_rows) + TILE - 1) / TILE);
    const int64_t length = outer ? n_rows : n_cols;
    steps = static_cast<int>((length + 63) / 64);
    const int blocks = (steps + 1) / 2;
    int want = (one ? 148 : 296) / tiles;
    const int most = (blocks + 1) / 2;
    if (want > most) want = most;
    if (want > 32) want = 32;
    if (want < 1) want = 1;
    steps_per_split = (blocks + want - 1) / want * 2;
    splits = (steps + steps_per_split - 1) / steps_per_split;
  }
};

// The arguments of a launch. x: the activation; other: W parts [2 RP, n_cols] (INNER) or T parts
// [n_rows, pair_width] (OUTER).
struct Call {
  CUtensorMap tm_x, tm_o;
  Params p;
  Plan plan;
};

template <int RP, bool OUTER, bool MASK>
int make_call(const Plan& plan, const void* x, int64_t ld, int64_t n_rows, int64_t n_cols,
              const void* other, const float* down, const Dropout& d, float* part, Call* c) {
  c->plan = plan;
  c->p = Params{n_rows, static_cast<int>(n_cols), c->plan.steps, c->plan.steps_per_split,
                down,   part,                     d};
  int st = talm_make_tmap_2d_f16(&c->tm_x, x, n_cols, n_rows, ld, 64, OUTER ? 64 : TILE);
  if (st == TALM_OK)
    st = OUTER ? talm_make_tmap_2d_f16(&c->tm_o, other, pair_width(RP), n_rows, pair_width(RP), 64,
                                       64)
               : talm_make_tmap_2d_f16(&c->tm_o, other, n_cols, 2 * RP, n_cols, 64, 2 * RP);
  return st;
}

template <int RP, bool OUTER, bool MASK>
int launch(const Plan& plan, const void* x, int64_t ld, int64_t n_rows, int64_t n_cols,
           const void* other, const float* down, const Dropout& d, float* part,
           cudaStream_t stream) {
  constexpr int smem = smem_bytes<RP, OUTER, MASK>();
  static_assert(smem <= 232448 && (MASK || 2 * smem <= 232448), "shared memory");
  auto kernel = sums_kernel<RP, OUTER, MASK>;
  // before the tensor maps, as in up::launch
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return set_error(TALM_ECUDA, "smem: %s", cudaGetErrorString(e));
  Call c;
  const int st = make_call<RP, OUTER, MASK>(plan, x, ld, n_rows, n_cols, other, down, d, part, &c);
  if (st != TALM_OK) return st;
  return launch_dependent(
      kernel, dim3(static_cast<unsigned>(c.plan.tiles), static_cast<unsigned>(c.plan.splits), 1),
      threads(MASK), smem, stream, c.tm_x, c.tm_o, c.p);
}

// dt = g B and dB = g^T t (see sums_pair_kernel).
template <int RP>
int launch_pair(const Plan& dt_plan, const Plan& db_plan, const void* g, int64_t ld, int64_t n_rows,
                int64_t n_cols, const void* w_parts, const float* w_down, float* dt_part,
                const void* t_parts, const float* t_down, float* db_part, cudaStream_t stream) {
  constexpr int a = smem_bytes<RP, false, false>(), b = smem_bytes<RP, true, false>();
  constexpr int smem = a > b ? a : b;
  auto kernel = sums_pair_kernel<RP>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return set_error(TALM_ECUDA, "smem: %s", cudaGetErrorString(e));
  const Dropout none{nullptr, 0, 1.0f};
  Call in, out;
  int st = make_call<RP, false, false>(dt_plan, g, ld, n_rows, n_cols, w_parts, w_down, none,
                                       dt_part, &in);
  if (st == TALM_OK)
    st = make_call<RP, true, false>(db_plan, g, ld, n_rows, n_cols, t_parts, t_down, none, db_part,
                                    &out);
  if (st != TALM_OK) return st;
  const int inner = dt_plan.tiles * dt_plan.splits, outer = db_plan.tiles * db_plan.splits;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(inner + outer)), threads(false), smem,
                          stream, in.tm_x, in.tm_o, in.p, dt_plan.splits, out.tm_x, out.tm_o, out.p,
                          db_plan.tiles, outer);
}

}  // namespace sums
}  // namespace adapter
}  // namespace talm
