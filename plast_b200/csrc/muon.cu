// Muon: momentum, orthogonalisation of the update by Newton-Schulz products, weight update.
//
// For a weight of rows x cols (a tensor of more dims counts as shape[0] x the rest) with gradient g
// and momentum v:
//   v = mu v + g,  u = nesterov ? g + mu v : v
//   X = u / (|u|_F + eps), transposed where rows > cols, so that X is m x n with m <= n
//   repeated:  A = X X^T,  B = b A + c A A,  X = a X + B X
//   w = w (1 - lr decay) - lr s X (turned back),  s by the scale rule
// The polynomial a x + b x^3 + c x^5 keeps singular values within [0, 1.2025] and lifts those above
// about 10^-3 to about 1 in five steps.
#include "plast_b200_optim.h"
#include "row_map.cuh"
#include "split_gemm.cuh"
#include "ew_kernel_device.cuh" // pdl_wait / pdl_launch_dependents

#include <algorithm>
#include <math.h>
#include <mutex>
#include <stdlib.h>
#include <unordered_map>
#include <vector>

namespace pb {

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr int kMuonMax = 32;                       // matrices per launch (256 bytes hold their counters)
static_assert(kMuonMax * sizeof(unsigned) <= 256, "");
constexpr u64 kMuonScratch = (u64)2 << 30;         // scratch of one group of matrices
constexpr int kMuonThreads = 256;
constexpr int kMuonChunk = kMuonThreads * 16;      // elements per CTA of the momentum pass

struct MuonMat {
  const float *g;  // gradient, or the input of orthogonalise
  float *v;        // momentum; NULL: u = g
  float *w;        // weight (w = w * keep - rate * X) or, with keep == 0 and rate == -1, the output
  char *x[2], *a, *b; // panels: X (two, in turn), A, B
  double *partial; // sums of squares of the momentum pass, then partial[0] holds their total
  float keep, rate;
  unsigned rows, cols; // as stored
  unsigned m, n;       // m <= n
  unsigned first;      // first CTA of this matrix in the launch at hand
  unsigned first_tile[3], tiles[3]; // of this matrix in the products gram, polynomial, apply
  unsigned chunks;
};
struct MuonTable {
  MuonMat mat[kMuonMax];
  int count;
  unsigned total;     // CTAs of the launch at hand
  unsigned tiles[3];  // of each product
  int narrow[3];      // tiles of 128 x 64 instead of 128 x 128
  unsigned *stored;   // per matrix: warps that have stored their part of a tile, over all products so far
  float mu, epsilon;
  int nesterov;
};

__device__ __forceinline__ int matrix_of(const MuonTable &t, unsigned block) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.mat[mid].first <= block) lo = mid; else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ float update_of(const MuonTable &t, float g, float v) {
  return t.nesterov ? __fmaf_rn(t.mu, v, g) : v;
}

// v = mu v + g and the chunk's sum of u^2 (in 64 bits: the squares of fp32 numbers may leave fp32)
__global__ void __launch_bounds__(kMuonThreads) muon_momentum_kernel(const __grid_constant__ MuonTable t) {
  pdl_wait();
  pdl_launch_dependents();
  const MuonMat &q = t.mat[matrix_of(t, blockIdx.x)];
  const u64 total = (u64)q.rows * q.cols, begin = (u64)(blockIdx.x - q.first) * kMuonChunk;
  double sum = 0.0;
  for (int i = 0; i < kMuonChunk / kMuonThreads; ++i) {
    const u64 j = begin + (u64)i * kMuonThreads + threadIdx.x;
    if (j >= total) break;
    float u = q.g[j];
    if (q.v) {
      const float v = __fmaf_rn(t.mu, q.v[j], u);
      q.v[j] = v;
      u = update_of(t, u, v);
    }
    sum += (double)u * (double)u;
  }
  __shared__ double part[kMuonThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kMuonThreads / 32; ++i) sum += part[i];
    q.partial[1 + blockIdx.x - q.first] = sum;
  }
}

// one CTA per matrix: the chunks' sums in a fixed order
__global__ void __launch_bounds__(kMuonThreads) muon_norm_kernel(const __grid_constant__ MuonTable t) {
  pdl_wait();
  pdl_launch_dependents();
  const MuonMat &q = t.mat[blockIdx.x];
  __shared__ double part[kMuonThreads];
  double sum = 0.0;
  for (unsigned i = threadIdx.x; i < q.chunks; i += kMuonThreads) sum += q.partial[1 + i];
  part[threadIdx.x] = sum;
  __syncthreads();
  for (int o = kMuonThreads / 2; o; o >>= 1) {
    if ((int)threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    q.partial[0] = part[0];
    t.stored[blockIdx.x] = 0; // for the steps
  }
}

// X = u / (|u| + eps), turned so that it has at most as many rows as columns, into its panel: one CTA
// per 128 x 64 block, eight values to a thread; what lies outside the matrix is zero.
__global__ void __launch_bounds__(kMuonThreads) muon_load_kernel(const __grid_constant__ MuonTable t) {
  pdl_wait();
  pdl_launch_dependents();
  const MuonMat &q = t.mat[matrix_of(t, blockIdx.x)];
  __shared__ float tile[kPanelCols][kPanelRows + 1]; // the block, turned
  // in 64 bits: the norm may be outside fp32's range where the quotient is not
  const double inv = (double)kSplitScale / (sqrt(q.partial[0]) + (double)t.epsilon);
  const unsigned col_blocks = panel_col_blocks(q.n), at = blockIdx.x - q.first;
  const unsigned rb = at / col_blocks, cb = at % col_blocks;
  const bool turned = q.rows > q.cols;
  auto value = [&](u64 j) {
    float u = q.g[j];
    if (q.v) u = update_of(t, u, q.v[j]);
    return (float)((double)u * inv);
  };
  if (turned) { // stored row = panel column
    for (unsigned e = threadIdx.x; e < kPanelRows * kPanelCols; e += kMuonThreads) {
      const unsigned i = e % kPanelRows, k = e / kPanelRows; // panel row, panel column
      const unsigned r = cb * kPanelCols + k, c = rb * kPanelRows + i;
      tile[k][i] = r < q.rows && c < q.cols ? value((u64)r * q.cols + c) : 0.0f;
    }
    __syncthreads();
  }
  char *block = q.x[0] + panel_block(rb, cb, col_blocks);
  for (unsigned e = threadIdx.x; e < kPanelRows * 8; e += kMuonThreads) {
    const unsigned row = e / 8, chunk = e % 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (turned) v[i] = tile[chunk * 8 + i][row];
      else {
        const unsigned r = rb * kPanelRows + row, c = cb * kPanelCols + chunk * 8 + i;
        v[i] = r < q.rows && c < q.cols ? value((u64)r * q.cols + c) : 0.0f;
      }
    }
    uint4 hi, lo;
    split8(v, hi, lo);
    *reinterpret_cast<uint4 *>(block + panel_chunk(row, chunk)) = hi;
    *reinterpret_cast<uint4 *>(block + kPanelHalf + panel_chunk(row, chunk)) = lo;
  }
}

// ---- the products --------------------------------------------------------------------------------------
// Three kinds, all on panels of split fp16 numbers (split_gemm.cuh), all values scaled by 2^14:
//   gram        A = X X^T          both operands X, K-major, K = n
//   polynomial  B = b A + c A A    both operands A, K = m
//   apply       X = a X + B X      left B; right X, MN-major (its rows are K), K = m
// A and B are symmetric: only tiles on and above the diagonal are computed and stored. An operand
// block below it is fetched as the block above it and read MN-major, which is its transpose.
//
// One launch goes through all products of all matrices. A persistent CTA takes every gridDim-th tile,
// of 128 x 128 (or 128 x 64); a pair of CTAs (CTAS = 2) tiles of 256 x 256, each CTA holding half of
// either operand. One thread brings 64 KB stages (64 of K, hi and lo of both operands) with bulk
// copies, one warp (of the pair) issues the twelve tcgen05.mma of a stage, small products first, and
// eight warps drain the accumulators. Tensor-core accumulation truncates; every kNsChunk stages the
// accumulator (one of two in tensor memory) is therefore added in fp32 registers, rounded to nearest,
// while the next one fills.
//
// A product of a matrix starts when all tiles of its product before are stored, which a counter per
// matrix in global memory tells; the tiles of other matrices do not wait. The grid is launched
// cooperatively (all of it is resident, so the waits end) and every wait is limited.
enum MuonProduct { kGram = 0, kPolynomial = 1, kApply = 2 };
constexpr int kNsStages = 3;
constexpr unsigned kNsStageBytes = 4 * kPanelHalf; // left hi, left lo, right hi, right lo
constexpr int kNsEpilogueWarps = 8, kNsThreads = (kNsEpilogueWarps + 2) * 32;
#ifndef NS_CHUNK
#define NS_CHUNK 2
#endif
constexpr int kNsChunk = NS_CHUNK;
constexpr unsigned kNsTurnBytes = kNsEpilogueWarps * 32 * 17 * 4; // a 32 x 16 piece per warp, to store rows in order
constexpr unsigned kNsSmem = kNsStages * kNsStageBytes + 1024 + kNsTurnBytes;

__device__ unsigned g_ns_gave_up; // a wait ran out: results are NaN from then on, see plast_b200_muon_status

// tiles along a side, and of a product; `wide`: columns of a tile (256, 128 or 64)
__host__ __device__ inline unsigned ns_along(unsigned size, unsigned tile) { return (size + tile - 1) / tile; }
template <int CTAS> __host__ __device__ inline unsigned ns_wide(bool narrow) { return narrow ? 64 : 128 * CTAS; }
template <int CTAS> __host__ __device__ inline u64 ns_tiles_of(const MuonMat &q, int what, bool narrow) {
  const u64 r = ns_along(q.m, 128 * CTAS), per_diagonal = 128 * CTAS / ns_wide<CTAS>(narrow);
  const u64 c = ns_along(what == kApply ? q.n : q.m, ns_wide<CTAS>(narrow));
  return what == kApply ? r * c : r * c - per_diagonal * (r * (r - 1) / 2); // row i starts at its diagonal block
}

struct NsTile {
  unsigned i, j, k_blocks; // tile row, tile column, K / 64
};
template <int CTAS, int WHAT>
__device__ __forceinline__ const MuonMat &tile_at(const MuonTable &t, unsigned tile, NsTile &out) {
  int lo = 0, hi = t.count - 1; // the last matrix whose first tile is not beyond
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.mat[mid].first_tile[WHAT] <= tile) lo = mid; else hi = mid - 1;
  }
  const MuonMat &q = t.mat[lo];
  const unsigned wide = ns_wide<CTAS>(t.narrow[WHAT]), across = ns_along(WHAT == kApply ? q.n : q.m, wide);
  unsigned at = tile - q.first_tile[WHAT];
  if (WHAT == kApply) {
    out.i = at / across;
    out.j = at % across;
  } else { // rows of the upper triangle
    const unsigned per_diagonal = 128 * CTAS / wide;
    unsigned i = 0, length = across;
    while (at >= length) {
      at -= length;
      length -= per_diagonal;
      ++i;
    }
    out.i = i;
    out.j = i * per_diagonal + at;
  }
  out.k_blocks = panel_col_blocks(WHAT == kGram ? q.n : q.m);
  return q;
}

// 128 rows (block row rb) by 64 of K (block kb) of a panel into `dst`: hi, then lo. `flip`: as the
// transpose of the block above the diagonal, two pieces of 64 K rows by 64 columns each. `narrow`: 64
// rows, rb counts in 64. Returns the bytes; what lies outside the panel is not fetched (it only feeds
// results that are not stored).
__device__ __forceinline__ unsigned operand_bytes(unsigned rb, unsigned row_blocks, unsigned col_blocks, bool flip, bool narrow) {
  if (narrow) return (flip ? rb < col_blocks : rb / 2 < row_blocks) ? kPanelHalf : 0;
  if (!flip) return rb < row_blocks ? 2 * kPanelHalf : 0;
  return 2 * rb + 1 < col_blocks ? 2 * kPanelHalf : (2 * rb < col_blocks ? kPanelHalf : 0);
}
__device__ __forceinline__ void load_operand(uint32_t dst, const char *panel, unsigned rb, unsigned kb, unsigned row_blocks,
                                             unsigned col_blocks, bool flip, bool narrow, uint32_t bar) {
  constexpr unsigned kPiece = kPanelHalf / 2; // 64 rows
  if (narrow) {
    if (flip ? rb >= col_blocks : rb / 2 >= row_blocks) return;
    const char *src = flip ? panel + panel_block(kb / 2, rb, col_blocks) + (kb & 1) * kPiece
                           : panel + panel_block(rb / 2, kb, col_blocks) + (rb & 1) * kPiece;
    bulk_load(dst, src, kPiece, bar);
    bulk_load(dst + kPanelHalf, src + kPanelHalf, kPiece, bar);
    return;
  }
  if (!flip) {
    if (rb < row_blocks) bulk_load(dst, panel + panel_block(rb, kb, col_blocks), 2 * kPanelHalf, bar);
    return;
  }
#pragma unroll
  for (unsigned c = 0; c < 2; ++c)
    if (2 * rb + c < col_blocks) {
      const char *src = panel + panel_block(kb / 2, 2 * rb + c, col_blocks) + (kb & 1) * kPiece;
      bulk_load(dst + c * kPiece, src, kPiece, bar);
      bulk_load(dst + kPanelHalf + c * kPiece, src + kPanelHalf, kPiece, bar);
    }
}

struct NsShared {
  uint64_t full[kNsStages], peer_full[kNsStages], empty[kNsStages], acc_full[2], acc_empty[2], drained;
  uint32_t tmem;
  volatile unsigned gave_up;
  MuonTable table; // a copy: the roles index it at every tile, which is slow in constant memory
};
// A role's place in the rings of stages and accumulators, kept from one product to the next.
struct NsRing {
  uint32_t stages; // shared memory
  unsigned rank;   // in the pair
  unsigned first;  // this CTA's (pair's) first tile of the product at hand
  unsigned it, round;
};

// Waits until matrix q's products up to this one (step s, product what) are stored. Relaxed polling, then
// one fence: an acquiring load would fence at every turn.
template <int CTAS, int WHAT>
__device__ __forceinline__ bool ns_wait_stored(const MuonTable &t, const MuonMat &q, int s, volatile unsigned *gave_up) {
  unsigned target = s * (q.tiles[0] + q.tiles[1] + q.tiles[2]);
  if (WHAT > kGram) target += q.tiles[kGram];
  if (WHAT > kPolynomial) target += q.tiles[kPolynomial];
  target *= CTAS * kNsEpilogueWarps;
  const unsigned *counter = t.stored + (&q - t.mat);
  long long start = 0;
  for (unsigned spins = 0;; ++spins) {
    unsigned now;
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(counter) : "memory");
    if (now >= target) break;
    if (spins == 0) start = clock64();
    if ((spins & 63) == 63) {
      if (*gave_up) return false;
      if (clock64() - start > kWaitCycles) {
        *gave_up = 1;
        return false;
      }
    }
  }
  asm volatile("fence.acq_rel.gpu;" ::: "memory");
  return true;
}

// ---- the thread that loads
template <int CTAS, int WHAT>
__device__ bool ns_load(NsShared &sh, NsRing &ring, int s) {
  const MuonTable &t = sh.table;
  const int from = s & 1;
  const bool narrow = CTAS == 1 && t.narrow[WHAT];
  for (unsigned tile = ring.first; tile < t.tiles[WHAT]; tile += gridDim.x / CTAS) {
    NsTile at;
    const MuonMat &q = tile_at<CTAS, WHAT>(t, tile, at);
    if (!ns_wait_stored<CTAS, WHAT>(t, q, s, &sh.gave_up)) return false;
    asm volatile("fence.proxy.async.global;" ::: "memory"); // panels are written with plain stores
    const unsigned rows = panel_row_blocks(q.m), xcb = panel_col_blocks(q.n), mcb = panel_col_blocks(q.m);
    const char *left = WHAT == kGram ? q.x[from] : WHAT == kPolynomial ? q.a : q.b;
    const char *right = WHAT == kPolynomial ? q.a : q.x[from];
    const unsigned left_cb = WHAT == kGram ? xcb : mcb, right_cb = WHAT == kPolynomial ? mcb : xcb;
    const unsigned i = at.i * CTAS + ring.rank, j = at.j * CTAS + ring.rank;
    const unsigned j_diagonal = narrow ? at.j / 2 : at.j;
    for (unsigned k = 0; k < at.k_blocks; ++k, ++ring.it) {
      const unsigned st = ring.it % kNsStages, phase = (ring.it / kNsStages) & 1;
      const bool flip_left = WHAT != kGram && k / (2 * CTAS) < at.i;
      const bool flip_right = WHAT == kApply || (WHAT == kPolynomial && k / (2 * CTAS) < j_diagonal);
      if (!barrier_wait(smem_address(&sh.empty[st]), phase ^ 1, &sh.gave_up)) return false;
      const uint32_t bar = smem_address(&sh.full[st]), dst = ring.stages + st * kNsStageBytes;
      barrier_expect(bar, operand_bytes(i, rows, left_cb, flip_left, false) + operand_bytes(j, rows, right_cb, flip_right, narrow));
      load_operand(dst, left, i, k, rows, left_cb, flip_left, false, bar);
      load_operand(dst + 2 * kPanelHalf, right, j, k, rows, right_cb, flip_right, narrow, bar);
    }
  }
  return true;
}

// ---- the warp that issues the products (in the second CTA of a pair: passes on that its half is there).
// All lanes walk the loops together, so that descriptors stay in uniform registers; one lane issues.
template <int CTAS, int WHAT>
__device__ bool ns_multiply(NsShared &sh, NsRing &ring) {
  constexpr unsigned kColumns = 128 * CTAS;
  const MuonTable &t = sh.table;
  const bool narrow = CTAS == 1 && t.narrow[WHAT];
  const uint32_t tmem = sh.tmem;
  for (unsigned tile = ring.first; tile < t.tiles[WHAT]; tile += gridDim.x / CTAS) {
    NsTile at;
    tile_at<CTAS, WHAT>(t, tile, at);
    const unsigned j_diagonal = narrow ? at.j / 2 : at.j;
    for (unsigned k = 0; k < at.k_blocks; ++k, ++ring.it) {
      const unsigned st = ring.it % kNsStages, phase = (ring.it / kNsStages) & 1, buf = ring.round & 1;
      if (!__all_sync(0xffffffffu, barrier_wait(smem_address(&sh.full[st]), phase, &sh.gave_up))) return false;
      if (CTAS > 1 && ring.rank != 0) {
        if (elect_one()) barrier_arrive_at(smem_address(&sh.peer_full[st]), 0);
        __syncwarp();
        continue;
      }
      const bool first = k % kNsChunk == 0;
      if (first && !__all_sync(0xffffffffu, barrier_wait(smem_address(&sh.acc_empty[buf]), ((ring.round >> 1) & 1) ^ 1, &sh.gave_up)))
        return false;
      if (CTAS > 1 && !__all_sync(0xffffffffu, barrier_wait(smem_address(&sh.peer_full[st]), phase, &sh.gave_up))) return false;
      tmem_fence_after();
      const bool flip_left = WHAT != kGram && k / (2 * CTAS) < at.i;
      const bool flip_right = WHAT == kApply || (WHAT == kPolynomial && k / (2 * CTAS) < j_diagonal);
      const uint32_t stage = ring.stages + st * kNsStageBytes;
      const uint64_t left = operand_desc(stage, kPanelHalf / 2, 1024);
      const uint64_t right = operand_desc(stage + 2 * kPanelHalf, kPanelHalf / 2, 1024);
      const uint32_t acc = tmem + buf * kColumns;
      const uint32_t desc = mma_desc(128 * CTAS, ns_wide<CTAS>(narrow), flip_left, flip_right);
      // 16 of K: 32 bytes along K-major rows, or 16 rows of 128 bytes; descriptors count in 16 bytes
      const unsigned left_step = flip_left ? 128 : 2, right_step = flip_right ? 128 : 2;
      const bool last = k % kNsChunk == kNsChunk - 1 || k + 1 == at.k_blocks;
      if (elect_one()) {
#pragma unroll
        for (int part = 0; part < 3; ++part) { // lo hi, hi lo, hi hi
          const uint64_t l = left + (part == 0 ? kPanelHalf >> 4 : 0), r = right + (part == 1 ? kPanelHalf >> 4 : 0);
#pragma unroll
          for (int step = 0; step < 4; ++step)
            mma_f16<CTAS>(acc, l + step * left_step, r + step * right_step, desc, !(first && part == 0 && step == 0));
        }
        mma_commit<CTAS>(smem_address(&sh.empty[st]));
        if (last) mma_commit<CTAS>(smem_address(&sh.acc_full[buf]));
      }
      __syncwarp();
      if (last) ++ring.round;
    }
  }
  return true;
}

// ---- the warps that drain: warp w takes rows 32 (w % 4) .. and half of the tile's columns
template <int CTAS, int WHAT>
__device__ bool ns_drain(NsShared &sh, NsRing &ring, int s, bool last, float *turn) {
  constexpr unsigned kColumns = 128 * CTAS;
  const MuonTable &t = sh.table;
  const int from = s & 1;
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned row_in_tile = (warp & 3) * 32 + lane, half = warp >> 2;
  const bool narrow = CTAS == 1 && t.narrow[WHAT];
  const unsigned groups = narrow ? 1 : 2 * CTAS; // of 32 columns
  for (unsigned tile = ring.first; tile < t.tiles[WHAT]; tile += gridDim.x / CTAS) {
    NsTile at;
    const MuonMat &q = tile_at<CTAS, WHAT>(t, tile, at);
    float acc[64 * CTAS];
#pragma unroll
    for (int i = 0; i < 64 * CTAS; ++i) acc[i] = 0.0f;
    const unsigned rounds = (at.k_blocks + kNsChunk - 1) / kNsChunk;
#pragma unroll 1
    for (unsigned c = 0; c < rounds; ++c, ++ring.round) {
      const unsigned buf = ring.round & 1;
      if (!__all_sync(0xffffffffu, barrier_wait(smem_address(&sh.acc_full[buf]), (ring.round >> 1) & 1, &sh.gave_up))) return false;
      tmem_fence_after();
      const uint32_t columns = sh.tmem + (((warp & 3) * 32) << 16) + buf * kColumns + half * groups * 32;
#pragma unroll
      for (int g = 0; g < 2 * CTAS; ++g) {
        if (g >= groups) continue;
        float v[32];
        tmem_load32(columns + g * 32, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[g * 32 + i] += v[i];
      }
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (ring.rank == 0) barrier_arrive(smem_address(&sh.acc_empty[buf]));
        else barrier_arrive_at(smem_address(&sh.acc_empty[buf]), 0);
      }
    }
    const unsigned width = WHAT == kApply ? q.n : q.m, rb = at.i * CTAS + ring.rank;
    const unsigned col_blocks = panel_col_blocks(width), row_blocks = panel_row_blocks(q.m);
    const char *old = WHAT == kPolynomial ? q.a : q.x[from]; // the linear term
    char *out = WHAT == kGram ? q.a : WHAT == kPolynomial ? q.b : q.x[from ^ 1];
    const unsigned row = rb * 128 + row_in_tile;
    // The linear term is other CTAs' work; the accumulators came after it was stored (the loads waited),
    // which orders it for the thread that loaded: this warp looks for itself.
    if (WHAT != kGram) {
      bool ok = true;
      if (lane == 0) ok = ns_wait_stored<CTAS, WHAT>(t, q, s, &sh.gave_up);
      if (!__all_sync(0xffffffffu, ok)) return false;
    }
    // 32 columns at a time: half of a block column. All its loads are issued before its stores: the
    // compiler cannot move a load over a store that may alias it, and a load waits for L2.
#pragma unroll
    for (int g = 0; g < 2 * CTAS; ++g) {
      if (g >= groups || rb >= row_blocks) continue;
      const unsigned col0 = at.j * ns_wide<CTAS>(narrow) + (half * groups + g) * 32;
      const unsigned cb = col0 / kPanelCols, chunk0 = (col0 % kPanelCols) / 8;
      if (cb >= col_blocks) continue;
      const u64 offset = panel_block(rb, cb, col_blocks);
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = acc[g * 32 + i] * kSplitUnscale;
      if (WHAT != kGram) {
        uint4 hi[4], lo[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) { // past L1, which may hold an earlier step's values
          const char *here = old + offset + panel_chunk(row_in_tile, chunk0 + c);
          hi[c] = __ldcg(reinterpret_cast<const uint4 *>(here));
          lo[c] = __ldcg(reinterpret_cast<const uint4 *>(here + kPanelHalf));
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float z[8];
          join8(hi[c], lo[c], z);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float &r = v[c * 8 + i];
            r = WHAT == kPolynomial ? __fmaf_rn(kNsB, z[i], kNsC * r) : __fmaf_rn(kNsA, z[i], r);
          }
        }
      }
      if (WHAT != kApply || !last) {
        if (row >= q.m) { // padding stays zero (an operand read from beyond the panel may leave anything here)
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint4 hi, lo;
          split8(v + c * 8, hi, lo);
          char *here = out + offset + panel_chunk(row_in_tile, chunk0 + c);
          *reinterpret_cast<uint4 *>(here) = hi;
          *reinterpret_cast<uint4 *>(here + kPanelHalf) = lo;
        }
        continue;
      }
      // the weights (or the output), 32 neighbours to an access: where the matrix was turned, the lanes'
      // rows are neighbours as they are, else a piece is turned in shared memory first
      const float scale = g_ns_gave_up ? NAN : kSplitUnscale * q.rate;
      if (q.rows > q.cols) {
        if (row < q.m)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (col0 + i < q.n) {
              float *w = q.w + (u64)(col0 + i) * q.m + row;
              *w = q.keep == 0.0f ? -scale * v[i] : q.keep * *w - scale * v[i];
            }
      } else {
        float *mine = turn + warp * (32 * 17);
        const unsigned row0 = rb * 128 + (warp & 3) * 32 + (lane >> 4);
#pragma unroll
        for (int piece = 0; piece < 2; ++piece) {
#pragma unroll
          for (int i = 0; i < 16; ++i) mine[lane * 17 + i] = v[piece * 16 + i];
          __syncwarp();
          const unsigned col = col0 + piece * 16 + (lane & 15);
          if (col < q.n)
#pragma unroll 8
            for (int r = 0; r < 32; r += 2)
              if (row0 + r < q.m) {
                float *w = q.w + (u64)(row0 + r) * q.n + col;
                const float x = scale * mine[(r + (lane >> 4)) * 17 + (lane & 15)];
                *w = q.keep == 0.0f ? -x : q.keep * *w - x;
              }
          __syncwarp();
        }
      }
    }
    __syncwarp();
    if (lane == 0) asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(t.stored + (&q - t.mat)) : "memory");
  }
  return true;
}

template <int CTAS>
__global__ void __launch_bounds__(kNsThreads, 1) muon_steps_kernel(const __grid_constant__ MuonTable param, int steps) {
  extern __shared__ char dynamic_smem[];
  __shared__ __align__(16) NsShared sh;
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (unsigned i = threadIdx.x; i < sizeof(MuonTable) / 4; i += kNsThreads)
    reinterpret_cast<unsigned *>(&sh.table)[i] = reinterpret_cast<const unsigned *>(&param)[i];
  NsRing ring = {(smem_address(dynamic_smem) + 1023) & ~1023u, CTAS == 1 ? 0 : blockIdx.x % CTAS, 0, 0, 0};
  float *turn = reinterpret_cast<float *>(dynamic_smem + kNsStages * kNsStageBytes + 1024);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kNsStages; ++s) {
      barrier_init(smem_address(&sh.full[s]), 1);
      barrier_init(smem_address(&sh.peer_full[s]), 1);
      barrier_init(smem_address(&sh.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      barrier_init(smem_address(&sh.acc_full[b]), 1);
      barrier_init(smem_address(&sh.acc_empty[b]), kNsEpilogueWarps * CTAS);
    }
    barrier_init(smem_address(&sh.drained), 1);
    sh.gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  if (warp == kNsEpilogueWarps + 1) tmem_alloc<CTAS>(smem_address(&sh.tmem), 2 * 128 * CTAS);
  tmem_fence_before();
  __syncthreads();
  if (CTAS > 1) cluster_sync_all(); // the other CTA's barriers exist
  tmem_fence_after();

  // Tiles are numbered through all products, so that a product that ends between two turns of the grid
  // leaves the next one's first tiles to the CTAs that are free.
  const MuonTable &t = sh.table;
  const unsigned workers = gridDim.x / CTAS, me = blockIdx.x / CTAS;
  unsigned before = 0; // tiles of the products so far, modulo the number of workers
  auto advance = [&](int what) { before = (before + t.tiles[what]) % workers; };
  auto begin = [&] { ring.first = (me + workers - before) % workers; };
  bool ok = true;
  if (warp == kNsEpilogueWarps) {
    if (lane == 0) {
      for (int s = 0; ok && s < steps; ++s) {
        begin();
        ok = ok && ns_load<CTAS, kGram>(sh, ring, s);
        advance(kGram);
        begin();
        ok = ok && ns_load<CTAS, kPolynomial>(sh, ring, s);
        advance(kPolynomial);
        begin();
        ok = ok && ns_load<CTAS, kApply>(sh, ring, s);
        advance(kApply);
      }
      if (!ok) // copies in flight end before shared memory goes away
        for (unsigned back = 1; back <= kNsStages && back <= ring.it; ++back) {
          const unsigned i = ring.it - back, st = i % kNsStages, phase = (i / kNsStages) & 1;
          const long long start = clock64();
          while (!barrier_try(smem_address(&sh.full[st]), phase) && clock64() - start < 10000000) {}
        }
    }
  } else if (warp == kNsEpilogueWarps + 1) {
    for (int s = 0; ok && s < steps; ++s) {
      begin();
      ok = ok && ns_multiply<CTAS, kGram>(sh, ring);
      advance(kGram);
      begin();
      ok = ok && ns_multiply<CTAS, kPolynomial>(sh, ring);
      advance(kPolynomial);
      begin();
      ok = ok && ns_multiply<CTAS, kApply>(sh, ring);
      advance(kApply);
    }
    if (!ok && ring.rank == 0 && lane == 0) { // products in flight end before tensor memory is freed
      mma_commit<CTAS>(smem_address(&sh.drained));
      const long long start = clock64();
      while (!barrier_try(smem_address(&sh.drained), 0) && clock64() - start < 10000000) {}
    }
  } else {
    for (int s = 0; ok && s < steps; ++s) {
      begin();
      ok = ok && ns_drain<CTAS, kGram>(sh, ring, s, false, turn);
      advance(kGram);
      begin();
      ok = ok && ns_drain<CTAS, kPolynomial>(sh, ring, s, false, turn);
      advance(kPolynomial);
      begin();
      ok = ok && ns_drain<CTAS, kApply>(sh, ring, s, s + 1 == steps, turn);
      advance(kApply);
    }
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if (CTAS > 1) cluster_sync_all(); // nothing of this CTA is used by the other one any more
  tmem_fence_after();
  if (threadIdx.x == 0 && sh.gave_up) atomicOr(&g_ns_gave_up, 1u);
  if (warp == kNsEpilogueWarps + 1) tmem_free<CTAS>(sh.tmem, 2 * 128 * CTAS);
}

// steps == 0: X itself
__global__ void __launch_bounds__(kMuonThreads) muon_store_kernel(const __grid_constant__ MuonTable t) {
  pdl_wait();
  pdl_launch_dependents();
  const MuonMat &q = t.mat[matrix_of(t, blockIdx.x)];
  const u64 total = (u64)q.rows * q.cols, begin = (u64)(blockIdx.x - q.first) * kMuonChunk;
  const unsigned col_blocks = panel_col_blocks(q.n);
  for (u64 j = begin + threadIdx.x; j < begin + kMuonChunk && j < total; j += kMuonThreads) {
    unsigned r = (unsigned)(j / q.cols), c = (unsigned)(j % q.cols);
    if (q.rows > q.cols) {
      const unsigned s = r;
      r = c;
      c = s;
    }
    const char *at = q.x[0] + panel_block(r / kPanelRows, c / kPanelCols, col_blocks) +
                     panel_chunk(r % kPanelRows, (c % kPanelCols) / 8) + (c & 7) * 2;
    const float v = (__half2float(*(const __half *)at) + __half2float(*(const __half *)(at + kPanelHalf))) * kSplitUnscale;
    q.w[j] = q.keep == 0.0f ? -q.rate * v : __fmaf_rn(-q.rate, v, q.keep * q.w[j]);
  }
}

// ---- host --------------------------------------------------------------------------------------------
static u64 padded(u64 bytes) { return (bytes + 255) & ~(u64)255; }
static u64 scratch_bytes(const MuonMat &q) {
  return 2 * panel_bytes(q.m, q.n) + 2 * panel_bytes(q.m, q.m) + padded((u64)(q.chunks + 1) * 8);
}

// Numbers the CTAs (or tiles) of a launch over the matrices.
template <class Blocks>
static void number(MuonTable &t, Blocks blocks) {
  u64 n = 0;
  for (int i = 0; i < t.count; ++i) {
    t.mat[i].first = (unsigned)n;
    n += blocks(t.mat[i]);
  }
  t.total = (unsigned)n; // a group's scratch bounds it far below 2^32
}
static bool check_cuda(cudaError_t e) {
  if (e == cudaSuccess) return true;
  cudaGetLastError();
  set_error(PLAST_B200_ERR_CUDA, "muon: %s", cudaGetErrorString(e));
  return false;
}
template <class Blocks>
static bool launch_over(MuonTable &t, Blocks blocks, void (*kernel)(const MuonTable)) {
  number(t, blocks);
  if (!check_cuda(launch_k(kernel, dim3(t.total), dim3(kMuonThreads), 0, stream(), t))) return false;
  count_launch();
  return true;
}
template <int CTAS>
static void run_steps(MuonTable &t, int steps) {
  for (int what = kGram; what <= kApply; ++what) {
    // tiles of 128 x 64 where the GPU has an SM for each
    u64 n = 0;
    for (int i = 0; i < t.count; ++i) n += ns_tiles_of<1>(t.mat[i], what, true);
    t.narrow[what] = CTAS == 1 && n <= (u64)sm_count();
    n = 0;
    for (int i = 0; i < t.count; ++i) {
      MuonMat &q = t.mat[i];
      q.first_tile[what] = (unsigned)n;
      q.tiles[what] = (unsigned)ns_tiles_of<CTAS>(q, what, t.narrow[what]);
      n += q.tiles[what];
    }
    t.tiles[what] = (unsigned)n;
  }
  const auto kernel = muon_steps_kernel<CTAS>;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kNsThreads);
  cfg.dynamicSmemBytes = kNsSmem;
  cfg.stream = stream();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CTAS > 1 ? 2 : 1;
  if (!check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNsSmem))) return;
  // what is resident at once: one CTA per SM, pairs where a GPU partition has two SMs for them
  unsigned most = (unsigned)sm_count();
  if (CTAS > 1) {
    int clusters = 0;
    cfg.gridDim = dim3(CTAS);
    cfg.numAttrs = 1;
    cfg.attrs = attr + 1;
    if (!check_cuda(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg))) return;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    most = (unsigned)clusters;
  }
  const unsigned tiles = std::max(t.tiles[kGram], std::max(t.tiles[kPolynomial], t.tiles[kApply]));
  cfg.gridDim = dim3(std::min(tiles, most) * CTAS);
  if (check_cuda(cudaLaunchKernelEx(&cfg, kernel, t, steps))) count_launch();
}

// One group of matrices whose scratch is `base`.
static void run_group(MuonTable &t, char *base, int steps) {
  auto take = [&](u64 bytes) {
    char *p = base;
    base += bytes;
    return p;
  };
  for (int i = 0; i < t.count; ++i) {
    MuonMat &q = t.mat[i];
    q.x[0] = take(panel_bytes(q.m, q.n));
    q.x[1] = take(panel_bytes(q.m, q.n));
    q.a = take(panel_bytes(q.m, q.m));
    q.b = take(panel_bytes(q.m, q.m));
    q.partial = (double *)take(padded((u64)(q.chunks + 1) * 8));
  }
  t.stored = (unsigned *)take(256);
  auto chunks = [](const MuonMat &q) { return (u64)q.chunks; };
  auto blocks = [](const MuonMat &q) { return (u64)panel_row_blocks(q.m) * panel_col_blocks(q.n); };
  if (!launch_over(t, chunks, muon_momentum_kernel)) return;
  if (!launch_over(t, [](const MuonMat &) { return (u64)1; }, muon_norm_kernel)) return;
  if (!launch_over(t, blocks, muon_load_kernel)) return;
  if (steps > 0) {
    u64 tiles = 0;
    for (int i = 0; i < t.count; ++i) tiles += ns_tiles_of<2>(t.mat[i], kApply, false);
    const bool pairs = tuned(kTuneMuonPairs) >= 0 ? tuned(kTuneMuonPairs) != 0 : tiles >= (u64)sm_count() / 2;
    if (pairs) run_steps<2>(t, steps);
    else run_steps<1>(t, steps);
    return;
  }
  launch_over(t, chunks, muon_store_kernel);
}

// All matrices, in groups that share one piece of scratch.
static void run_matrices(const std::vector<MuonMat> &mats, float mu, float epsilon, int nesterov, int steps) {
  u64 largest = 0;
  std::vector<size_t> ends;
  for (size_t i = 0; i < mats.size();) {
    u64 bytes = 256; // the counters of stored tiles
    size_t k = i;
    while (k < mats.size() && k - i < (size_t)kMuonMax && (k == i || bytes + scratch_bytes(mats[k]) <= kMuonScratch))
      bytes += scratch_bytes(mats[k++]);
    largest = std::max(largest, bytes);
    ends.push_back(i = k);
  }
  char *scratch = nullptr;
  PB_CUDA(scratch_alloc_async((void **)&scratch, largest));
  size_t i = 0;
  for (size_t end : ends) {
    MuonTable t = {};
    t.mu = mu;
    t.epsilon = epsilon;
    t.nesterov = nesterov;
    for (; i < end; ++i) t.mat[t.count++] = mats[i];
    run_group(t, scratch, steps);
    if (failed()) break;
  }
  cudaFreeAsync(scratch, stream());
}

// shape[0] x the rest; false (with an error) for what is not a matrix of ordinary size
static bool matrix_dims(const char *name, int i, const Tensor *t, MuonMat *q) {
  if (t->ndim < 2 || t->ndim > MAX_NDIM) {
    set_error(PLAST_B200_ERR_SHAPE, "%s: tensor %d is not a matrix (2 to %d dims)", name, i, MAX_NDIM);
    return false;
  }
  u64 rest = 1;
  for (u64 d = 1; d < t->ndim; ++d) rest *= t->shape[d];
  if (t->shape[0] > PLAST_MUON_MAX_DIM || rest > PLAST_MUON_MAX_DIM) {
    set_error(PLAST_B200_ERR_LIMIT, "%s: tensor %d has more than %d rows or columns", name, i, PLAST_MUON_MAX_DIM);
    return false;
  }
  q->rows = (unsigned)t->shape[0];
  q->cols = (unsigned)rest;
  q->m = std::min(q->rows, q->cols);
  q->n = std::max(q->rows, q->cols);
  q->chunks = (unsigned)(((u64)q->rows * q->cols + kMuonChunk - 1) / kMuonChunk);
  return true;
}

static bool check_matrix(const char *name, int i, const Tensor *t, const char *what) {
  if (t->dtype != FLOAT32) {
    set_error(PLAST_B200_ERR_DTYPE, "%s: %s %d is not FLOAT32", name, what, i);
    return false;
  }
  if (!t->data && numel(t) > 0) {
    set_error(PLAST_B200_ERR_NULL, "%s: %s %d has no data", name, what, i);
    return false;
  }
  if (!is_packed(t)) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: %s %d is not contiguous", name, what, i);
    return false;
  }
  return true;
}

// A buffer that is written must appear once.
static bool all_distinct(const char *name, std::vector<const void *> written) {
  std::sort(written.begin(), written.end());
  if (std::adjacent_find(written.begin(), written.end()) == written.end()) return true;
  set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: one buffer would be written twice", name);
  return false;
}

static bool check_steps(const char *name, int steps, float epsilon) {
  if (steps < 0 || steps > PLAST_MUON_MAX_STEPS || !(epsilon >= 0.0f) || !(epsilon < INFINITY)) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: 0 to %d steps, epsilon not negative", name, PLAST_MUON_MAX_STEPS);
    return false;
  }
  return true;
}

// ---- momenta owned by the library (as those of Adam) ---------------------------------------------------
struct MuonState {
  Tensor *structs;
  void *slab;
  int n;
};
static std::mutex g_muon_mutex;
static std::unordered_map<Tensor **, MuonState> g_muon_states; // keyed by the m array

// m[i] = zeros like parameters[i], for every parameter that a step updates
static Tensor **create_momenta(Tensor **parameters, int n) {
  Tensor **m = (Tensor **)calloc(n > 0 ? n : 1, sizeof(Tensor *));
  Tensor *structs = (Tensor *)calloc(n > 0 ? n : 1, sizeof(Tensor));
  void *slab = nullptr;
  u64 bytes = 0;
  for (int i = 0; i < n; ++i)
    if (parameters[i]) bytes += padded(numel(parameters[i]) * 4);
  bytes = bytes ? bytes : 256;
  bool ok = m && structs;
  if (!ok) set_error(PLAST_B200_ERR_CUDA, "muon: out of host memory");
  if (ok && cudaMalloc(&slab, bytes) != cudaSuccess) {
    cudaGetLastError();
    set_error(PLAST_B200_ERR_CUDA, "muon: cannot allocate %llu bytes for the momenta", (unsigned long long)bytes);
    ok = false;
  }
  if (ok && cudaMemsetAsync(slab, 0, bytes, stream()) != cudaSuccess) {
    set_error(PLAST_B200_ERR_CUDA, "muon: cannot zero the momenta");
    ok = false;
  }
  if (!ok) {
    if (slab) cudaFree(slab);
    free(m);
    free(structs);
    return nullptr;
  }
  char *cursor = (char *)slab;
  for (int i = 0; i < n; ++i) {
    if (!parameters[i]) continue;
    Tensor *t = &structs[i];
    t->data = cursor;
    t->ndim = parameters[i]->ndim;
    u64 stride = 1;
    for (u64 d = t->ndim; d-- > 0;) {
      t->shape[d] = parameters[i]->shape[d];
      t->strides[d] = stride;
      stride *= t->shape[d];
    }
    t->dtype = FLOAT32;
    t->device = parameters[i]->device;
    cursor += padded(stride * 4);
    m[i] = t;
  }
  std::lock_guard<std::mutex> lock(g_muon_mutex);
  g_muon_states[m] = MuonState{structs, slab, n};
  return m;
}

static void muon_step(Muon *opt, Tensor **parameters, int num_parameters) {
  const char *name = "muon";
  if (!opt) return set_error(PLAST_B200_ERR_NULL, "Muon is NULL");
  if (!parameters && num_parameters > 0) return set_error(PLAST_B200_ERR_NULL, "muon: parameters is NULL");
  if (!check_steps(name, opt->ns_steps, opt->epsilon)) return;
  if (opt->scale != PLAST_MUON_SCALE_ASPECT && opt->scale != PLAST_MUON_SCALE_RMS && opt->scale != PLAST_MUON_SCALE_NONE)
    return set_error(PLAST_B200_ERR_UNSUPPORTED, "muon: unknown scale rule");
  std::vector<MuonMat> mats;
  std::vector<int> index;
  std::vector<const void *> written;
  for (int i = 0; i < num_parameters; ++i) {
    const Tensor *p = parameters[i];
    if (!p || !p->grad) continue;
    MuonMat q = {};
    if (!matrix_dims(name, i, p, &q) || !check_matrix(name, i, p, "parameter") || !check_matrix(name, i, p->grad, "gradient"))
      return;
    if (numel(p->grad) != numel(p)) return set_error(PLAST_B200_ERR_SHAPE, "muon: gradient %d differs in size", i);
    if (numel(p) == 0) continue;
    q.g = (const float *)p->grad->data;
    q.w = (float *)p->data;
    const float r = (float)q.rows, c = (float)q.cols;
    const float s = opt->scale == PLAST_MUON_SCALE_NONE  ? 1.0f
                    : opt->scale == PLAST_MUON_SCALE_RMS ? 0.2f * sqrtf(r > c ? r : c)
                                                         : sqrtf(r > c ? r / c : 1.0f);
    q.rate = opt->lr * s;
    q.keep = 1.0f - opt->lr * opt->weight_decay;
    mats.push_back(q);
    index.push_back(i);
    written.push_back(q.w);
  }
  if (!all_distinct(name, written)) return;
  // momenta: the caller's, or made here on the first step
  bool made = false;
  if (opt->m) {
    std::lock_guard<std::mutex> lock(g_muon_mutex);
    auto it = g_muon_states.find(opt->m);
    if (it != g_muon_states.end() && num_parameters > it->second.n)
      return set_error(PLAST_B200_ERR_SHAPE, "muon: %d parameters, but the momenta were created for %d", num_parameters, it->second.n);
  } else if (!mats.empty()) {
    opt->m = create_momenta(parameters, num_parameters);
    if (!opt->m) return;
    made = true;
  }
  for (size_t k = 0; k < mats.size(); ++k) {
    const Tensor *m = opt->m[index[k]];
    if (!m) return set_error(PLAST_B200_ERR_NULL, "muon: parameter %d has no momentum", index[k]);
    if (!made && (!check_matrix(name, index[k], m, "momentum"))) return;
    if (numel(m) != (u64)mats[k].rows * mats[k].cols)
      return set_error(PLAST_B200_ERR_SHAPE, "muon: momentum %d differs in size", index[k]);
    mats[k].v = (float *)m->data;
    written.push_back(m->data);
  }
  if (!all_distinct(name, written)) return;
  if (mats.empty()) return;
  run_matrices(mats, opt->momentum, opt->epsilon, opt->nesterov != 0, opt->ns_steps);
  note_kernel("muon");
  end_call();
}

static void orthogonalise(const Tensor **inputs, Tensor **outputs, int count, int steps, float epsilon) {
  const char *name = "orthogonalise";
  if ((!inputs || !outputs) && count > 0) return set_error(PLAST_B200_ERR_NULL, "%s: inputs or outputs is NULL", name);
  if (!check_steps(name, steps, epsilon)) return;
  std::vector<MuonMat> mats;
  std::vector<const void *> written;
  for (int i = 0; i < count; ++i) {
    MuonMat q = {};
    if (!inputs[i] || !outputs[i]) return set_error(PLAST_B200_ERR_NULL, "%s: tensor %d is NULL", name, i);
    if (!matrix_dims(name, i, inputs[i], &q) || !check_matrix(name, i, inputs[i], "input") ||
        !check_tensor(outputs[i], "orthogonalise: output", false) || !check_matrix(name, i, outputs[i], "output"))
      return;
    if (!same_shape(inputs[i], outputs[i])) return set_error(PLAST_B200_ERR_SHAPE, "%s: output %d differs in shape", name, i);
    if (numel(inputs[i]) == 0) continue;
    q.g = (const float *)inputs[i]->data;
    q.w = (float *)outputs[i]->data;
    q.keep = 0.0f;
    q.rate = -1.0f;
    mats.push_back(q);
    written.push_back(q.w);
  }
  if (!all_distinct(name, written)) return;
  // an output may be its own input, but not another one's
  std::sort(written.begin(), written.end());
  for (const MuonMat &q : mats)
    if (q.g != q.w && std::binary_search(written.begin(), written.end(), (const void *)q.g))
      return set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: an output is another matrix's input", name);
  if (mats.empty()) return;
  run_matrices(mats, 0.0f, epsilon, 0, steps);
  note_kernel("orthogonalise");
  end_call();
}

} // namespace pb

using namespace pb;

extern "C" {

void muon_step_cuda(Muon *optimizer, Tensor **parameters, int num_parameters) {
  begin_call();
  try {
    muon_step(optimizer, parameters, num_parameters);
  } catch (...) { // std::bad_alloc
    set_error(PLAST_B200_ERR_CUDA, "muon: out of host memory");
  }
}

void plast_b200_orthogonalise(const Tensor **inputs, Tensor **outputs, int count, int steps, float epsilon) {
  begin_call();
  try {
    orthogonalise(inputs, outputs, count, steps, epsilon);
  } catch (...) {
    set_error(PLAST_B200_ERR_CUDA, "orthogonalise: out of host memory");
  }
}

int plast_b200_muon_status(void) {
  begin_call();
  unsigned status = 0;
  PB_CUDA_RET(cudaStreamSynchronize(stream()), -1);
  PB_CUDA_RET(cudaMemcpyFromSymbol(&status, g_ns_gave_up, sizeof status), -1);
  if (status) {
    const unsigned none = 0;
    PB_CUDA_RET(cudaMemcpyToSymbol(g_ns_gave_up, &none, sizeof none), -1);
  }
  return (int)status;
}

void plast_b200_muon_state_release(Tensor **m) {
  MuonState st = {};
  {
    std::lock_guard<std::mutex> lock(g_muon_mutex);
    auto it = g_muon_states.find(m);
    if (it == g_muon_states.end()) return;
    st = it->second;
    g_muon_states.erase(it);
  }
  cudaStreamSynchronize(stream());
  cudaFree(st.slab);
  free(st.structs);
  free(m);
}

} // extern "C"
