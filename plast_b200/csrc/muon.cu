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
constexpr int kMuonMax = 32;                       // matrices per launch
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
  unsigned first_tile[3]; // first tile of this matrix in the products gram, polynomial, apply
  unsigned chunks;
};
struct MuonTable {
  MuonMat mat[kMuonMax];
  int count;
  unsigned total;     // CTAs of the launch at hand
  unsigned tiles[3];  // of each product
  int narrow[3];      // tiles of 128 x 64 instead of 128 x 128
  unsigned *arrived;  // grid barrier of the fused steps
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
    if (blockIdx.x == 0) *t.arrived = 0; // for the grid barrier of the steps
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
// A persistent CTA walks tiles of 128 x 128 (or 128 x 64); a pair of CTAs (CTAS = 2) walks tiles of
// 256 x 256, each CTA holding half of either operand. One thread brings 64 KB stages (64 of K, hi and
// lo of both operands) with bulk copies, one thread (of the pair) issues the twelve tcgen05.mma of a
// stage, small products first, and eight warps drain the accumulators. Tensor-core accumulation
// truncates; every kNsChunk stages the accumulator (one of two in tensor memory) is therefore added in
// fp32 registers, rounded to nearest, while the next one fills.
enum MuonProduct { kGram = 0, kPolynomial = 1, kApply = 2 };
constexpr int kNsStages = 3;
constexpr unsigned kNsStageBytes = 4 * kPanelHalf; // left hi, left lo, right hi, right lo
constexpr int kNsEpilogueWarps = 8, kNsThreads = (kNsEpilogueWarps + 2) * 32;
#ifndef NS_CHUNK
#define NS_CHUNK 2
#endif
constexpr int kNsChunk = NS_CHUNK;
constexpr unsigned kNsTurnBytes = kNsEpilogueWarps * 32 * 33 * 4; // a 32 x 32 piece per warp, to store rows in order
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
  int lo = 0, hi = t.count - 1;
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
};
// A role's place in the rings of stages and accumulators, kept from one product to the next.
struct NsRing {
  uint32_t stages; // shared memory
  unsigned rank;   // in the pair
  unsigned it, round;
};

// ---- the thread that loads
template <int CTAS, int WHAT>
__device__ bool ns_load(const MuonTable &t, int from, NsShared &sh, NsRing &ring) {
  const bool narrow = CTAS == 1 && t.narrow[WHAT];
  for (unsigned tile = blockIdx.x / CTAS; tile < t.tiles[WHAT]; tile += gridDim.x / CTAS) {
    NsTile at;
    const MuonMat &q = tile_at<CTAS, WHAT>(t, tile, at);
    const unsigned rows = panel_row_blocks(q.m), xcb = panel_col_blocks(q.n), mcb = panel_col_blocks(q.m);
    const char *left = WHAT == kGram ? q.x[from] : WHAT == kPolynomial ? q.a : q.b;
    const char *right = WHAT == kPolynomial ? q.a : q.x[from];
    const unsigned left_cb = WHAT == kGram ? xcb : mcb, right_cb = WHAT == kPolynomial ? mcb : xcb;
    const unsigned i = at.i * CTAS + ring.rank, j = at.j * CTAS + ring.rank;
    const unsigned j_diagonal = narrow ? at.j / 2 : at.j;
    for (unsigned k = 0; k < at.k_blocks; ++k, ++ring.it) {
      const unsigned s = ring.it % kNsStages, phase = (ring.it / kNsStages) & 1;
      const bool flip_left = WHAT != kGram && k / (2 * CTAS) < at.i;
      const bool flip_right = WHAT == kApply || (WHAT == kPolynomial && k / (2 * CTAS) < j_diagonal);
      if (!barrier_wait(smem_address(&sh.empty[s]), phase ^ 1, &sh.gave_up)) return false;
      const uint32_t bar = smem_address(&sh.full[s]), dst = ring.stages + s * kNsStageBytes;
      barrier_expect(bar, operand_bytes(i, rows, left_cb, flip_left, false) + operand_bytes(j, rows, right_cb, flip_right, narrow));
      load_operand(dst, left, i, k, rows, left_cb, flip_left, false, bar);
      load_operand(dst + 2 * kPanelHalf, right, j, k, rows, right_cb, flip_right, narrow, bar);
    }
  }
  return true;
}

// ---- the thread that issues the products (in the second CTA of a pair: passes on that its half is there)
template <int CTAS, int WHAT>
__device__ bool ns_multiply(const MuonTable &t, NsShared &sh, NsRing &ring) {
  constexpr unsigned kColumns = 128 * CTAS;
  const bool narrow = CTAS == 1 && t.narrow[WHAT];
  for (unsigned tile = blockIdx.x / CTAS; tile < t.tiles[WHAT]; tile += gridDim.x / CTAS) {
    NsTile at;
    tile_at<CTAS, WHAT>(t, tile, at);
    const unsigned j_diagonal = narrow ? at.j / 2 : at.j;
    for (unsigned k = 0; k < at.k_blocks; ++k, ++ring.it) {
      const unsigned s = ring.it % kNsStages, phase = (ring.it / kNsStages) & 1, buf = ring.round & 1;
      if (CTAS > 1 && ring.rank != 0) {
        if (!barrier_wait(smem_address(&sh.full[s]), phase, &sh.gave_up)) return false;
        barrier_arrive_at(smem_address(&sh.peer_full[s]), 0);
        continue;
      }
      const bool flip_left = WHAT != kGram && k / (2 * CTAS) < at.i;
      const bool flip_right = WHAT == kApply || (WHAT == kPolynomial && k / (2 * CTAS) < j_diagonal);
      const bool first = k % kNsChunk == 0;
      if (first && !barrier_wait(smem_address(&sh.acc_empty[buf]), ((ring.round >> 1) & 1) ^ 1, &sh.gave_up)) return false;
      if (!barrier_wait(smem_address(&sh.full[s]), phase, &sh.gave_up)) return false;
      if (CTAS > 1 && !barrier_wait(smem_address(&sh.peer_full[s]), phase, &sh.gave_up)) return false;
      tmem_fence_after();
      const uint32_t left = ring.stages + s * kNsStageBytes, right = left + 2 * kPanelHalf;
      const uint32_t acc = sh.tmem + buf * kColumns;
      const uint32_t desc = mma_desc(128 * CTAS, ns_wide<CTAS>(narrow), flip_left, flip_right);
      // 16 of K: 32 bytes along K-major rows, or 16 rows of 128 bytes
      const unsigned left_step = flip_left ? 2048 : 32, right_step = flip_right ? 2048 : 32;
#pragma unroll
      for (int part = 0; part < 3; ++part) { // lo hi, hi lo, hi hi
        const uint32_t l = left + (part == 0 ? kPanelHalf : 0), r = right + (part == 1 ? kPanelHalf : 0);
#pragma unroll
        for (int step = 0; step < 4; ++step)
          mma_f16<CTAS>(acc, operand_desc(l + step * left_step, kPanelHalf / 2, 1024),
                        operand_desc(r + step * right_step, kPanelHalf / 2, 1024), desc, !(first && part == 0 && step == 0));
      }
      mma_commit<CTAS>(smem_address(&sh.empty[s]));
      if (k % kNsChunk == kNsChunk - 1 || k + 1 == at.k_blocks) {
        mma_commit<CTAS>(smem_address(&sh.acc_full[buf]));
        ++ring.round;
      }
    }
  }
  return true;
}

// ---- the warps that drain: warp w takes rows 32 (w % 4) .. and half of the tile's columns
template <int CTAS, int WHAT>
__device__ bool ns_drain(const MuonTable &t, int from, bool last, NsShared &sh, NsRing &ring, float *turn) {
  constexpr unsigned kColumns = 128 * CTAS;
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned row_in_tile = (warp & 3) * 32 + lane, half = warp >> 2;
  const bool narrow = CTAS == 1 && t.narrow[WHAT];
  const unsigned pieces = narrow ? 2 : 4 * CTAS; // of 16 columns
  for (unsigned tile = blockIdx.x / CTAS; tile < t.tiles[WHAT]; tile += gridDim.x / CTAS) {
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
      const uint32_t columns = sh.tmem + (((warp & 3) * 32) << 16) + buf * kColumns + half * pieces * 16;
#pragma unroll
      for (int h = 0; h < 4 * CTAS; ++h) {
        if (h >= pieces) continue;
        float v[16];
        tmem_load16(columns + h * 16, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[h * 16 + i] += v[i];
      }
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (ring.rank == 0) barrier_arrive(smem_address(&sh.acc_empty[buf]));
        else barrier_arrive_at(smem_address(&sh.acc_empty[buf]), 0);
      }
    }
    const unsigned width = WHAT == kApply ? q.n : q.m, rb = at.i * CTAS + ring.rank;
    const unsigned col_blocks = panel_col_blocks(width);
    if (rb >= panel_row_blocks(q.m)) continue;
    const char *old = WHAT == kPolynomial ? q.a : q.x[from]; // the linear term
    char *out = WHAT == kGram ? q.a : WHAT == kPolynomial ? q.b : q.x[from ^ 1];
    const unsigned row = rb * 128 + row_in_tile;
    // 32 columns at a time: half of a block column. All its loads are issued before its stores: the
    // compiler cannot move a load over a store that may alias it, and a load waits for L2.
#pragma unroll
    for (int g = 0; g < 2 * CTAS; ++g) {
      if (g * 2 >= pieces) continue;
      const unsigned col0 = at.j * ns_wide<CTAS>(narrow) + (half * pieces + g * 2) * 16;
      const unsigned cb = col0 / kPanelCols, chunk0 = (col0 % kPanelCols) / 8;
      if (cb >= col_blocks) continue;
      const u64 offset = panel_block(rb, cb, col_blocks);
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = acc[g * 32 + i] * kSplitUnscale;
      if (WHAT != kGram) {
        uint4 hi[4], lo[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const char *here = old + offset + panel_chunk(row_in_tile, chunk0 + c);
          hi[c] = *reinterpret_cast<const uint4 *>(here);
          lo[c] = *reinterpret_cast<const uint4 *>(here + kPanelHalf);
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
              *w = q.keep == 0.0f ? -scale * v[i] : __fmaf_rn(-scale, v[i], q.keep * *w);
            }
      } else {
        float *mine = turn + warp * (32 * 33);
#pragma unroll
        for (int i = 0; i < 32; ++i) mine[lane * 33 + i] = v[i];
        __syncwarp();
        const unsigned row0 = rb * 128 + (warp & 3) * 32, col = col0 + lane;
        if (col < q.n)
#pragma unroll 8
          for (int r = 0; r < 32; ++r)
            if (row0 + r < q.m) {
              float *w = q.w + (u64)(row0 + r) * q.n + col;
              *w = q.keep == 0.0f ? -scale * mine[r * 33 + lane] : __fmaf_rn(-scale, mine[r * 33 + lane], q.keep * *w);
            }
        __syncwarp();
      }
    }
  }
  return true;
}

// Barriers and tensor memory at the start and end of a kernel of products.
template <int CTAS>
__device__ __forceinline__ void ns_begin(NsShared &sh) {
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
  if (threadIdx.x >> 5 == kNsEpilogueWarps + 1) tmem_alloc<CTAS>(smem_address(&sh.tmem), 2 * 128 * CTAS);
  tmem_fence_before();
  __syncthreads();
  if (CTAS > 1) cluster_sync_all(); // the other CTA's barriers exist
  tmem_fence_after();
}
template <int CTAS>
__device__ __forceinline__ void ns_end(NsShared &sh) {
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if (CTAS > 1) cluster_sync_all(); // nothing of this CTA is used by the other one any more
  tmem_fence_after();
  if (threadIdx.x == 0 && sh.gave_up) atomicOr(&g_ns_gave_up, 1u);
  if (threadIdx.x >> 5 == kNsEpilogueWarps + 1) tmem_free<CTAS>(sh.tmem, 2 * 128 * CTAS);
}
// After a wait that ran out: copies (or products) in flight end before shared and tensor memory go away.
__device__ __forceinline__ void ns_abandon_loads(NsShared &sh, const NsRing &ring) {
  for (unsigned back = 1; back <= kNsStages && back <= ring.it; ++back) {
    const unsigned i = ring.it - back, s = i % kNsStages, phase = (i / kNsStages) & 1;
    const long long start = clock64();
    while (!barrier_try(smem_address(&sh.full[s]), phase) && clock64() - start < 10000000) {}
  }
}
template <int CTAS>
__device__ __forceinline__ void ns_abandon_products(NsShared &sh) {
  mma_commit<CTAS>(smem_address(&sh.drained));
  const long long start = clock64();
  while (!barrier_try(smem_address(&sh.drained), 0) && clock64() - start < 10000000) {}
}

// One product over all matrices.
template <int CTAS, int WHAT>
__global__ void __launch_bounds__(kNsThreads, 1) muon_product_kernel(const __grid_constant__ MuonTable t, int from, int last) {
  extern __shared__ char dynamic_smem[];
  __shared__ __align__(8) NsShared sh;
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  NsRing ring = {(smem_address(dynamic_smem) + 1023) & ~1023u, CTAS == 1 ? 0 : blockIdx.x % CTAS, 0, 0};
  float *turn = reinterpret_cast<float *>(dynamic_smem + kNsStages * kNsStageBytes + 1024);
  ns_begin<CTAS>(sh);
  pdl_wait();
  pdl_launch_dependents();
  if (warp == kNsEpilogueWarps) {
    if (lane == 0) {
      asm volatile("fence.proxy.async;" ::: "memory"); // the panels were written with plain stores
      if (!ns_load<CTAS, WHAT>(t, from, sh, ring)) ns_abandon_loads(sh, ring);
    }
  } else if (warp == kNsEpilogueWarps + 1) {
    if (lane == 0 && !ns_multiply<CTAS, WHAT>(t, sh, ring) && ring.rank == 0) ns_abandon_products<CTAS>(sh);
  } else {
    ns_drain<CTAS, WHAT>(t, from, last != 0, sh, ring, turn);
  }
  ns_end<CTAS>(sh);
}

// ---- all steps in one launch ---------------------------------------------------------------------------
// For matrices whose products are short a launch per product is most of the time (measured: 10 to 13
// us a product of 256 x 640). Here one cooperative grid goes through all of them; a product starts
// when every CTA has stored its tiles of the one before (a counter in global memory).
__device__ __forceinline__ void grid_arrive(unsigned *arrived) {
  __threadfence();
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(arrived) : "memory");
}
__device__ __forceinline__ bool grid_wait(const unsigned *arrived, unsigned target, volatile unsigned *gave_up) {
  const long long start = clock64();
  for (unsigned spins = 0;; ++spins) {
    unsigned now;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(arrived) : "memory");
    if (now >= target) return true;
    if ((spins & 255) == 255) {
      if (*gave_up) return false;
      if (clock64() - start > kWaitCycles) {
        *gave_up = 1;
        return false;
      }
    }
  }
}

__global__ void __launch_bounds__(kNsThreads, 1) muon_steps_kernel(const __grid_constant__ MuonTable t, int steps) {
  extern __shared__ char dynamic_smem[];
  __shared__ __align__(8) NsShared sh;
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  NsRing ring = {(smem_address(dynamic_smem) + 1023) & ~1023u, 0, 0, 0};
  float *turn = reinterpret_cast<float *>(dynamic_smem + kNsStages * kNsStageBytes + 1024);
  ns_begin<1>(sh);
  if (warp == kNsEpilogueWarps) {
    if (lane == 0) {
      bool ok = true;
      for (int s = 0; ok && s < steps; ++s) {
        const int from = s & 1;
        ok = grid_wait(t.arrived, 3 * s * gridDim.x, &sh.gave_up);
        asm volatile("fence.proxy.async;" ::: "memory"); // panels are written with plain stores
        ok = ok && ns_load<1, kGram>(t, from, sh, ring) && grid_wait(t.arrived, (3 * s + 1) * gridDim.x, &sh.gave_up);
        asm volatile("fence.proxy.async;" ::: "memory");
        ok = ok && ns_load<1, kPolynomial>(t, from, sh, ring) && grid_wait(t.arrived, (3 * s + 2) * gridDim.x, &sh.gave_up);
        asm volatile("fence.proxy.async;" ::: "memory");
        ok = ok && ns_load<1, kApply>(t, from, sh, ring);
      }
      if (!ok) ns_abandon_loads(sh, ring);
    }
  } else if (warp == kNsEpilogueWarps + 1) {
    if (lane == 0) {
      bool ok = true;
      for (int s = 0; ok && s < steps; ++s)
        ok = ns_multiply<1, kGram>(t, sh, ring) && ns_multiply<1, kPolynomial>(t, sh, ring) && ns_multiply<1, kApply>(t, sh, ring);
      if (!ok) ns_abandon_products<1>(sh);
    }
  } else {
    // The draining warps read what other CTAs stored (the linear term), so they wait for the grid too.
    // After a wait that ran out they go on through the block's barriers, all of them, without work.
    auto live = [&] { return !__any_sync(0xffffffffu, sh.gave_up != 0); };
    auto next = [&](unsigned product) {
      asm volatile("fence.proxy.async;" ::: "memory");
      asm volatile("bar.sync 1, %0;" ::"r"(kNsEpilogueWarps * 32) : "memory");
      if (threadIdx.x == 0 && !sh.gave_up) {
        grid_arrive(t.arrived);
        grid_wait(t.arrived, product * gridDim.x, &sh.gave_up);
      }
      asm volatile("bar.sync 1, %0;" ::"r"(kNsEpilogueWarps * 32) : "memory");
    };
    for (int s = 0; s < steps; ++s) {
      const int from = s & 1;
      if (live()) ns_drain<1, kGram>(t, from, false, sh, ring, turn);
      next(3 * s + 1);
      if (live()) ns_drain<1, kPolynomial>(t, from, false, sh, ring, turn);
      next(3 * s + 2);
      if (live()) ns_drain<1, kApply>(t, from, s + 1 == steps, sh, ring, turn);
      if (s + 1 < steps) next(3 * s + 3);
    }
  }
  ns_end<1>(sh);
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
static bool launched(cudaError_t e) {
  if (e == cudaSuccess) {
    count_launch();
    return true;
  }
  set_error(PLAST_B200_ERR_CUDA, "muon: %s", cudaGetErrorString(e));
  return false;
}
template <class Blocks>
static bool launch_over(MuonTable &t, Blocks blocks, void (*kernel)(const MuonTable)) {
  number(t, blocks);
  return launched(launch_k(kernel, dim3(t.total), dim3(kMuonThreads), 0, stream(), t));
}
template <int CTAS> static void number_tiles(MuonTable &t) {
  for (int what = kGram; what <= kApply; ++what) {
    u64 n = 0;
    for (int i = 0; i < t.count; ++i) {
      t.mat[i].first_tile[what] = (unsigned)n;
      n += ns_tiles_of<CTAS>(t.mat[i], what, t.narrow[what]);
    }
    t.tiles[what] = (unsigned)n;
  }
}
template <int CTAS, int WHAT>
static bool launch_product(MuonTable &t, int from, int last) {
  const auto kernel = muon_product_kernel<CTAS, WHAT>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNsSmem);
  if (e != cudaSuccess) return launched(e);
  const unsigned most = (unsigned)sm_count() / CTAS, grid = std::min(t.tiles[WHAT], most) * CTAS;
  return launched(launch_kc(CTAS, kernel, dim3(grid), dim3(kNsThreads), kNsSmem, stream(), t, from, last));
}
// Tiles of 256 x 256 by pairs of CTAs, a launch per product.
static void run_pairs(MuonTable &t, int steps) {
  for (int &narrow : t.narrow) narrow = 0;
  number_tiles<2>(t);
  for (int s = 0; s < steps; ++s) {
    const int from = s & 1;
    if (!launch_product<2, kGram>(t, from, 0) || !launch_product<2, kPolynomial>(t, from, 0) ||
        !launch_product<2, kApply>(t, from, s + 1 == steps))
      return;
  }
}
// Tiles of 128 x 128 (128 x 64 where that still leaves one each), all steps in one launch.
static void run_fused(MuonTable &t, int steps) {
  const unsigned sms = (unsigned)sm_count();
  for (int what = kGram; what <= kApply; ++what) {
    u64 n = 0;
    for (int i = 0; i < t.count; ++i) n += ns_tiles_of<1>(t.mat[i], what, true);
    t.narrow[what] = n <= sms;
  }
  number_tiles<1>(t);
  const unsigned tiles = std::max(t.tiles[kGram], std::max(t.tiles[kPolynomial], t.tiles[kApply]));
  cudaError_t e = cudaFuncSetAttribute(muon_steps_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNsSmem);
  if (e == cudaSuccess) {
    void *args[] = {&t, &steps};
    e = cudaLaunchCooperativeKernel((const void *)muon_steps_kernel, dim3(std::min(tiles, sms)), dim3(kNsThreads), args, kNsSmem, stream());
  }
  launched(e);
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
  t.arrived = (unsigned *)take(256);
  auto chunks = [](const MuonMat &q) { return (u64)q.chunks; };
  auto blocks = [](const MuonMat &q) { return (u64)panel_row_blocks(q.m) * panel_col_blocks(q.n); };
  if (!launch_over(t, chunks, muon_momentum_kernel)) return;
  if (!launch_over(t, [](const MuonMat &) { return (u64)1; }, muon_norm_kernel)) return;
  if (!launch_over(t, blocks, muon_load_kernel)) return;
  if (steps > 0) {
    u64 tiles = 0;
    for (int i = 0; i < t.count; ++i) tiles += ns_tiles_of<2>(t.mat[i], kApply, false);
    const bool pairs = tuned(kTuneMuonPairs) >= 0 ? tuned(kTuneMuonPairs) != 0 : tiles >= (u64)sm_count() / 2;
    if (pairs) run_pairs(t, steps);
    else run_fused(t, steps);
    return;
  }
  launch_over(t, chunks, muon_store_kernel);
}

// All matrices, in groups that share one piece of scratch.
static void run_matrices(const std::vector<MuonMat> &mats, float mu, float epsilon, int nesterov, int steps) {
  u64 largest = 0;
  std::vector<size_t> ends;
  for (size_t i = 0; i < mats.size();) {
    u64 bytes = 256; // the grid barrier
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
