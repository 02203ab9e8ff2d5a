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
//
// What bounds it, on a B200: large matrices the way of the operands from L2 to the SMs (a pair of CTAs brings
// 128 KB for every 1,536 cycles of products on its 256 x 256 tile; it takes 1,900) and the power cap: one
// 4096 x 8192 in 6.6 ms, 1.10 PFLOP/s of fp16 products. Matrices of 1024: 16 square and 8 of 4096 x 1024 in
// 3.57 ms, 0.76 PFLOP/s, as every 16 K blocks a tile is stored. Small ones the chain of 3 products a step: 8 us
// each where a tile has a CTA of its own (six matrices of up to 512: 130 us).
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
constexpr int kMuonChunk = kMuonThreads * 32;      // elements per CTA of the momentum pass

struct MuonMat {
  const float *g;  // gradient, or the input of orthogonalise
  float *v;        // momentum; NULL: u = g
  float *w;        // weight (w = w * keep - rate * X) or, with keep == 0 and rate == -1, the output
  char *x[2], *a; // panels: X (two, in turn), A, B behind A
  double *partial; // sums of squares of the momentum pass, then partial[0] holds their total
  float keep, rate;
  unsigned rows, cols; // as stored
  unsigned m, n;       // m <= n
  unsigned first;      // first CTA of this matrix in the launch at hand
  unsigned chunks;
};
struct MuonTable {
  MuonMat mat[kMuonMax];
  int count;
  unsigned total;     // CTAs of the launch at hand
  unsigned *tickets, ticket_count; // see NsTable
  float4 *parts;
  unsigned *stored;   // per matrix: draining warps that have stored their part of a tile, over all products so far
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
  auto one = [&](float g, float &v) {
    float u = g;
    if (q.v) {
      v = __fmaf_rn(t.mu, v, g);
      u = update_of(t, g, v);
    }
    sum += (double)u * (double)u;
  };
  if (total - begin >= (u64)kMuonChunk && (((uintptr_t)q.g | (uintptr_t)q.v) & 15) == 0) {
    const float4 *g4 = reinterpret_cast<const float4 *>(q.g + begin) + threadIdx.x;
    float4 *v4 = q.v ? reinterpret_cast<float4 *>(q.v + begin) + threadIdx.x : nullptr;
#pragma unroll 1
    for (int batch = 0; batch < kMuonChunk / kMuonThreads / 16; ++batch, g4 += 4 * kMuonThreads) {
      float4 g[4], v[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = g4[i * kMuonThreads];
      if (v4)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = v4[i * kMuonThreads];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        one(g[i].x, v[i].x);
        one(g[i].y, v[i].y);
        one(g[i].z, v[i].z);
        one(g[i].w, v[i].w);
        if (v4) v4[i * kMuonThreads] = v[i];
      }
      if (v4) v4 += 4 * kMuonThreads;
    }
  } else {
#pragma unroll 4
    for (u64 j = begin + threadIdx.x; j < begin + kMuonChunk && j < total; j += kMuonThreads) {
      float v = q.v ? q.v[j] : 0.0f;
      one(q.g[j], v);
      if (q.v) q.v[j] = v;
    }
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
#pragma unroll 8
  for (unsigned i = threadIdx.x; i < q.chunks; i += kMuonThreads) sum += q.partial[1 + i];
  if (blockIdx.x == 0)
    for (unsigned i = threadIdx.x; i < t.ticket_count; i += kMuonThreads) t.tickets[i] = 0;
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
  __shared__ float tile[kPanelRows][kPanelCols + 1];
  // the factor in 64 bits: the norm may be outside fp32's range where the quotient is not; the products
  // too, unless it is an ordinary number
  const double square = q.partial[0]; // infinite where an element is: NaN then, as the steps would make it
  const double inv = square < INFINITY ? (double)kSplitScale / (sqrt(square) + (double)t.epsilon) : NAN;
  const float inv32 = (float)inv;
  const bool ordinary = inv32 > 1e-30f && inv32 < 1e30f;
  auto value = [&](float u, float v) {
    if (q.v) u = update_of(t, u, v);
    return ordinary ? u * inv32 : (float)((double)u * inv);
  };
  const unsigned col_blocks = panel_col_blocks(q.n), at = blockIdx.x - q.first;
  const unsigned rb = at / col_blocks, cb = at % col_blocks;
  const bool turned = q.rows > q.cols;
  // the block in the matrix as it is stored
  const unsigned r0 = turned ? cb * kPanelCols : rb * kPanelRows, c0 = turned ? rb * kPanelRows : cb * kPanelCols;
  constexpr int kEach = kPanelRows * kPanelCols / 4 / kMuonThreads; // float4 per thread
  const unsigned wide = turned ? kPanelRows / 4 : kPanelCols / 4;     // float4 along a stored row of the block
  float x[kEach][4];
  const bool vec = (((uintptr_t)q.g | (uintptr_t)q.v) & 15) == 0 && q.cols % 4 == 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const unsigned item = e * kMuonThreads + threadIdx.x, r = r0 + item / wide, c = c0 + item % wide * 4;
    const u64 j = (u64)r * q.cols + c;
    float4 g = make_float4(0.0f, 0.0f, 0.0f, 0.0f), v = g;
    if (r < q.rows && c < q.cols) {
      if (vec) {
        g = *reinterpret_cast<const float4 *>(q.g + j);
        if (q.v) v = *reinterpret_cast<const float4 *>(q.v + j);
      } else {
        float *gs = &g.x, *vs = &v.x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c + i < q.cols) {
            gs[i] = q.g[j + i];
            if (q.v) vs[i] = q.v[j + i];
          }
      }
      x[e][0] = value(g.x, v.x);
      x[e][1] = c + 1 < q.cols ? value(g.y, v.y) : 0.0f;
      x[e][2] = c + 2 < q.cols ? value(g.z, v.z) : 0.0f;
      x[e][3] = c + 3 < q.cols ? value(g.w, v.w) : 0.0f;
    } else x[e][0] = x[e][1] = x[e][2] = x[e][3] = 0.0f;
  }
  // through shared memory to eight neighbours along a panel row per thread
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const unsigned item = e * kMuonThreads + threadIdx.x, r = item / wide, c = item % wide * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) tile[turned ? c + i : r][turned ? r : c + i] = x[e][i];
  }
  __syncthreads();
  char *block = q.x[0] + panel_block(rb, cb, col_blocks);
#pragma unroll
  for (unsigned e = threadIdx.x; e < kPanelRows * 8; e += kMuonThreads) {
    const unsigned row = e / 8, chunk = e % 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = tile[row][chunk * 8 + i];
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
// What is kept of A and B is moved towards 0 along the diagonal, S = A - T I and Q = B + s I:
//   c A A + b A = c S S + (b + 2 c T) S + ((b + 2 c T) T - c T^2) I,   X = (a - s) X + Q X
// With singular values of X near 1, A is near I and B near -2.74 I, and a X + B X would lose two bits to
// cancellation, of numbers that have 22: 2e-6 off on 64 x 1000, 6e-7 with T = 0.7, s = 2.3 (plain fp32:
// 1.3e-6). All the way (T = -b / 2c, s = a: no linear terms) A and B start near -1.2 I and 3.4 I
// instead, and their rounding hurts: 3 to 6e-6.
//
// One launch goes through all products of all matrices. A persistent CTA takes every gridDim-th tile,
// of 128 x 128 (or 128 x 64); a pair of CTAs (CTAS = 2) tiles of 256 x 256, each CTA holding half of
// either operand. One thread brings 64 KB stages (64 of K, hi and lo of both operands) with bulk
// copies, one warp (of the pair) issues the twelve tcgen05.mma of a stage, small products first, and
// sixteen warps drain the accumulators. Tensor-core accumulation truncates; every one or two stages the
// accumulator (one of two in tensor memory) is therefore added in fp32 registers, rounded to nearest,
// while the next one fills.
//
// A product of a matrix starts when all tiles of its product before are stored, which a counter per
// matrix in global memory tells; the tiles of other matrices do not wait. The grid is launched
// cooperatively (all of it is resident, so the waits end) and every wait is limited.
enum MuonProduct { kGram = 0, kPolynomial = 1, kApply = 2 };
constexpr int kNsStages = 3;
constexpr unsigned kNsStageBytes = 4 * kPanelHalf; // left hi, left lo, right hi, right lo
constexpr int kNsEpilogueWarps = 16, kNsThreads = (kNsEpilogueWarps + 4) * 32;
// Stages summed in tensor memory before they are added in registers (for pairs one costs 15 %).
template <int CTAS> constexpr int kNsChunk = CTAS == 1 ? 1 : 2;
// The truncation of such a sum shortens it by about one (single) to three units of 2^-23 on average,
// which the addition in registers puts back: it multiplies by this. Sums that truncate nothing come out that much too
// large, which is below what the operands' 22 bits cost: a permutation matrix of 256 is 4.7e-7 off after five
// steps, with products in fp32 5.8e-7; 1024 x 4096 6.2e-7 (pairs 1.1e-6) and 3.7e-6.
template <int CTAS> constexpr float kNsRaise = 1.0f + (CTAS == 1 ? 1 : 3) / 8388608.0f;
// What the diagonals of A and B are moved by, see above, and what follows for the linear terms.
constexpr double kNsT = 0.7, kNsS = 2.3;
constexpr double kNsLinear = (double)kNsB + 2.0 * kNsC * kNsT; // of B in A - T
constexpr unsigned kNsMostParts = 8;   // of a split K
constexpr unsigned kNsPieceBytes = 2048; // per draining warp: 32 rows of 32 columns of hi or lo, or 32 x 16 floats

struct NsMat {
  char *x[2], *a; // B lies behind A
  float *w;
  float keep, rate;
  unsigned m, n;
  unsigned first_tile[3], tiles[3]; // a tile whose K is split counts once for each part
  unsigned char splits[3];
  bool turned; // stored as n x m
  __device__ __forceinline__ char *b() const { return a + panel_block(panel_row_blocks(m), 0, panel_col_blocks(m)); }
};
struct NsTable {
  NsMat mat[kMuonMax];
  unsigned *stored;
  unsigned *tickets; // of tiles whose K is split: per draining warp, how many parts are there
  float4 *parts;     // their sums
  unsigned room;     // tiles, per product
  unsigned tiles[3]; // of each product
  int narrow[3];     // tiles of 128 x 64 instead of 128 x 128
  int count;
  long long wait_cycles; // limit of every wait
};

__device__ unsigned g_ns_gave_up; // CTAs in which a wait has run out, over all calls: see plast_b200_muon_status

// tiles along a side, and of a product; `wide`: columns of a tile (256, 128 or 64)
__host__ __device__ inline unsigned ns_along(unsigned size, unsigned tile) { return (size + tile - 1) / tile; }
template <int CTAS> __host__ __device__ inline unsigned ns_wide(bool narrow) { return narrow ? 64 : 128 * CTAS; }
template <int CTAS> inline u64 ns_tiles_of(unsigned m, unsigned n, int what, bool narrow) {
  const u64 r = ns_along(m, 128 * CTAS), per_diagonal = 128 * CTAS / ns_wide<CTAS>(narrow);
  const u64 c = ns_along(what == kApply ? n : m, ns_wide<CTAS>(narrow));
  return what == kApply ? r * c : r * c - per_diagonal * (r * (r - 1) / 2); // row i starts at its diagonal block
}

// K blocks of one part (single CTAs only)
__host__ __device__ inline unsigned ns_part_blocks(unsigned k_blocks, unsigned parts) {
  return (k_blocks + parts - 1) / parts;
}

struct NsTile {
  unsigned i, j;         // tile row, tile column
  unsigned k0, k_blocks; // first K block (of 64) and their number
  unsigned part, parts;  // of K
};
template <int CTAS>
__device__ __forceinline__ const NsMat &tile_at(const NsTable &t, int what, unsigned tile, NsTile &out) {
  int lo = 0, hi = t.count - 1; // the last matrix whose first tile is not beyond
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.mat[mid].first_tile[what] <= tile) lo = mid; else hi = mid - 1;
  }
  const NsMat &q = t.mat[lo];
  const unsigned wide = ns_wide<CTAS>(t.narrow[what]), across = ns_along(what == kApply ? q.n : q.m, wide);
  unsigned at = tile - q.first_tile[what];
  const unsigned k_all = panel_col_blocks(what == kGram ? q.n : q.m);
  out.parts = CTAS == 1 ? q.splits[what] : 1;
  out.part = 0;
  out.k0 = 0;
  out.k_blocks = k_all;
  if (CTAS == 1 && out.parts > 1) {
    out.part = at % out.parts;
    at /= out.parts;
    const unsigned each = ns_part_blocks(k_all, out.parts);
    out.k0 = out.part * each;
    out.k_blocks = k_all - out.k0 < each ? k_all - out.k0 : each;
  }
  if (what == kApply) {
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
  return q;
}

// The linear term of a tile comes through the same ring of stages, after the first four K blocks (eight
// for pairs; or after the last): by then the draining warps are done with the tile before and take it at once. The
// gram matrix has none, nor have the other parts of a split K.
template <int CTAS>
__device__ __forceinline__ unsigned ns_linear_after(const NsTile &at, int what) {
  constexpr unsigned kAfter = 4 * CTAS;
  if (what == kGram || at.part != 0) return ~0u;
  return at.k_blocks < kAfter ? at.k_blocks : kAfter;
}

// One operand of a tile: 128 rows (64 where narrow) by 64 of K per stage. `plain`: the block in block
// row rb, 32 KB at once. `flip`: read MN-major from the blocks above the diagonal (or, for X, always),
// pieces of 64 K rows by 64 columns, 8 KB of hi and of lo each. What lies outside the panel is not
// fetched (it only feeds results that are not stored).
struct NsOperand {
  const char *plain, *flip;   // of K block 0; the flipped one moves on every second block
  u64 flip_step;              // bytes from one block row to the next
  unsigned plain_bytes, flip_bytes; // per stage
  bool narrow;
};
__device__ __forceinline__ NsOperand operand_of(const char *panel, unsigned rb, unsigned row_blocks, unsigned col_blocks, bool narrow) {
  NsOperand o;
  o.narrow = narrow;
  o.flip_step = panel_block(1, 0, col_blocks);
  if (narrow) { // rb counts in 64
    o.plain = panel + panel_block(rb / 2, 0, col_blocks) + (rb & 1) * (kPanelHalf / 2);
    o.flip = panel + panel_block(0, rb, col_blocks);
    o.plain_bytes = rb / 2 < row_blocks ? kPanelHalf : 0;
    o.flip_bytes = rb < col_blocks ? kPanelHalf : 0;
  } else {
    o.plain = panel + panel_block(rb, 0, col_blocks);
    o.flip = panel + panel_block(0, 2 * rb, col_blocks);
    o.plain_bytes = rb < row_blocks ? 2 * kPanelHalf : 0;
    o.flip_bytes = 2 * rb + 1 < col_blocks ? 2 * kPanelHalf : (2 * rb < col_blocks ? kPanelHalf : 0);
  }
  return o;
}
__device__ __forceinline__ void load_operand(const NsOperand &o, uint32_t dst, unsigned k, bool flip, uint32_t bar) {
  constexpr unsigned kPiece = kPanelHalf / 2; // 64 rows
  if (!flip) {
    if (!o.plain_bytes) return;
    const char *src = o.plain + (u64)k * (2 * kPanelHalf);
    if (!o.narrow) bulk_load(dst, src, 2 * kPanelHalf, bar);
    else {
      bulk_load(dst, src, kPiece, bar);
      bulk_load(dst + kPanelHalf, src + kPanelHalf, kPiece, bar);
    }
    return;
  }
  if (!o.flip_bytes) return;
  const char *src = o.flip + (k >> 1) * o.flip_step + (k & 1) * kPiece;
  bulk_load(dst, src, kPiece, bar);
  bulk_load(dst + kPanelHalf, src + kPanelHalf, kPiece, bar);
  if (o.flip_bytes == 2 * kPanelHalf) { // the neighbouring block column
    src += 2 * kPanelHalf;
    bulk_load(dst + kPiece, src, kPiece, bar);
    bulk_load(dst + kPanelHalf + kPiece, src + kPanelHalf, kPiece, bar);
  }
}

struct NsShared {
  // A wait knows a turn of a barrier by its parity alone: it must not begin before the turn before is over, nor be left
  // behind by two. So every barrier has waiters that wait for each of its turns: `full` is of operands (the issuing
  // warp), `linear_full` of linear terms (by their part, which the same draining warps read each time, and stage).
  uint64_t full[kNsStages], peer_full[kNsStages], empty[kNsStages], linear_full[2][kNsStages], acc_full[2], acc_empty[2], drained;
  NsTable table; // a copy: the roles index it at every tile, which is slow in constant memory
  uint32_t tmem;
  WaitLimit wait;
  volatile unsigned allowed; // tiles whose operands are stored, as the looking-out thread has seen
  alignas(16) unsigned written[kNsEpilogueWarps]; // per draining warp: tiles that it has written its part of
  unsigned linear_read[kNsStages]; // draining warps that have read a linear term in this stage, over all tiles
};
constexpr unsigned kNsSmem = kNsStages * kNsStageBytes + kNsEpilogueWarps * kNsPieceBytes + sizeof(NsShared);
static_assert(kNsSmem <= 232448, "227 KB of shared memory per CTA");

// a stage as an address for plain loads
__device__ __forceinline__ const char *dynamic_stage(uint32_t stages, unsigned stage) {
  return reinterpret_cast<const char *>(__cvta_shared_to_generic(stages + stage * kNsStageBytes));
}
// A role's place in the rings of stages and accumulators, kept from one product to the next.
struct NsRing {
  uint32_t stages;      // shared memory
  unsigned rank;        // in the pair
  unsigned first;       // this CTA's (pair's) first tile of the product at hand
  unsigned stage, phase; // of the next stage; the phase is that of its `empty`
  unsigned turns;       // by stage, a bit: the parity of the next turn of its `full` or `linear_full` for this role
  unsigned buf, turn;   // of the next accumulator
  unsigned tiles;       // so far, for the roles that count them
  __device__ __forceinline__ void skip_stages(unsigned n) {
    stage += n;
    phase ^= (stage / kNsStages) & 1;
    stage %= kNsStages;
  }
  __device__ __forceinline__ void next_stage() {
    if (++stage == kNsStages) {
      stage = 0;
      phase ^= 1;
    }
  }
  // parity of the turn that is waited for (once)
  __device__ __forceinline__ unsigned take_turn(unsigned at) {
    const unsigned parity = (turns >> at) & 1;
    turns ^= 1u << at;
    return parity;
  }
  __device__ __forceinline__ void next_accumulator() {
    buf ^= 1;
    turn ^= buf == 0;
  }
};

// Waits until matrix q's products up to this one (step s, product what) are stored. The look-out thread begins to wait
// when the product before begins, which may take longer than the limit: it counts from the last tile that was stored.
template <int CTAS>
__device__ __noinline__ bool ns_wait_stored(const NsTable &t, const NsMat &q, int s, int what, WaitLimit *wait) {
  unsigned target = 0;
  for (int w = 0; w < 3; ++w) target += q.tiles[w] / q.splits[w] * (s + (w < what));
  target *= CTAS * kNsEpilogueWarps;
  const unsigned *counter = t.stored + (&q - t.mat);
  long long start = 0;
  unsigned last = 0;
  for (unsigned spins = 0;; ++spins) {
    unsigned now;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(counter) : "memory");
    if (now >= target) return true;
    if (spins == 0 || now != last) start = clock64();
    last = now;
    if ((spins & 63) == 63 && wait->over(start)) return false;
  }
}

// The same for a counter in shared memory.
__device__ __noinline__ bool ns_wait_counter(const volatile unsigned *counter, unsigned target, WaitLimit *wait) {
  const long long start = clock64();
  for (unsigned spins = 0; *counter < target; ++spins)
    if ((spins & 63) == 63 && wait->over(start)) return false;
  __threadfence_block();
  return true;
}

// Until every draining warp has written its part of `target` tiles. (One count for all of them would not tell: a warp
// may be two tiles ahead of another, as far as the two accumulators go.)
__device__ __noinline__ bool ns_wait_written(const unsigned *written, unsigned target, WaitLimit *wait) {
  const uint32_t at = smem_address(written);
  const long long start = clock64();
  for (unsigned spins = 0;; ++spins) {
    bool all = true;
#pragma unroll
    for (int i = 0; i < kNsEpilogueWarps / 4; ++i) {
      uint4 v;
      asm volatile("ld.volatile.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at + 16 * i) : "memory");
      all = all && v.x >= target && v.y >= target && v.z >= target && v.w >= target;
    }
    if (all) break;
    if ((spins & 63) == 63 && wait->over(start)) return false;
  }
  __threadfence_block();
  return true;
}

// The roles below take the product as an argument, not as a template: three copies of each do not fit
// the instruction cache, and a tile of a small matrix runs its code once (measured with three copies,
// 180 KB: 2,400 cycles to store a tile of 128 x 64, all of it fetching instructions).

// ---- the thread that loads
template <int CTAS>
__device__ bool ns_load(NsShared &sh, NsRing &ring, int s, int what) {
  const NsTable &t = sh.table;
  const int from = s & 1;
  const bool narrow = CTAS == 1 && t.narrow[what];
  for (unsigned tile = ring.first; tile < t.tiles[what]; tile += gridDim.x / CTAS) {
    NsTile at;
    const NsMat &q = tile_at<CTAS>(t, what, tile, at);
    const unsigned rows = panel_row_blocks(q.m), xcb = panel_col_blocks(q.n), mcb = panel_col_blocks(q.m);
    const NsOperand left = operand_of(what == kGram ? q.x[from] : what == kPolynomial ? q.a : q.b(), at.i * CTAS + ring.rank, rows,
                                      what == kGram ? xcb : mcb, false);
    const NsOperand right = operand_of(what == kPolynomial ? q.a : q.x[from], at.j * CTAS + ring.rank, rows,
                                       what == kPolynomial ? mcb : xcb, narrow);
    // K blocks before these are above the diagonal
    const unsigned flip_left = what == kGram ? 0 : 2 * CTAS * at.i;
    const unsigned flip_right = what == kGram ? 0 : what == kApply ? ~0u : 2 * CTAS * (narrow ? at.j / 2 : at.j);
    if (!ns_wait_counter(&sh.allowed, ++ring.tiles, &sh.wait)) return false;
    asm volatile("fence.proxy.async.global;" ::: "memory"); // panels are written with plain stores
    const unsigned k_linear = ns_linear_after<CTAS>(at, what);
    for (unsigned k = 0; k <= at.k_blocks; ++k) {
      if (k == k_linear) {
        // the linear term, b A or a X: two block columns of this CTA's rows to a stage
        const char *old = what == kPolynomial ? q.a : q.x[from];
        const unsigned rb = at.i * CTAS + ring.rank, cbs = what == kPolynomial ? mcb : xcb;
        const unsigned cb0 = narrow ? at.j : at.j * 2 * CTAS, cb_end = cb0 + (narrow ? 1 : 2 * CTAS);
        for (unsigned c = 0; c < CTAS; ++c, ring.next_stage()) {
          if (!barrier_wait(smem_address(&sh.empty[ring.stage]), ring.phase ^ 1, &sh.wait)) return false;
          const uint32_t bar = smem_address(&sh.linear_full[c][ring.stage]), dst = ring.stages + ring.stage * kNsStageBytes;
          const unsigned first = cb0 + 2 * c;
          unsigned n = 0; // block columns that exist
          if (rb < rows)
            while (n < 2 && first + n < cb_end && first + n < cbs) ++n;
          barrier_expect(bar, n * 2 * kPanelHalf);
          ring.turns ^= 1u << (kNsStages * (1 + c) + ring.stage);
          if (n) bulk_load(dst, old + panel_block(rb, first, cbs), n * 2 * kPanelHalf, bar); // neighbours in memory
        }
      }
      if (k == at.k_blocks) break;
      if (!barrier_wait(smem_address(&sh.empty[ring.stage]), ring.phase ^ 1, &sh.wait)) return false;
      const uint32_t bar = smem_address(&sh.full[ring.stage]), dst = ring.stages + ring.stage * kNsStageBytes;
      const unsigned kb = at.k0 + k;
      const bool fl = kb < flip_left, fr = kb < flip_right;
      barrier_expect(bar, (fl ? left.flip_bytes : left.plain_bytes) + (fr ? right.flip_bytes : right.plain_bytes));
      ring.turns ^= 1u << ring.stage;
      load_operand(left, dst, kb, fl, bar);
      load_operand(right, dst + 2 * kPanelHalf, kb, fr, bar);
      ring.next_stage();
    }
  }
  return true;
}

// ---- the thread that looks out for the tiles' operands, ahead of the one that loads (to which a look and
// its fence at every tile cost 3,000 to 4,000 cycles without a load in flight)
template <int CTAS>
__device__ bool ns_look_out(NsShared &sh, NsRing &ring, int s, int what) {
  const NsTable &t = sh.table;
  for (unsigned tile = ring.first; tile < t.tiles[what]; tile += gridDim.x / CTAS) {
    NsTile at;
    const NsMat &q = tile_at<CTAS>(t, what, tile, at);
    if (!ns_wait_stored<CTAS>(t, q, s, what, &sh.wait)) return false;
    __threadfence_block();
    sh.allowed = ++ring.tiles;
  }
  return true;
}

// ---- the warp that issues the products (in the second CTA of a pair: passes on that its half is there).
// All lanes walk the loops together, so that descriptors stay in uniform registers; one lane issues.
template <int CTAS>
__device__ bool ns_multiply(NsShared &sh, NsRing &ring, int what) {
  constexpr unsigned kColumns = 128 * CTAS;
  const NsTable &t = sh.table;
  const bool narrow = CTAS == 1 && t.narrow[what];
  const uint32_t tmem = sh.tmem;
  for (unsigned tile = ring.first; tile < t.tiles[what]; tile += gridDim.x / CTAS) {
    NsTile at;
    tile_at<CTAS>(t, what, tile, at);
    const unsigned flip_left = what == kGram ? 0 : 2 * CTAS * at.i;
    const unsigned flip_right = what == kGram ? 0 : what == kApply ? ~0u : 2 * CTAS * (narrow ? at.j / 2 : at.j);
    const unsigned k_linear = ns_linear_after<CTAS>(at, what);
    for (unsigned k = 0; k <= at.k_blocks; ++k, ring.next_stage()) {
      if (k == k_linear) ring.skip_stages(CTAS); // not for the tensor cores
      if (k == at.k_blocks) break;
      const uint32_t full = smem_address(&sh.full[ring.stage]);
      const unsigned parity = ring.take_turn(ring.stage);
      if (!__all_sync(0xffffffffu, barrier_wait(full, parity, &sh.wait))) return false;
      if (CTAS > 1 && ring.rank != 0) {
        if (elect_one()) barrier_arrive_at(smem_address(&sh.peer_full[ring.stage]), 0);
        __syncwarp();
        continue;
      }
      const bool first = k % kNsChunk<CTAS> == 0, last = k % kNsChunk<CTAS> == kNsChunk<CTAS> - 1 || k + 1 == at.k_blocks;
      if (first && !__all_sync(0xffffffffu, barrier_wait(smem_address(&sh.acc_empty[ring.buf]), ring.turn ^ 1, &sh.wait)))
        return false;
      if (CTAS > 1 && !__all_sync(0xffffffffu, barrier_wait(smem_address(&sh.peer_full[ring.stage]), parity, &sh.wait)))
        return false;
      tmem_fence_after();
      const bool fl = at.k0 + k < flip_left, fr = at.k0 + k < flip_right;
      const uint32_t stage = ring.stages + ring.stage * kNsStageBytes;
      const uint64_t left = operand_desc(stage, kPanelHalf / 2, 1024);
      const uint64_t right = operand_desc(stage + 2 * kPanelHalf, kPanelHalf / 2, 1024);
      const uint32_t acc = tmem + ring.buf * kColumns;
      const uint32_t desc = mma_desc(128 * CTAS, ns_wide<CTAS>(narrow), fl, fr);
      // 16 of K: 32 bytes along K-major rows, or 16 rows of 128 bytes; descriptors count in 16 bytes
      const unsigned left_step = fl ? 128 : 2, right_step = fr ? 128 : 2;
      if (elect_one()) {
#pragma unroll
        for (int part = 0; part < 3; ++part) { // lo hi, hi lo, hi hi
          const uint64_t l = left + (part == 0 ? kPanelHalf >> 4 : 0), r = right + (part == 1 ? kPanelHalf >> 4 : 0);
#pragma unroll
          for (int step = 0; step < 4; ++step)
            mma_f16<CTAS>(acc, l + step * left_step, r + step * right_step, desc, !(first && part == 0 && step == 0));
        }
        mma_commit<CTAS>(smem_address(&sh.empty[ring.stage]));
        if (last) mma_commit<CTAS>(smem_address(&sh.acc_full[ring.buf]));
      }
      __syncwarp();
      if (last) ring.next_accumulator();
    }
  }
  return true;
}

// ---- the warps that drain: warp w takes rows 32 (w % 4) .. and a quarter of the tile's columns (64, 32 or
// 16), 32 at a time.
//
// A lane holds a row, so it would touch 32 different lines per access to a panel; the rows go through
// shared memory instead and a warp's access covers whole 64-byte pieces of eight rows.
template <int CTAS>
__device__ bool ns_drain(NsShared &sh, NsRing &ring, int s, int what, bool last, char *piece) {
  constexpr unsigned kColumns = 128 * CTAS;
  constexpr int kGroups = 2 * CTAS; // of 16 columns
  const NsTable &t = sh.table;
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp >> 2;
  const unsigned row_in_tile = (warp & 3) * 32 + lane;
  const bool narrow = CTAS == 1 && t.narrow[what];
  const unsigned columns = narrow ? 16 : 32 * CTAS;
  const unsigned part_of_linear = CTAS > 1 ? quarter / 2 : 0; // whose stage holds the warp's columns
  const float init = (float)(what == kPolynomial ? kNsLinear / kNsC : (double)kNsA - kNsS) * kSplitScale;
  const float diagonal = (float)(what == kGram ? -kNsT : what == kPolynomial ? kNsLinear * kNsT - kNsC * kNsT * kNsT + kNsS : 0.0) * kSplitScale;
  const float finish = what == kPolynomial ? kNsC * kSplitUnscale : kSplitUnscale;
  // a group's 32 columns: four 16-byte chunks of a row (two where narrow)
  const unsigned shift = narrow ? 1 : 2, mask = (1u << shift) - 1;
  for (unsigned tile = ring.first; tile < t.tiles[what]; tile += gridDim.x / CTAS) {
    NsTile at;
    const NsMat &q = tile_at<CTAS>(t, what, tile, at);
    const unsigned rb = at.i * CTAS + ring.rank, col_blocks = panel_col_blocks(what == kApply ? q.n : q.m);
    const unsigned col0 = at.j * ns_wide<CTAS>(narrow) + quarter * columns; // first column of the warp
    const unsigned row = rb * 128 + row_in_tile;
    const bool rows_exist = rb < panel_row_blocks(q.m);
    float acc[16 * kGroups];
#pragma unroll
    for (int i = 0; i < 16 * kGroups; ++i) acc[i] = 0.0f;
    const unsigned rounds = (at.k_blocks + kNsChunk<CTAS> - 1) / kNsChunk<CTAS>;
    const unsigned k_linear = ns_linear_after<CTAS>(at, what);
#pragma unroll 1
    for (unsigned c = 0; c <= rounds; ++c) {
      if (k_linear != ~0u && c == (k_linear + kNsChunk<CTAS> - 1) / kNsChunk<CTAS>) {
        // the lane's row of the linear term, from the stage that holds the warp's block column
        NsRing here = ring;
        here.skip_stages(k_linear + part_of_linear);
        if (!__all_sync(0xffffffffu, barrier_wait(smem_address(&sh.linear_full[part_of_linear][here.stage]), ring.take_turn(here.stage),
                                                  &sh.wait)))
          return false;
        const unsigned block = CTAS > 1 ? (quarter & 1) : narrow ? 0 : quarter / 2;
        const unsigned chunk0 = CTAS > 1 ? 0 : narrow ? quarter * 2 : (quarter & 1) * 4;
        const char *old = dynamic_stage(ring.stages, here.stage) + block * (2 * kPanelHalf);
        if (rows_exist && col0 / kPanelCols < col_blocks) {
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int k = 0; k < 2 * kGroups; ++k) {
              if (k >= 2 && narrow) continue;
              const uint4 h = *reinterpret_cast<const uint4 *>(old + part * kPanelHalf + panel_chunk(row_in_tile, chunk0 + k));
              const unsigned w[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                float &x = acc[k * 8 + 2 * i], &y = acc[k * 8 + 2 * i + 1];
                x = __fmaf_rn(f.x, init, x);
                y = __fmaf_rn(f.y, init, y);
              }
            }
        }
        // the last of the warps that share the stage gives it back (counted by stage: warps that are ahead read the
        // next tile's term in another one, and none in this one before it is given back)
        __syncwarp();
        if (lane == 0) {
          __threadfence_block();
          const unsigned share = kNsEpilogueWarps / CTAS;
          if (atomicAdd(&sh.linear_read[here.stage], 1u) % share == share - 1) {
            __threadfence_block();
            barrier_arrive(smem_address(&sh.empty[here.stage]));
          }
        }
      }
      if (c == rounds) break;
      if (!__all_sync(0xffffffffu, barrier_wait(smem_address(&sh.acc_full[ring.buf]), ring.turn, &sh.wait))) return false;
      tmem_fence_after();
      const uint32_t from = sh.tmem + (((warp & 3) * 32) << 16) + ring.buf * kColumns + quarter * columns;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        if (g > 0 && narrow) continue;
        float v[16];
        tmem_load16(from + g * 16, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[g * 16 + i] = __fmaf_rn(v[i], kNsRaise<CTAS>, acc[g * 16 + i]);
      }
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (ring.rank == 0) barrier_arrive(smem_address(&sh.acc_empty[ring.buf]));
        else barrier_arrive_at(smem_address(&sh.acc_empty[ring.buf]), 0);
      }
      ring.next_accumulator();
    }
    ring.skip_stages(at.k_blocks + (k_linear == ~0u ? 0 : CTAS));
    bool mine = true; // this warp stores its part of the tile
    if (CTAS == 1 && at.parts > 1) {
      // The warp's sums go to memory; the last of the parts' warps (a ticket) adds all of them up, always in
      // the same order. Each product has its own room, where a place belongs to one matrix: another matrix
      // may be ahead by any number of products.
      const unsigned whole = ((what * t.room + tile - at.part)) * kNsEpilogueWarps + warp; // the tile's first part
      float4 *out = t.parts + ((u64)whole + at.part * kNsEpilogueWarps) * (8 * 32) + lane;
#pragma unroll
      for (int i = 0; i < 4 * kGroups; ++i)
        if (i < 4 || !narrow) out[i * 32] = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
      __syncwarp();
      unsigned before = 0;
      if (lane == 0) {
        asm volatile("fence.acq_rel.gpu;" ::: "memory");
        before = atomicAdd(t.tickets + whole, 1u);
        if (before == at.parts - 1) t.tickets[whole] = 0; // for the next product
        asm volatile("fence.acq_rel.gpu;" ::: "memory");
      }
      mine = __shfl_sync(0xffffffffu, before, 0) == at.parts - 1;
      __syncwarp(); // what lane 0 has acquired is there for all lanes (a shuffle orders no memory)
      if (mine) {
#pragma unroll
        for (int i = 0; i < 16 * kGroups; ++i) acc[i] = 0.0f;
        const float4 *in = t.parts + (u64)whole * (8 * 32) + lane;
#pragma unroll 1
        for (unsigned part = 0; part < at.parts; ++part, in += kNsEpilogueWarps * 8 * 32) {
          float4 v[4 * kGroups];
#pragma unroll
          for (int i = 0; i < 4 * kGroups; ++i)
            if (i < 4 || !narrow) v[i] = __ldcg(in + i * 32);
#pragma unroll
          for (int i = 0; i < 4 * kGroups; ++i)
            if (i < 4 || !narrow) {
              acc[4 * i] += v[i].x;
              acc[4 * i + 1] += v[i].y;
              acc[4 * i + 2] += v[i].z;
              acc[4 * i + 3] += v[i].w;
            }
        }
      }
    }
    if (rows_exist && mine) {
      if (what != kApply || !last) {
        char *out = what == kGram ? q.a : what == kPolynomial ? q.b() : q.x[(s & 1) ^ 1];
        if (rb * 128 + 128 > q.m && row >= q.m) {
          // padding stays zero (an operand read from beyond the panel may leave anything in the sums)
#pragma unroll
          for (int i = 0; i < 16 * kGroups; ++i) acc[i] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < CTAS; ++u) { // 32 columns
          const unsigned col = col0 + u * 32, cb = col / kPanelCols, chunk0 = (col % kPanelCols) / 8;
          if (cb >= col_blocks) continue;
          // where the lane writes and reads the piece, and its first line in the panel; the k-th of its up to
          // four 16-byte chunks lies k * 32 / chunks rows on
          char *const mine = piece + lane * 64, *const theirs = piece + (lane >> shift) * 64 +
                                                                (((lane & mask) ^ ((lane >> (shift + 1)) & 3)) << 4);
          char *line = out + panel_block(rb, cb, col_blocks) + panel_chunk((warp & 3) * 32 + (lane >> shift), chunk0 + (lane & mask));
          const unsigned piece_step = narrow ? 1024 : 512, line_step = 2 * piece_step;
          const bool on_diagonal = what != kApply && col / 32 == row / 32;
          unsigned lo[16];
#pragma unroll
          for (int part = 0; part < 2; ++part, line += kPanelHalf) {
#pragma unroll
            for (unsigned c = 0; c < 4; ++c) {
              if (c > mask) continue;
              unsigned w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (part == 0) {
                  float x = acc[u * 32 + c * 8 + 2 * i] * finish, y = acc[u * 32 + c * 8 + 2 * i + 1] * finish;
                  if (on_diagonal) {
                    if (col + c * 8 + 2 * i == row && row < q.m) x += diagonal;
                    if (col + c * 8 + 2 * i + 1 == row && row < q.m) y += diagonal;
                  }
                  const __half2 h = __floats2half2_rn(x, y);
                  const float2 f = __half22float2(h);
                  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
                  w[i] = *reinterpret_cast<const unsigned *>(&h);
                  lo[c * 4 + i] = *reinterpret_cast<const unsigned *>(&l);
                } else w[i] = lo[c * 4 + i];
              }
              *reinterpret_cast<uint4 *>(mine + ((c ^ ((lane >> 1) & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
#pragma unroll
            for (unsigned k = 0; k < 4; ++k)
              if (k <= mask)
                *reinterpret_cast<uint4 *>(line + k * line_step) = *reinterpret_cast<const uint4 *>(theirs + k * piece_step);
            __syncwarp();
          }
        }
      } else {
        // the weights (or the output), along the matrix's rows as they are stored: the lanes' rows where it
        // was turned, else 16 columns of two rows through shared memory
        const float scale = finish * kSplitUnscale * q.rate;
        float *mine = reinterpret_cast<float *>(piece);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          if (g > 0 && narrow) continue;
          const unsigned c0 = col0 + g * 16;
          if (q.turned) {
            float *w = q.w + (u64)c0 * q.m + row;
            if (row < q.m)
#pragma unroll
              for (int i = 0; i < 16; ++i, w += q.m)
                if (c0 + i < q.n) {
                  const float x = scale * acc[g * 16 + i];
                  *w = q.keep == 0.0f ? -x : q.keep * *w - x;
                }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) mine[lane * 16 + (i ^ (lane & 15))] = acc[g * 16 + i];
            __syncwarp();
            const unsigned col = c0 + (lane & 15), r0 = lane >> 4, row0 = rb * 128 + (warp & 3) * 32;
            float *w = q.w + (u64)(row0 + r0) * q.n + col;
            if (col < q.n)
#pragma unroll 4
              for (unsigned r = r0; r < 32; r += 2, w += 2 * (u64)q.n)
                if (row0 + r < q.m) {
                  const float x = scale * mine[r * 16 + ((lane & 15) ^ (r & 15))];
                  *w = q.keep == 0.0f ? -x : q.keep * *w - x;
                }
            __syncwarp();
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) {
      if (CTAS == 1 && at.parts > 1) { // parts of one tile end in different CTAs: every warp tells for itself
        if (mine) asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(t.stored + (&q - t.mat)) : "memory");
      }
      __threadfence_block();
      *(volatile unsigned *)&sh.written[warp] = ++ring.tiles;
    }
  }
  return true;
}

// ---- the thread that tells the other CTAs: its fence waits for the stores of the draining warps, which go
// on to their next tile meanwhile (a release of their own cost each of them 1,500 to 2,000 cycles a tile)
template <int CTAS>
__device__ bool ns_publish(NsShared &sh, NsRing &ring, int what) {
  const NsTable &t = sh.table;
  for (unsigned tile = ring.first; tile < t.tiles[what]; tile += gridDim.x / CTAS) {
    NsTile at;
    const NsMat &q = tile_at<CTAS>(t, what, tile, at);
    if (!ns_wait_written(sh.written, ++ring.tiles, &sh.wait)) return false;
    if (at.parts == 1)
      asm volatile("red.release.gpu.global.add.u32 [%0], %1;" ::"l"(t.stored + (&q - t.mat)), "n"(kNsEpilogueWarps) : "memory");
  }
  return true;
}

// After a wait that ran out: NaN over this CTA's tiles of the results. What other CTAs have stored was made of
// complete operands; what they could not store they overwrite themselves (of a split K every CTA with a part).
template <int CTAS>
__device__ __noinline__ void ns_spoil(const NsTable &t, unsigned first, unsigned rank) {
  for (unsigned tile = first; tile < t.tiles[kApply]; tile += gridDim.x / CTAS) {
    NsTile at;
    const NsMat &q = tile_at<CTAS>(t, kApply, tile, at);
    const unsigned wide = ns_wide<CTAS>(CTAS == 1 && t.narrow[kApply]), row0 = (at.i * CTAS + rank) * 128, col0 = at.j * wide;
    for (unsigned e = threadIdx.x; e < 128 * wide; e += kNsThreads) {
      const unsigned row = row0 + e / wide, col = col0 + e % wide;
      if (row < q.m && col < q.n) q.w[q.turned ? (u64)col * q.m + row : (u64)row * q.n + col] = NAN;
    }
  }
}

template <int CTAS>
__global__ void __launch_bounds__(kNsThreads, 1) muon_steps_kernel(const __grid_constant__ NsTable param, int steps) {
  extern __shared__ __align__(1024) char dynamic_smem[];
  NsShared &sh = *reinterpret_cast<NsShared *>(dynamic_smem + kNsStages * kNsStageBytes + kNsEpilogueWarps * kNsPieceBytes);
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (unsigned i = threadIdx.x; i < sizeof(NsTable) / 4; i += kNsThreads)
    reinterpret_cast<unsigned *>(&sh.table)[i] = reinterpret_cast<const unsigned *>(&param)[i];
  NsRing ring = {smem_address(dynamic_smem), CTAS == 1 ? 0 : blockIdx.x % CTAS, 0, 0, 0, 0, 0, 0, 0};
  if (threadIdx.x == 0) {
    for (int s = 0; s < kNsStages; ++s) {
      barrier_init(smem_address(&sh.full[s]), 1);
      barrier_init(smem_address(&sh.peer_full[s]), 1);
      barrier_init(smem_address(&sh.empty[s]), 1);
      for (int c = 0; c < 2; ++c) barrier_init(smem_address(&sh.linear_full[c][s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      barrier_init(smem_address(&sh.acc_full[b]), 1);
      barrier_init(smem_address(&sh.acc_empty[b]), kNsEpilogueWarps * CTAS);
    }
    barrier_init(smem_address(&sh.drained), 1);
    sh.wait.limit = param.wait_cycles;
    sh.wait.gave_up = sh.allowed = 0;
    for (int w = 0; w < kNsEpilogueWarps; ++w) sh.written[w] = 0;
    for (int s = 0; s < kNsStages; ++s) sh.linear_read[s] = 0;
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
  const NsTable &t = sh.table;
  const unsigned workers = gridDim.x / CTAS, me = blockIdx.x / CTAS;
  char *piece = dynamic_smem + kNsStages * kNsStageBytes + warp * kNsPieceBytes;
  unsigned before = 0; // tiles of the products so far, modulo the number of workers
  bool ok = true;
#pragma unroll 1
  for (int product = 0; ok && product < 3 * steps; ++product) {
    const int s = product / 3, what = product - 3 * s;
    ring.first = (me + workers - before) % workers;
    if (warp < kNsEpilogueWarps) ok = ns_drain<CTAS>(sh, ring, s, what, s + 1 == steps, piece);
    else if (warp == kNsEpilogueWarps + 1) ok = ns_multiply<CTAS>(sh, ring, what);
    else if (lane == 0) {
      if (warp == kNsEpilogueWarps) ok = ns_load<CTAS>(sh, ring, s, what);
      else if (warp == kNsEpilogueWarps + 2) ok = ns_publish<CTAS>(sh, ring, what);
      else ok = ns_look_out<CTAS>(sh, ring, s, what);
    }
    before = (before + t.tiles[what]) % workers;
  }
  __syncwarp();
  __syncthreads();
  if (sh.wait.gave_up) { // what is in flight ends before its memory goes away
    const long long start = clock64();
    if (warp == kNsEpilogueWarps && lane == 0)
      for (int i = 0; i < 3 * kNsStages; ++i) { // the last copy of each barrier
        const uint32_t bar = i < kNsStages ? smem_address(&sh.full[i]) : smem_address(&sh.linear_full[i / kNsStages - 1][i % kNsStages]);
        while (!barrier_try(bar, ((ring.turns >> i) & 1) ^ 1) && clock64() - start < 10000000) {}
      }
    if (warp == kNsEpilogueWarps + 1 && ring.rank == 0 && elect_one()) {
      mma_commit<CTAS>(smem_address(&sh.drained));
      while (!barrier_try(smem_address(&sh.drained), 0) && clock64() - start < 10000000) {}
    }
    __syncwarp();
    const unsigned skipped = (unsigned)((u64)(steps - 1) * (t.tiles[kGram] + t.tiles[kPolynomial] + t.tiles[kApply]) % workers);
    before = (skipped + t.tiles[kGram] + t.tiles[kPolynomial]) % workers; // the last product's, as in the loop
    ns_spoil<CTAS>(t, (me + workers - before) % workers, ring.rank);
    if (threadIdx.x == 0) atomicAdd(&g_ns_gave_up, 1u);
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if (CTAS > 1) cluster_sync_all(); // nothing of this CTA is used by the other one any more
  tmem_fence_after();
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

// Tickets and sums of the tiles whose K is split: at most one turn of the GPU, for each product.
static u64 ns_ticket_bytes() { return padded((u64)3 * sm_count() * kNsEpilogueWarps * sizeof(unsigned)); }
static u64 ns_parts_bytes() { return padded((u64)3 * sm_count() * kNsEpilogueWarps * 8 * 32 * sizeof(float4)); }

// Numbers the CTAs of a launch over the matrices.
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
// What a product over all matrices costs, in thousands of SM cycles as traced on a B200, for tiles and K
// parts of one kind: K blocks of 64 take 1.7 (pairs, 256 x 256), 1.25 (128 x 128) or 1.05 (128 x 64); a
// tile ends with 3 that its CTA's next one does not hide, a split one with 14; the product as a whole
// starts and ends with 9 (20 for pairs).
template <int CTAS>
static double ns_cost(const NsTable &t, int what, bool narrow, unsigned part_blocks, u64 *units) {
  const double per_block = CTAS == 2 ? 1.7 : narrow ? 1.05 : 1.25;
  double total = 0.0, longest = 0.0;
  *units = 0;
  for (int i = 0; i < t.count; ++i) {
    const unsigned k_blocks = panel_col_blocks(what == kGram ? t.mat[i].n : t.mat[i].m), parts = ns_along(k_blocks, part_blocks);
    const double one = std::min(k_blocks, part_blocks) * per_block + (parts > 1 ? 14.0 : 3.0);
    const u64 n = ns_tiles_of<CTAS>(t.mat[i].m, t.mat[i].n, what, narrow) * parts;
    *units += n;
    total += (double)n * one;
    longest = std::max(longest, one);
  }
  const double workers = (double)(sm_count() / CTAS), turns = ceil((double)*units / workers);
  return std::max(longest, turns * total / (double)*units) + (CTAS == 2 ? 20.0 : 9.0);
}
// Chooses the tiles and K parts of a product; returns its cost.
template <int CTAS>
static double ns_shape(NsTable &t, int what, unsigned *part_blocks) {
  unsigned longest = 0;
  for (int i = 0; i < t.count; ++i) longest = std::max(longest, panel_col_blocks(what == kGram ? t.mat[i].n : t.mat[i].m));
  u64 units = 0;
  t.narrow[what] = 0;
  *part_blocks = longest;
  double best = ns_cost<CTAS>(t, what, false, longest, &units);
  for (int narrow = 0; narrow < (CTAS == 1 ? 2 : 0); ++narrow)
    for (unsigned parts = 1; parts <= kNsMostParts; ++parts) {
      const unsigned blocks = parts == 1 ? longest : ns_part_blocks(longest, parts);
      const double cost = ns_cost<CTAS>(t, what, narrow != 0, blocks, &units);
      if (cost < best && (parts == 1 || units <= (u64)sm_count())) { // the parts' sums have room for one turn
        best = cost;
        t.narrow[what] = narrow;
        *part_blocks = blocks;
      }
    }
  return best;
}

static NsTable steps_table(const MuonTable &mt) {
  NsTable t = {};
  t.count = mt.count;
  t.stored = mt.stored;
  t.tickets = mt.tickets;
  t.parts = mt.parts;
  t.room = (unsigned)sm_count();
  t.wait_cycles = tuned(kTuneMuonWait) >= 0 ? tuned(kTuneMuonWait) * 1000ll : kWaitCycles;
  for (int i = 0; i < mt.count; ++i) {
    const MuonMat &q = mt.mat[i];
    NsMat &d = t.mat[i];
    d.x[0] = q.x[0];
    d.x[1] = q.x[1];
    d.a = q.a;
    d.w = q.w;
    d.keep = q.keep;
    d.rate = q.rate;
    d.m = q.m;
    d.n = q.n;
    d.turned = q.rows > q.cols;
  }
  return t;
}

template <int CTAS>
static void run_steps(NsTable &t, int steps) {
  for (int what = kGram; what <= kApply; ++what) {
    unsigned part_blocks = 0;
    ns_shape<CTAS>(t, what, &part_blocks);
    u64 n = 0;
    for (int i = 0; i < t.count; ++i) {
      NsMat &q = t.mat[i];
      const unsigned k_blocks = panel_col_blocks(what == kGram ? q.n : q.m);
      q.splits[what] = (unsigned char)ns_along(k_blocks, part_blocks);
      q.first_tile[what] = (unsigned)n;
      q.tiles[what] = (unsigned)ns_tiles_of<CTAS>(q.m, q.n, what, t.narrow[what]) * q.splits[what];
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
    take(panel_bytes(q.m, q.m)); // B
    q.partial = (double *)take(padded((u64)(q.chunks + 1) * 8));
  }
  t.stored = (unsigned *)take(256);
  t.tickets = (unsigned *)take(ns_ticket_bytes());
  t.parts = (float4 *)take(ns_parts_bytes());
  t.ticket_count = (unsigned)(ns_ticket_bytes() / sizeof(unsigned));
  auto chunks = [](const MuonMat &q) { return (u64)q.chunks; };
  auto blocks = [](const MuonMat &q) { return (u64)panel_row_blocks(q.m) * panel_col_blocks(q.n); };
  if (!launch_over(t, chunks, muon_momentum_kernel)) return;
  if (!launch_over(t, [](const MuonMat &) { return (u64)1; }, muon_norm_kernel)) return;
  if (!launch_over(t, blocks, muon_load_kernel)) return;
  if (steps > 0) {
    NsTable table = steps_table(t);
    double single = 0.0, paired = 0.0;
    unsigned blocks;
    for (int what = kGram; what <= kApply; ++what) {
      single += ns_shape<1>(table, what, &blocks);
      paired += ns_shape<2>(table, what, &blocks);
    }
    const bool pairs = tuned(kTuneMuonPairs) >= 0 ? tuned(kTuneMuonPairs) != 0 : paired < single;
    if (pairs) run_steps<2>(table, steps);
    else run_steps<1>(table, steps);
    return;
  }
  launch_over(t, chunks, muon_store_kernel);
}

// All matrices, in groups that share one piece of scratch.
static void run_matrices(std::vector<MuonMat> &mats, float mu, float epsilon, int nesterov, int steps) {
  // longest products first: what ends a product is short then, and the next ones have begun
  std::stable_sort(mats.begin(), mats.end(), [](const MuonMat &a, const MuonMat &b) { return a.n != b.n ? a.n > b.n : a.m > b.m; });
  u64 largest = 0;
  std::vector<size_t> ends;
  for (size_t i = 0; i < mats.size();) {
    u64 bytes = 256 + ns_ticket_bytes() + ns_parts_bytes();
    size_t k = i;
    while (k < mats.size() && k - i < (size_t)kMuonMax && (k == i || bytes + scratch_bytes(mats[k]) <= kMuonScratch))
      bytes += scratch_bytes(mats[k++]);
    largest = std::max(largest, bytes);
    ends.push_back(i = k);
  }
  char *scratch = nullptr;
  if (!check_cuda(scratch_alloc_async((void **)&scratch, largest))) return;
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

// The buffers of a call. One that is written overlaps no other, but that it may be its own matrix's input.
struct MuonSpan {
  const char *begin, *end;
  bool written;
  int matrix;
};
static MuonSpan span_of(const Tensor *t, bool written, int matrix) {
  const char *p = (const char *)t->data;
  return MuonSpan{p, p + numel(t) * 4, written, matrix};
}
static bool apart(const char *name, std::vector<MuonSpan> spans, bool in_place) {
  std::sort(spans.begin(), spans.end(), [](const MuonSpan &a, const MuonSpan &b) { return a.begin < b.begin; });
  for (size_t i = 0; i < spans.size(); ++i)
    for (size_t k = i + 1; k < spans.size() && spans[k].begin < spans[i].end; ++k) {
      const MuonSpan &a = spans[i], &b = spans[k];
      if (!a.written && !b.written) continue;
      if (in_place && a.written != b.written && a.matrix == b.matrix && a.begin == b.begin && a.end == b.end) continue;
      set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: a buffer that is written overlaps another one", name);
      return false;
    }
  return true;
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

// A call that needs the host's view of the device cannot be part of a graph; refused before it spoils the capture.
static bool check_not_captured(const char *what) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (!check_cuda(cudaStreamIsCapturing(stream(), &status))) return false;
  if (status == cudaStreamCaptureStatusNone) return true;
  set_error(PLAST_B200_ERR_UNSUPPORTED, "muon: %s cannot be captured into a graph", what);
  return false;
}

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
  std::vector<MuonSpan> spans;
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
    spans.push_back(span_of(p, true, i));
    spans.push_back(span_of(p->grad, false, i));
  }
  if (!apart(name, spans, false)) return;
  // momenta: the caller's, or made here on the first step
  bool made = false;
  if (opt->m) {
    std::lock_guard<std::mutex> lock(g_muon_mutex);
    auto it = g_muon_states.find(opt->m);
    if (it != g_muon_states.end() && num_parameters > it->second.n)
      return set_error(PLAST_B200_ERR_SHAPE, "muon: %d parameters, but the momenta were created for %d", num_parameters, it->second.n);
  } else if (!mats.empty()) {
    if (!check_not_captured("a first step, which creates the momenta,")) return;
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
    if (!made) spans.push_back(span_of(m, true, index[k]));
  }
  if (!made && !apart(name, spans, false)) return;
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
  std::vector<MuonSpan> spans;
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
    spans.push_back(span_of(inputs[i], false, i));
    spans.push_back(span_of(outputs[i], true, i));
  }
  if (!apart(name, spans, true)) return;
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
  static std::mutex mutex;
  static std::unordered_map<int, unsigned> told; // per device: what an earlier look has seen
  int device = 0;
  unsigned now = 0;
  if (!check_not_captured("a look at the status")) return -1;
  PB_CUDA_RET(cudaGetDevice(&device), -1);
  PB_CUDA_RET(cudaMemcpyFromSymbolAsync(&now, g_ns_gave_up, sizeof now, 0, cudaMemcpyDeviceToHost, stream()), -1);
  PB_CUDA_RET(cudaStreamSynchronize(stream()), -1);
  try {
    std::lock_guard<std::mutex> lock(mutex);
    unsigned &seen = told[device];
    const bool more = now != seen;
    seen = now;
    return more;
  } catch (...) { // std::bad_alloc
    set_error(PLAST_B200_ERR_CUDA, "muon: out of host memory");
    return -1;
  }
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
