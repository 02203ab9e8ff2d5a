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
  unsigned first;      // first CTA (or tile) of this matrix in the launch at hand
  unsigned chunks;
};
struct MuonTable {
  MuonMat mat[kMuonMax];
  int count;
  unsigned total; // CTAs or tiles of the launch at hand
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
  if (threadIdx.x == 0) q.partial[0] = part[0];
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
//   polynomial  B = b A + c A A    both operands A (symmetric), K-major, K = m
//   apply       X = a X + B X      left B, K-major; right X, MN-major (its rows are K), K = m
// A persistent CTA walks tiles of 128 x 128. One thread brings 64 KB stages (64 of K, hi and lo of
// both operands) with bulk copies, one thread issues the twelve tcgen05.mma of a stage, small products
// first, and eight warps drain the accumulators. Tensor-core accumulation truncates; every kNsChunk
// stages the accumulator (one of two in tensor memory) is therefore added in fp32 registers, rounded
// to nearest, while the next one fills.
enum MuonProduct { kGram = 0, kPolynomial = 1, kApply = 2 };
constexpr int kNsStages = 3;
constexpr unsigned kNsStageBytes = 4 * kPanelHalf; // left hi, left lo, right hi, right lo
constexpr int kNsEpilogueWarps = 8, kNsThreads = (kNsEpilogueWarps + 2) * 32;
#ifndef NS_CHUNK
#define NS_CHUNK 4
#endif
constexpr int kNsChunk = NS_CHUNK;
constexpr unsigned kNsSmem = kNsStages * kNsStageBytes + 1024;

__device__ unsigned g_ns_gave_up; // a wait ran out: results are NaN from then on, see plast_b200_muon_status

struct NsTile {
  unsigned i, j, k_blocks; // tile row, tile column, K / 64
};
template <int WHAT>
__device__ __forceinline__ const MuonMat &tile_at(const MuonTable &t, unsigned tile, NsTile &out) {
  const MuonMat &q = t.mat[matrix_of(t, tile)];
  const unsigned across = panel_row_blocks(WHAT == kApply ? q.n : q.m), at = tile - q.first;
  out.i = at / across;
  out.j = at % across;
  out.k_blocks = panel_col_blocks(WHAT == kGram ? q.n : q.m);
  return q;
}

template <int WHAT>
__global__ void __launch_bounds__(kNsThreads, 1) muon_product_kernel(const __grid_constant__ MuonTable t, int from, int last) {
  extern __shared__ char dynamic_smem[];
  __shared__ __align__(8) uint64_t full[kNsStages], empty[kNsStages], acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t tmem_base;
  __shared__ volatile unsigned gave_up;
  const uint32_t stages = (smem_address(dynamic_smem) + 1023) & ~1023u;
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr unsigned kColumns = 128; // of one accumulator

  if (threadIdx.x == 0) {
    for (int s = 0; s < kNsStages; ++s) {
      barrier_init(smem_address(&full[s]), 1);
      barrier_init(smem_address(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      barrier_init(smem_address(&acc_full[b]), 1);
      barrier_init(smem_address(&acc_empty[b]), kNsEpilogueWarps);
    }
    barrier_init(smem_address(&drained), 1);
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kNsEpilogueWarps + 1) tmem_alloc<1>(smem_address(&tmem_base), 2 * kColumns);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = tmem_base;
  pdl_wait();
  pdl_launch_dependents();

  if (warp == kNsEpilogueWarps) { // ---- loads
    if (lane == 0) {
      asm volatile("fence.proxy.async;" ::: "memory"); // the panels were written with plain stores
      unsigned it = 0;
      bool ok = true;
      for (unsigned tile = blockIdx.x; ok && tile < t.total; tile += gridDim.x) {
        NsTile at;
        const MuonMat &q = tile_at<WHAT>(t, tile, at);
        const unsigned xcb = panel_col_blocks(q.n), mcb = panel_col_blocks(q.m);
        const char *left = WHAT == kGram ? q.x[from] : WHAT == kPolynomial ? q.a : q.b;
        const unsigned left_cb = WHAT == kGram ? xcb : mcb;
        const char *right = WHAT == kApply ? q.x[from] : left;
        for (unsigned k = 0; k < at.k_blocks; ++k, ++it) {
          const unsigned s = it % kNsStages, phase = (it / kNsStages) & 1;
          if (!(ok = barrier_wait(smem_address(&empty[s]), phase ^ 1, &gave_up))) break;
          const uint32_t bar = smem_address(&full[s]), dst = stages + s * kNsStageBytes;
          if (WHAT != kApply) {
            barrier_expect(bar, kNsStageBytes);
            bulk_load(dst, left + panel_block(at.i, k, left_cb), 2 * kPanelHalf, bar);
            bulk_load(dst + 2 * kPanelHalf, right + panel_block(at.j, k, left_cb), 2 * kPanelHalf, bar);
          } else {
            // right: rows 64 k .. 64 k + 63 of two neighbouring blocks of X, the second of which may
            // lie beyond its last column (then those columns of the tile are not stored)
            const bool both = 2 * at.j + 1 < xcb;
            barrier_expect(bar, 2 * kPanelHalf + (both ? 2 : 1) * kPanelHalf);
            bulk_load(dst, left + panel_block(at.i, k, left_cb), 2 * kPanelHalf, bar);
            for (unsigned c = 0; c < (both ? 2u : 1u); ++c) {
              const char *src = right + panel_block(k / 2, 2 * at.j + c, xcb) + (k & 1) * (kPanelHalf / 2);
              bulk_load(dst + 2 * kPanelHalf + c * (kPanelHalf / 2), src, kPanelHalf / 2, bar);
              bulk_load(dst + 3 * kPanelHalf + c * (kPanelHalf / 2), src + kPanelHalf, kPanelHalf / 2, bar);
            }
          }
        }
      }
      if (!ok) // copies in flight end before shared memory goes away
        for (unsigned back = 1; back <= kNsStages && back <= it; ++back) {
          const unsigned i = it - back, s = i % kNsStages, phase = (i / kNsStages) & 1;
          const long long start = clock64();
          while (!barrier_try(smem_address(&full[s]), phase) && clock64() - start < 10000000) {}
        }
    }
  } else if (warp == kNsEpilogueWarps + 1) { // ---- products
    if (lane == 0) {
      constexpr uint32_t desc = mma_desc(128, 128, false, WHAT == kApply);
      unsigned it = 0, round = 0;
      bool ok = true;
      for (unsigned tile = blockIdx.x; ok && tile < t.total; tile += gridDim.x) {
        NsTile at;
        tile_at<WHAT>(t, tile, at);
        for (unsigned k = 0; k < at.k_blocks; ++k, ++it) {
          const unsigned s = it % kNsStages, phase = (it / kNsStages) & 1, buf = round & 1;
          const bool first = k % kNsChunk == 0;
          if (first && !(ok = barrier_wait(smem_address(&acc_empty[buf]), ((round >> 1) & 1) ^ 1, &gave_up))) break;
          if (!(ok = barrier_wait(smem_address(&full[s]), phase, &gave_up))) break;
          tmem_fence_after();
          const uint32_t left = stages + s * kNsStageBytes, right = left + 2 * kPanelHalf;
          const uint32_t acc = tmem + buf * kColumns;
#pragma unroll
          for (int part = 0; part < 3; ++part) { // lo hi, hi lo, hi hi
            const uint32_t l = left + (part == 0 ? kPanelHalf : 0), r = right + (part == 1 ? kPanelHalf : 0);
#pragma unroll
            for (int step = 0; step < 4; ++step) { // 16 of K
              const uint64_t da = operand_desc(l + step * 32, 16, 1024);
              const uint64_t db = WHAT == kApply ? operand_desc(r + step * 2048, kPanelHalf / 2, 1024)
                                                 : operand_desc(r + step * 32, 16, 1024);
              mma_f16<1>(acc, da, db, desc, !(first && part == 0 && step == 0));
            }
          }
          mma_commit<1>(smem_address(&empty[s]));
          if (k % kNsChunk == kNsChunk - 1 || k + 1 == at.k_blocks) {
            mma_commit<1>(smem_address(&acc_full[buf]));
            ++round;
          }
        }
      }
      if (!ok) {
        mma_commit<1>(smem_address(&drained));
        const long long start = clock64();
        while (!barrier_try(smem_address(&drained), 0) && clock64() - start < 10000000) {}
      }
    }
  } else { // ---- accumulators to results: warp w takes rows 32 (w % 4) .. and columns 64 (w / 4) ..
    const unsigned row_in_tile = (warp & 3) * 32 + lane, half = warp >> 2;
    unsigned round = 0;
    bool ok = true;
    for (unsigned tile = blockIdx.x; ok && tile < t.total; tile += gridDim.x) {
      NsTile at;
      const MuonMat &q = tile_at<WHAT>(t, tile, at);
      float acc[64];
      const unsigned rounds = (at.k_blocks + kNsChunk - 1) / kNsChunk;
      for (unsigned c = 0; c < rounds; ++c, ++round) {
        const unsigned buf = round & 1;
        ok = __all_sync(0xffffffffu, barrier_wait(smem_address(&acc_full[buf]), (round >> 1) & 1, &gave_up));
        if (!ok) break;
        tmem_fence_after();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[32];
          tmem_load32(tmem + (((warp & 3) * 32) << 16) + buf * kColumns + half * 64 + h * 32, v);
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[h * 32 + i] = c == 0 ? v[i] : acc[h * 32 + i] + v[i];
        }
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) barrier_arrive(smem_address(&acc_empty[buf]));
      }
      if (!ok) break;
      // the warp's 64 columns are one block column of the result
      const unsigned width = WHAT == kApply ? q.n : q.m;
      const unsigned col_blocks = panel_col_blocks(width), cb = 2 * at.j + half;
      if (cb >= col_blocks) continue;
      const u64 offset = panel_block(at.i, cb, col_blocks);
      const char *old = WHAT == kPolynomial ? q.a : q.x[from]; // the linear term
      char *out = WHAT == kGram ? q.a : WHAT == kPolynomial ? q.b : q.x[from ^ 1];
#pragma unroll
      for (int chunk = 0; chunk < 8; ++chunk) {
        const u64 here = offset + panel_chunk(row_in_tile, chunk);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = acc[chunk * 8 + i] * kSplitUnscale;
        if (WHAT != kGram) {
          float z[8];
          join8(*reinterpret_cast<const uint4 *>(old + here), *reinterpret_cast<const uint4 *>(old + here + kPanelHalf), z);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[i] = WHAT == kPolynomial ? __fmaf_rn(kNsB, z[i], kNsC * v[i]) : __fmaf_rn(kNsA, z[i], v[i]);
        }
        if (WHAT != kApply || !last) {
          uint4 hi, lo;
          split8(v, hi, lo);
          *reinterpret_cast<uint4 *>(out + here) = hi;
          *reinterpret_cast<uint4 *>(out + here + kPanelHalf) = lo;
        } else {
          const unsigned row = at.i * 128 + row_in_tile;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const unsigned col = cb * kPanelCols + chunk * 8 + i;
            if (row >= q.m || col >= q.n) continue;
            float *w = q.w + (q.rows <= q.cols ? (u64)row * q.n + col : (u64)col * q.m + row);
            const float x = g_ns_gave_up ? NAN : v[i] * kSplitUnscale;
            *w = q.keep == 0.0f ? -q.rate * x : __fmaf_rn(-q.rate, x, q.keep * *w);
          }
        }
      }
    }
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (threadIdx.x == 0 && gave_up) atomicOr(&g_ns_gave_up, 1u);
  if (warp == kNsEpilogueWarps + 1) tmem_free<1>(tmem, 2 * kColumns);
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
template <int WHAT>
static bool launch_product(MuonTable &t, int from, int last) {
  number(t, [](const MuonMat &q) {
    return (u64)panel_row_blocks(q.m) * panel_row_blocks(WHAT == kApply ? q.n : q.m);
  });
  const cudaError_t e = cudaFuncSetAttribute(muon_product_kernel<WHAT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kNsSmem);
  if (e != cudaSuccess) return launched(e);
  const unsigned grid = t.total < (unsigned)sm_count() ? t.total : (unsigned)sm_count();
  return launched(launch_k(muon_product_kernel<WHAT>, dim3(grid), dim3(kNsThreads), kNsSmem, stream(), t, from, last));
}

// One group of matrices whose scratch is `base`.
static void run_group(MuonTable &t, char *base, int steps) {
  for (int i = 0; i < t.count; ++i) {
    MuonMat &q = t.mat[i];
    auto take = [&](u64 bytes) {
      char *p = base;
      base += bytes;
      return p;
    };
    q.x[0] = take(panel_bytes(q.m, q.n));
    q.x[1] = take(panel_bytes(q.m, q.n));
    q.a = take(panel_bytes(q.m, q.m));
    q.b = take(panel_bytes(q.m, q.m));
    q.partial = (double *)take(padded((u64)(q.chunks + 1) * 8));
  }
  auto chunks = [](const MuonMat &q) { return (u64)q.chunks; };
  auto blocks = [](const MuonMat &q) { return (u64)panel_row_blocks(q.m) * panel_col_blocks(q.n); };
  if (!launch_over(t, chunks, muon_momentum_kernel)) return;
  if (!launch_over(t, [](const MuonMat &) { return (u64)1; }, muon_norm_kernel)) return;
  if (!launch_over(t, blocks, muon_load_kernel)) return;
  for (int s = 0; s < steps; ++s) {
    const int from = s & 1, last = s + 1 == steps;
    if (!launch_product<kGram>(t, from, 0) || !launch_product<kPolynomial>(t, from, 0) || !launch_product<kApply>(t, from, last))
      return;
  }
  if (steps == 0) launch_over(t, chunks, muon_store_kernel);
}

// All matrices, in groups that share one piece of scratch.
static void run_matrices(const std::vector<MuonMat> &mats, float mu, float epsilon, int nesterov, int steps) {
  u64 largest = 0;
  std::vector<size_t> ends;
  for (size_t i = 0; i < mats.size();) {
    u64 bytes = 0;
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
