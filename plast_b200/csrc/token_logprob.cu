// Log probabilities of given tokens with their entropy, log normaliser and top alternatives.
//
// For one row x of C logits at temperature T, z = x / T, m = max z, e_j = exp(z_j - m):
//   L = m + log S,  S = sum e_j                       log normaliser
//   logprob = z_t - L                                 of the given token t
//   H = log S - U / S,  U = sum e_j (z_j - m)         entropy; both terms are >= 0, nothing cancels
// One pass over the row keeps (m, S, U) per thread; a new maximum m' rescales with d = m - m':
//   S' = S e^d,  U' = (U + S d) e^d.
// The k best logits come out of the same pass (see "alternatives" below).
// Backward, with upstream gradients gl (logprob), gH (entropy), gL (log_norm):
//   dx_j += ( gl (1[j == t] - p_j) - gH p_j (log p_j + H) + gL p_j ) / T,
//   p_j = e^(z_j - m) / S,  log p_j = (z_j - m) - log S.
// m and S travel from forward to backward as two numbers per row: L alone would round p_j by half an
// ulp of L, which for logits far from 0 (a row at the type's lowest value) leaves nothing of it.
#include "row_map.cuh"
#include "ew_kernel_device.cuh" // pdl_wait / pdl_launch_dependents

#include <cooperative_groups.h>
#include <math.h>

namespace pb {

constexpr int kLpMaxThreads = 512;
constexpr int kLpUnroll = 4;      // float4 per thread and trip
constexpr int kLpCandidates = 1024;
constexpr int kLpMaxCluster = 8;  // portable cluster size
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;

typedef unsigned long long u64key;

struct LpParams {
  const float *x;
  const int *token;
  float *logprob, *entropy, *log_norm; // the last two may be NULL
  float2 *stats;                       // (max logit, S), may be NULL
  float *top_logprob;
  int *top_index;
  RowMap map;      // 0: logits, 1: tokens
  u64 col_stride;  // of the logits
  unsigned cols;
  int top;
  unsigned cluster;
  float scale_log2; // log2(e) / T
  double temperature;
};

__device__ __forceinline__ float ex2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
// max that keeps a NaN; bounds the exponent of masked logits so that 0 * (-inf) does not arise
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
constexpr float kFloorLog2 = -1000.0f; // 2^-1000 is 0 in fp32

// Running statistics of a slice, in log2 units: m is a raw logit, t = (x - m) * log2(e) / T.
struct LpStat {
  float m, s, u;
  __device__ __forceinline__ void init() { m = -3.402823466e38f; s = 0.0f; u = 0.0f; }
  // moves to a maximum m1 >= m
  __device__ __forceinline__ void raise(float m1, float c) {
    const float t = max_nan((m - m1) * c, kFloorLog2);
    const float f = ex2(t);
    u = __fmaf_rn(s, t, u) * f;
    s = s * f;
    m = m1;
  }
  __device__ __forceinline__ void add(float x, float c) {
    const float t = max_nan((x - m) * c, kFloorLog2);
    const float e = ex2(t);
    s += e;
    u = __fmaf_rn(e, t, u);
  }
  __device__ __forceinline__ void merge(float om, float os, float ou, float c) {
    LpStat o = {om, os, ou};
    const float m1 = fmaxf(m, om);
    raise(m1, c);
    o.raise(m1, c);
    s += o.s;
    u += o.u;
  }
};

// ---- alternatives ------------------------------------------------------------------------------------
// A logit and its index as one number: larger logits first, of equal logits the lower index first
// (-0 and +0 are equal). NaN has no place in the order and is never a candidate.
__device__ __forceinline__ u64key key_of(float v, unsigned index) {
  unsigned b = __float_as_uint(v + 0.0f);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((u64key)b << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ float value_of(u64key k) {
  const unsigned b = (unsigned)(k >> 32);
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}
__device__ __forceinline__ unsigned index_of(u64key k) { return 0xffffffffu - (unsigned)k; }

struct LpShared {
  u64key cand[kLpCandidates];
  u64key best[PLAST_TOKEN_TOP_MAX];
  u64key join[kLpMaxCluster * PLAST_TOKEN_TOP_MAX];
  float stat[kLpMaxCluster][3];
  float warp_stat[kLpMaxThreads / 32][3];
  float warp_k[kLpMaxThreads / 32], warp_j[kLpMaxThreads / 32];
  unsigned count;
  double log_s, shift;
  int empty;
};

// The k best of the n keys in `from` go to sh.best in order, by counting for each key how many are
// larger (keys are distinct); `n <= kLpCandidates`. Threads share a key where there are few.
__device__ void select_best(LpShared &sh, const u64key *from, unsigned n, int k) {
  unsigned share = 1;
  while (share < 32 && n * share * 2 <= blockDim.x) share *= 2;
  const unsigned lane = threadIdx.x & (share - 1), per_trip = blockDim.x / share;
  for (unsigned base = 0; base < n; base += per_trip) { // the trip count is uniform
    const unsigned at = base + threadIdx.x / share;
    const u64key mine = at < n ? from[at] : 0;
    unsigned larger = 0;
    if (mine)
      for (unsigned i = lane; i < n; i += share) larger += from[i] > mine;
    for (unsigned o = share / 2; o; o >>= 1) larger += __shfl_xor_sync(0xffffffffu, larger, o);
    if (mine && lane == 0 && larger < (unsigned)k) sh.best[larger] = mine;
  }
}

// A lower bound on the k-th largest logit of the rows' elements seen in one trip, from the largest
// logit of each thread: k threads of one warp hold k distinct elements at or above that warp's k-th
// largest, and so do ceil(k / warps) threads of every warp.
__device__ __forceinline__ float trip_bound(LpShared &sh, float mine, int k) {
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float v = mine;
#pragma unroll
  for (unsigned size = 2; size <= 32; size *= 2)
#pragma unroll
    for (unsigned o = size / 2; o; o >>= 1) { // bitonic sort, largest first
      const float other = __shfl_xor_sync(0xffffffffu, v, o);
      const bool keep_max = ((lane & o) == 0) == ((lane & size) == 0 || size == 32);
      v = keep_max ? fmaxf(v, other) : fminf(v, other);
    }
  const int j = (k + (int)warps - 1) / (int)warps;
  if ((int)lane == k - 1) sh.warp_k[warp] = v;
  if ((int)lane == j - 1) sh.warp_j[warp] = v;
  __syncthreads();
  float a = sh.warp_k[0], b = sh.warp_j[0];
  for (unsigned w = 1; w < warps; ++w) {
    a = fmaxf(a, sh.warp_k[w]);
    b = fminf(b, sh.warp_j[w]);
  }
  __syncthreads();
  return fmaxf(a, b);
}

// ---- forward -----------------------------------------------------------------------------------------
// One cluster of CTAs per row (1 where the rows fill the GPU; up to 8 where there are few rows, whose
// slices are joined through distributed shared memory). A trip moves 16 logits per thread.
//
// Alternatives: logits that can still be among the k best are pushed into a shared list with an
// atomic counter (their order does not matter: the list is ranked by key at the end). The threshold
// starts as trip_bound() of the first trip, about the hundredth part of random logits; if the list
// fills up it is cut to its k best, whose last key is the new threshold, and the trip's other
// candidates are tried again, so any order and any number of ties ends with the exact answer.
template <bool UNIT, bool TOP>
__global__ void __launch_bounds__(kLpMaxThreads) token_logprob_kernel(const __grid_constant__ LpParams p) {
  __shared__ LpShared sh;
  namespace cg = cooperative_groups;
  pdl_wait();
  pdl_launch_dependents();
  const unsigned rank = blockIdx.x % p.cluster, row = blockIdx.x / p.cluster;
  if (p.cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  u64 off[3];
  row_offsets(p.map, row, off);
  const float *x = p.x + off[0];
  const float c = p.scale_log2;
  const int k = p.top;
  // thread 0 of the row's first CTA reports; its two dependent loads start now
  int token = -1;
  float x_token = 0.0f;
  if (rank == 0 && threadIdx.x == 0) {
    token = p.token[off[1]];
    if (token >= 0 && (unsigned)token < p.cols) x_token = x[(u64)token * p.col_stride];
    else token = -1;
  }
  if (TOP && threadIdx.x == 0) sh.count = 0;
  // vectors of four logits; the first one starts at the 16-byte boundary at or before the row
  const unsigned lead = UNIT ? (unsigned)(((uintptr_t)x >> 2) & 3) : 0u;
  const unsigned vectors = (unsigned)(((u64)p.cols + lead + 3) >> 2);
  const unsigned slice = (vectors + p.cluster - 1) / p.cluster;
  const unsigned first = rank * slice < vectors ? rank * slice : vectors;
  const unsigned last = vectors - first < slice ? vectors : first + slice;
  const unsigned trip = blockDim.x * kLpUnroll;

  LpStat st;
  st.init();
  u64key threshold = 0;
  float threshold_value = -INFINITY;
  bool first_trip = true;
  for (unsigned base = first; base < last; base += trip) {
    float v[kLpUnroll * 4];
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      const unsigned at = base + u * blockDim.x + threadIdx.x;
      const long long j = (long long)at * 4 - lead; // logit index of the vector's first lane
      if (at < last && j >= 0 && j + 4 <= (long long)p.cols) {
        if (UNIT) {
          const float4 q = __ldcs(reinterpret_cast<const float4 *>(x + j));
          v[4 * u] = q.x; v[4 * u + 1] = q.y; v[4 * u + 2] = q.z; v[4 * u + 3] = q.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[4 * u + i] = x[(u64)(j + i) * p.col_stride];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[4 * u + i] = (at < last && j + i >= 0 && j + i < (long long)p.cols) ? x[(u64)(j + i) * p.col_stride] : -INFINITY;
      }
    }
    float top = v[0];
#pragma unroll
    for (int i = 1; i < kLpUnroll * 4; ++i) top = fmaxf(top, v[i]);
    if (top > st.m) st.raise(top, c);
#pragma unroll
    for (int i = 0; i < kLpUnroll * 4; ++i) st.add(v[i], c);

    if (TOP) {
      if (first_trip) {
        threshold_value = trip_bound(sh, fmaxf(top, -INFINITY), k); // fmaxf drops a NaN
        threshold = ((u64key)(unsigned)(key_of(threshold_value, 0) >> 32) << 32) - 1;
        first_trip = false;
      }
      unsigned todo = 0;
      if (top >= threshold_value) {
#pragma unroll
        for (int i = 0; i < kLpUnroll * 4; ++i) todo |= (v[i] >= threshold_value ? 1u : 0u) << i;
      }
      while (__syncthreads_or(todo != 0)) {
        unsigned left = 0;
        for (; todo; todo &= todo - 1) { // few: the logit is fetched again instead of held in registers
          const unsigned i = __ffs(todo) - 1;
          const unsigned at = base + (i / 4) * blockDim.x + threadIdx.x;
          const long long j = (long long)at * 4 - lead + (i & 3);
          if (at >= last || j < 0 || j >= (long long)p.cols) continue;
          const u64key key = key_of(x[(u64)j * p.col_stride], (unsigned)j);
          if (key <= threshold) continue;
          const unsigned slot = atomicAdd(&sh.count, 1u);
          if (slot < kLpCandidates) sh.cand[slot] = key;
          else left |= 1u << i;
        }
        todo = left;
        __syncthreads();
        if (sh.count > kLpCandidates) { // cut the list, tighten the threshold, try the rest again
          select_best(sh, sh.cand, kLpCandidates, k);
          __syncthreads();
          for (int i = threadIdx.x; i < k; i += blockDim.x) sh.cand[i] = sh.best[i];
          if (threadIdx.x == 0) sh.count = k;
          threshold = sh.best[k - 1];
          threshold_value = value_of(threshold);
          __syncthreads();
        }
      }
    }
  }

  // ---- the CTA's statistics
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, st.m, o), os = __shfl_xor_sync(0xffffffffu, st.s, o),
                ou = __shfl_xor_sync(0xffffffffu, st.u, o);
    st.merge(om, os, ou, c);
  }
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0) {
    sh.warp_stat[warp][0] = st.m;
    sh.warp_stat[warp][1] = st.s;
    sh.warp_stat[warp][2] = st.u;
  }
  __syncthreads();
  if (TOP) {
    // slots that the selection does not fill stay 0 (a key is never 0)
    for (int i = threadIdx.x; i < k; i += blockDim.x) sh.best[i] = 0;
    __syncthreads();
    select_best(sh, sh.cand, sh.count < kLpCandidates ? sh.count : kLpCandidates, k);
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    st.m = sh.warp_stat[0][0]; st.s = sh.warp_stat[0][1]; st.u = sh.warp_stat[0][2];
    for (unsigned w = 1; w < warps; ++w) st.merge(sh.warp_stat[w][0], sh.warp_stat[w][1], sh.warp_stat[w][2], c);
  }
  __syncwarp();
  if (p.cluster > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); // every CTA of the cluster runs
    LpShared *lead_sh = cg::this_cluster().map_shared_rank(&sh, 0);
    if (threadIdx.x == 0) {
      lead_sh->stat[rank][0] = st.m;
      lead_sh->stat[rank][1] = st.s;
      lead_sh->stat[rank][2] = st.u;
    }
    if (TOP)
      for (int i = threadIdx.x; i < k; i += blockDim.x) lead_sh->join[rank * k + i] = sh.best[i];
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0) return;
    if (threadIdx.x == 0) {
      st.m = sh.stat[0][0]; st.s = sh.stat[0][1]; st.u = sh.stat[0][2];
      for (unsigned r = 1; r < p.cluster; ++r) st.merge(sh.stat[r][0], sh.stat[r][1], sh.stat[r][2], c);
    }
    if (TOP) {
      for (int i = threadIdx.x; i < k; i += blockDim.x) sh.best[i] = 0;
      __syncthreads();
      select_best(sh, sh.join, p.cluster * k, k);
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) {
    // the last few operations of a row in 64 bits, each result rounded once
    const bool empty = st.s == 0.0f; // every logit is -inf
    const double log_s = log((double)st.s);
    const double L = empty ? -INFINITY : (double)st.m / p.temperature + log_s;
    const double shift = (double)st.m; // log p = (x - m) / T - log S keeps its digits where L has none
    double h = empty ? 0.0 : log_s - kLn2 * ((double)st.u / (double)st.s);
    if (h < 0.0) h = 0.0; // rounding of U; a NaN passes
    double lp = 0.0;
    if (token >= 0) lp = empty ? -INFINITY : ((double)x_token - shift) / p.temperature - log_s;
    p.logprob[row] = (float)lp;
    if (p.entropy) p.entropy[row] = (float)h;
    if (p.log_norm) p.log_norm[row] = (float)L;
    if (p.stats) p.stats[row] = make_float2(st.m, st.s);
    sh.log_s = log_s;
    sh.shift = shift;
    sh.empty = empty;
  }
  if (TOP) {
    __syncthreads();
    if ((int)threadIdx.x < k) {
      const u64key key = sh.best[threadIdx.x];
      const u64 at = (u64)row * k + threadIdx.x;
      p.top_index[at] = key ? (int)index_of(key) : -1;
      p.top_logprob[at] = !key ? NAN : sh.empty ? -INFINITY : (float)(((double)value_of(key) - sh.shift) / p.temperature - sh.log_s);
    }
  }
}

// ---- backward ----------------------------------------------------------------------------------------
struct LpGradParams {
  const float *x;
  const int *token;
  float *dx;
  const float2 *stats;                             // (max logit, S) of the forward
  const float *entropy;                            // may be NULL when g_entropy is
  const float *g_logprob, *g_entropy, *g_log_norm; // any may be NULL
  RowMap map;                                      // 0: logits, 1: tokens, 2: gradient
  u64 col_stride, grad_stride;
  unsigned cols;
  float scale_log2, inv_t;
};

// A streaming pass over the row: 4 B read and 8 B for the += per logit.
template <bool VEC>
__global__ void __launch_bounds__(kLpMaxThreads) token_logprob_backward_kernel(const __grid_constant__ LpGradParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const unsigned row = blockIdx.x;
  const float2 stat = p.stats[row];
  if (stat.y == 0.0f) return; // an empty row has no gradient
  u64 off[3];
  row_offsets(p.map, row, off);
  const float *x = p.x + off[0];
  float *dx = p.dx + off[2];
  int token = p.token[off[1]];
  const bool valid = token >= 0 && (unsigned)token < p.cols;
  const float gl = valid && p.g_logprob ? p.g_logprob[row] : 0.0f;
  const float gh = p.g_entropy ? p.g_entropy[row] : 0.0f;
  const float gn = p.g_log_norm ? p.g_log_norm[row] : 0.0f;
  const unsigned hit = valid ? (unsigned)token : 0xffffffffu;
  // the gradient is p_j (base + slope t_j), t_j = (x_j - m) log2(e) / T, all constants with 1 / T in them
  const float m = stat.x, c = p.scale_log2, inv_s = p.inv_t / stat.y, at_token = gl * p.inv_t;
  const float slope = -gh * (float)kLn2;
  const float base = (gn - gl) + gh * (logf(stat.y) - (p.g_entropy ? p.entropy[row] : 0.0f));
  // one element; the exponent is bounded below so that a masked logit (p = 0) adds exactly 0
  auto grad = [&](float xv, unsigned j) {
    const float t = max_nan((xv - m) * c, kFloorLog2);
    const float g = ex2(t) * inv_s * __fmaf_rn(slope, t, base);
    return j == hit ? g + at_token : g;
  };
  if (VEC) {
    const unsigned lead = (unsigned)(((uintptr_t)x >> 2) & 3);
    const unsigned vectors = (unsigned)(((u64)p.cols + lead + 3) >> 2);
    for (unsigned at0 = threadIdx.x; at0 < vectors; at0 += blockDim.x * 2) {
      float4 q[2], d[2];
      bool full[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned at = at0 + u * blockDim.x;
        const long long j = (long long)at * 4 - lead;
        full[u] = at < vectors && j >= 0 && j + 4 <= (long long)p.cols;
        if (full[u]) {
          q[u] = __ldcs(reinterpret_cast<const float4 *>(x + j));
          d[u] = __ldcs(reinterpret_cast<const float4 *>(dx + j));
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned at = at0 + u * blockDim.x;
        const long long j = (long long)at * 4 - lead;
        if (full[u]) {
          d[u].x += grad(q[u].x, (unsigned)j);
          d[u].y += grad(q[u].y, (unsigned)j + 1);
          d[u].z += grad(q[u].z, (unsigned)j + 2);
          d[u].w += grad(q[u].w, (unsigned)j + 3);
          __stcs(reinterpret_cast<float4 *>(dx + j), d[u]);
        } else if (at < vectors) {
          for (int i = 0; i < 4; ++i)
            if (j + i >= 0 && j + i < (long long)p.cols) dx[j + i] += grad(x[j + i], (unsigned)(j + i));
        }
      }
    }
  } else {
    for (unsigned j = threadIdx.x; j < p.cols; j += blockDim.x) {
      float *d = dx + (u64)j * p.grad_stride;
      *d += grad(x[(u64)j * p.col_stride], j);
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------
struct LpShape {
  u64 rows, cols;
  u64 col_stride;
};

static bool check_row_output(const Tensor *t, u64 n, DTYPE dtype, const char *what) {
  if (!check_typed(t, dtype, what)) return false;
  if (numel(t) != n) {
    set_error(PLAST_B200_ERR_SHAPE, "%s: %llu elements, expected %llu", what, (unsigned long long)numel(t),
              (unsigned long long)n);
    return false;
  }
  if (!is_packed(t)) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: must be contiguous", what);
    return false;
  }
  return true;
}

static bool check_logits(const Tensor *logits, const Tensor *tokens, float temperature, LpShape *s) {
  if (!check_typed(logits, FLOAT32, "token_logprob: logits") || !check_typed(tokens, INT32, "token_logprob: tokens"))
    return false;
  if (logits->ndim < 1) {
    set_error(PLAST_B200_ERR_SHAPE, "token_logprob: logits must have at least one dim");
    return false;
  }
  const u64 lead = logits->ndim - 1;
  bool same = tokens->ndim == lead;
  for (u64 d = 0; same && d < lead; ++d) same = tokens->shape[d] == logits->shape[d];
  if (lead == 0 && numel(tokens) == 1) same = true;
  if (!same) {
    set_error(PLAST_B200_ERR_SHAPE, "token_logprob: tokens must have the logits' shape without the last dim");
    return false;
  }
  // 1 / T has to be a normal fp32 number
  if (!(temperature >= 1e-30f) || !(temperature <= 1e30f)) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "token_logprob: temperature must be in [1e-30, 1e30]");
    return false;
  }
  s->cols = logits->shape[lead];
  s->col_stride = logits->strides[lead];
  s->rows = 1;
  for (u64 d = 0; d < lead; ++d) s->rows *= logits->shape[d];
  if (s->cols == 0) {
    set_error(PLAST_B200_ERR_SHAPE, "token_logprob: no logits to choose from");
    return false;
  }
  if (s->cols >= 0x7ffffff0ull || s->rows >= 0x7fffffffull / kLpMaxCluster) {
    set_error(PLAST_B200_ERR_LIMIT, "token_logprob: more than 2^31 - 16 logits in a row or 2^28 rows");
    return false;
  }
  return true;
}

static bool check_stats(const Tensor *t, u64 rows) {
  if (!check_row_output(t, 2 * rows, FLOAT32, "token_logprob: stats")) return false;
  if ((uintptr_t)t->data & 7) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "token_logprob: stats must be aligned to 8 bytes");
    return false;
  }
  return true;
}

static unsigned lp_threads(u64 cols) { // one trip of the CTA covers threads * 16 logits
  unsigned t = kLpMaxThreads;
  while (t > 64 && (u64)t * 8 >= cols) t /= 2;
  return t;
}

} // namespace pb

using namespace pb;

extern "C" {

void plast_b200_token_logprob(const Tensor *logits, const Tensor *tokens, Tensor *logprob, Tensor *entropy,
                              Tensor *log_norm, Tensor *stats, Tensor *top_logprob, Tensor *top_index,
                              float temperature) {
  begin_call();
  LpShape s;
  if (!check_logits(logits, tokens, temperature, &s)) return;
  if (!check_row_output(logprob, s.rows, FLOAT32, "token_logprob: logprob")) return;
  if (entropy && !check_row_output(entropy, s.rows, FLOAT32, "token_logprob: entropy")) return;
  if (log_norm && !check_row_output(log_norm, s.rows, FLOAT32, "token_logprob: log_norm")) return;
  if (stats && !check_stats(stats, s.rows)) return;
  u64 top = 0;
  if (top_logprob || top_index) {
    if (!top_logprob || !top_index) {
      set_error(PLAST_B200_ERR_NULL, "token_logprob: top_logprob and top_index come together");
      return;
    }
    if (!check_tensor(top_index, "token_logprob: top_index")) return;
    if (top_index->ndim < 1) {
      set_error(PLAST_B200_ERR_SHAPE, "token_logprob: top_index must have a last dim");
      return;
    }
    top = top_index->shape[top_index->ndim - 1];
    if (top > s.cols) {
      set_error(PLAST_B200_ERR_SHAPE, "token_logprob: %llu alternatives of %llu logits", (unsigned long long)top,
                (unsigned long long)s.cols);
      return;
    }
    if (top > PLAST_TOKEN_TOP_MAX) {
      set_error(PLAST_B200_ERR_LIMIT, "token_logprob: more than %d alternatives", PLAST_TOKEN_TOP_MAX);
      return;
    }
    if (!check_row_output(top_logprob, s.rows * top, FLOAT32, "token_logprob: top_logprob") ||
        !check_row_output(top_index, s.rows * top, INT32, "token_logprob: top_index"))
      return;
  }
  if (s.rows == 0) return; // nothing to do

  LpParams p = {};
  p.x = (const float *)logits->data;
  p.token = (const int *)tokens->data;
  p.logprob = (float *)logprob->data;
  p.entropy = entropy ? (float *)entropy->data : nullptr;
  p.log_norm = log_norm ? (float *)log_norm->data : nullptr;
  p.stats = stats ? (float2 *)stats->data : nullptr;
  p.top_logprob = top ? (float *)top_logprob->data : nullptr;
  p.top_index = top ? (int *)top_index->data : nullptr;
  make_row_map(&p.map, logits->shape, logits->ndim - 1, logits->strides, tokens->strides, nullptr);
  p.col_stride = s.col_stride;
  p.cols = (unsigned)s.cols;
  p.top = (int)top;
  p.scale_log2 = (float)(1.4426950408889634 / (double)temperature);
  p.temperature = temperature;
  const unsigned threads = lp_threads(s.cols);
  // few rows: split each over a cluster while every CTA keeps at least one full trip
  p.cluster = 1;
  while (p.cluster < kLpMaxCluster && s.rows * p.cluster < (u64)sm_count() &&
         s.cols / (p.cluster * 2) >= (u64)threads * 4 * kLpUnroll)
    p.cluster *= 2;
  const bool unit = s.col_stride == 1 || s.cols == 1;
  const dim3 grid((unsigned)(s.rows * p.cluster)), block(threads);
  cudaError_t e;
  if (top) e = unit ? launch_kc(p.cluster, token_logprob_kernel<true, true>, grid, block, 0, stream(), p)
                    : launch_kc(p.cluster, token_logprob_kernel<false, true>, grid, block, 0, stream(), p);
  else e = unit ? launch_kc(p.cluster, token_logprob_kernel<true, false>, grid, block, 0, stream(), p)
                : launch_kc(p.cluster, token_logprob_kernel<false, false>, grid, block, 0, stream(), p);
  PB_CUDA(e);
  count_launch();
  note_kernel(top ? "token_logprob_top" : "token_logprob");
  end_call();
}

void plast_b200_token_logprob_backward(Tensor *logits, const Tensor *tokens, const Tensor *stats,
                                       const Tensor *logprob, const Tensor *entropy, const Tensor *log_norm,
                                       float temperature) {
  begin_call();
  LpShape s;
  if (!check_logits(logits, tokens, temperature, &s)) return;
  if (!logits->requires_grad) return; // nothing to do
  if (!check_grad(logits, "token_logprob: logits") || !check_stats(stats, s.rows)) return;
  const Tensor *upstream[3] = {logprob, entropy, log_norm};
  static const char *const names[3] = {"token_logprob: gradient of logprob", "token_logprob: gradient of entropy",
                                       "token_logprob: gradient of log_norm"};
  const float *g[3] = {};
  for (int i = 0; i < 3; ++i) {
    if (!upstream[i] || !upstream[i]->grad) continue;
    if (!check_row_output(upstream[i]->grad, s.rows, FLOAT32, names[i])) return;
    g[i] = (const float *)upstream[i]->grad->data;
  }
  if (g[1] && !check_row_output(entropy, s.rows, FLOAT32, "token_logprob: entropy")) return;
  if (s.rows == 0 || (!g[0] && !g[1] && !g[2])) return; // nothing to do

  LpGradParams p = {};
  const Tensor *dx = logits->grad;
  p.x = (const float *)logits->data;
  p.token = (const int *)tokens->data;
  p.dx = (float *)dx->data;
  p.entropy = g[1] ? (const float *)entropy->data : nullptr;
  p.stats = (const float2 *)stats->data;
  p.g_logprob = g[0];
  p.g_entropy = g[1];
  p.g_log_norm = g[2];
  const u64 lead = logits->ndim - 1;
  make_row_map(&p.map, logits->shape, lead, logits->strides, tokens->strides, dx->strides);
  p.col_stride = s.col_stride;
  p.grad_stride = dx->strides[lead];
  p.cols = (unsigned)s.cols;
  p.inv_t = (float)(1.0 / (double)temperature);
  p.scale_log2 = (float)(1.4426950408889634 / (double)temperature);
  // float4 where logits and gradient share their phase against 16 bytes in every row
  bool vec = (s.col_stride == 1 && p.grad_stride == 1) &&
             (((uintptr_t)p.x ^ (uintptr_t)p.dx) & 15) == 0;
  for (int d = 0; d < p.map.nd && vec; ++d)
    if (p.map.size[d] > 1) vec = ((p.map.stride[0][d] ^ p.map.stride[2][d]) & 3) == 0;
  const dim3 grid((unsigned)s.rows), block(lp_threads(s.cols));
  PB_CUDA(vec ? launch_k(token_logprob_backward_kernel<true>, grid, block, 0, stream(), p)
              : launch_k(token_logprob_backward_kernel<false>, grid, block, 0, stream(), p));
  count_launch();
  note_kernel(vec ? "token_logprob_backward_vec4" : "token_logprob_backward");
  end_call();
}

} // extern "C"
