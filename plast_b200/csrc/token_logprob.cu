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

#include <algorithm>
#include <cooperative_groups.h>
#include <math.h>

namespace pb {

constexpr int kLpMaxThreads = 512;
constexpr int kLpUnroll = 4;      // float4 per thread and trip
constexpr int kLpCandidates = 1024;
constexpr int kLpMaxCluster = 8;  // portable cluster size
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
  double inv_temperature;
};

// 2^t by the special function unit, up to 2^-22 off relative to itself: one instruction per logit in loops that have to keep
// up with HBM. A row's results stay within 1e-7 of 64 bits (4.7e-8 to 9.6e-8 for 1 to 8192 rows of 32768 to 131072, the
// same formulas in elementary fp32 steps 6.5e-8 to 1.7e-7).
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
  // all lanes of a warp, in a tree (every lane ends with the same bits: the merge is symmetric)
  __device__ __forceinline__ void merge_warp(float c, int lanes = 32) {
#pragma unroll 1
    for (int o = lanes / 2; o; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o),
                  ou = __shfl_xor_sync(0xffffffffu, u, o);
      merge(om, os, ou, c);
    }
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
  u64key cand[kLpCandidates]; // a list per warp while the row streams
  u64key last[kLpCandidates]; // what is left of them at the end
  u64key best[PLAST_TOKEN_TOP_MAX];   // of the CTA
  u64key chosen[PLAST_TOKEN_TOP_MAX]; // of the cluster
  u64key join[kLpMaxCluster * PLAST_TOKEN_TOP_MAX];
  float stat[kLpMaxCluster][3];
  float warp_stat[kLpMaxThreads / 32][3];
  volatile float warp_bound[kLpMaxThreads / 32];
  unsigned count;
  double log_s, shift;
  int empty;
};

// The k best of the n distinct keys in `from` (0 = none) go to `to` in order, by counting for each key
// how many are larger. `threads` lanes (a power of two, whole warps) take part, several to a key where
// there are few.
__device__ __forceinline__ void select_best(u64key *to, const u64key *from, unsigned n, int k, unsigned thread, unsigned threads) {
  unsigned share = 1;
  while (share < 32 && n * share * 2 <= threads) share *= 2;
  const unsigned lane = thread & (share - 1), per_trip = threads / share;
  for (unsigned base = 0; base < n; base += per_trip) { // the trip count is uniform
    const unsigned at = base + thread / share;
    const u64key mine = at < n ? from[at] : 0;
    unsigned larger = 0;
    if (mine)
      for (unsigned i = lane; i < n; i += share) larger += from[i] > mine;
    for (unsigned o = share / 2; o; o >>= 1) larger += __shfl_xor_sync(0xffffffffu, larger, o);
    if (mine && lane == 0 && larger < (unsigned)k) to[larger] = mine;
  }
}

// fp32 numbers as unsigned ones in the same order, for the warp-wide integer reductions
__device__ __forceinline__ unsigned ordered(float v) {
  const unsigned b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(unsigned b) {
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}
// The j-th largest of the lanes' values: the largest, j times, without the lanes that had it.
__device__ __forceinline__ float warp_nth(float v, int j) {
  unsigned mine = ordered(v), best = 0;
  for (int i = 0; i < j; ++i) {
    best = __reduce_max_sync(0xffffffffu, mine);
    if ((threadIdx.x & 31) == __ffs(__ballot_sync(0xffffffffu, mine == best)) - 1) mine = 0;
  }
  return unordered(best);
}

// The k-th largest of the lanes' values: a bitonic sort, largest first.
__device__ __forceinline__ float warp_kth(float v, int k) {
  const unsigned lane = threadIdx.x & 31;
#pragma unroll
  for (unsigned size = 2; size <= 32; size *= 2)
#pragma unroll
    for (unsigned o = size / 2; o; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, v, o);
      v = ((lane & o) == 0) == ((lane & size) == 0) ? fmaxf(v, other) : fminf(v, other);
    }
  return __shfl_sync(0xffffffffu, v, k - 1);
}
// A value that at least k distinct logits reach, from the warps' `nth`-th largest lane maxima: where one
// per warp does (nth == 1), the k-th largest of them, else the smallest.
__device__ __forceinline__ float common_bound(const LpShared &sh, int k, int nth) {
  const unsigned lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const float mine = sh.warp_bound[lane < warps ? lane : 0];
  if (nth == 1 && k < (int)warps) {
    int larger = 0;
    for (unsigned w = 0; w < warps; ++w) {
      const float other = __shfl_sync(0xffffffffu, mine, w); // one look at shared memory: others change it
      larger += other > mine || (other == mine && w < lane);
    }
    const unsigned which = __ballot_sync(0xffffffffu, lane < warps && larger == k - 1);
    return __shfl_sync(0xffffffffu, mine, __ffs(which) - 1);
  }
  return unordered(__reduce_min_sync(0xffffffffu, ordered(mine)));
}
// the next fp32 number above (NaN above infinity)
__device__ __forceinline__ float next_above(float v) {
  const int b = __float_as_int(v);
  return __int_as_float(v == 0.0f ? 1 : b > 0 ? b + 1 : b - 1);
}

// Cuts a warp's list of candidates to its k best, in order; returns the last of them, the new threshold.
// k times the warp's largest: a lane looks after every 32nd place and looks again when it has lost one.
__device__ __forceinline__ u64key cut_list(u64key *list, unsigned count, u64key *spare, int k) {
  const unsigned lane = threadIdx.x & 31;
  __syncwarp();
  u64key mine = 0;
  unsigned at = 0;
  auto look = [&] {
    mine = 0;
    for (unsigned i = lane; i < count; i += 32)
      if (list[i] > mine) {
        mine = list[i];
        at = i;
      }
  };
  look();
  u64key best = 0;
  for (int r = 0; r < k; ++r) {
    const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(mine >> 32));
    const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(mine >> 32) == hi ? (unsigned)mine : 0u);
    best = ((u64key)hi << 32) | lo;
    if (mine == best) { // one lane: keys are distinct
      spare[r] = best;
      list[at] = 0;
      look();
    }
    __syncwarp();
  }
  if ((int)lane < k) list[lane] = spare[lane];
  __syncwarp();
  return best;
}

// What is reported of a row besides its alternatives: the last few operations in 64 bits, each result
// rounded once. `log_s` and `shift`: log p of a logit x is (x - shift) / T - log_s, which keeps its
// digits where the log normaliser has none.
__device__ __forceinline__ void report_row(const LpParams &p, unsigned row, const LpStat &st, int token, float x_token, double &log_s,
                                           double &shift, int &empty) {
  empty = st.s == 0.0f; // every logit is -inf
  log_s = log((double)st.s);
  shift = (double)st.m;
  const double L = empty ? -INFINITY : shift * p.inv_temperature + log_s;
  double h = empty ? 0.0 : log_s - kLn2 * ((double)st.u / (double)st.s);
  if (h < 0.0) h = 0.0; // rounding of U; a NaN passes
  double lp = 0.0;
  if (token >= 0) lp = empty ? -INFINITY : ((double)x_token - shift) * p.inv_temperature - log_s;
  p.logprob[row] = (float)lp;
  if (p.entropy) p.entropy[row] = (float)h;
  if (p.log_norm) p.log_norm[row] = (float)L;
  if (p.stats) p.stats[row] = make_float2(st.m, st.s);
}
__device__ __forceinline__ void report_alternative(const LpParams &p, unsigned row, int i, u64key key, double log_s, double shift, int empty) {
  const u64 at = (u64)row * p.top + i;
  p.top_index[at] = key ? (int)index_of(key) : -1;
  p.top_logprob[at] = !key ? NAN : empty ? -INFINITY : (float)(((double)value_of(key) - shift) * p.inv_temperature - log_s);
}

// A row (or slice) as vectors of four logits; the first one starts at the 16-byte boundary at or before it.
template <bool UNIT> struct LpRow {
  const float *x;
  u64 stride;
  unsigned cols, lead, vectors;
  __device__ __forceinline__ LpRow(const float *x, const LpParams &p) : x(x), stride(p.col_stride), cols(p.cols) {
    lead = UNIT ? (unsigned)(((uintptr_t)x >> 2) & 3) : 0u;
    vectors = (unsigned)(((u64)cols + lead + 3) >> 2);
  }
  __device__ __forceinline__ long long index(unsigned at) const { return (long long)at * 4 - lead; } // of its first lane
  // four logits of vector `at`, -inf where there are none
  __device__ __forceinline__ void fetch(unsigned at, unsigned last, float *v) const {
    const long long j = index(at);
    if (at < last && j >= 0 && j + 4 <= (long long)cols) {
      if (UNIT) {
        const float4 q = __ldcs(reinterpret_cast<const float4 *>(x + j));
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = x[(u64)(j + i) * stride];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = (at < last && j + i >= 0 && j + i < (long long)cols) ? x[(u64)(j + i) * stride] : -INFINITY;
    }
  }
};

// ---- forward, few rows --------------------------------------------------------------------------------
// One cluster of CTAs per row (1 where the rows fill the GPU; up to 8 where there are few rows, whose
// slices are joined through distributed shared memory). A trip moves 16 logits per thread.
//
// Alternatives: logits that can still be among the k best go to a list that each warp keeps for itself,
// without a barrier in the stream. What is wanted follows from the largest logit that every lane has
// seen: j = ceil(k / warps) lanes of each warp hold at least k distinct logits, so the smallest of the
// warps' j-th largest lane maxima is below the k-th best (a value that another warp has raised since is
// only better). About 3 k logits of a random row pass. A list that is full is cut to its k best, so any
// order and any number of ties ends with the exact answer.
template <bool UNIT, bool TOP>
__global__ void __launch_bounds__(kLpMaxThreads, 2) token_logprob_kernel(const __grid_constant__ LpParams p) {
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
  // thread 0 of the row's first CTA reports; of its two dependent loads the second starts with the stream
  const bool reports = rank == 0 && threadIdx.x == 0;
  int token = reports ? p.token[off[1]] : -1;
  float x_token = 0.0f;
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  // the warp's candidates: `room` places of the shared list; keys above `threshold` are wanted
  const unsigned room = kLpCandidates / warps;
  u64key *const list = sh.cand + warp * room;
  unsigned count = 0;
  u64key threshold = 0;
  const int nth = TOP ? (k + (int)warps - 1) / (int)warps : 1;
  float seen = -INFINITY; // the lane's largest logit so far
  if (TOP) {
    if (lane == 0) sh.warp_bound[warp] = -INFINITY;
    if (threadIdx.x == 0) sh.count = 0;
    // places that a selection does not fill stay 0 (a key is never 0)
    if (threadIdx.x < PLAST_TOKEN_TOP_MAX) sh.best[threadIdx.x] = sh.chosen[threadIdx.x] = 0;
    __syncthreads();
  }
  const LpRow<UNIT> r(x, p);
  const unsigned lead = r.lead, vectors = r.vectors;
  const unsigned slice = (vectors + p.cluster - 1) / p.cluster;
  const unsigned first = rank * slice < vectors ? rank * slice : vectors;
  const unsigned last = vectors - first < slice ? vectors : first + slice;
  const unsigned trip = blockDim.x * kLpUnroll;

  LpStat st;
  st.init();
  float bound = -INFINITY;
  for (unsigned base = first; base < last; base += trip) {
    float v[kLpUnroll * 4];
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) r.fetch(base + u * blockDim.x + threadIdx.x, last, v + 4 * u);
    if (reports && base == first) {
      if (token >= 0 && (unsigned)token < p.cols) x_token = x[(u64)token * p.col_stride];
      else token = -1;
    }
    float top = v[0];
#pragma unroll
    for (int i = 1; i < kLpUnroll * 4; ++i) top = fmaxf(top, v[i]);
    if (top > st.m) st.raise(top, c);
#pragma unroll
    for (int i = 0; i < kLpUnroll * 4; ++i) st.add(v[i], c);

    if (TOP) {
      seen = fmaxf(seen, top); // drops a NaN
      // a logit that equals the last of a cut list comes after it (the stream's indices grow)
      const float least = threshold ? max_nan(bound, next_above(value_of(threshold))) : bound;
      unsigned todo = 0;
      if (base == first || __any_sync(0xffffffffu, top >= least)) {
        const float nth_seen = warp_nth(seen, nth);
        if (lane == 0) sh.warp_bound[warp] = nth_seen;
        if (base == first) __syncthreads(); // once: every warp has a first bound (all have the same trips)
        bound = fmaxf(bound, common_bound(sh, k, nth));
        const float wanted = max_nan(least, bound);
        if (top >= wanted) {
#pragma unroll
          for (int i = 0; i < kLpUnroll * 4; ++i) todo |= (v[i] >= wanted ? 1u : 0u) << i;
        }
      }
      while (__any_sync(0xffffffffu, todo != 0)) { // few
        u64key key = 0;
        if (todo) {
          const unsigned i = __ffs(todo) - 1;
          todo &= todo - 1;
          float mine = v[0];
#pragma unroll
          for (int n = 1; n < kLpUnroll * 4; ++n) mine = i == n ? v[n] : mine;
          const unsigned at = base + (i / 4) * blockDim.x + threadIdx.x;
          const long long j = (long long)at * 4 - lead + (i & 3);
          if (at < last && j >= 0 && j < (long long)p.cols) key = key_of(mine, (unsigned)j);
          if (key <= threshold) key = 0;
        }
        const unsigned with = __ballot_sync(0xffffffffu, key != 0), n = __popc(with);
        if (count + n > room) { // after the cut there is room for 32: room >= 64 >= k + 32
          threshold = cut_list(list, count, sh.last + warp * room, k);
          count = k;
        }
        if (key) list[count + __popc(with & ((1u << lane) - 1))] = key;
        count += n;
      }
    }
  }

  // ---- the CTA's statistics
  st.merge_warp(c);
  const float warp_low = TOP ? warp_nth(seen, nth) : 0.0f;
  if (lane == 0) {
    if (TOP) sh.warp_bound[warp] = warp_low;
    sh.warp_stat[warp][0] = st.m;
    sh.warp_stat[warp][1] = st.s;
    sh.warp_stat[warp][2] = st.u;
  }
  __syncthreads();
  if (TOP) { // what the final bound leaves of the lists
    const float low = common_bound(sh, k, nth);
    const u64key floor_key = (key_of(low, 0) >> 32) << 32; // larger keys have at least this value
    for (unsigned i = lane; i < count; i += 32) {
      const u64key key = list[i];
      if (key > floor_key) sh.last[atomicAdd(&sh.count, 1u)] = key;
    }
    __syncthreads();
  }

  // ---- the row's results: the upper half of the CTA selects while thread 0 does the scalars
  const unsigned upper = blockDim.x / 2;
  if (TOP && threadIdx.x >= upper) select_best(sh.best, sh.last, sh.count, k, threadIdx.x - upper, upper);
  if (warp == 0) {
    st.init();
    if (lane < warps) { st.m = sh.warp_stat[lane][0]; st.s = sh.warp_stat[lane][1]; st.u = sh.warp_stat[lane][2]; }
    st.merge_warp(c);
    if (p.cluster == 1 && threadIdx.x == 0) report_row(p, row, st, token, x_token, sh.log_s, sh.shift, sh.empty);
  }
  if (TOP) __syncthreads();
  const u64key *chosen = sh.best;
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
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0) return;
    if (TOP && threadIdx.x >= upper) select_best(sh.chosen, sh.join, p.cluster * k, k, threadIdx.x - upper, upper);
    if (warp == 0) {
      st.init();
      if (lane < p.cluster) { st.m = sh.stat[lane][0]; st.s = sh.stat[lane][1]; st.u = sh.stat[lane][2]; }
      st.merge_warp(c);
      if (threadIdx.x == 0) report_row(p, row, st, token, x_token, sh.log_s, sh.shift, sh.empty);
    }
    if (TOP) __syncthreads();
    chosen = sh.chosen;
  }
  if (TOP && (int)threadIdx.x < k) report_alternative(p, row, threadIdx.x, chosen[threadIdx.x], sh.log_s, sh.shift, sh.empty);
}

// ---- forward, many rows -------------------------------------------------------------------------------
// A persistent CTA whose eight warps stream one row after the other while a ninth finishes the row before.
// The end of a row is a chain of short steps (joining statistics, alternatives, logarithms) of 3 us, with
// alternatives 6 to 7 beside the stream; in the streaming warps it leaves HBM idle for as long. Measured: 8192
// rows of 65536 in 318 to 330 us without alternatives (6.5 to 6.8 TB/s) and 360 with sixteen, 2048 rows of 32768 in
// 48 and 57 (the last row's end among them). With short rows the finishing warp is the bound, hence the rule at the launch.
//
// The stream notes the largest logit of every thread and piece (one or more trips). A lane of the finishing
// warp looks after eight threads; the k-th largest of the lanes' largest notes (above 16: of the largest
// notes of the lanes' halves) is a bound, since k distinct logits reach it. The pieces whose note reaches it
// are fetched again and the k best of what reaches it are kept: some 1.5 k logits of a random row. A list
// that gets long is cut to its k best, whose last is a threshold from then on, so any order and any number
// of ties ends with the exact answer.
constexpr int kLpRowCtas = 4, kLpStream = 256, kLpRowThreads = kLpStream + 32, kLpPieces = 16, kLpHits = 256;
struct LpRowShared {
  float note[2][kLpPieces * kLpStream], whole[2][kLpStream];
  float stat[2][kLpStream / 32][3];
  unsigned trips[2];
  u64key list[kLpCandidates], spare[PLAST_TOKEN_TOP_MAX];
  unsigned short hits[kLpHits];
  unsigned char reach[kLpStream];
};
// named barriers: a row's notes are there / may be overwritten (two buffers)
__device__ __forceinline__ void rows_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kLpRowThreads) : "memory"); }
__device__ __forceinline__ void rows_arrive(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kLpRowThreads) : "memory"); }

template <bool UNIT, bool TOP>
__global__ void __launch_bounds__(kLpRowThreads, kLpRowCtas) token_logprob_rows_kernel(const __grid_constant__ LpParams p, unsigned rows) {
  __shared__ LpRowShared sh;
  pdl_wait();
  pdl_launch_dependents();
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float c = p.scale_log2;
  constexpr unsigned kTrip = kLpStream * kLpUnroll;
  // the same for every row but for its lead, which adds at most one vector
  const unsigned most_trips = (unsigned)((((u64)p.cols + 6) / 4 + kTrip - 1) / kTrip);
  unsigned piece_log = 0;
  while (((most_trips + (1u << piece_log) - 1) >> piece_log) > kLpPieces) ++piece_log;
  unsigned turn = 0;

  if (warp < kLpStream / 32) { // ---- stream
    for (unsigned row = blockIdx.x; row < rows; row += gridDim.x, ++turn) {
      const unsigned buf = turn & 1;
      u64 off[3];
      row_offsets(p.map, row, off);
      const LpRow<UNIT> r(p.x + off[0], p);
      LpStat st;
      st.init();
      if (turn >= 2) rows_sync(3 + buf);
      float note = -INFINITY, whole = -INFINITY;
      unsigned trips = 0;
      for (unsigned base = 0; base < r.vectors; base += kTrip) {
        float v[kLpUnroll * 4];
#pragma unroll
        for (int u = 0; u < kLpUnroll; ++u) r.fetch(base + u * kLpStream + threadIdx.x, r.vectors, v + 4 * u);
        float top = v[0];
#pragma unroll
        for (int i = 1; i < kLpUnroll * 4; ++i) top = fmaxf(top, v[i]);
        if (top > st.m) st.raise(top, c);
#pragma unroll
        for (int i = 0; i < kLpUnroll * 4; ++i) st.add(v[i], c);
        if (TOP) {
          note = fmaxf(note, top); // drops a NaN
          ++trips;
          if ((trips & ((1u << piece_log) - 1)) == 0 || base + kTrip >= r.vectors) {
            sh.note[buf][((trips - 1) >> piece_log) * kLpStream + threadIdx.x] = note;
            whole = fmaxf(whole, note);
            note = -INFINITY;
          }
        }
      }
      if (TOP) sh.whole[buf][threadIdx.x] = whole;
      st.merge_warp(c);
      if (lane == 0) {
        sh.stat[buf][warp][0] = st.m;
        sh.stat[buf][warp][1] = st.s;
        sh.stat[buf][warp][2] = st.u;
      }
      if (TOP && threadIdx.x == 0) sh.trips[buf] = trips;
      rows_arrive(1 + buf);
    }
    return;
  }

  // ---- finish
  const int k = p.top;
  for (unsigned row = blockIdx.x; row < rows; row += gridDim.x, ++turn) {
    const unsigned buf = turn & 1;
    u64 off[3];
    row_offsets(p.map, row, off);
    const LpRow<UNIT> r(p.x + off[0], p);
    int token = p.token[off[1]];
    float x_token = 0.0f;
    if (token >= 0 && (unsigned)token < p.cols) x_token = r.x[(u64)token * p.col_stride];
    else token = -1;
    rows_sync(1 + buf);
    LpStat st;
    st.init();
    if (lane < kLpStream / 32) { st.m = sh.stat[buf][lane][0]; st.s = sh.stat[buf][lane][1]; st.u = sh.stat[buf][lane][2]; }
    st.merge_warp(c, kLpStream / 32);
    unsigned count = 0;
    bool used_up = false; // the notes
    if (TOP) {
      const unsigned trips = sh.trips[buf], here = (trips + (1u << piece_log) - 1) >> piece_log;
      const float *note = sh.note[buf];
      // A lane looks after eight threads; the k-th largest of the lanes' largest logits is the bound.
      // (of more than 16: of the lanes' two halves)
      float top[kLpStream / 32];
#pragma unroll
      for (int i = 0; i < kLpStream / 32; ++i) top[i] = sh.whole[buf][i * 32 + lane];
      float low = top[0], high = top[kLpStream / 64];
#pragma unroll
      for (int i = 1; i < kLpStream / 64; ++i) {
        low = fmaxf(low, top[i]);
        high = fmaxf(high, top[kLpStream / 64 + i]);
      }
      float bound;
      if (k <= 4) bound = warp_nth(fmaxf(low, high), k);
      else if (k <= 16) bound = warp_kth(fmaxf(low, high), k);
      else { // the largest of 64, k times, each time without the one that had it
        unsigned a = ordered(fmaxf(low, high)), b = ordered(fminf(low, high)), best = 0;
        for (int n = 0; n < k; ++n) {
          best = __reduce_max_sync(0xffffffffu, a);
          if (lane == __ffs(__ballot_sync(0xffffffffu, a == best)) - 1u) {
            a = b;
            b = 0;
          }
        }
        bound = unordered(best);
      }
      u64key threshold = 0; // larger keys are wanted
      unsigned hits = 0;
      // the pieces behind the first `hits` notes of the list, one per lane
      auto look_again = [&] {
        __syncwarp();
        for (unsigned h0 = 0; h0 < hits; h0 += 32) {
          const bool mine = h0 + lane < hits;
          const unsigned hit = mine ? sh.hits[h0 + lane] : 0, thread = hit % kLpStream, piece = hit / kLpStream;
          for (unsigned t = piece << piece_log, n = 0; n < (1u << piece_log); ++n, ++t) {
            const unsigned at0 = t * kTrip + thread;
            float v[kLpUnroll * 4];
            unsigned todo = 0;
#pragma unroll
            for (int u = 0; u < kLpUnroll; ++u) {
              v[4 * u] = v[4 * u + 1] = v[4 * u + 2] = v[4 * u + 3] = -INFINITY;
              if (mine) r.fetch(at0 + u * kLpStream, r.vectors, v + 4 * u);
            }
            if (mine) {
#pragma unroll
              for (int i = 0; i < kLpUnroll * 4; ++i) todo |= (v[i] >= bound ? 1u : 0u) << i;
              if (threshold) { // of many equal logits only those before the last of the list are wanted
                const float least = value_of(threshold);
                const long long before = index_of(threshold), j0 = r.index(at0);
#pragma unroll
                for (int i = 0; i < kLpUnroll * 4; ++i)
                  if (v[i] < least || (v[i] == least && j0 + (i / 4) * (4 * kLpStream) + (i & 3) >= before)) todo &= ~(1u << i);
              }
            }
            while (__any_sync(0xffffffffu, todo != 0)) {
              u64key key = 0;
              if (todo) {
                const unsigned i = __ffs(todo) - 1;
                todo &= todo - 1;
                float value = v[0];
#pragma unroll
                for (int m = 1; m < kLpUnroll * 4; ++m) value = i == m ? v[m] : value;
                const unsigned at = at0 + (i / 4) * kLpStream;
                const long long j = r.index(at) + (i & 3);
                if (at < r.vectors && j >= 0 && j < (long long)p.cols) key = key_of(value, (unsigned)j);
                if (key <= threshold) key = 0;
              }
              const unsigned with = __ballot_sync(0xffffffffu, key != 0), n_with = __popc(with);
              if (count + n_with > kLpCandidates) {
                threshold = cut_list(sh.list, count, sh.spare, k);
                count = k;
              }
              if (key) sh.list[count + __popc(with & ((1u << lane) - 1))] = key;
              count += n_with;
            }
          }
          if (count > 128) { // many equal logits: most of the rest need not be looked at
            threshold = cut_list(sh.list, count, sh.spare, k);
            count = k;
          }
        }
        hits = 0;
        __syncwarp();
      };
      // the threads that reach it, then their pieces that do
      unsigned threads = 0;
#pragma unroll
      for (int i = 0; i < kLpStream / 32; ++i) {
        const unsigned with = __ballot_sync(0xffffffffu, top[i] >= bound);
        if (top[i] >= bound) sh.reach[threads + __popc(with & ((1u << lane) - 1))] = (unsigned char)(i * 32 + lane);
        threads += __popc(with);
      }
      __syncwarp();
      // Ties: where the k-th best is as large as the best, the first k logits of that value are the answer, in an
      // empty row the first k of all. They are looked for at the start of the row.
      bool found = false;
      if (threads > 32 && __all_sync(0xffffffffu, fmaxf(low, high) <= bound)) {
        float v[16];
#pragma unroll
        for (unsigned i = 0; i < 16; ++i) v[i] = i * 32 + lane < p.cols ? r.x[(u64)(i * 32 + lane) * r.stride] : NAN;
#pragma unroll
        for (unsigned i = 0; i < 16; ++i) {
          const unsigned with = __ballot_sync(0xffffffffu, v[i] == bound), at = count + __popc(with & ((1u << lane) - 1));
          if (v[i] == bound && at < (unsigned)k) sh.spare[at] = key_of(v[i], i * 32 + lane);
          count += __popc(with);
        }
        found = count >= (unsigned)k;
        count = found ? k : 0;
      }
      if (!found) {
        // a thread per lane (two where k is large), its pieces as bits
        bool listed = threads <= 64;
        for (unsigned i = 0; listed && i < threads; i += 32) {
          const unsigned thread = i + lane < threads ? sh.reach[i + lane] : 0;
          unsigned pieces = 0;
          if (i + lane < threads) {
#pragma unroll
            for (unsigned piece = 0; piece < (unsigned)kLpPieces; ++piece)
              if (piece < here && note[piece * kLpStream + thread] >= bound) pieces |= 1u << piece;
          }
          unsigned at = __popc(pieces);
#pragma unroll
          for (int o = 1; o < 32; o *= 2) {
            const unsigned before = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= (unsigned)o) at += before;
          }
          const unsigned more = __shfl_sync(0xffffffffu, at, 31);
          listed = hits + more <= (unsigned)kLpHits;
          if (!listed) break;
          at += hits - __popc(pieces);
          for (; pieces; pieces &= pieces - 1)
            sh.hits[at++] = (unsigned short)((__ffs(pieces) - 1) * kLpStream + thread);
          hits += more;
        }
        if (listed) {
          used_up = true;
          __syncwarp();
          rows_arrive(3 + buf);
        } else hits = 0;
        if (!listed)
          for (unsigned piece = 0; piece < here; ++piece) {
            // a logit that equals the last of a cut list comes after it: pieces follow the row
            const float least = threshold ? max_nan(bound, next_above(value_of(threshold))) : bound;
            for (unsigned i = 0; i < threads; i += 32) {
              const unsigned thread = i + lane < threads ? sh.reach[i + lane] : 0;
              const bool hit = i + lane < threads && note[piece * kLpStream + thread] >= least;
              const unsigned with = __ballot_sync(0xffffffffu, hit);
              if (!with) continue;
              if (hit) sh.hits[hits + __popc(with & ((1u << lane) - 1))] = (unsigned short)(piece * kLpStream + thread);
              hits += __popc(with);
              if (hits > kLpHits - 32) look_again();
            }
            if (hits > 96) look_again();
          }
        look_again();
        if (count > 96) cut_list(sh.list, count, sh.spare, k);
        else {
          sh.spare[lane] = 0;
          __syncwarp();
          select_best(sh.spare, sh.list, count, k, lane, 32);
        }
      }
      __syncwarp();
    }
    if (!used_up) rows_arrive(3 + buf);
    double log_s, shift;
    int empty;
    if (lane == 0) report_row(p, row, st, token, x_token, log_s, shift, empty);
    if (TOP) {
      log_s = __shfl_sync(0xffffffffu, log_s, 0);
      shift = __shfl_sync(0xffffffffu, shift, 0);
      empty = __shfl_sync(0xffffffffu, empty, 0);
      if ((int)lane < k) report_alternative(p, row, lane, sh.spare[lane], log_s, shift, empty);
      __syncwarp();
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
  unsigned cols, piece; // piece: vectors of four (or logits) per CTA
  float scale_log2, inv_t;
};

// A streaming pass: 4 B read and 8 B for the += per logit. A CTA takes a piece of one row (grid.y), so that a
// thousand long rows end together: whole rows of 50001 run in 3.4 turns of the GPU.
template <bool VEC>
__global__ void __launch_bounds__(256) token_logprob_backward_kernel(const __grid_constant__ LpGradParams p) {
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
    const unsigned begin = blockIdx.y * p.piece, end = vectors - begin < p.piece ? vectors : begin + p.piece;
    if (begin >= vectors) return; // the row's lead made one piece fewer
    for (unsigned at0 = begin + threadIdx.x; at0 < end; at0 += blockDim.x * 2) {
      float4 q[2], d[2];
      bool full[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned at = at0 + u * blockDim.x;
        const long long j = (long long)at * 4 - lead;
        full[u] = at < end && j >= 0 && j + 4 <= (long long)p.cols;
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
        } else if (at < end) {
          for (int i = 0; i < 4; ++i)
            if (j + i >= 0 && j + i < (long long)p.cols) dx[j + i] += grad(x[j + i], (unsigned)(j + i));
        }
      }
    }
  } else {
    const unsigned begin = blockIdx.y * p.piece, end = p.cols - begin < p.piece ? p.cols : begin + p.piece;
    for (unsigned j = begin + threadIdx.x; j < end; j += blockDim.x) {
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

// Whether the kernel for many rows serves. Against the other one, measured in us with 0 / 1 / 16 / 32 alternatives:
//   rows for every resident CTA, four to an SM: where a row's stream covers the end of the row before
//     2048 rows of 32768: 48 / 54 / 56 / 77  (49 / 61 / 80 / 93)
//     4096 rows of 16384: 46 / 58 / 67 / 106 (52 / 74 / 97 / 112)
//     4096 rows of 8192:  27 / 47 / 56 / 93  (32 / 53 / 65 / 77)
//     4096 rows of 4096:  19 / 41 / 49 / 85  (23 / 42 / 47 / 57)
//     4096 rows of 2048:  21 / 42 / 49 / 83  (12 / 21 / 26 / 36)
// Fewer rows, measured in captured graphs over inputs larger than L2, as the other one's time over this one's with
// 1 / 9 / 16 / 17 / 20 / 24 / 32 alternatives (0 / 1 / 16 / 20 / 32 from 300 rows on):
//   more rows than the other one has resident CTAs, two to an SM: always
//     590 rows of 8192: 1.40 / 1.52 / 1.51 / 1.83 / 1.31, of 65536 (60000 up to 16): 1.15 / 1.23 / 1.61 / 1.51 / 1.39
//     300 rows of 8192: 1.23 / 1.31 / 1.20 / 1.30 / 0.94, of 65536 (60000 up to 16): 1.13 / 1.16 / 1.36 / 1.42 / 1.20
//   more than one to an SM: for 9 to 24 alternatives, whose selection a CTA of the other one does after its stream
//     200 rows of 8192:   -   / 1.00 / 1.06 / 1.38 / 1.29 / 1.02 / 0.88
//     200 rows of 32768: 0.91 / 1.07 / 1.10 / 1.27 / 1.23 / 1.09 / 0.97
//     200 rows of 65536: 0.81 / 0.98 / 1.02 / 1.20 / 1.17 /  -   /  -
//   up to one to an SM, where the other one shares a row among up to eight CTAs: for 17 to 22 alternatives (two of each of
//   its sixteen warps' lanes have to be in its bound) and rows that are not long
//     148 rows of 8192:   -   / 0.83 / 0.98 / 1.30 / 1.21 / 0.96 / 0.81, of 32768: 0.82 / 0.90 / 0.96 / 1.14 / 1.08 / 1.01 / 0.86
//     24 rows of 8192:    -   / 0.86 / 0.92 / 1.12 / 1.02 / 0.83 / 0.70, of 32768:  -   / 0.60 / 0.71 / 0.95 / 0.92 / 0.82 / 0.76
//     1 row of 8192 / 16384 / 40960 with 17: 0.91 / 0.97 / 0.92, with 32: 0.56 / 0.67 / 0.72
static bool rows_kernel_serves(u64 rows, u64 cols, u64 top) {
  const u64 sms = (u64)sm_count();
  if (rows >= sms * kLpRowCtas) return cols >= (top == 0 ? 4096 : top <= 16 ? 8192 : 16384);
  if (cols < 8192) return false;
  if (rows > sms * 2) return true;
  if (rows > sms) return top >= 9 && top <= 24 && cols <= 65536;
  return top >= 17 && top <= 22 && rows >= 8 && cols <= (rows >= sms / 2 ? 32768 : 24576);
}

static unsigned lp_threads(u64 cols, unsigned most) { // one trip of the CTA covers threads * 16 logits
  unsigned t = most;
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
  // rows are read while others are written
  const Extent all[8] = {extent_of(logits), extent_of(tokens), extent_of(logprob), extent_of(entropy), extent_of(log_norm), extent_of(stats),
                         extent_of(top ? top_logprob : nullptr), extent_of(top ? top_index : nullptr)};
  for (int i = 2; i < 8; ++i)
    if (!check_apart("token_logprob", "an output", all[i], Extent{}, all, i)) return;

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
  p.inv_temperature = 1.0 / (double)temperature;
  const u64 resident = (u64)sm_count() * kLpRowCtas;
  const bool by_rows = rows_kernel_serves(s.rows, s.cols, top);
  // The other one: with rows for all resident CTAs smaller ones, so that the ends of some rows overlap the
  // streams of others (4096 rows of 16384, 16 alternatives: 132 us with 512 threads, 98 with 256)
  const unsigned threads = lp_threads(s.cols, s.rows >= resident ? 256 : kLpMaxThreads);
  // few rows: split each over a cluster while every CTA keeps at least one full trip
  p.cluster = 1;
  while (p.cluster < kLpMaxCluster && s.rows * p.cluster < (u64)sm_count() &&
         s.cols / (p.cluster * 2) >= (u64)threads * 4 * kLpUnroll)
    p.cluster *= 2;
  const bool unit = s.col_stride == 1 || s.cols == 1;
  if (by_rows) {
    const dim3 row_grid((unsigned)std::min(s.rows, resident));
    const unsigned rows = (unsigned)s.rows;
    PB_CUDA(top ? (unit ? launch_k(token_logprob_rows_kernel<true, true>, row_grid, dim3(kLpRowThreads), 0, stream(), p, rows)
                        : launch_k(token_logprob_rows_kernel<false, true>, row_grid, dim3(kLpRowThreads), 0, stream(), p, rows))
                : (unit ? launch_k(token_logprob_rows_kernel<true, false>, row_grid, dim3(kLpRowThreads), 0, stream(), p, rows)
                        : launch_k(token_logprob_rows_kernel<false, false>, row_grid, dim3(kLpRowThreads), 0, stream(), p, rows)));
    count_launch();
    note_kernel(top ? "token_logprob_rows_top" : "token_logprob_rows");
    return end_call();
  }
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

  const Tensor *dx = logits->grad;
  const Extent others[6] = {extent_of(tokens), extent_of(stats), extent_of(g[0] ? logprob->grad : nullptr), extent_of(g[1] ? entropy->grad : nullptr),
                            extent_of(g[1] ? entropy : nullptr), extent_of(g[2] ? log_norm->grad : nullptr)};
  if (!check_apart("token_logprob", "the gradient of the logits", extent_of(dx), extent_of(logits), others, 6)) return;
  LpGradParams p = {};
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
  // Pieces of at least 8192 logits (16384 where that leaves 16 turns of the GPU and more), at most 65535 of them; a
  // row may start up to three before its first vector. 1021 rows of 50001: 98 us (100 with 16384, 102 with 16384
  // and 512 threads), 8192 of 65536: 953 us (965 with 8192, 975), 4000 of 8000: 60 us (63 with 512 threads).
  const unsigned items = vec ? (unsigned)((s.cols + 3 + 3) / 4) : (unsigned)s.cols;
  const bool many = s.rows * (items / 4096) >= (u64)sm_count() * 4 * 16;
  p.piece = std::max(!vec ? 16384u : many ? 4096u : 2048u, items / 65535 + 1);
  const dim3 grid((unsigned)s.rows, (items + p.piece - 1) / p.piece), block(lp_threads(s.cols, 256));
  PB_CUDA(vec ? launch_k(token_logprob_backward_kernel<true>, grid, block, 0, stream(), p)
              : launch_k(token_logprob_backward_kernel<false>, grid, block, 0, stream(), p));
  count_launch();
  note_kernel(vec ? "token_logprob_backward_vec4" : "token_logprob_backward");
  end_call();
}

} // extern "C"
