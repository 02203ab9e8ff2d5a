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
  float *x[2], *a, *b;
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

// X = u / (|u| + eps), turned so that it has at most as many rows as columns
__global__ void __launch_bounds__(kMuonThreads) muon_load_kernel(const __grid_constant__ MuonTable t) {
  pdl_wait();
  pdl_launch_dependents();
  const MuonMat &q = t.mat[matrix_of(t, blockIdx.x)];
  __shared__ float tile[32][33];
  const float norm = (float)sqrt(q.partial[0]) + t.epsilon;
  const unsigned per_row = (q.cols + 31) / 32, at = blockIdx.x - q.first;
  const unsigned r0 = at / per_row * 32, c0 = at % per_row * 32;
  const unsigned tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (unsigned i = ty; i < 32; i += 8) {
    const unsigned r = r0 + i, c = c0 + tx;
    float u = 0.0f;
    if (r < q.rows && c < q.cols) {
      const u64 j = (u64)r * q.cols + c;
      u = q.g[j];
      if (q.v) u = update_of(t, u, q.v[j]);
      u = u / norm;
      if (q.rows <= q.cols) q.x[0][j] = u;
    }
    tile[i][tx] = u;
  }
  if (q.rows <= q.cols) return;
  __syncthreads();
  for (unsigned i = ty; i < 32; i += 8) {
    const unsigned r = r0 + tx, c = c0 + i;
    if (r < q.rows && c < q.cols) q.x[0][(u64)c * q.rows + r] = tile[tx][i];
  }
}

// One 64 x 64 tile of a product, 4 x 4 per thread.
enum MuonProduct { kGram = 0, kPolynomial = 1, kApply = 2 };
template <int WHAT>
__global__ void __launch_bounds__(kMuonThreads) muon_product_kernel(const __grid_constant__ MuonTable t, int from, int last) {
  pdl_wait();
  pdl_launch_dependents();
  const MuonMat &q = t.mat[matrix_of(t, blockIdx.x)];
  const float *x = q.x[from];
  const float *p = WHAT == kGram ? x : WHAT == kPolynomial ? q.a : q.b;      // left operand, rows of length k
  const float *r = WHAT == kApply ? x : p;                                    // right operand
  const unsigned k = WHAT == kGram ? q.n : q.m, width = WHAT == kApply ? q.n : q.m;
  const unsigned tiles = (width + 63) / 64, at = blockIdx.x - q.first;
  const unsigned i0 = at / tiles * 64, j0 = at % tiles * 64;
  __shared__ float sp[16][65], sr[16][65];
  float acc[4][4] = {};
  const unsigned tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (unsigned k0 = 0; k0 < k; k0 += 16) {
    for (unsigned e = threadIdx.x; e < 64 * 16; e += kMuonThreads) {
      const unsigned kk = e & 15, i = e >> 4;
      sp[kk][i] = i0 + i < q.m && k0 + kk < k ? p[(u64)(i0 + i) * k + k0 + kk] : 0.0f;
      if (WHAT != kApply) sr[kk][i] = j0 + i < q.m && k0 + kk < k ? r[(u64)(j0 + i) * k + k0 + kk] : 0.0f;
      else {
        const unsigned j = e & 63, kr = e >> 6;
        sr[kr][j] = j0 + j < q.n && k0 + kr < k ? r[(u64)(k0 + kr) * q.n + j0 + j] : 0.0f;
      }
    }
    __syncthreads();
    for (int kk = 0; kk < 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(sp[kk][ty * 4 + i], sr[kk][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned row = i0 + ty * 4 + i, col = j0 + tx * 4 + j;
      if (row >= q.m || col >= width) continue;
      const u64 at_ij = (u64)row * width + col;
      if (WHAT == kGram) q.a[at_ij] = acc[i][j];
      if (WHAT == kPolynomial) q.b[at_ij] = __fmaf_rn(kNsB, q.a[at_ij], kNsC * acc[i][j]);
      if (WHAT == kApply) {
        const float v = __fmaf_rn(kNsA, x[at_ij], acc[i][j]);
        if (!last) q.x[from ^ 1][at_ij] = v;
        else {
          float *w = q.w + (q.rows <= q.cols ? at_ij : (u64)col * q.m + row);
          *w = q.keep == 0.0f ? -q.rate * v : __fmaf_rn(-q.rate, v, q.keep * *w);
        }
      }
    }
}

// steps == 0: X itself
__global__ void __launch_bounds__(kMuonThreads) muon_store_kernel(const __grid_constant__ MuonTable t, int from) {
  pdl_wait();
  pdl_launch_dependents();
  const MuonMat &q = t.mat[matrix_of(t, blockIdx.x)];
  const u64 total = (u64)q.rows * q.cols, begin = (u64)(blockIdx.x - q.first) * kMuonChunk;
  for (u64 j = begin + threadIdx.x; j < begin + kMuonChunk && j < total; j += kMuonThreads) {
    const u64 r = j / q.cols, c = j - r * q.cols;
    const float v = q.x[from][q.rows <= q.cols ? j : c * q.rows + r];
    q.w[j] = q.keep == 0.0f ? -q.rate * v : __fmaf_rn(-q.rate, v, q.keep * q.w[j]);
  }
}

// ---- host --------------------------------------------------------------------------------------------
static u64 padded(u64 bytes) { return (bytes + 255) & ~(u64)255; }
static u64 scratch_bytes(const MuonMat &q) {
  return 2 * padded((u64)q.m * q.n * 4) + 2 * padded((u64)q.m * q.m * 4) + padded((u64)(q.chunks + 1) * 8);
}

template <class Blocks, class... KArgs, class... Args>
static bool launch_over(MuonTable &t, Blocks blocks, void (*kernel)(KArgs...), Args... args) {
  u64 n = 0;
  for (int i = 0; i < t.count; ++i) {
    t.mat[i].first = (unsigned)n;
    n += blocks(t.mat[i]);
  }
  const cudaError_t e = launch_k(kernel, dim3((unsigned)n), dim3(kMuonThreads), 0, stream(), t, args...);
  if (e != cudaSuccess) {
    set_error(PLAST_B200_ERR_CUDA, "muon: %s", cudaGetErrorString(e));
    return false;
  }
  count_launch();
  return true;
}

// One group of matrices whose scratch is `base`.
static void run_group(MuonTable &t, char *base, int steps) {
  for (int i = 0; i < t.count; ++i) {
    MuonMat &q = t.mat[i];
    for (int k = 0; k < 2; ++k) {
      q.x[k] = (float *)base;
      base += padded((u64)q.m * q.n * 4);
    }
    q.a = (float *)base;
    base += padded((u64)q.m * q.m * 4);
    q.b = (float *)base;
    base += padded((u64)q.m * q.m * 4);
    q.partial = (double *)base;
    base += padded((u64)(q.chunks + 1) * 8);
  }
  auto chunks = [](const MuonMat &q) { return (u64)q.chunks; };
  auto tiles = [](unsigned a, unsigned b, unsigned s) { return (u64)((a + s - 1) / s) * ((b + s - 1) / s); };
  if (!launch_over(t, chunks, muon_momentum_kernel)) return;
  if (!launch_over(t, [](const MuonMat &) { return (u64)1; }, muon_norm_kernel)) return;
  if (!launch_over(t, [&](const MuonMat &q) { return tiles(q.rows, q.cols, 32); }, muon_load_kernel)) return;
  int from = 0;
  for (int s = 0; s < steps; ++s) {
    const int last = s + 1 == steps;
    if (!launch_over(t, [&](const MuonMat &q) { return tiles(q.m, q.m, 64); }, muon_product_kernel<kGram>, from, 0)) return;
    if (!launch_over(t, [&](const MuonMat &q) { return tiles(q.m, q.m, 64); }, muon_product_kernel<kPolynomial>, from, 0)) return;
    if (!launch_over(t, [&](const MuonMat &q) { return tiles(q.m, q.n, 64); }, muon_product_kernel<kApply>, from, last)) return;
    from ^= 1;
  }
  if (steps == 0) launch_over(t, chunks, muon_store_kernel, 0);
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
