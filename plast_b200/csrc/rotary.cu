// Rotary position embedding and the root-mean-square norm of query and key heads with it.
//
// Per head x of D elements, with weight w and the rotation R of its first 2n elements:
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  u = w n,  y = R u
// and backwards, from dy:
//   du = R^T dy,  dw = sum du n,  dn = w du,  dx = r (dn - n mean(dn n)).
// The rotary op alone is y = R x, dx = R^T dy.
//
// All of it is bound by HBM: 8 B per element forward, 12 B (rotary) or 16 B (with the norm) backward.
// A group of lanes holds one head in registers; a lane holds "slots" of two vectors, the two partners
// of a pair (halves) or eight consecutive elements (interleaved, or the part that is not rotated), so
// rotating needs no exchange between lanes and the norm only a shuffle sum. A group keeps the angles of
// its position for several heads.
#include "plast_b200_rotary.h"
#include "row_map.cuh"
#include "ew_kernel_device.cuh" // pdl_wait / pdl_launch_dependents
#include "iter.h"
#include "peer_link.cuh"

#include <math.h>

namespace pb {

constexpr int kHeadThreads = 256;
constexpr int kHeadStreams = 4; // strides of: 0 first streamed tensor, 1 second, 2 gradient, 3 positions

// One tensor of heads. Which tensors the streams are: forward x, out; rotary backward dout, dx;
// norm backward x, dout, dx.
struct HeadSide {
  const float *in0, *in1;
  float *out;
  const int *position;
  const float *weight;   // NULL: ones
  float *partial;        // [blocks][D] sums of the weight's gradient, or NULL
  u64 weight_stride;
  u64 elem_stride[3];    // along the head: in0, in1 (or out in the forward), out
  u64 head_stride[3];
  int nd;                // dims before the head dim and without the "heads" dim
  unsigned size[MAX_NDIM];
  u64 stride[kHeadStreams][MAX_NDIM];
  unsigned heads, heads_per_item, chunks, items, blocks;
};

struct HeadParams {
  HeadSide side[2];
  const float *freq;
  u64 freq_stride;
  unsigned head, half; // D, n
  unsigned slots, rotated_slots, log_group;
  int interleaved;
  float amplitude, epsilon;
};

// cos and sin of position * frequency. The product and its reduction to r in [-pi/4, pi/4] are done in
// 64 bits: in 32 a position of 10^6 would lose 0.06 rad. On that range the Taylor series up to r^11 and
// r^10 are within 3e-10 of the functions, so their fp32 evaluation is as good as its last rounding; the
// quadrant is put back afterwards.
__device__ __forceinline__ void turn(int position, float freq, float amplitude, float &c, float &s) {
  const double a = (double)position * (double)freq;
  const double q = rint(a * 0.63661977236758134308);
  double rd = __fma_rn(-q, 1.57079632679489655800, a);
  rd = __fma_rn(-q, 6.12323399573676603587e-17, rd);
  const float r = (float)rd, z = r * r;
  float ps = -1.0f / 39916800.0f;
  ps = __fmaf_rn(ps, z, 1.0f / 362880.0f);
  ps = __fmaf_rn(ps, z, -1.0f / 5040.0f);
  ps = __fmaf_rn(ps, z, 1.0f / 120.0f);
  ps = __fmaf_rn(ps, z, -1.0f / 6.0f);
  const float rs = __fmaf_rn(ps * z, r, r);
  float pc = -1.0f / 3628800.0f;
  pc = __fmaf_rn(pc, z, 1.0f / 40320.0f);
  pc = __fmaf_rn(pc, z, -1.0f / 720.0f);
  pc = __fmaf_rn(pc, z, 1.0f / 24.0f);
  pc = __fmaf_rn(pc, z, -0.5f);
  const float rc = __fmaf_rn(pc, z, 1.0f);
  const int quadrant = (int)(__double2ll_rn(q) & 3);
  const float cc = (quadrant & 1) ? rs : rc, ss = (quadrant & 1) ? rc : rs;
  c = ((quadrant == 1 || quadrant == 2) ? -cc : cc) * amplitude;
  s = ((quadrant & 2) ? -ss : ss) * amplitude;
}

template <int VEC> struct Slot { float a[VEC], b[VEC]; };

template <int VEC>
__device__ __forceinline__ void load_part(float (&v)[VEC], const float *p, u64 es) {
  if (VEC == 4) {
    const float4 q = __ldcs(reinterpret_cast<const float4 *>(p));
    v[0] = q.x; v[1 % VEC] = q.y; v[2 % VEC] = q.z; v[3 % VEC] = q.w;
  } else {
    v[0] = *p;
  }
}
template <int VEC>
__device__ __forceinline__ void store_part(const float (&v)[VEC], float *p) {
  if (VEC == 4) __stcs(reinterpret_cast<float4 *>(p), make_float4(v[0], v[1 % VEC], v[2 % VEC], v[3 % VEC]));
  else *p = v[0];
}

// (a, b) -> (a c - b s, a s + b c) over the pairs of a slot
template <int VEC>
__device__ __forceinline__ void rotate(Slot<VEC> &v, const float *c, const float *s, bool interleaved) {
  if (VEC == 1 || !interleaved) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float a = v.a[i], b = v.b[i];
      v.a[i] = __fmaf_rn(a, c[i], -(b * s[i]));
      v.b[i] = __fmaf_rn(a, s[i], b * c[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float a0 = v.a[i], a1 = v.a[i + 1 < VEC ? i + 1 : i], b0 = v.b[i], b1 = v.b[i + 1 < VEC ? i + 1 : i];
      const float c0 = c[i / 2], s0 = s[i / 2], c1 = c[VEC / 2 + i / 2], s1 = s[VEC / 2 + i / 2];
      v.a[i] = __fmaf_rn(a0, c0, -(a1 * s0));
      v.a[i + 1 < VEC ? i + 1 : i] = __fmaf_rn(a0, s0, a1 * c0);
      v.b[i] = __fmaf_rn(b0, c1, -(b1 * s1));
      v.b[i + 1 < VEC ? i + 1 : i] = __fmaf_rn(b0, s1, b1 * c1);
    }
  }
}

// Heads in flight per group and CTAs per SM (registers limit their product). For heads of up to 128
// elements, measured on 8192 positions of 32 + 8 heads of 128 (forward 336 MB, backward 671 MB): the
// norm forward 62 us with 2 heads and 4 CTAs (68 with 3, 81 with 4 heads and 2); its backward 121 us with
// 2 heads and 2 CTAs (150 with 1 head and 3). The rotation alone differs by 3 % between these.
template <int SLOTS, bool NORM, bool BACK> struct HeadShape {
  static constexpr int kHeads = SLOTS > 1 ? 1 : 2;
  static constexpr int kBlocks = SLOTS > 2 ? 1 : SLOTS == 2 || (NORM && BACK) ? 2 : 4;
};
template <int VEC, int SLOTS, bool NORM, bool BACK>
__global__ void __launch_bounds__(kHeadThreads, HeadShape<SLOTS, NORM, BACK>::kBlocks)
heads_kernel(const __grid_constant__ HeadParams p) {
  constexpr int U = HeadShape<SLOTS, NORM, BACK>::kHeads;
  pdl_wait();
  pdl_launch_dependents();
  const bool second = blockIdx.x >= p.side[0].blocks;
  const HeadSide &sd = p.side[second ? 1 : 0];
  const unsigned block = second ? blockIdx.x - p.side[0].blocks : blockIdx.x;
  const unsigned group_lanes = 1u << p.log_group, lane = threadIdx.x & (group_lanes - 1);
  const unsigned groups = kHeadThreads >> p.log_group;

  // where the lane's slots lie in a head
  unsigned offa[SLOTS], offb[SLOTS];
  bool has_a[SLOTS], has_b[SLOTS], turns[SLOTS];
  float w[SLOTS][2 * VEC], acc[SLOTS][2 * VEC];
#pragma unroll
  for (int t = 0; t < SLOTS; ++t) {
    const unsigned s = lane + t * group_lanes;
    turns[t] = s < p.rotated_slots;
    if (turns[t]) {
      offa[t] = p.interleaved ? 2 * VEC * s : VEC * s;
      offb[t] = p.interleaved ? offa[t] + VEC : offa[t] + p.half;
      has_a[t] = has_b[t] = true;
    } else {
      offa[t] = 2 * p.half + 2 * VEC * (s - p.rotated_slots);
      offb[t] = offa[t] + VEC;
      has_a[t] = s < p.slots && offa[t] < p.head;
      has_b[t] = s < p.slots && offb[t] < p.head;
    }
    if (NORM) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        w[t][i] = sd.weight && has_a[t] ? sd.weight[(offa[t] + i) * sd.weight_stride] : 1.0f;
        w[t][VEC + i] = sd.weight && has_b[t] ? sd.weight[(offb[t] + i) * sd.weight_stride] : 1.0f;
        acc[t][i] = acc[t][VEC + i] = 0.0f;
      }
    }
  }

  // every lane of a warp stays in the loop together: the norm's shuffles need them
  const u64 step = (u64)sd.blocks * groups;
  const unsigned group_in_warp = (threadIdx.x & 31) >> p.log_group;
  for (u64 item0 = (u64)block * groups + (threadIdx.x >> p.log_group); item0 - group_in_warp < sd.items; item0 += step) {
    const bool live = item0 < sd.items;
    const unsigned item = live ? (unsigned)item0 : 0;
    const unsigned token = item / sd.chunks, chunk = item - token * sd.chunks;
    u64 at[kHeadStreams] = {};
    unsigned rest = token;
    for (int d = sd.nd - 1; d > 0; --d) {
      const unsigned q = rest / sd.size[d], i = rest - q * sd.size[d];
      rest = q;
#pragma unroll
      for (int a = 0; a < kHeadStreams; ++a) at[a] += i * sd.stride[a][d];
    }
#pragma unroll
    for (int a = 0; a < kHeadStreams; ++a) at[a] += rest * sd.stride[a][0];
    const int position = sd.position[at[3]];
    float c[SLOTS][VEC], sn[SLOTS][VEC];
#pragma unroll
    for (int t = 0; t < SLOTS; ++t) {
      const unsigned s = lane + t * group_lanes;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        c[t][i] = 1.0f;
        sn[t][i] = 0.0f;
        if (turns[t]) turn(position, p.freq[(s * VEC + i) * p.freq_stride], p.amplitude, c[t][i], sn[t][i]);
        if (BACK) sn[t][i] = -sn[t][i];
      }
    }
    const unsigned h_begin = chunk * sd.heads_per_item;
    const unsigned h_end = sd.heads - h_begin < sd.heads_per_item ? sd.heads : h_begin + sd.heads_per_item;
    const unsigned trips = (sd.heads_per_item + U - 1) / U; // the same for all lanes
    for (unsigned trip = 0; trip < trips; ++trip) {
      Slot<VEC> x[U][SLOTS], dy[U][SLOTS], old[U][SLOTS];
      bool on[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const unsigned h = h_begin + trip * U + u;
        on[u] = live && h < h_end;
        const float *p0 = sd.in0 + at[0] + (u64)h * sd.head_stride[0];
        const float *p1 = sd.in1 + at[1] + (u64)h * sd.head_stride[1];
        const float *po = sd.out + at[2] + (u64)h * sd.head_stride[2];
#pragma unroll
        for (int t = 0; t < SLOTS; ++t) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            x[u][t].a[i] = x[u][t].b[i] = 0.0f;
            dy[u][t].a[i] = dy[u][t].b[i] = 0.0f;
          }
          if (on[u] && has_a[t]) {
            load_part<VEC>(x[u][t].a, p0 + offa[t] * sd.elem_stride[0], 0);
            if (NORM && BACK) load_part<VEC>(dy[u][t].a, p1 + offa[t] * sd.elem_stride[1], 0);
            if (BACK && sd.out) load_part<VEC>(old[u][t].a, po + offa[t] * sd.elem_stride[2], 0);
          }
          if (on[u] && has_b[t]) {
            load_part<VEC>(x[u][t].b, p0 + offb[t] * sd.elem_stride[0], 0);
            if (NORM && BACK) load_part<VEC>(dy[u][t].b, p1 + offb[t] * sd.elem_stride[1], 0);
            if (BACK && sd.out) load_part<VEC>(old[u][t].b, po + offb[t] * sd.elem_stride[2], 0);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (NORM) {
          float sum = 0.0f, dot = 0.0f;
#pragma unroll
          for (int t = 0; t < SLOTS; ++t) {
            if (BACK && turns[t]) rotate<VEC>(dy[u][t], c[t], sn[t], p.interleaved);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              sum = __fmaf_rn(x[u][t].a[i], x[u][t].a[i], sum);
              sum = __fmaf_rn(x[u][t].b[i], x[u][t].b[i], sum);
              if (BACK) {
                dot = __fmaf_rn(dy[u][t].a[i] * w[t][i], x[u][t].a[i], dot);
                dot = __fmaf_rn(dy[u][t].b[i] * w[t][VEC + i], x[u][t].b[i], dot);
              }
            }
          }
          for (unsigned o = group_lanes / 2; o; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (BACK) dot += __shfl_xor_sync(0xffffffffu, dot, o);
          }
          const float r = 1.0f / sqrtf(sum / (float)p.head + p.epsilon);
          const float back = BACK ? (dot * r / (float)p.head) : 0.0f; // mean(dn n)
#pragma unroll
          for (int t = 0; t < SLOTS; ++t)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float na = x[u][t].a[i] * r, nb = x[u][t].b[i] * r;
              if (BACK) {
                const float da = dy[u][t].a[i], db = dy[u][t].b[i];
                if (on[u]) { // an idle group's r may be anything
                  acc[t][i] = __fmaf_rn(da, na, acc[t][i]);
                  acc[t][VEC + i] = __fmaf_rn(db, nb, acc[t][VEC + i]);
                }
                x[u][t].a[i] = r * __fmaf_rn(-na, back, da * w[t][i]);
                x[u][t].b[i] = r * __fmaf_rn(-nb, back, db * w[t][VEC + i]);
              } else {
                x[u][t].a[i] = na * w[t][i];
                x[u][t].b[i] = nb * w[t][VEC + i];
              }
            }
        }
        if (!(NORM && BACK)) {
#pragma unroll
          for (int t = 0; t < SLOTS; ++t)
            if (turns[t]) rotate<VEC>(x[u][t], c[t], sn[t], p.interleaved);
        }
        if (on[u] && sd.out) {
          const unsigned h = h_begin + trip * U + u;
          float *po = sd.out + at[2] + (u64)h * sd.head_stride[2];
#pragma unroll
          for (int t = 0; t < SLOTS; ++t) {
            if (BACK) {
#pragma unroll
              for (int i = 0; i < VEC; ++i) {
                x[u][t].a[i] += old[u][t].a[i];
                x[u][t].b[i] += old[u][t].b[i];
              }
            }
            if (has_a[t]) store_part<VEC>(x[u][t].a, po + offa[t] * sd.elem_stride[2]);
            if (has_b[t]) store_part<VEC>(x[u][t].b, po + offb[t] * sd.elem_stride[2]);
          }
        }
      }
    }
  }

  // the block's part of the weight's gradient: its groups in a fixed order
  if (NORM && BACK) {
    if (!sd.partial) return; // the whole block
    __shared__ float part[kHeadThreads * SLOTS * 2 * VEC];
#pragma unroll
    for (int t = 0; t < SLOTS; ++t)
#pragma unroll
      for (int i = 0; i < 2 * VEC; ++i) part[(t * 2 * VEC + i) * kHeadThreads + threadIdx.x] = acc[t][i];
    __syncthreads();
    const unsigned values = group_lanes * SLOTS * 2 * VEC;
    for (unsigned v = threadIdx.x; v < values; v += kHeadThreads) {
      const unsigned l = v & (group_lanes - 1), ti = v >> p.log_group;
      const unsigned t = ti / (2 * VEC), i = ti % (2 * VEC), s = l + t * group_lanes;
      unsigned off;
      if (s < p.rotated_slots) {
        const unsigned oa = p.interleaved ? 2 * VEC * s : VEC * s;
        off = i < VEC ? oa + i : (p.interleaved ? oa + VEC : oa + p.half) + (i - VEC);
      } else {
        off = 2 * p.half + 2 * VEC * (s - p.rotated_slots) + i;
      }
      if (s >= p.slots || off >= p.head) continue;
      float sum = 0.0f;
      for (unsigned g = 0; g < groups; ++g) sum += part[ti * kHeadThreads + g * group_lanes + l];
      sd.partial[(u64)block * p.head + off] = sum;
    }
  }
}

// dw += sum over blocks of the partial sums, 32 columns per CTA, rows in a fixed order
struct WeightGradParams {
  const float *partial[2];
  float *dw[2];
  u64 stride[2];
  unsigned rows[2];
  unsigned head;
  bool shared; // queries and keys have one weight: both sums go to dw[0]
};
__global__ void __launch_bounds__(1024) head_weight_grad_kernel(const WeightGradParams p) {
  __shared__ float part[32][33];
  pdl_wait();
  pdl_launch_dependents();
  const int side = blockIdx.y;
  const unsigned col = blockIdx.x * 32 + threadIdx.x;
  float sum = 0.0f;
  for (int from = side; from <= (p.shared ? 1 : side); ++from)
    if (p.partial[from] && col < p.head)
      for (unsigned r = threadIdx.y; r < p.rows[from]; r += 32) sum += p.partial[from][(u64)r * p.head + col];
  part[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && p.dw[side] && col < p.head) {
    float total = 0.0f;
    for (int i = 0; i < 32; ++i) total += part[i][threadIdx.x];
    p.dw[side][col * p.stride[side]] += total;
  }
}

// ---- host --------------------------------------------------------------------------------------------
static bool check_layout(const char *name, u64 layout, float amplitude) {
  if (layout != PLAST_ROTARY_HALVES && layout != PLAST_ROTARY_INTERLEAVED) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: unknown pair layout", name);
    return false;
  }
  if (!(amplitude > 0.0f) || !(amplitude < INFINITY)) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: the amplitude must be positive and finite", name);
    return false;
  }
  return true;
}

// Positions and frequencies against a tensor of heads; fills what does not depend on the side.
static bool check_turns(const char *name, const Tensor *x, const Tensor *positions, const Tensor *freq, HeadParams *p) {
  char what[96];
  snprintf(what, sizeof what, "%s: positions", name);
  if (!check_typed(positions, INT32, what)) return false;
  snprintf(what, sizeof what, "%s: inv_freq", name);
  if (!check_typed(freq, FLOAT32, what)) return false;
  if (x->ndim < 1) {
    set_error(PLAST_B200_ERR_SHAPE, "%s: a tensor of heads has at least one dim", name);
    return false;
  }
  const u64 head = x->shape[x->ndim - 1];
  if (head > PLAST_ROTARY_MAX_HEAD) {
    set_error(PLAST_B200_ERR_LIMIT, "%s: heads of more than %d elements", name, PLAST_ROTARY_MAX_HEAD);
    return false;
  }
  if (freq->ndim != 1 || freq->shape[0] == 0 || 2 * freq->shape[0] > head) {
    set_error(PLAST_B200_ERR_SHAPE, "%s: inv_freq must have one dim of 1 to head / 2 elements", name);
    return false;
  }
  if (positions->requires_grad || freq->requires_grad) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: no gradient for positions or inv_freq", name);
    return false;
  }
  p->freq = (const float *)freq->data;
  p->freq_stride = freq->strides[0];
  p->head = (unsigned)head;
  p->half = (unsigned)freq->shape[0];
  return true;
}

// The dims before the last one, planned over up to three tensors and the positions.
static bool plan_side(const char *name, HeadSide *sd, const Tensor *const streams[3], const Tensor *positions) {
  const Tensor *x = streams[0];
  const u64 lead = x->ndim - 1;
  u64 strides[kHeadStreams][MAX_NDIM] = {};
  if (!broadcast_strides(positions, x->shape, lead, strides[3])) {
    set_error(PLAST_B200_ERR_SHAPE, "%s: positions do not broadcast against the dims before the last", name);
    return false;
  }
  u64 rows = 1;
  for (u64 d = 0; d < lead; ++d) rows *= x->shape[d];
  if (rows >= 0x7fffffffull) {
    set_error(PLAST_B200_ERR_LIMIT, "%s: more than 2^31 - 2 heads", name);
    return false;
  }
  for (int a = 0; a < 3; ++a) {
    const Tensor *t = streams[a] ? streams[a] : x;
    for (u64 d = 0; d < lead; ++d) strides[a][d] = t->strides[d];
    sd->elem_stride[a] = t->strides[lead];
  }
  IterPlan plan;
  make_plan(&plan, x->shape, lead, kHeadStreams, strides, nullptr, 0);
  // the heads: the largest dim along which the position stays
  int hd = -1;
  for (int d = 0; d < plan.ndim; ++d)
    if (plan.stride[3][d] == 0 && plan.size[d] > 1 && (hd < 0 || plan.size[d] > plan.size[hd])) hd = d;
  sd->heads = hd < 0 ? 1 : (unsigned)plan.size[hd];
  for (int a = 0; a < 3; ++a) sd->head_stride[a] = hd < 0 ? 0 : plan.stride[a][hd];
  sd->nd = 0;
  for (int d = plan.ndim - 1; d >= 0; --d) { // outermost first
    if (d == hd) continue;
    sd->size[sd->nd] = (unsigned)plan.size[d];
    for (int a = 0; a < kHeadStreams; ++a) sd->stride[a][sd->nd] = plan.stride[a][d];
    ++sd->nd;
  }
  if (sd->nd == 0) {
    sd->nd = 1;
    sd->size[0] = 1;
  }
  sd->items = (unsigned)(rows / (sd->heads ? sd->heads : 1));
  sd->position = (const int *)positions->data;
  return true;
}

static bool side_vec4(const HeadSide &sd, int streams) {
  const void *ptr[3] = {sd.in0, sd.in1, sd.out};
  for (int a = 0; a < 3; ++a) {
    if (streams == 2 && a == 1) continue;
    if ((uintptr_t)ptr[a] & 15 || sd.elem_stride[a] != 1) return false;
    if (sd.heads > 1 && (sd.head_stride[a] & 3)) return false;
    for (int d = 0; d < sd.nd; ++d)
      if (sd.size[d] > 1 && (sd.stride[a][d] & 3)) return false;
  }
  return true;
}

// Chooses vector width, lanes per head and heads per item, and launches. `max_blocks`: 0 = one trip
// per block, else a fixed grid whose blocks keep partial sums.
template <bool NORM, bool BACK>
static void launch_heads(HeadParams &p, int sides, unsigned max_blocks) {
  bool vec4 = p.head % 4 == 0 && p.half % 4 == 0;
  for (int i = 0; i < sides; ++i) vec4 = vec4 && side_vec4(p.side[i], NORM && BACK ? 3 : 2);
  const unsigned vec = vec4 ? 4 : 1;
  p.rotated_slots = p.half / vec;
  p.slots = p.rotated_slots + (p.head - 2 * p.half + 2 * vec - 1) / (2 * vec);
  p.log_group = 0;
  while (p.log_group < 5 && (1u << p.log_group) < p.slots) ++p.log_group;
  const unsigned per_lane = (p.slots + (1u << p.log_group) - 1) >> p.log_group;
  const unsigned groups = kHeadThreads >> p.log_group;
  // Heads per item, which share its angles: 1 to 8, whichever makes the turns of the GPU cheapest. A turn costs its
  // heads and the angles, the latter in heads: 1.5 where little else is done, less beside more traffic. Measured
  // with 1 .. 8 heads: rotary of 3000 positions, 32 heads, half rotated, with gradient 49 / 48 / 55 us for 2 / 4 / 8 (of
  // 8196 positions 119 / 112 / 116); norm and rotation of 8192 positions, 32 + 8 heads, with gradient 209 / 190 / 182.
  const unsigned per_sm = NORM && BACK ? 2 : per_lane * vec <= 4 && vec4 ? 4 : per_lane <= 2 ? 2 : 1;
  const double angles = 2.0 * p.half / p.head * (BACK ? (NORM ? 0.4 : 0.8) : 1.5);
  unsigned share = 1;
  double least = 0.0;
  for (unsigned n = 1; n <= 8; n *= 2) {
    u64 blocks = 0;
    for (int i = 0; i < sides; ++i) {
      const HeadSide &sd = p.side[i];
      const unsigned each = n < sd.heads ? n : sd.heads;
      blocks += ((u64)sd.items * ((sd.heads + each - 1) / each) + groups - 1) / groups;
    }
    const u64 turns = (blocks + (u64)sm_count() * per_sm - 1) / ((u64)sm_count() * per_sm);
    const double cost = (double)turns * ((n == 1 ? 1.6 : n) + angles); // one head alone leaves memory waiting
    if (n == 1 || cost < least) {
      least = cost;
      share = n;
    }
    if (turns <= 1) break; // more heads per item take longer
  }
  u64 want = 0;
  for (int i = 0; i < sides; ++i) {
    HeadSide &sd = p.side[i];
    sd.heads_per_item = share < sd.heads ? share : sd.heads;
    sd.chunks = (sd.heads + sd.heads_per_item - 1) / sd.heads_per_item;
    sd.items *= sd.chunks;
    sd.blocks = (sd.items + groups - 1) / groups;
    want += sd.blocks;
  }
  if (max_blocks && want > max_blocks) // in proportion, at least one each
    for (int i = 0; i < sides; ++i) {
      const u64 b = (u64)p.side[i].blocks * max_blocks / want;
      p.side[i].blocks = b ? (unsigned)b : 1;
    }
  unsigned grid = 0;
  for (int i = 0; i < sides; ++i) grid += p.side[i].blocks;
  const dim3 g(grid), b(kHeadThreads);
  cudaError_t e;
  if (vec4) {
    if (per_lane <= 1) e = launch_k(heads_kernel<4, 1, NORM, BACK>, g, b, 0, stream(), p);
    else if (per_lane <= 2) e = launch_k(heads_kernel<4, 2, NORM, BACK>, g, b, 0, stream(), p);
    else e = launch_k(heads_kernel<4, 4, NORM, BACK>, g, b, 0, stream(), p);
  } else {
    if (per_lane <= 2) e = launch_k(heads_kernel<1, 2, NORM, BACK>, g, b, 0, stream(), p);
    else e = launch_k(heads_kernel<1, 16, NORM, BACK>, g, b, 0, stream(), p);
  }
  PB_CUDA(e);
  count_launch();
}

static bool check_same_heads(const char *name, const Tensor *x, const Tensor *y, const char *what) {
  char text[96];
  snprintf(text, sizeof text, "%s: %s", name, what);
  if (!check_typed(y, FLOAT32, text)) return false;
  if (!same_shape(x, y)) {
    set_error(PLAST_B200_ERR_SHAPE, "%s: shape differs from its input's", text);
    return false;
  }
  return true;
}

static bool check_output(const char *name, const Tensor *x, const Tensor *y) {
  if (!check_same_heads(name, x, y, "output")) return false;
  if (has_repeated_elements(y)) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: the output holds an element at two indices", name);
    return false;
  }
  return true;
}

static bool check_weight(const char *name, const Tensor *w, unsigned head) {
  if (!w) return true;
  char text[96];
  snprintf(text, sizeof text, "%s: weight", name);
  if (!check_typed(w, FLOAT32, text)) return false;
  if (w->ndim < 1 || w->shape[w->ndim - 1] != head || numel(w) != head) {
    set_error(PLAST_B200_ERR_SHAPE, "%s: must have one element per element of a head", text);
    return false;
  }
  return true;
}

} // namespace pb

using namespace pb;

extern "C" {

void rotary_cuda_forward(const Tensor **inputs, Tensor *output, KernelParams params) {
  begin_call();
  if (!inputs) return set_error(PLAST_B200_ERR_NULL, "rotary: inputs is NULL");
  const Tensor *x = inputs[0];
  HeadParams p = {};
  if (!check_typed(x, FLOAT32, "rotary: x") || !check_layout("rotary", params.dim, params.fval) ||
      !check_turns("rotary", x, inputs[1], inputs[2], &p) || !check_output("rotary", x, output))
    return;
  const Tensor *const streams[3] = {x, nullptr, output};
  if (!plan_side("rotary", &p.side[0], streams, inputs[1])) return;
  const Extent others[2] = {extent_of(inputs[1]), extent_of(inputs[2])};
  if (!check_apart("rotary", "the output", extent_of(output), extent_of(x), others, 2)) return;
  if (numel(x) == 0) return; // nothing to do
  p.side[0].in0 = p.side[0].in1 = (const float *)x->data;
  p.side[0].out = (float *)output->data;
  p.interleaved = params.dim == PLAST_ROTARY_INTERLEAVED;
  p.amplitude = params.fval;
  launch_heads<false, false>(p, 1, 0);
  note_kernel("rotary");
  end_call();
}

void rotary_cuda_backward(Tensor **inputs, const Tensor *output, KernelParams params) {
  begin_call();
  if (!inputs) return set_error(PLAST_B200_ERR_NULL, "rotary: inputs is NULL");
  const Tensor *x = inputs[0];
  HeadParams p = {};
  if (!check_typed(x, FLOAT32, "rotary: x") || !check_layout("rotary", params.dim, params.fval) ||
      !check_turns("rotary", x, inputs[1], inputs[2], &p))
    return;
  if (!x->requires_grad) return; // nothing to do
  if (!check_tensor(output, "rotary: output", false) || !check_grad(x, "rotary: x") ||
      !check_same_heads("rotary", x, output->grad, "gradient of the output"))
    return;
  const Tensor *const streams[3] = {output->grad, nullptr, x->grad};
  if (!plan_side("rotary", &p.side[0], streams, inputs[1])) return;
  const Extent others[2] = {extent_of(inputs[1]), extent_of(inputs[2])};
  if (!check_apart("rotary", "the gradient of x", extent_of(x->grad), extent_of(output->grad), others, 2)) return;
  if (numel(x) == 0) return; // nothing to do
  p.side[0].in0 = p.side[0].in1 = (const float *)output->grad->data;
  p.side[0].out = (float *)x->grad->data;
  p.interleaved = params.dim == PLAST_ROTARY_INTERLEAVED;
  p.amplitude = params.fval;
  launch_heads<false, true>(p, 1, 0);
  note_kernel("rotary_backward");
  end_call();
}

int plast_b200_rotary_frequencies(const PlastRotaryScaling *scaling, u64 rotated, float base, float *host_inv_freq,
                                  float *amplitude) {
  begin_call();
  PlastRotaryScaling sc = {PLAST_ROTARY_SCALING_NONE, 1.0f, 0.0f, 0.0f, 0};
  if (scaling) sc = *scaling;
  if (!host_inv_freq) {
    set_error(PLAST_B200_ERR_NULL, "rotary_frequencies: no table to write to");
    return plast_b200_last_error();
  }
  if (rotated < 2 || rotated % 2 || rotated > PLAST_ROTARY_MAX_HEAD) {
    set_error(PLAST_B200_ERR_SHAPE, "rotary_frequencies: rotated must be even, 2 to %d", PLAST_ROTARY_MAX_HEAD);
    return plast_b200_last_error();
  }
  const bool scaled = sc.kind != PLAST_ROTARY_SCALING_NONE;
  const bool ranged = sc.kind == PLAST_ROTARY_SCALING_PARTS || sc.kind == PLAST_ROTARY_SCALING_BANDS;
  if (sc.kind < PLAST_ROTARY_SCALING_NONE || sc.kind > PLAST_ROTARY_SCALING_BANDS || !(base > 1.0f) || !(base < INFINITY) ||
      (scaled && (!(sc.factor >= 1.0f) || !(sc.factor < INFINITY))) ||
      (ranged && (!(sc.slow > 0.0f) || !(sc.fast > sc.slow) || !(sc.fast < INFINITY) || sc.context == 0)) ||
      (sc.kind == PLAST_ROTARY_SCALING_BASE && rotated < 4)) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "rotary_frequencies: base, factor, slow, fast or context out of range");
    return plast_b200_last_error();
  }
  const double d = (double)rotated, two_pi = 6.283185307179586476925;
  double b = base;
  if (sc.kind == PLAST_ROTARY_SCALING_BASE) b *= pow((double)sc.factor, d / (d - 2.0));
  // the pair that makes `turns` turns over the context: context * b^(-2 i / d) = 2 pi turns
  auto pair_of = [&](double turns) { return d * log((double)sc.context / (turns * two_pi)) / (2.0 * log(b)); };
  double low = 0.0, high = 0.0;
  if (sc.kind == PLAST_ROTARY_SCALING_PARTS) {
    low = floor(pair_of(sc.fast));
    high = ceil(pair_of(sc.slow));
    low = low < 0.0 ? 0.0 : low;
    high = high > d - 1.0 ? d - 1.0 : high;
    if (high <= low) high = low + 0.001;
  }
  for (u64 i = 0; i < rotated / 2; ++i) {
    const double f = pow(b, -2.0 * (double)i / d);
    double g = f;
    if (sc.kind == PLAST_ROTARY_SCALING_LINEAR) g = f / sc.factor;
    if (sc.kind == PLAST_ROTARY_SCALING_PARTS) {
      double ramp = ((double)i - low) / (high - low);
      ramp = ramp < 0.0 ? 0.0 : (ramp > 1.0 ? 1.0 : ramp);
      g = f / sc.factor * ramp + f * (1.0 - ramp);
    }
    if (sc.kind == PLAST_ROTARY_SCALING_BANDS) {
      const double turns = (double)sc.context * f / two_pi; // context / wavelength
      double keep = (turns - sc.slow) / ((double)sc.fast - sc.slow);
      keep = keep < 0.0 ? 0.0 : (keep > 1.0 ? 1.0 : keep);
      g = f * keep + f / sc.factor * (1.0 - keep);
    }
    host_inv_freq[i] = (float)g;
  }
  if (amplitude) *amplitude = sc.kind == PLAST_ROTARY_SCALING_PARTS ? (float)(0.1 * log((double)sc.factor) + 1.0) : 1.0f;
  return PLAST_B200_OK;
}

static bool check_qk(const char *name, const Tensor *q, const Tensor *k, const Tensor *qw, const Tensor *kw,
                     const Tensor *positions, const Tensor *freq, const Tensor *k_out, const PlastQkNormParams &params,
                     HeadParams *p) {
  if (!check_typed(q, FLOAT32, "qk_norm_rotary: q") || !check_layout(name, (u64)(unsigned)params.layout, params.amplitude))
    return false;
  if (!(params.epsilon >= 0.0f) || !(params.epsilon < INFINITY)) {
    set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: epsilon must not be negative", name);
    return false;
  }
  if (!check_turns(name, q, positions, freq, p) || !check_weight(name, qw, p->head)) return false;
  if (!k && (kw || k_out)) {
    set_error(PLAST_B200_ERR_NULL, "%s: k is NULL but its weight or output is not", name);
    return false;
  }
  if (k) {
    if (!check_typed(k, FLOAT32, "qk_norm_rotary: k")) return false;
    if (k->ndim < 1 || k->shape[k->ndim - 1] != p->head) {
      set_error(PLAST_B200_ERR_SHAPE, "%s: q and k have different head sizes", name);
      return false;
    }
    if (!check_weight(name, kw, p->head)) return false;
  }
  p->interleaved = params.layout == PLAST_ROTARY_INTERLEAVED;
  p->amplitude = params.amplitude;
  p->epsilon = params.epsilon;
  return true;
}

void plast_b200_qk_norm_rotary(const Tensor *q, const Tensor *k, const Tensor *q_weight, const Tensor *k_weight,
                               const Tensor *positions, const Tensor *inv_freq, Tensor *q_out, Tensor *k_out,
                               PlastQkNormParams params) {
  begin_call();
  const char *name = "qk_norm_rotary";
  HeadParams p = {};
  if (!check_qk(name, q, k, q_weight, k_weight, positions, inv_freq, k_out, params, &p)) return;
  const Tensor *xs[2] = {q, k}, *ws[2] = {q_weight, k_weight};
  Tensor *outs[2] = {q_out, k_out};
  int sides = 0;
  for (int i = 0; i < 2; ++i) {
    if (!xs[i]) continue;
    if (!check_output(name, xs[i], outs[i])) return;
    HeadSide &sd = p.side[sides];
    const Tensor *const streams[3] = {xs[i], nullptr, outs[i]};
    if (!plan_side(name, &sd, streams, positions)) return;
    if (numel(xs[i]) == 0) { // nothing on this side; the slot is used by the next one
      sd = HeadSide{};
      continue;
    }
    sd.in0 = sd.in1 = (const float *)xs[i]->data;
    sd.out = (float *)outs[i]->data;
    sd.weight = ws[i] ? (const float *)ws[i]->data : nullptr;
    sd.weight_stride = ws[i] ? ws[i]->strides[ws[i]->ndim - 1] : 0;
    ++sides;
  }
  // both sides run at once: an output lies over its own input at most
  const Extent in[2] = {extent_of(q), extent_of(k)}, out[2] = {extent_of(q_out), extent_of(k_out)};
  for (int i = 0; i < (k ? 2 : 1); ++i) {
    const Extent others[6] = {in[1 - i], out[1 - i], extent_of(q_weight), extent_of(k_weight), extent_of(positions), extent_of(inv_freq)};
    if (!check_apart(name, i ? "k_out" : "q_out", out[i], in[i], others, 6)) return;
  }
  if (sides) launch_heads<true, false>(p, sides, 0);
  note_kernel("qk_norm_rotary");
  end_call();
}

void plast_b200_qk_norm_rotary_backward(Tensor *q, Tensor *k, Tensor *q_weight, Tensor *k_weight,
                                        const Tensor *positions, const Tensor *inv_freq, const Tensor *q_out,
                                        const Tensor *k_out, PlastQkNormParams params) {
  begin_call();
  const char *name = "qk_norm_rotary";
  HeadParams p = {};
  if (!check_qk(name, q, k, q_weight, k_weight, positions, inv_freq, k_out, params, &p)) return;
  const Tensor *xs[2] = {q, k}, *ws[2] = {q_weight, k_weight}, *outs[2] = {q_out, k_out};
  int sides = 0;
  bool wants_weight[2] = {};
  WeightGradParams wg = {};
  Extent in[2] = {}, dout[2] = {}; // of the sides that are computed
  for (int i = 0; i < 2; ++i) {
    if (!xs[i]) continue;
    const bool need_x = xs[i]->requires_grad, need_w = ws[i] && ws[i]->requires_grad;
    if (!need_x && !need_w) continue;
    if (!check_tensor(outs[i], "qk_norm_rotary: output", false) ||
        (need_x && !check_grad(xs[i], "qk_norm_rotary: input")) ||
        !check_same_heads(name, xs[i], outs[i]->grad, "gradient of the output"))
      return;
    if (need_w && !check_grad(ws[i], "qk_norm_rotary: weight")) return;
    in[i] = extent_of(xs[i]);
    dout[i] = extent_of(outs[i]->grad);
    if (need_w && peer_bracket_open())
      return set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: weight gradients are not combined inside a peer bracket", name);
    HeadSide &sd = p.side[sides];
    const Tensor *const streams[3] = {xs[i], outs[i]->grad, need_x ? xs[i]->grad : nullptr};
    if (!plan_side(name, &sd, streams, positions)) return;
    if (numel(xs[i]) == 0) {
      sd = HeadSide{};
      continue;
    }
    sd.in0 = (const float *)xs[i]->data;
    sd.in1 = (const float *)outs[i]->grad->data;
    sd.out = need_x ? (float *)xs[i]->grad->data : nullptr; // NULL: the weight's gradient alone
    sd.weight = ws[i] ? (const float *)ws[i]->data : nullptr;
    sd.weight_stride = ws[i] ? ws[i]->strides[ws[i]->ndim - 1] : 0;
    wants_weight[sides] = need_w;
    if (need_w) {
      const Tensor *dw = ws[i]->grad;
      wg.dw[sides] = (float *)dw->data;
      wg.stride[sides] = dw->strides[dw->ndim - 1];
    }
    ++sides;
  }
  if (!sides) return; // nothing to do
  // Both sides run at once: the gradient of an input lies over the gradient of its output at most, that of a weight (added
  // afterwards) over the other weight's at most.
  auto written = [](const Tensor *t) { return extent_of(t && t->requires_grad ? t->grad : nullptr); };
  for (int i = 0; i < (k ? 2 : 1); ++i) {
    const Extent others[8] = {in[0], in[1], dout[1 - i], written(xs[1 - i]), extent_of(q_weight), extent_of(k_weight), extent_of(positions), extent_of(inv_freq)};
    if (!check_apart(name, i ? "the gradient of k" : "the gradient of q", written(xs[i]), dout[i], others, 8)) return;
  }
  const Extent dqw = written(q_weight), dkw = written(k_weight);
  if (share_an_element(dqw, dkw) && // but for a shared weight, whose dims before the last may differ
      (dqw.t->data != dkw.t->data || dqw.t->strides[dqw.t->ndim - 1] != dkw.t->strides[dkw.t->ndim - 1]))
    return set_error(PLAST_B200_ERR_UNSUPPORTED, "%s: the gradients of the weights overlap", name);
  const unsigned max_blocks = (unsigned)sm_count() * 2; // all resident: each keeps one partial sum
  float *scratch = nullptr;
  if (wants_weight[0] || wants_weight[1]) {
    const cudaError_t e = scratch_alloc_async((void **)&scratch, (size_t)2 * max_blocks * p.head * sizeof(float));
    if (e != cudaSuccess) {
      cudaGetLastError(); // reported here, not by the next call
      return set_error(PLAST_B200_ERR_CUDA, "%s: no scratch for the weight gradients: %s", name, cudaGetErrorString(e));
    }
    for (int i = 0; i < sides; ++i)
      if (wants_weight[i]) p.side[i].partial = scratch + (size_t)i * max_blocks * p.head;
  }
  launch_heads<true, true>(p, sides, max_blocks);
  if (scratch) {
    if (!failed()) {
      for (int i = 0; i < sides; ++i) {
        wg.partial[i] = p.side[i].partial;
        wg.rows[i] = p.side[i].blocks;
      }
      wg.head = p.head;
      wg.shared = sides == 2 && wg.dw[0] && wg.dw[0] == wg.dw[1];
      const cudaError_t e = launch_k(head_weight_grad_kernel, dim3((p.head + 31) / 32, wg.shared ? 1u : (unsigned)sides), dim3(32, 32), 0, stream(), wg);
      if (e != cudaSuccess) set_error(PLAST_B200_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
      else count_launch();
    }
    cudaFreeAsync(scratch, stream());
  }
  note_kernel("qk_norm_rotary_backward");
  end_call();
}

} // extern "C"
