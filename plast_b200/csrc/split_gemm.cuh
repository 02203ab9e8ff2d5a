// Matrix products of 22-bit operands with fp32 sums on the tensor cores: panels of split fp16 operands, and the
// device-side pieces (barriers, bulk copies, tcgen05) that a kernel over them is made of.
//
// An fp32 value v, scaled by 2^14, is kept as two fp16 numbers, hi = fp16(v) and lo = fp16(v - hi):
// 22 bits. A product x y is then hi hi + hi lo + lo hi; the missing lo lo is below 2^-22 of it. The
// three products run on tcgen05.mma kind::f16 with fp32 accumulators in tensor memory.
//
// Values must stay below 65504 / 2^14 = 3.99 in magnitude (fp16's range), and keep all 22 bits down
// to 2^-14 (where lo leaves fp16's normal range); below that the absolute error stays at 2^-39.
//
// Panels: a matrix of R rows and C columns is cut into blocks of 128 x 64, stored one after the other
// by block row and block column, each as 16 KB of hi and 16 KB of lo. A block holds 128 rows of 128
// bytes whose eight 16-byte chunks are permuted by the row, chunk ^ (row & 7): the 128-byte swizzle
// that tcgen05 reads, so a plain contiguous bulk copy brings an operand into shared memory, and the
// same block serves as an operand whose long side is K (K-major: rows are M or N) or whose rows are K
// (MN-major). No tensor map is needed, and padding is part of the panel (zeros).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace pb {

constexpr int kPanelRows = 128, kPanelCols = 64;
constexpr unsigned kPanelHalf = kPanelRows * kPanelCols * 2; // bytes of hi, or of lo
constexpr float kSplitScale = 16384.0f, kSplitUnscale = 1.0f / 16384.0f;

__host__ __device__ inline unsigned panel_row_blocks(unsigned rows) { return (rows + kPanelRows - 1) / kPanelRows; }
__host__ __device__ inline unsigned panel_col_blocks(unsigned cols) { return (cols + kPanelCols - 1) / kPanelCols; }
inline uint64_t panel_bytes(unsigned rows, unsigned cols) {
  return (uint64_t)panel_row_blocks(rows) * panel_col_blocks(cols) * (2 * kPanelHalf);
}

#ifdef __CUDACC__
// byte offset of block (rb, cb) of a panel with `col_blocks` block columns
__device__ __forceinline__ uint64_t panel_block(unsigned rb, unsigned cb, unsigned col_blocks) {
  return ((uint64_t)rb * col_blocks + cb) * (2 * kPanelHalf);
}
// byte offset inside a block's hi (or lo) of 8 columns: row 0..127, chunk 0..7
__device__ __forceinline__ unsigned panel_chunk(unsigned row, unsigned chunk) {
  return row * 128 + ((chunk ^ (row & 7)) << 4);
}

// eight scaled values as hi and lo chunks
__device__ __forceinline__ void split8(const float *v, uint4 &hi, uint4 &lo) {
  unsigned h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 a = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    const float2 f = __half22float2(a);
    const __half2 b = __floats2half2_rn(v[2 * i] - f.x, v[2 * i + 1] - f.y);
    h[i] = *reinterpret_cast<const unsigned *>(&a);
    l[i] = *reinterpret_cast<const unsigned *>(&b);
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}
// ---- barriers ----------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void barrier_init(uint32_t bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// the same barrier of another CTA of the cluster
__device__ __forceinline__ void barrier_arrive_at(uint32_t bar, unsigned cta) {
  asm volatile("{\n\t.reg .b32 remote;\n\t"
               "mapa.shared::cluster.u32 remote, %0, %1;\n\t"
               "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [remote];\n\t}" ::"r"(bar), "r"(cta)
               : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, unsigned parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\t"
               "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
               "selp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok)
               : "r"(bar), "r"(parity)
               : "memory");
  return ok != 0;
}
// A wait that always ends: after `limit` cycles, or when another role of the CTA has given up, it raises
// `gave_up` and returns false; the caller then leaves its loop.
constexpr long long kWaitCycles = 4000000000ll; // about two seconds
struct WaitLimit { // shared memory
  long long limit;
  volatile unsigned gave_up;
  __device__ __forceinline__ bool over(long long start) { // looked at now and then
    if (gave_up) return true;
    if (clock64() - start <= limit) return false;
    gave_up = 1;
    return true;
  }
};
__device__ __noinline__ bool barrier_wait_long(uint32_t bar, unsigned parity, WaitLimit *wait) {
  const long long start = clock64();
  for (;;) {
    for (int i = 0; i < 64; ++i)
      if (barrier_try(bar, parity)) return true;
    if (wait->over(start)) return false;
  }
}

__device__ __forceinline__ bool barrier_wait(uint32_t bar, unsigned parity, WaitLimit *wait) {
  return barrier_try(bar, parity) || barrier_wait_long(bar, parity, wait);
}

// ---- copies and tensor core ----------------------------------------------------------------------------
// contiguous global -> shared copy; addresses and size are multiples of 16 bytes
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, unsigned bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Shared-memory operand descriptor: 128-byte swizzle, start on a 1024-byte atom plus the K step.
//   K-major: `sbo` = bytes from 8 rows to the next 8; `lbo` unused
//   MN-major: `lbo` = bytes from 64 elements along M or N to the next 64, `sbo` = from 8 K rows to the next
__device__ __forceinline__ uint64_t operand_desc(uint32_t address, unsigned lbo, unsigned sbo) {
  return (uint64_t)((address & 0x3ffff) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// Instruction descriptor of kind::f16: fp16 operands, fp32 accumulators.
__host__ __device__ constexpr uint32_t mma_desc(unsigned m, unsigned n, bool a_mn_major, bool b_mn_major) {
  return (1u << 4) | ((a_mn_major ? 1u : 0u) << 15) | ((b_mn_major ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
template <int CTAS>
__device__ __forceinline__ void mma_f16(uint32_t tmem, uint64_t a, uint64_t b, uint32_t desc, bool accumulate) {
  if (CTAS == 1)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                 "l"(a), "l"(b), "r"(desc), "r"((uint32_t)accumulate)
                 : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                 "l"(a), "l"(b), "r"(desc), "r"((uint32_t)accumulate)
                 : "memory");
}
// arrives on the barrier (of both CTAs of a pair) when every product issued so far is done
template <int CTAS>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if (CTAS == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"((uint16_t)3)
                 : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tmem_alloc(uint32_t where, unsigned columns) { // one whole warp
  if (CTAS == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t tmem, unsigned columns) { // the warp that allocated
  if (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 16 columns of the warp's 32 lanes (the wait belongs to the load: nothing may use the values before)
__device__ __forceinline__ void tmem_load16(uint32_t tmem, float (&v)[16]) {
  uint32_t *r = reinterpret_cast<uint32_t *>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
               "tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(tmem)
               : "memory");
}
// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t chosen;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
  return chosen != 0;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
#endif

} // namespace pb
