// SPDX-License-Identifier: Apache-2.0
// The fifth-generation tensor core (tcgen05) as the cross-attention kernels
// use it: 128-row products D (+)= A B^T with 32-bit sums in tensor memory, A
// and B in shared memory (128-byte swizzled panels of 64 16-bit columns) or A
// in tensor memory, one thread issuing, completion on an mbarrier.
#pragma once
#include "features.cuh"

namespace gsa {
namespace tc {

__device__ __forceinline__ uint32_t smem_address(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

// ---- mbarriers ------------------------------------------------------------

__device__ __forceinline__ void barrier_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)
               : "memory");
}

__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar)
               : "memory");
}
// Arrives and adds the bytes of the copies that the phase waits for.
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(
                   bar),
               "r"(bytes)
               : "memory");
}
// The barriers that this thread initialised, visible to the block's threads
// (after a barrier of theirs) and to copies and products.
__device__ __forceinline__ void barriers_ready() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Every wait is for work of the same block that is under way and takes
// microseconds; the limit (seconds) turns a fault of the program into an
// error.  The loop is written out so that the common case, a phase that is
// complete, falls through (270 against 276 us of a forward pass).
constexpr int kWaitLimit = 1 << 22;
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity) {
  uint32_t left;
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .u32 n;\n mov.u32 n, %3;\n"
      "WAIT_AGAIN_%=:\n"
      " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " @p bra WAIT_DONE_%=;\n"
      " sub.u32 n, n, 1;\n setp.ne.u32 q, n, 0;\n"
      " @q bra WAIT_AGAIN_%=;\n"
      "WAIT_DONE_%=:\n mov.u32 %0, n;\n}\n"
      : "=r"(left)
      : "r"(bar), "r"(parity), "n"(kWaitLimit)
      : "memory");
  return left != 0;
}

// Some warps of a block meet: `threads` of them in all, by a number of their
// own (1 to 15).
__device__ __forceinline__ void meet(int number, int threads) {
  asm volatile("barrier.sync %0, %1;" ::"r"(number), "r"(threads) : "memory");
}

// ---- tensor memory --------------------------------------------------------

// By one whole warp; columns: a power of two of at least 32.
__device__ __forceinline__ void tmem_alloc(uint32_t out, uint32_t columns) {
  asm volatile(
      "tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
          out),
      "r"(columns)
      : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(
                   at),
               "r"(columns));
}

__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void wait_load() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void wait_store() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 32 columns of the warp's 32 rows: a row per lane.  The registers hold the
// values after wait_load().
__device__ __forceinline__ void load32(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]),
        "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}

__device__ __forceinline__ void load16(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]),
        "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15])
      : "r"(at));
}

__device__ __forceinline__ void load8(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]),
        "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(at));
}

__device__ __forceinline__ void store8(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
      "r"(r[6]), "r"(r[7])
      : "memory");
}

__device__ __forceinline__ void store16(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
      "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// ---- operands -------------------------------------------------------------

// A tile of `rows` rows (a multiple of 8) and up to 128 16-bit columns lies in
// panels of 64 columns: a panel row is 128 bytes, its 16-byte chunks swizzled
// by the row (chunk ^ row % 8).  Panels start on 1,024 bytes.
__device__ __forceinline__ uint32_t tile_offset(int rows, int row, int chunk) {
  return (uint32_t)((chunk >> 3) * rows * 128 + row * 128 +
                    (((chunk & 7) ^ (row & 7)) << 4));
}

constexpr uint64_t kDescriptor = (1ull << 46) |  // descriptor version
                                 (2ull << 61);   // 128-byte swizzle

// The tile as an operand whose columns are summed over (K-major): 8-row
// groups are 1,024 bytes apart.  Step: 16 columns, 32 bytes within a panel.
__device__ __forceinline__ uint64_t by_columns(uint32_t tile) {
  return kDescriptor | ((tile >> 4) & 0x3fffu) | (1ull << 16) |
         ((uint64_t)(1024 >> 4) << 32);
}
// The tile as an operand whose rows are summed over (MN-major): panels of 64
// columns lie `panel` bytes apart, 8-row groups 1,024.  Step: 16 rows, 2,048.
__device__ __forceinline__ uint64_t by_rows(uint32_t tile, uint32_t panel) {
  return kDescriptor | ((tile >> 4) & 0x3fffu) |
         ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32);
}

// A tile of 16 columns without swizzle, summed over its columns: per 8 rows
// their first 16 bytes, then their second.
__device__ __forceinline__ uint32_t narrow_offset(int row, int chunk) {
  return (uint32_t)((row >> 3) * 256 + chunk * 128 + (row & 7) * 16);
}
__device__ __forceinline__ uint64_t by_columns_narrow(uint32_t tile) {
  return (1ull << 46) | ((tile >> 4) & 0x3fffu) |
         ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(256 >> 4) << 32);
}

// Instruction: 128 x n products of fp16 or bf16 pairs summed in 32 bits.
template <typename T>
__device__ __forceinline__ uint32_t instruction(int n, bool b_by_rows) {
  const uint32_t type = __is_same(T, __nv_bfloat16) ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) |
         ((b_by_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((128u >> 4) << 24);
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b,
                                    uint32_t instr, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add)
      : "memory");
}
// A in tensor memory: two 16-bit values per 32-bit column.
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b,
                                         uint32_t instr, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(
          d),
      "r"(a), "l"(b), "r"(instr), "r"((uint32_t)add)
      : "memory");
}
// The barrier's phase completes when all products issued so far have.
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 "
      "[%0];" ::"r"(bar)
      : "memory");
}

// One lane of a converged warp.  Products are issued under it by warps that
// run as one, so that their operands are known to be uniform: from a lone
// thread each took 70 clocks to issue.
__device__ __forceinline__ bool elect() {
  uint32_t yes;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(yes));
  return yes != 0;
}

// D[128][n] (+)= A[128][16 steps] B[n][16 steps]^T, both by columns; a and b
// of kA and kB rows, at most kSteps steps.
template <typename T, int kA, int kB, int kSteps>
__device__ __forceinline__ void product_by_columns(uint32_t d, uint32_t a,
                                                   uint32_t b, int steps) {
  const uint32_t instr = instruction<T>(kB, false);
  const uint64_t a0 = by_columns(a), b0 = by_columns(b);
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
    if (s < steps)
      mma(d, a0 + ((s >> 2) * kA * 128 + (s & 3) * 32) / 16,
          b0 + ((s >> 2) * kB * 128 + (s & 3) * 32) / 16, instr, s > 0);
}

// D[128][n] (+)= A[128][kB] B[kB][n], A in tensor memory, B's tile of kB rows
// by rows.
template <typename T, int kB>
__device__ __forceinline__ void product_by_rows(uint32_t d, uint32_t a,
                                                uint32_t b, int n, bool add) {
  const uint32_t instr = instruction<T>(n, true);
  const uint64_t b0 = by_rows(b, kB * 128);
#pragma unroll
  for (int s = 0; s < kB / 16; ++s)
    mma_tmem(d, a + s * 8, b0 + s * 2048 / 16, instr, add || s > 0);
}

// ---- copies ---------------------------------------------------------------

// A box of a tensor map (columns, head, row) into a panel of shared memory;
// the barrier gets its bytes.  The column is a multiple of 64.
__device__ __forceinline__ void copy_box(uint32_t to, const void* map,
                                         uint32_t bar, int column, int head,
                                         int row) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(to),
      "l"(map), "r"(bar), "r"(column), "r"(head), "r"(row)
      : "memory");
}

// 16 bytes from global to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t to, const void* from,
                                       bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to),
               "l"(from), "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Shared memory written by this thread's copies becomes visible to the tensor
// core (after the block's barrier).
__device__ __forceinline__ void fence_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// ---- pairs of 32-bit values -------------------------------------------------

__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float* lo, float* hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*lo), "=f"(*hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

}  // namespace tc
}  // namespace gsa
