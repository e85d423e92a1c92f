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

__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n"
      " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

// Every wait is for products already issued, which take microseconds; the
// limit (seconds) turns a fault of the program into an error.
constexpr int kWaitLimit = 1 << 22;
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < kWaitLimit; ++i)
    if (barrier_try(bar, parity)) return true;
  return false;
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

// D[128][n] (+)= A[128][16 steps] B[n][16 steps]^T, both by columns; a and b
// of `a_rows` and `b_rows` rows.
template <typename T>
__device__ __forceinline__ void product_by_columns(uint32_t d, uint32_t a,
                                                   int a_rows, uint32_t b,
                                                   int b_rows, int n,
                                                   int steps) {
  const uint32_t instr = instruction<T>(n, false);
  for (int s = 0; s < steps; ++s) {
    const uint32_t in = (s & 3) * 32;
    mma(d, by_columns(a + (s >> 2) * a_rows * 128 + in),
        by_columns(b + (s >> 2) * b_rows * 128 + in), instr, s > 0);
  }
}

// D[128][n] (+)= A[128][16 steps] B[16 steps][n], A in tensor memory, B's
// tile of b_rows rows by rows.
template <typename T>
__device__ __forceinline__ void product_by_rows(uint32_t d, uint32_t a,
                                                uint32_t b, int b_rows, int n,
                                                int steps, bool add) {
  const uint32_t instr = instruction<T>(n, true);
  for (int s = 0; s < steps; ++s)
    mma_tmem(d, a + s * 8, by_rows(b + s * 2048, b_rows * 128), instr,
             add || s > 0);
}

// ---- copies ---------------------------------------------------------------

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

}  // namespace tc
}  // namespace gsa
