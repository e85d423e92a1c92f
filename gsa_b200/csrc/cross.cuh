// SPDX-License-Identifier: Apache-2.0
// Arguments and tile loads shared by the cross-attention kernels.
//
// The query rows of a scene and of one head of keys are packed: `group` query
// heads share the keys' head, and packed row r is query row r / group of head
// kv_head * group + r % group.  So shared heads fill a tile's rows, and a
// tile's keys are read once for all of them.
#pragma once
#include <cuda.h>
#include "tensor_core.cuh"

namespace gsa {

struct CrossArgs {
  const void *q, *k, *v, *out, *dout;
  const unsigned char* mask;  // [n_k], 0 shuts a key out; may be null
  const int *q_seg, *k_seg;
  float* lse;  // [n_q][heads], natural
  // what the keys' pass needs of a packed row, [kv_heads][n_q * group]: its
  // -lse in units of q k^T (less the factor that P carries) and its -delta, in
  // four parts of the inputs' type each
  uint4* row_values;
  // fp16 gradients, [scenes][kv_heads][2 + value_chunks]: the bits of the
  // largest |dout|^2 of a packed row and of the largest |v|^2 of an open key,
  // and the latter in every `value_rows` keys
  unsigned* sizes;
  void *o, *dq, *dk, *dv;
  float* part;      // [splits][rows][heads][dim] partial results
  float* part_lse;  // [splits][n_q][heads]
  int* error;       // set where a bounded wait ran out
  long long n_q, n_k;
  long long q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, d_row,
      d_head;
  int scenes, heads, kv_heads, group, dim, tiles, splits;
  int value_chunks, value_rows;
  float scale, scale_log2e;
};

constexpr int kRows = 128;     // rows of a resident tile
constexpr int kThreads = 192;  // of a block: a thread per row, a warp that
                               // issues the products, a warp that loads tiles

// Where a thread's 16-byte chunks of a tile lie: a fixed chunk, every
// `step`-th row of those that `threads` threads share.  `chunks` covers dim
// rounded up to 16 columns.
struct Chunks {
  int chunk, row, step;
  bool live, data;
};
__device__ __forceinline__ Chunks chunks_of(int dim, int thread, int threads) {
  const int chunks = (dim + 15) / 16 * 2;
  const int shift = chunks <= 2 ? 1 : chunks <= 4 ? 2 : chunks <= 8 ? 3 : 4;
  Chunks c;
  c.chunk = thread & ((1 << shift) - 1);
  c.row = thread >> shift;
  c.step = threads >> shift;
  c.live = c.chunk < chunks;
  c.data = c.chunk * 8 < dim;
  return c;
}

// kN packed rows r0 .. of a scene (`n` of them in all) into a tile; rows and
// columns behind the last are zeros.
template <typename T, int kN>
__device__ __forceinline__ void load_packed(const Chunks& c, uint32_t tile,
                                            const T* base, long long row,
                                            long long head, int group, int r0,
                                            int n) {
  if (!c.live) return;
  for (int i = c.row; i < kN; i += c.step) {
    const int r = r0 + i;
    const bool there = c.data && r < n;
    const int qr = group == 1 ? r : r / group;
    const T* from =
        there ? base + qr * row + (r - qr * group) * head + c.chunk * 8 : base;
    tc::copy16(tile + tc::tile_offset(kN, i, c.chunk), from, there);
  }
}

// Zeros in the rows of a tile of kN rows whose bit is not set in `open` (a
// word per 32 rows), by one warp: four rows at a time, 16 bytes a lane.  A
// small loop: it runs once in a block's life, and its instructions come from
// far.
template <int kN>
__device__ __forceinline__ void clear_rows(uint32_t tile, int panels,
                                           const uint32_t* open) {
  const int lane = threadIdx.x & 31;
  tile += (lane >> 3) * 128 + (lane & 7) * 16;
#pragma unroll
  for (int w = 0; w < kN / 32; ++w) {
    uint32_t shut = ~open[w] >> (lane >> 3);
#pragma unroll 1
    for (int i = 0; shut; i += 4, shut >>= 4)
      if (shut & 1)
        for (int p = 0; p < panels; ++p)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                           tile + p * kN * 128 + (w * 32 + i) * 128),
                       "r"(0)
                       : "memory");
  }
}

// Which of kN keys from k0 on are open, a bit each, in every lane of a warp.
template <int kN>
__device__ __forceinline__ void key_words(uint32_t* words,
                                          const unsigned char* mask, int k0,
                                          int n) {
#pragma unroll
  for (int w = 0; w < kN / 32; ++w) {
    if (mask) {
      const int r = k0 + w * 32 + (threadIdx.x & 31);
      words[w] = __ballot_sync(kFull, r < n && __ldg(mask + r));
    } else {
      const int left = n - k0 - w * 32;
      words[w] = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1 : 0u;
    }
  }
}

// A block's share [begin, end) of n items among `splits`.
__device__ __forceinline__ void share(int n, int splits, int which, int* begin,
                                      int* end) {
  const int each = n / splits, rest = n % splits;
  *begin = which * each + (which < rest ? which : rest);
  *end = *begin + each + (which < rest ? 1 : 0);
}

// 2^x of a pair without the exponential unit, to 2^-22 (2.2e-7 at most, of them
// 1.6e-7 the fit's): n = round(x), then a polynomial of degree 5 in x - n (a Remez
// fit of 2^f on [-1/2, 1/2]).
// x = -inf gives exactly 0; x is not NaN and below 128.
__device__ __forceinline__ void exp2_polynomial(uint64_t x, float* lo,
                                                float* hi) {
  float a, b;
  tc::unpair(x, &a, &b);
  x = tc::pair(fmaxf(a, -127.f), fmaxf(b, -127.f));
  const float magic = 12582912.f;  // 1.5 * 2^23: its last bit is one
  const uint64_t y = tc::add2(x, tc::pair(magic, magic));
  const uint64_t n = tc::add2(y, tc::pair(-magic, -magic));
  const uint64_t f = tc::fma2(n, tc::pair(-1.f, -1.f), x);
  uint64_t p = tc::fma2(f, tc::pair(1.3276472e-3f, 1.3276472e-3f),
                        tc::pair(9.6755413e-3f, 9.6755413e-3f));
  p = tc::fma2(f, p, tc::pair(5.5507133e-2f, 5.5507133e-2f));
  p = tc::fma2(f, p, tc::pair(2.4022120e-1f, 2.4022120e-1f));
  p = tc::fma2(f, p, tc::pair(6.9314697e-1f, 6.9314697e-1f));
  p = tc::fma2(f, p, tc::pair(1.f, 1.f));
  float pa, pb, ya, yb;
  tc::unpair(p, &pa, &pb);
  tc::unpair(y, &ya, &yb);
  *lo = __int_as_float(__float_as_int(pa) + (__float_as_int(ya) << 23));
  *hi = __int_as_float(__float_as_int(pb) + (__float_as_int(yb) << 23));
}

// Host side (cross_forward.cu): the argument checks, the split rule and the
// tensor maps that both directions share.
int multiprocessors();
int split_count(long long blocks, long long tiles, int room);
bool cross_sizes(const attention_args* a);
CrossArgs cross_arguments(const attention_args* in);
// (columns, heads, rows) of a tensor of rows in boxes of 64 x `heads_box` x
// `rows_box`, 128-byte swizzled; what lies outside reads as zero.
cudaError_t row_map(CUtensorMap* map, long long type, const feature_rows& t,
                    long long dim, long long heads, long long rows,
                    int heads_box, int rows_box);

}  // namespace gsa
