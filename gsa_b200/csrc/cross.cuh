// SPDX-License-Identifier: Apache-2.0
// Arguments and tile loads shared by the cross-attention kernels.
//
// The query rows of a scene and of one head of keys are packed: `group` query
// heads share the keys' head, and packed row r is query row r / group of head
// kv_head * group + r % group.  So shared heads fill a tile's rows, and a
// tile's keys are read once for all of them.
#pragma once
#include "tensor_core.cuh"

namespace gsa {

struct CrossArgs {
  const void *q, *k, *v, *out, *dout;
  const unsigned char* mask;  // [n_k], 0 shuts a key out; may be null
  const int *q_seg, *k_seg;
  float* lse;    // [n_q][heads], natural
  float* delta;  // [n_q][heads]
  void *o, *dq, *dk, *dv;
  float* part;      // [splits][rows][heads][dim] partial results
  float* part_lse;  // [splits][n_q][heads]
  int* error;       // set where a bounded wait ran out
  long long n_q, n_k;
  long long q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, d_row,
      d_head;
  int scenes, heads, kv_heads, group, dim, tiles, splits;
  float scale, scale_log2e;
};

constexpr int kRows = 128;     // rows of a resident tile, threads of a block
constexpr int kThreads = 128;

// Where a thread's 16-byte chunks of a tile lie: a fixed chunk, every
// `step`-th row.  `chunks` covers dim rounded up to 16 columns.
struct Chunks {
  int chunk, row, step;
  bool live, data;
};
__device__ __forceinline__ Chunks chunks_of(int dim) {
  const int chunks = (dim + 15) / 16 * 2;
  const int shift = chunks <= 2 ? 1 : chunks <= 4 ? 2 : chunks <= 8 ? 3 : 4;
  Chunks c;
  c.chunk = threadIdx.x & ((1 << shift) - 1);
  c.row = threadIdx.x >> shift;
  c.step = kThreads >> shift;
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

// kN key (or value) rows from k0 on; shut and absent keys are zeros, so that
// whatever lies there takes no part in any product.
template <typename T, int kN>
__device__ __forceinline__ void load_keys(const Chunks& c, uint32_t tile,
                                          const T* base, long long row,
                                          const unsigned char* mask, int k0,
                                          int n) {
  if (!c.live) return;
  for (int i = c.row; i < kN; i += c.step) {
    const int r = k0 + i;
    const bool there = c.data && r < n && (!mask || __ldg(mask + r));
    const T* from = there ? base + r * row + c.chunk * 8 : base;
    tc::copy16(tile + tc::tile_offset(kN, i, c.chunk), from, there);
  }
}

// Which of kN keys from k0 on are open, a bit each.
template <int kN>
__device__ __forceinline__ void key_words(uint32_t* words,
                                          const unsigned char* mask, int k0,
                                          int n) {
  if (threadIdx.x < kN) {
    const int r = k0 + (int)threadIdx.x;
    const bool open = r < n && (!mask || __ldg(mask + r));
    const uint32_t w = __ballot_sync(kFull, open);
    if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = w;
  }
}

// Host side (cross_forward.cu): the argument checks and the split rule that
// both directions share.
int multiprocessors();
int split_count(long long blocks, long long tiles, int room);
bool cross_sizes(const attention_args* a);
CrossArgs cross_arguments(const attention_args* in);

// A block's share [begin, end) of n items among `splits`.
__device__ __forceinline__ void share(int n, int splits, int which, int* begin,
                                      int* end) {
  const int each = n / splits, rest = n % splits;
  *begin = which * each + (which < rest ? which : rest);
  *end = *begin + each + (which < rest ? 1 : 0);
}

}  // namespace gsa
