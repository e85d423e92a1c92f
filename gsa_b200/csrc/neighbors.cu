// SPDX-License-Identifier: Apache-2.0
// Attention along the rows of a neighbour query.  Query row r of scene i,
// head h, reads the entries j of its row of scene-local key IDs:
//
//   s_j = scale <q, k_j>,  p = softmax(s),  out = sum_j p_j v_j,
//   lse = log sum_j exp s_j,
//
// over the entries that name a row of the scene's keys and, in padded rows
// (the radius query's: ascending IDs, then the first again), do not repeat
// the first entry.  A row without entries gives 0 and lse = -inf, one whose
// scores are all -inf has no softmax and gives NaN for both.  Backward,
// with p_j = exp(s_j - lse) and delta = <dout, out>:
//
//   ds_j = p_j (<dout, v_j> - delta),   dq = scale sum_j ds_j k_j,
//   dv[key] = sum p dout,   dk[key] = scale sum ds q
//
// over all (row, entry) that name the key: the entries are sorted by key
// first (stable), so the sums have one fixed order and need no atomics.
//
// The bound is the gather and what each gathered element costs: an entry reads
// a key's and a value's head through L2, and its elements are unpacked,
// multiplied and added in 32 bits.  So nothing is done twice: a block first
// lists the entries that count of its rows (once for all heads) in shared
// memory; a head is a group of lanes with a 16-byte vector each, with several
// entries' loads in flight, multiplying pairs at a time.  Every lane of a group
// takes the whole sum of a product: sharing the entries' sums and exponentials
// out among the lanes saves instructions but lengthens the chain from load to
// result (397 us for 388 forward, 488 for 464 forward and back).
//
// 192,000 rows of 32 entries, 8 heads of 32 in bf16: 391 us, 1.07 TB/s of
// tensors in device memory (418 MB) and 12 TB/s of gathered heads through L1
// and L2.  48,000 rows, 4 heads of 32 in FP32, forward and back: 467 us, of them
// about 98 forward, 87 for the order of the entries, 103 for dq and 173 for dk
// and dv.
#include "features.cuh"
#include "tensor_core.cuh"

namespace gsa {
namespace {

struct NeighborArgs {
  const void *q, *k, *v, *out, *dout;
  void *o, *dq, *dk, *dv;
  float *lse_out, *delta;
  const float* lse;
  const int* ids;    // [n_q][width], scene-local
  const int *q_seg, *k_seg;
  const int* starts;  // [n_k + 1]: a key's entries in `order`
  const int* order;   // query rows, sorted by the key they name
  long long n_q, n_k;
  long long q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, d_row,
      d_head;
  // rows' strides in bytes, of what is gathered: a 32-bit one times a row is
  // one instruction
  uint32_t q_step, k_step, v_step, d_step;
  int scenes, heads, kv_heads, group, dim, width, padded;
  float scale, scale_log2e;
};

constexpr int kBlock = 128;
// Blocks of an SM (64 registers a thread): the forward pass of 192,000 rows
// took 388 us, with 7 (72 registers) 431, with 9 (spills) 476.
constexpr int kResident = 8;
// Entries of a group whose loads are in flight (an earlier form of the forward
// pass: 514 us with 4, 654 with 8, 549 with 2).
constexpr int kAhead = 4;
constexpr int kListStride = 36;    // of a row's list, clear of bank conflicts

template <int L>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int o = L / 2; o; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
  return x;
}

// A vector's elements as pairs of 32-bit values.
template <typename T>
struct Pairs {
  static constexpr int N = Vec<T>::V / 2;
  uint64_t v[N];
  __device__ __forceinline__ Pairs() {}
  __device__ __forceinline__ explicit Pairs(const uint4& u) {
    float f[2 * N];
    Vec<T>::unpack(u, f);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = tc::pair(f[2 * i], f[2 * i + 1]);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0;
  }
  __device__ __forceinline__ float dot(const Pairs& o) const {
    uint64_t s = tc::mul2(v[0], o.v[0]);
#pragma unroll
    for (int i = 1; i < N; ++i) s = tc::fma2(v[i], o.v[i], s);
    float a, b;
    tc::unpair(s, &a, &b);
    return a + b;
  }
  // this += w * o
  __device__ __forceinline__ void add(float w, const Pairs& o) {
    const uint64_t w2 = tc::pair(w, w);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = tc::fma2(w2, o.v[i], v[i]);
  }
  __device__ __forceinline__ void scale(float w) {
    const uint64_t w2 = tc::pair(w, w);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = tc::mul2(v[i], w2);
  }
  __device__ __forceinline__ uint4 pack() const {
    float f[2 * N];
#pragma unroll
    for (int i = 0; i < N; ++i) tc::unpair(v[i], &f[2 * i], &f[2 * i + 1]);
    return Vec<T>::pack(f);
  }
};

// The products of two words' 16-bit elements, added to 32 bits without being
// unpacked.
template <typename T>
__device__ __forceinline__ float fma_word(uint32_t a, uint32_t b, float c) {
  if constexpr (__is_same(T, __nv_bfloat16))
    asm("{\n .reg .b16 a0, a1, b0, b1;\n mov.b32 {a0, a1}, %1;\n"
        " mov.b32 {b0, b1}, %2;\n fma.rn.f32.bf16 %0, a0, b0, %0;\n"
        " fma.rn.f32.bf16 %0, a1, b1, %0;\n}\n"
        : "+f"(c)
        : "r"(a), "r"(b));
  else
    asm("{\n .reg .b16 a0, a1, b0, b1;\n mov.b32 {a0, a1}, %1;\n"
        " mov.b32 {b0, b1}, %2;\n fma.rn.f32.f16 %0, a0, b0, %0;\n"
        " fma.rn.f32.f16 %0, a1, b1, %0;\n}\n"
        : "+f"(c)
        : "r"(a), "r"(b));
  return c;
}
template <typename T>
__device__ __forceinline__ float dot(const uint4& a, const uint4& b) {
  if constexpr (sizeof(T) == 4) {
    return Pairs<T>(a).dot(Pairs<T>(b));
  } else {
    return fma_word<T>(a.x, b.x, fma_word<T>(a.z, b.z, 0.f)) +
           fma_word<T>(a.y, b.y, fma_word<T>(a.w, b.w, 0.f));
  }
}

// A row's vector; rows from 0 on.
__device__ __forceinline__ uint4 gather(const void* base, int row,
                                        uint32_t step) {
  return __ldg(reinterpret_cast<const uint4*>(
      static_cast<const char*>(base) + (uint64_t)(uint32_t)row * step));
}

template <typename T>
__device__ __forceinline__ uint4 vector_at(const void* base,
                                           long long element) {
  return __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(base) +
                                              element));
}

// The block's rows from `first` on: the keys (global rows) that a row's
// entries name, those that count, in their order; behind the last, the first
// again up to a multiple of kAhead.
template <int kRowsMax>
struct RowLists {
  int keys[kRowsMax][kListStride];
  int count[kRowsMax];

  __device__ __forceinline__ void fill(const NeighborArgs& a, long long first,
                                       int rows) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = warp; i < rows; i += kBlock / 32) {
      const long long row = first + i;
      const int scene = scene_of(a.q_seg, a.scenes, (int)row);
      const int base = __ldg(a.k_seg + scene);
      const int n = __ldg(a.k_seg + scene + 1) - base;
      const int id = lane < a.width ? __ldg(a.ids + row * a.width + lane) : -1;
      const int head = __shfl_sync(kFull, id, 0);
      const bool there = (unsigned)id < (unsigned)n &&
                         !(a.padded && lane > 0 && id == head);
      const unsigned set = __ballot_sync(kFull, there);
      const int total = __popc(set);
      if (there) keys[i][__popc(set & ((1u << lane) - 1))] = base + id;
      const int one = __shfl_sync(kFull, base + id, set ? __ffs(set) - 1 : 0);
      const int padded = (total + kAhead - 1) / kAhead * kAhead;
      if (lane >= total && lane < padded) keys[i][lane] = one;
      if (lane == 0) count[i] = total;
    }
    __syncthreads();
  }
};

// A group of L lanes per (row, head).  What every kernel over query rows
// starts from.
template <typename T, int L>
struct Group {
  static constexpr int V = Vec<T>::V;
  long long unit, row;
  int h, j, n;        // head; lane of the group; entries
  const int* keys;
  bool live, mine;    // a unit of its own; a vector of its own
  const T *k, *v;

  __device__ __forceinline__ Group(
      const NeighborArgs& a, RowLists<kBlock / L + 1>& lists) {
    const long long unit0 = (long long)blockIdx.x * (kBlock / L);
    const long long total = a.n_q * a.heads;
    const long long last = min(unit0 + kBlock / L, total) - 1;
    const long long row0 = unit0 / a.heads;
    lists.fill(a, row0, (int)(last / a.heads - row0) + 1);
    unit = unit0 + threadIdx.x / L;
    j = threadIdx.x % L;
    live = unit < total;
    row = live ? unit / a.heads : row0;
    h = live ? (int)(unit - row * a.heads) : 0;
    mine = live && j * V < a.dim;
    keys = lists.keys[row - row0];
    n = live ? lists.count[row - row0] : 0;
    const int hk = h / a.group;
    // a lane without a vector reads the first, and takes no part (`sum`)
    const int at = mine ? j * V : 0;
    k = static_cast<const T*>(a.k) + hk * a.k_head + at;
    v = static_cast<const T*>(a.v) + hk * a.v_head + at;
  }

  // The group's sum of its lanes' parts.
  __device__ __forceinline__ float sum(float part) const {
    return group_sum<L>(mine ? part : 0.f);
  }

  // The vectors of kAhead entries from j0 on; behind the last entry they stay
  // as they are, and what comes of them is not used.
  __device__ __forceinline__ void load(const NeighborArgs& a, int j0,
                                       uint4* ku, uint4* vu) const {
    if (j0 >= n) return;
    int at[kAhead];
#pragma unroll
    for (int t = 0; t < kAhead; t += 4)
      *reinterpret_cast<int4*>(at + t) =
          *reinterpret_cast<const int4*>(keys + j0 + t);
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      ku[t] = gather(k, at[t], a.k_step);
      vu[t] = gather(v, at[t], a.v_step);
    }
  }
};

template <typename T, int L>
__global__ void __launch_bounds__(kBlock, kResident)
    neighbor_forward_kernel(const __grid_constant__ NeighborArgs a) {
  __shared__ __align__(16) RowLists<kBlock / L + 1> lists;
  const Group<T, L> g(a, lists);
  Pairs<T> acc;
  acc.clear();
  uint4 q = make_uint4(0, 0, 0, 0);
  if (g.mine)
    q = vector_at<T>(a.q, g.row * a.q_row + g.h * a.q_head + g.j * Vec<T>::V);
  float m = -kInf, l = 0.f;
  uint4 ku[kAhead] = {}, vu[kAhead] = {};
  for (int j0 = 0; __any_sync(kFull, j0 < g.n); j0 += kAhead) {
    g.load(a, j0, ku, vu);
    float s[kAhead], top = m;
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      s[t] = g.sum(dot<T>(ku[t], q)) * a.scale_log2e;
      if (j0 + t >= g.n) s[t] = -kInf;
      top = fmaxf(top, s[t]);
    }
    const float shift = top == -kInf ? 0.f : top;
    const float keep = exp2_fast(m - shift);
    m = top;
    l *= keep;
    acc.scale(keep);
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      const float p = exp2_fast(s[t] - shift);
      l += p;
      // behind the last entry: nothing, whatever the first one's value holds
      if (j0 + t < g.n) acc.add(p, Pairs<T>(vu[t]));
    }
  }
  if (!g.live) return;
  if (g.mine) {
    if (g.n) acc.scale(1.f / l); else acc.clear();
    *reinterpret_cast<uint4*>(static_cast<T*>(a.o) + g.row * a.o_row +
                              g.h * a.o_head + g.j * Vec<T>::V) = acc.pack();
  }
  if (g.j == 0 && a.lse_out)
    a.lse_out[g.unit] = !g.n     ? -kInf
                        : l == 0.f ? __int_as_float(0x7fffffff)
                                   : (m + log2f(l)) * kLn2;
}

// dq, and delta for the keys' pass.  Of few entries the rounding of a 16-bit
// `out` would be most of the error of ds, so that <dout, out> only serves as a
// start d0 there: with ds0 = p (dp - d0) and c = sum ds0, delta = d0 + c and
// dq = scale (sum ds0 k - c sum p k).  A single entry's ds is 0 (p is 1).
// The further sum costs registers: 48,000 rows in bf16, forward and back, with
// 7 blocks on an SM 396 us, with 8 (spills) 416, with 6 403.
template <typename T, int L>
__global__ void __launch_bounds__(kBlock, sizeof(T) == 2 ? 7 : kResident)
    neighbor_dq_kernel(const __grid_constant__ NeighborArgs a) {
  __shared__ __align__(16) RowLists<kBlock / L + 1> lists;
  const Group<T, L> g(a, lists);
  const int at = g.j * Vec<T>::V;
  constexpr bool kRounded = sizeof(T) == 2;
  Pairs<T> acc, mean;  // mean: sum p k
  acc.clear();
  mean.clear();
  float change = 0.f;
  uint4 q = make_uint4(0, 0, 0, 0), d = q;
  float part = 0.f;
  if (g.mine) {
    q = vector_at<T>(a.q, g.row * a.q_row + g.h * a.q_head + at);
    d = vector_at<T>(a.dout, g.row * a.d_row + g.h * a.d_head + at);
    part = dot<T>(
        vector_at<T>(a.out, g.row * a.o_row + g.h * a.o_head + at), d);
  }
  float delta = group_sum<L>(part);
  const float lse2 = g.live ? __ldg(a.lse + g.unit) * kLog2e : 0.f;
  uint4 ku[kAhead] = {}, vu[kAhead] = {};
  for (int j0 = 0; __any_sync(kFull, j0 < g.n); j0 += kAhead) {
    g.load(a, j0, ku, vu);
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      const float s = g.sum(dot<T>(ku[t], q));
      const float dp = g.sum(dot<T>(vu[t], d));
      const float p = exp2_fast(fmaf(s, a.scale_log2e, -lse2));
      if (j0 + t < g.n) {
        const float ds = p * (dp - delta);
        const Pairs<T> key(ku[t]);
        acc.add(ds, key);
        if constexpr (kRounded) {
          mean.add(p, key);
          change += ds;
        }
      }
    }
  }
  if constexpr (kRounded) {
    delta += change;
    acc.add(-change, mean);
  }
  if (__any_sync(kFull, g.n == 1)) {
    const float dp = g.sum(dot<T>(vu[0], d));  // of the first entry, if single
    if (g.n == 1) {
      delta = dp;
      acc.scale(dp - dp);
    }
  }
  if (g.live && g.j == 0) a.delta[g.unit] = delta;
  if (g.mine) {
    acc.scale(a.scale);
    *reinterpret_cast<uint4*>(static_cast<T*>(a.dq) + g.unit * a.dim + at) =
        acc.pack();
  }
}

// dk and dv: a warp per (key, head of keys); its 32 / L groups take the key's
// (entry, query head) pairs in turn and are added up at the end.
template <typename T, int L>
__global__ void __launch_bounds__(kBlock, kResident)
    neighbor_dkv_kernel(const __grid_constant__ NeighborArgs a) {
  constexpr int V = Vec<T>::V;
  constexpr int G = 32 / L;
  // Entries of a group in flight: more warps are worth more here (4 with 96
  // registers: 571 us of 48,000 rows forward and back, so: 503).
  constexpr int kDeep = 2;
  const long long unit =
      ((long long)blockIdx.x * kBlock + threadIdx.x) >> 5;
  if (unit >= a.n_k * a.kv_heads) return;  // the whole warp
  const int lane = threadIdx.x & 31, j = lane % L, who = lane / L;
  const long long key = unit / a.kv_heads;
  const int hk = (int)(unit - key * a.kv_heads);
  const bool mine = j * V < a.dim;
  const int first = mine ? j * V : 0;  // a lane without a vector: the first
  Pairs<T> dk, dv;
  dk.clear();
  dv.clear();
  const uint4 k =
      vector_at<T>(a.k, key * a.k_row + hk * a.k_head + first);
  const uint4 v =
      vector_at<T>(a.v, key * a.v_row + hk * a.v_head + first);
  uint4 qu[kDeep] = {}, du[kDeep] = {};
  const int from = __ldg(a.starts + key), to = __ldg(a.starts + key + 1);
  for (int e0 = from; e0 < to; e0 += 32) {
    // an entry's row and its values in a lane each
    const int n = min(32, to - e0);
    const int mine_row = lane < n ? __ldg(a.order + e0 + lane) : 0;
    for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
      const T* q = static_cast<const T*>(a.q) + h * a.q_head + first;
      const T* d = static_cast<const T*>(a.dout) + h * a.d_head + first;
      float mine_lse = 0.f, mine_delta = 0.f;
      if (lane < n) {
        const long long at = (long long)mine_row * a.heads + h;
        mine_lse = __ldg(a.lse + at) * kLog2e;
        mine_delta = __ldg(a.delta + at);
      }
      for (int t0 = 0; t0 < n; t0 += G * kDeep) {
        float lse2[kDeep], delta[kDeep];
#pragma unroll
        for (int t = 0; t < kDeep; ++t) {
          const int e = t0 + t * G + who;
          const int row = __shfl_sync(kFull, mine_row, e & 31);
          lse2[t] = __shfl_sync(kFull, mine_lse, e & 31);
          delta[t] = __shfl_sync(kFull, mine_delta, e & 31);
          if (e < n) {
            qu[t] = gather(q, row, a.q_step);
            du[t] = gather(d, row, a.d_step);
          }
        }
#pragma unroll
        for (int t = 0; t < kDeep; ++t) {
          const float s = group_sum<L>(mine ? dot<T>(qu[t], k) : 0.f);
          const float dp = group_sum<L>(mine ? dot<T>(du[t], v) : 0.f);
          if (t0 + t * G + who >= n) continue;
          const float p = exp2_fast(fmaf(s, a.scale_log2e, -lse2[t]));
          dk.add(p * (dp - delta[t]), Pairs<T>(qu[t]));
          dv.add(p, Pairs<T>(du[t]));
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < Pairs<T>::N; ++i) {
#pragma unroll
    for (int o = L; o < 32; o <<= 1) {
      dk.v[i] = tc::add2(dk.v[i], __shfl_xor_sync(kFull, dk.v[i], o));
      dv.v[i] = tc::add2(dv.v[i], __shfl_xor_sync(kFull, dv.v[i], o));
    }
  }
  if (who == 0 && mine) {
    dk.scale(a.scale);
    const long long at = unit * a.dim + j * V;
    *reinterpret_cast<uint4*>(static_cast<T*>(a.dk) + at) = dk.pack();
    *reinterpret_cast<uint4*>(static_cast<T*>(a.dv) + at) = dv.pack();
  }
}

// ---------------------------------------------------------------------------
// Entries sorted by key: a stable radix sort of (key, query row), absent
// entries last under the key n_k.  Per digit: counts per tile, their prefix
// per digit value, scatter.  Ranks inside a tile follow the entries' order.

constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortEach = 8;                     // entries per thread
constexpr int kTile = kSortThreads * kSortEach;  // entries per tile
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBins = 1 << kMaxDigitBits;

struct SortArgs {
  const unsigned* keys_in;
  const int* rows_in;
  unsigned* keys_out;
  int* rows_out;
  int* counts;  // [bins][tiles], then [bins] totals
  long long n;
  int tiles, shift, bits;
};

// keys[e]: the key row that entry e names, or n_k; rows[e]: its query row.
__global__ void __launch_bounds__(256)
    entry_keys_kernel(const __grid_constant__ NeighborArgs a, unsigned* keys,
                      int* rows) {
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
  if (e >= a.n_q * a.width) return;
  const long long row = e / a.width;
  const int scene = scene_of(a.q_seg, a.scenes, (int)row);
  const int base = __ldg(a.k_seg + scene);
  const int n = __ldg(a.k_seg + scene + 1) - base;
  int id = __ldg(a.ids + e);
  if (a.padded && e != row * a.width && id == __ldg(a.ids + row * a.width))
    id = -1;
  keys[e] = (unsigned)id < (unsigned)n ? (unsigned)(base + id)
                                       : (unsigned)a.n_k;
  rows[e] = (int)row;
}

__global__ void __launch_bounds__(kSortThreads)
    sort_count_kernel(const __grid_constant__ SortArgs a) {
  __shared__ int bins[kMaxBins];
  const int n_bins = 1 << a.bits;
  for (int i = threadIdx.x; i < n_bins; i += kSortThreads) bins[i] = 0;
  __syncthreads();
  const long long at = (long long)blockIdx.x * kTile;
#pragma unroll
  for (int t = 0; t < kSortEach; ++t) {
    const long long e = at + t * kSortThreads + threadIdx.x;
    if (e < a.n)
      atomicAdd(&bins[(a.keys_in[e] >> a.shift) & (n_bins - 1)], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n_bins; i += kSortThreads)
    a.counts[(long long)i * a.tiles + blockIdx.x] = bins[i];
}

// Inclusive sum over the block's kSortThreads values.
__device__ __forceinline__ int block_inclusive(int x, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(kFull, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < warp; ++w) before += warp_sums[w];
  return x + before;
}

// A block per digit value: its tiles' counts become their exclusive prefix.
__global__ void __launch_bounds__(kSortThreads)
    sort_scan_kernel(const __grid_constant__ SortArgs a) {
  __shared__ int warp_sums[kSortWarps];
  __shared__ int last;
  int* row = a.counts + (long long)blockIdx.x * a.tiles;
  int carry = 0;
  for (int t0 = 0; t0 < a.tiles; t0 += kSortThreads) {
    const int t = t0 + threadIdx.x;
    const int x = t < a.tiles ? row[t] : 0;
    const int sum = block_inclusive(x, warp_sums);
    if (t < a.tiles) row[t] = carry + sum - x;
    if (threadIdx.x == kSortThreads - 1) last = sum;
    __syncthreads();
    carry += last;
    __syncthreads();
  }
  if (threadIdx.x == 0)
    a.counts[(long long)(1 << a.bits) * a.tiles + blockIdx.x] = carry;
}

__global__ void __launch_bounds__(kSortThreads)
    sort_scatter_kernel(const __grid_constant__ SortArgs a) {
  __shared__ int count[kSortWarps][kMaxBins];  // then: where the warp's begin
  __shared__ int warp_sums[kSortWarps];
  const int n_bins = 1 << a.bits;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = lane; i < n_bins; i += 32) count[warp][i] = 0;
  __syncwarp();
  // a warp's entries are consecutive, 32 at a time in their order
  const long long at =
      (long long)blockIdx.x * kTile + warp * (32 * kSortEach);
  unsigned key[kSortEach];
  int row[kSortEach], rank[kSortEach];
#pragma unroll
  for (int t = 0; t < kSortEach; ++t) {
    const long long e = at + t * 32 + lane;
    key[t] = e < a.n ? a.keys_in[e] : 0u;
    row[t] = e < a.n ? a.rows_in[e] : 0;
  }
#pragma unroll
  for (int t = 0; t < kSortEach; ++t) {
    const bool live = at + t * 32 + lane < a.n;
    const unsigned digit = (key[t] >> a.shift) & (n_bins - 1);
    const unsigned peers =
        __match_any_sync(kFull, live ? digit : 0xffffffffu);
    const int before = __popc(peers & ((1u << lane) - 1));
    rank[t] = live ? count[warp][digit] + before : 0;
    __syncwarp();
    if (live && before == 0) count[warp][digit] += __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  // start of every digit value's run in the output, for this tile
  int carry = 0;
  for (int b0 = 0; b0 < n_bins; b0 += kSortThreads) {
    const int b = b0 + threadIdx.x;
    const int total =
        b < n_bins ? a.counts[(long long)n_bins * a.tiles + b] : 0;
    const int sum = block_inclusive(total, warp_sums);
    if (b < n_bins) {
      int begin = carry + sum - total +
                  a.counts[(long long)b * a.tiles + blockIdx.x];
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = count[w][b];
        count[w][b] = begin;
        begin += c;
      }
    }
    int all = 0;
    for (int w = 0; w < kSortWarps; ++w) all += warp_sums[w];
    carry += all;
    __syncthreads();
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < kSortEach; ++t) {
    if (at + t * 32 + lane >= a.n) continue;
    const int digit = (key[t] >> a.shift) & (n_bins - 1);
    const int to = count[warp][digit] + rank[t];
    a.keys_out[to] = key[t];
    a.rows_out[to] = row[t];
  }
}

// starts[key] for every key 0 .. n_k: the first sorted entry not below it.
__global__ void __launch_bounds__(256)
    key_starts_kernel(const unsigned* keys, int n, long long n_k,
                      int* starts) {
  const long long key = (long long)blockIdx.x * 256 + threadIdx.x;
  if (key > n_k) return;
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if (__ldg(keys + mid) < (unsigned)key) lo = mid + 1; else hi = mid;
  }
  starts[key] = lo;
}

struct SortPlan {
  int passes, bits, tiles;
};

SortPlan sort_plan(long long n, long long n_k) {
  int key_bits = 1;
  while ((1ll << key_bits) <= n_k) ++key_bits;
  SortPlan p;
  p.passes = (key_bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.bits = (key_bits + p.passes - 1) / p.passes;
  p.tiles = (int)ceil_div(n, kTile);
  return p;
}

long long align16(long long bytes) { return (bytes + 15) & ~15ll; }

// ---------------------------------------------------------------------------

template <typename T, int L>
cudaError_t forward(const NeighborArgs& a, cudaStream_t s) {
  const long long lanes = a.n_q * a.heads * L;
  count_launches(1);
  neighbor_forward_kernel<T, L>
      <<<(unsigned)ceil_div(lanes, kBlock), kBlock, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T, int L>
cudaError_t backward(const NeighborArgs& a, cudaStream_t s) {
  if (a.n_q) {
    const long long lanes = a.n_q * a.heads * L;
    count_launches(1);
    neighbor_dq_kernel<T, L>
        <<<(unsigned)ceil_div(lanes, kBlock), kBlock, 0, s>>>(a);
  }
  if (a.n_k) {
    count_launches(1);
    neighbor_dkv_kernel<T, L>
        <<<(unsigned)ceil_div(a.n_k * a.kv_heads, kBlock / 32), kBlock, 0, s>>>(
            a);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t run(const NeighborArgs& a, bool back, cudaStream_t s) {
  const int vectors = a.dim / Vec<T>::V;
#define GSA_LANES(L) \
  if (vectors <= L) return back ? backward<T, L>(a, s) : forward<T, L>(a, s)
  if constexpr (Vec<T>::V == 8) GSA_LANES(1);
  GSA_LANES(2);
  GSA_LANES(4);
  GSA_LANES(8);
  GSA_LANES(16);
  if constexpr (Vec<T>::V == 4) GSA_LANES(32);
#undef GSA_LANES
  return cudaErrorInvalidValue;
}

cudaError_t run_type(const NeighborArgs& a, int type, bool back,
                     cudaStream_t s) {
  if (type == kF32) return run<float>(a, back, s);
  if (type == kF16) return run<__half>(a, back, s);
  return run<__nv_bfloat16>(a, back, s);
}

// A gathered tensor's stride from row to row, in bytes.
bool step_of(const feature_rows& t, long long rows, long long type,
             uint32_t* step) {
  const long long bytes = rows > 1 ? t.row * (type == kF32 ? 4 : 2) : 0;
  *step = (uint32_t)bytes;
  return bytes >= 0 && bytes <= 0xffffffffll;
}

bool sizes_ok(const attention_args* a) {
  return attention_sizes(a) && a->width >= 1 && a->width <= 32 &&
         a->n_q * a->width < kMaxInt;
}

NeighborArgs arguments(const attention_args* in) {
  NeighborArgs a = {};
  a.q = in->q.data;
  a.k = in->k.data;
  a.v = in->v.data;
  a.ids = in->ids;
  a.q_seg = in->q_seg;
  a.k_seg = in->k_seg;
  a.scenes = (int)in->scenes;
  a.n_q = in->n_q;
  a.n_k = in->n_k;
  a.q_row = in->q.row;
  a.q_head = in->q.head;
  a.k_row = in->k.row;
  a.k_head = in->k.head;
  a.v_row = in->v.row;
  a.v_head = in->v.head;
  a.o_row = in->out.row;
  a.o_head = in->out.head;
  a.heads = (int)in->heads;
  a.kv_heads = (int)in->kv_heads;
  a.group = a.heads / a.kv_heads;
  a.dim = (int)in->dim;
  a.width = (int)in->width;
  a.padded = in->padded != 0;
  a.scale = (float)in->scale;
  a.scale_log2e = (float)(in->scale * (double)kLog2e);
  return a;
}

}  // namespace
}  // namespace gsa

using namespace gsa;

// See include/point_features.h.
GSA_API int neighbor_attention(const attention_args* in) {
  if (!sizes_ok(in) || !attention_scale(in->scale)) return -2;
  if (!in->n_q) return 0;
  if (!vector_rows(in->q, in->type) || !vector_rows(in->out, in->type) ||
      !in->ids || !in->q_seg || !in->k_seg)
    return -2;
  if (in->n_k &&
      (!vector_rows(in->k, in->type) || !vector_rows(in->v, in->type)))
    return -2;
  NeighborArgs a = arguments(in);
  if (!step_of(in->k, in->n_k, in->type, &a.k_step) ||
      !step_of(in->v, in->n_k, in->type, &a.v_step))
    return -2;
  a.o = const_cast<void*>(in->out.data);
  a.lse_out = in->lse;
  return run_type(a, (int)in->type, false, (cudaStream_t)in->stream);
}

// See include/point_features.h.
GSA_API int64_t neighbor_attention_grad_workspace(const attention_args* in) {
  if (!sizes_ok(in)) return -2;
  const long long n = in->n_q * in->width;
  const SortPlan p = sort_plan(n, in->n_k);
  return align16(in->n_q * in->heads * 4) + 4 * align16(n * 4) +
         align16((in->n_k + 1) * 4) +
         align16((1ll << p.bits) * (p.tiles + 1) * 4);
}

// See include/point_features.h.
GSA_API int neighbor_attention_grad(const attention_args* in) {
  if (!sizes_ok(in) || !attention_scale(in->scale) || !in->q_seg ||
      !in->k_seg)
    return -2;
  const long long type = in->type, n_q = in->n_q, n_k = in->n_k;
  if (n_q && (!vector_rows(in->q, type) || !vector_rows(in->out, type) ||
              !vector_rows(in->dout, type) || !vector_address(in->dq) ||
              !in->lse || !in->ids))
    return -2;
  if (n_k && (!vector_rows(in->k, type) || !vector_rows(in->v, type) ||
              !vector_address(in->dk) || !vector_address(in->dv)))
    return -2;
  if (!vector_address(in->workspace) ||
      in->workspace_bytes < neighbor_attention_grad_workspace(in))
    return -2;
  NeighborArgs a = arguments(in);
  if (!step_of(in->q, n_q, type, &a.q_step) ||
      !step_of(in->dout, n_q, type, &a.d_step) ||
      !step_of(in->k, n_k, type, &a.k_step) ||
      !step_of(in->v, n_k, type, &a.v_step))
    return -2;
  a.out = in->out.data;
  a.dout = in->dout.data;
  a.d_row = in->dout.row;
  a.d_head = in->dout.head;
  a.lse = in->lse;
  a.dq = in->dq;
  a.dk = in->dk;
  a.dv = in->dv;
  cudaStream_t s = (cudaStream_t)in->stream;
  const long long n = n_q * a.width;
  const SortPlan p = sort_plan(n, n_k);
  char* at = static_cast<char*>(in->workspace);
  auto take = [&](long long bytes) {
    char* r = at;
    at += align16(bytes);
    return r;
  };
  a.delta = reinterpret_cast<float*>(take(n_q * a.heads * 4));
  unsigned* keys[2];
  int* rows[2];
  for (int i = 0; i < 2; ++i) {
    keys[i] = reinterpret_cast<unsigned*>(take(n * 4));
    rows[i] = reinterpret_cast<int*>(take(n * 4));
  }
  int* starts = reinterpret_cast<int*>(take((n_k + 1) * 4));
  int* counts =
      reinterpret_cast<int*>(take((1ll << p.bits) * (p.tiles + 1) * 4));
  int from = 0;
  if (n && n_k) {
    count_launches(1 + 3 * p.passes);
    entry_keys_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, s>>>(a, keys[0],
                                                                 rows[0]);
    for (int pass = 0; pass < p.passes; ++pass, from ^= 1) {
      SortArgs t = {keys[from],     rows[from], keys[from ^ 1],
                    rows[from ^ 1], counts,     n,
                    p.tiles,        pass * p.bits, p.bits};
      sort_count_kernel<<<p.tiles, kSortThreads, 0, s>>>(t);
      sort_scan_kernel<<<1 << p.bits, kSortThreads, 0, s>>>(t);
      sort_scatter_kernel<<<p.tiles, kSortThreads, 0, s>>>(t);
    }
  }
  if (n_k) {
    count_launches(1);
    key_starts_kernel<<<(unsigned)ceil_div(n_k + 1, 256), 256, 0, s>>>(
        keys[from], (int)n, n_k, starts);
  }
  a.starts = starts;
  a.order = rows[from];
  return run_type(a, (int)type, true, s);
}
