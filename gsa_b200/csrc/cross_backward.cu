// SPDX-License-Identifier: Apache-2.0
// Gradients of cross attention.  With P = exp(scale q k^T - lse) and
// delta = rowsum(dout * out):
//
//   dv = P^T dout,  dP = dout v^T,  dS = P * (dP - delta),
//   dq = scale dS k,  dk = scale dS^T q.
//
// Two passes of one kernel, each recomputing P: one block per 128 packed query
// rows walks the keys and keeps dq in tensor memory (and finds delta for the
// other), one block per 128 keys walks the queries and keeps dk and dv.  Seven
// products instead of five, but every sum has one fixed order (no atomics, the
// same bits each time), and nothing but the results is written.  In the keys'
// pass the products are taken transposed (S^T = k q^T), so that P^T and dS^T
// come out with a key per thread and go back to tensor memory as the second
// products' left side; the walked tile serves as the right side of both its
// products, read by columns and by rows, without a transposed copy.
//
// A block has sixteen warps of rows (four threads share a row, a quarter of the
// walked columns each), a warp for the products that give scores, one for the
// others, which read what the rows make of them, and one that loads walked
// tiles (TMA; rows behind the scene's last and shut keys are cleared).  The
// scores of the next tile are taken as soon as this one's are in registers;
// P and dS have columns of their own.
//
// In the keys' pass lse and delta belong to the columns.  They come from the
// products themselves: 16 columns more, powers of two on the keys' side and on
// the walked side -lse / scale and -delta in four parts of the inputs' type
// (24 bits and more together), so that S and dP leave the tensor core less lse
// and delta.  Read from shared memory (131 KB for 128 x 128 scores) they took
// as long as all the exponentials.
//
// P and dS are rounded to the inputs' type for their products (half a step).
// For fp16, whose normals are 2^-14 to 2^16, P carries a factor of 2^15 (it is
// at most 1), and dS a power of two that brings its bound, 2 |dout| |v|, to
// between 2^14 and 2^15: a row's own in the queries' pass, one for a scene and a
// head of keys in the keys' pass, where rows are summed over.  So nothing
// overflows, and what is above 2^-28 of the bound keeps all its bits.  A small
// kernel before the passes finds |v| (8 x 1,500 keys of 8 x 64: 6 us), the
// queries' pass |dout|.
//
// What bounds it, for 128 x 128 scores and a head of 64: 1,400 clocks of
// products in the keys' pass (1,024 in the queries') beside 1,024 of
// exponentials.  A tile takes some 2,580 clocks there: its chain of scores,
// softmax, weights and products, of which only the next scores run ahead.  8 x
// 6,000 queries on 1,500 keys, 8 heads of 64 in bf16: about 330 us of the
// queries' pass and 350 of the keys', 540 TFLOP/s of the five products that
// count; 4 heads of 128 on 2 take 670 us, in fp16 the two take 707 and 680.
#include "cross.cuh"

namespace gsa {
namespace {


template <int kDim, bool kKeysPass>
struct Shape {
  // The queries' pass of heads up to 64 fits an SM twice, with walked tiles of
  // 64; the others walk 128 rows where tensor memory has room for their scores.
  static constexpr int kBlocks = kDim == 64 && !kKeysPass ? 2 : 1;
  static constexpr int kWalk =
      kBlocks == 2 || (kDim == 128 && kKeysPass) ? 64 : 128;
  static constexpr int kStages = kDim == 64 ? 4 : kKeysPass ? 3 : 2;
  static constexpr int kRowWarps = kBlocks == 2 ? 8 : 16;
  static constexpr int kShare = kRowWarps / 4;  // threads of a row
  static constexpr int kThreads = 32 * (kRowWarps + 3);
  static constexpr int kOwn = kRows * kDim * 2;   // bytes of a resident tile
  static constexpr int kTile = kWalk * kDim * 2;  // of a walked one
  // keys' pass: the further columns of a resident and of a walked tile
  static constexpr int kOwnMore = kKeysPass ? kRows * 32 : 0;
  static constexpr int kTileMore = kKeysPass ? kWalk * 32 : 0;
  static constexpr int kSmem = 1024 + 2 * (kOwn + kOwnMore) +
                               2 * kStages * (kTile + kTileMore);
  static constexpr uint32_t kColumns = 512 / kBlocks;
  static constexpr uint32_t kS = 0, kDp = kWalk, kDs = 2 * kWalk;
  static constexpr uint32_t kP = kDs + kWalk / 2;  // keys' pass
  static constexpr uint32_t kOut1 = kKeysPass ? kP + kWalk / 2 : kP;
  static constexpr uint32_t kOut2 = kOut1 + kDim;  // keys' pass: dv
  static constexpr uint32_t kEnd = kKeysPass ? kOut2 + kDim : kOut2;
  static_assert(kEnd <= kColumns, "tensor memory");
  static_assert(kBlocks * (kSmem + 5120) <= 227 * 1024, "shared memory");
};

struct BackMaps {
  CUtensorMap y1, y2;  // walked: queries and dout, or keys and values
};

enum Bar {
  kTileFull = 0,  // [stage] a walked tile is there
  kTileFree = 4,  // [stage] its products are complete
  kTileRaw = 8,   // [stage] a tile loaded, rows to be cleared
  kScores = 12,   // S and dP are complete
  kRead = 13,     // they are in registers (a count per warp)
  kWeights = 14,  // P and dS are there (a count per warp)
  kOutput = 15,   // the second products are complete
  kBars = 16
};

// The factor that P carries (2^x).
template <typename T>
__device__ __forceinline__ int p_bits() {
  return __is_same(T, __half) ? 15 : 0;
}
// An x with |dout| |v| < 2^x, from their squares.
__device__ __forceinline__ int size_exponent(float d2, float v2) {
  const int e = ((__float_as_int(d2 * v2) >> 23) & 255) - 127;
  return (e + 2) >> 1;
}
// The factor that dS carries (2^x), |dP| and |delta| being below 2^size.
template <typename T>
__device__ __forceinline__ int ds_bits(int size) {
  return __is_same(T, __half) ? 14 - size : 0;
}
__device__ __forceinline__ float power_of_two(int e) {  // -126 to 127
  return __int_as_float((127 + e) << 23);
}

// x as four values of T that stand for multiples of 2^15, 2^7, 2^-4 and 2^-24:
// together they hold an x below 2^31 to 24 bits, or to 2^-41, in fp16 too (what
// is beyond gives NaN there).
template <typename T>
__device__ __forceinline__ uint2 four_parts(float x) {
  constexpr int kExponents[4] = {15, 7, -4, -24};
  float part[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    part[i] = to_float(from_float<T>(x * power_of_two(-kExponents[i])));
    if (i == 0 && !(fabsf(part[0]) < kInf)) {
      if (fabsf(x) < kInf) part[0] = __int_as_float(0x7fffffff);
      break;
    }
    x -= part[i] * power_of_two(kExponents[i]);
  }
  return make_uint2(pack2<T>(part[0], part[1]), pack2<T>(part[2], part[3]));
}
// The other side of their product.
template <typename T>
__device__ __forceinline__ uint2 four_units() {
  return make_uint2(pack2<T>(power_of_two(15), power_of_two(7)),
                    pack2<T>(power_of_two(-4), power_of_two(-24)));
}

// The last 16 columns of a product by columns, from narrow tiles.
template <typename T, int kN>
__device__ __forceinline__ void product_more(uint32_t d, uint32_t a,
                                             uint32_t b) {
  tc::mma(d, tc::by_columns_narrow(a), tc::by_columns_narrow(b),
          tc::instruction<T>(kN, false), true);
}

// Whether one of n keys is open and no more.  By a whole warp.
__device__ __forceinline__ bool single_key(const unsigned char* mask, int n) {
  if (!mask) return n == 1;
  int open = 0;
  for (int k = threadIdx.x & 31; open < 2 && k - (int)(threadIdx.x & 31) < n;
       k += 8 * 32) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      open += __popc(__ballot_sync(
          kFull, k + i * 32 < n && __ldg(mask + k + i * 32)));
  }
  return open == 1;
}

// What the warps of a block share besides the tiles.
template <typename S, bool kKeysPass>
struct Shared {
  uint64_t bars[kBars];
  uint32_t tmem_at;
  float part_delta[kKeysPass ? 1 : S::kShare][kKeysPass ? 1 : kRows];
  float part_size[kKeysPass ? 1 : S::kShare][kKeysPass ? 1 : kRows];
};

// A block's work: rows from r0 on of a scene (n packed rows from q0 on, nk keys
// from k0 on) and of one head of keys, one share of the walked ones.  kOneTile
// (queries' pass): the scene's keys are in one tile; then delta is the sum of P *
// dP, without the rounding of `out`, which would be most of dS's error where
// keys are few.
template <typename T, int kDim, bool kKeysPass, bool kOneTile>
__device__ __forceinline__ void backward_block(
    const CrossArgs& a, const BackMaps& maps,
    Shared<Shape<kDim, kKeysPass>, kKeysPass>& shared, int scene, int q0,
    int n, int k0, int nk, int hk, int split, int r0) {
  using S = Shape<kDim, kKeysPass>;
  constexpr int W = S::kWalk, kRowWarps = S::kRowWarps;
  extern __shared__ uint8_t smem_raw[];
  auto& part_delta = shared.part_delta;

  const int own = kKeysPass ? nk : n, walked = kKeysPass ? n : nk;
  // a walked tile of packed rows holds whole query rows
  const int each = kKeysPass ? W / a.group * a.group : W;
  if (r0 >= own) return;
  int begin, end;
  share((walked + each - 1) / each, a.splits, split, &begin, &end);
  const int nt = end - begin;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t smem = (tc::smem_address(smem_raw) + 1023u) & ~1023u;
  const uint32_t x1 = smem, x2 = smem + S::kOwn, y1 = x2 + S::kOwn,
                 y2 = y1 + S::kStages * S::kTile;
  const uint32_t x1_more = y2 + S::kStages * S::kTile,
                 x2_more = x1_more + S::kOwnMore,
                 y1_more = x2_more + S::kOwnMore,
                 y2_more = y1_more + S::kStages * S::kTileMore;
  const uint32_t bar0 = tc::smem_address(shared.bars);
  const int steps = (a.dim + 15) / 16;
  const unsigned char* mask = a.mask ? a.mask + k0 : nullptr;
  bool ok = true;
  uint32_t tmem = 0;
  auto bar = [&](int which) { return bar0 + which * 8; };
  auto wait = [&](int which, int phase) {
    if (ok) ok = tc::barrier_wait(bar0 + which * 8, phase & 1);
  };
  auto store = [&](uint32_t at, uint32_t u0, uint32_t u1) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %3};" ::"r"(at), "r"(u0),
                 "r"(u1), "r"(0)
                 : "memory");
  };
  constexpr bool kSizes = __is_same(T, __half);
  unsigned* sizes =
      a.sizes + ((long long)scene * a.kv_heads + hk) * (2 + a.value_chunks);
  unsigned v_size = 0;  // queries' pass: of all keys, known to row warps

  // The loading warp: a tile's copies, and what is left to do when they are
  // there.
  const int panels = a.dim > 64 ? 2 : 1;
  int cleared = 0;  // a bit per stage: the phase of its raw barrier
  uint4 values[W / 32];
  const uint4 nothing =  // lse = inf: P = 0
      make_uint4(pack2<T>(-kInf, 0.f), 0, 0, 0);
  auto load_values = [&](int t) {
    const int first = (begin + t) * each;
    const long long at = ((long long)hk * a.n_q + q0) * a.group;
#pragma unroll
    for (int i = 0; i < W / 32; ++i) {
      const int r = first + i * 32 + lane;
      const bool there = t < nt && i * 32 + lane < each && r < n;
      values[i] = there ? a.row_values[at + r] : nothing;
    }
  };
  auto whole = [&](int t, uint32_t* open) {
    const int at = (begin + t) * each;
    if constexpr (kKeysPass) {
      key_words<W>(open, nullptr, 0, min(n - at, each));
      return n - at >= each;
    } else {
      key_words<W>(open, mask, at, nk);
      bool all = true;
#pragma unroll
      for (int i = 0; i < W / 32; ++i) all &= open[i] == 0xffffffffu;
      return all;
    }
  };
  auto issue = [&](int t) {
    const int stage = t % S::kStages;
    const int at = (begin + t) * each;
    const uint32_t t1 = y1 + stage * S::kTile, t2 = y2 + stage * S::kTile;
    uint32_t open[W / 32];
    const int full = (whole(t, open) ? kTileFull : kTileRaw) + stage;
    if (t >= S::kStages) wait(kTileFree + stage, t / S::kStages - 1);
    if (!__all_sync(kFull, ok)) return false;
    if (tc::elect()) {
      tc::barrier_expect(bar(full), 2 * panels * each * 128);
      const int head = kKeysPass ? hk * a.group : hk;
      const int row = kKeysPass ? q0 + at / a.group : k0 + at;
      for (int p = 0; p < panels; ++p) {
        tc::copy_box(t1 + p * W * 128, &maps.y1, bar(full), p * 64, head, row);
        tc::copy_box(t2 + p * W * 128, &maps.y2, bar(full), p * 64, head, row);
      }
    }
    __syncwarp();
    return true;
  };
  auto finish = [&](int t) {
    const int stage = t % S::kStages;
    if constexpr (kKeysPass) {
#pragma unroll
      for (int i = 0; i < W / 32; ++i) {
        const uint32_t to =
            stage * S::kTileMore + tc::narrow_offset(i * 32 + lane, 0);
        store(y1_more + to, values[i].x, values[i].y);
        store(y2_more + to, values[i].z, values[i].w);
      }
      // the next tile's are on their way while its place is waited for
      load_values(t + 1);
    }
    uint32_t open[W / 32];
    const bool all = whole(t, open);
    if (!all) {
      wait(kTileRaw + stage, cleared >> stage);
      cleared ^= 1 << stage;
      __syncwarp();
      clear_rows<W>(y1 + stage * S::kTile, panels, open);
      if constexpr (kKeysPass)
        clear_rows<W>(y2 + stage * S::kTile, panels, open);
    }
    if (!all || kKeysPass) {
      tc::fence_shared();
      __syncwarp();
      // in the keys' pass a tile is there with its copies and its values
      if (lane == 0) {
        tc::barrier_arrive(bar(kTileFull + stage));
        if (!all && kKeysPass) tc::barrier_arrive(bar(kTileFull + stage));
      }
    }
  };

  if (nt > 0) {
    if (warp == kRowWarps) {
      tc::tmem_alloc(tc::smem_address(&shared.tmem_at), S::kColumns);
    } else if (warp == kRowWarps + 1) {
      if (lane == 0) {
        for (int i = 0; i < kBars; ++i)
          tc::barrier_init(bar(i), i == kRead || i == kWeights ? kRowWarps
                                   : kKeysPass && i < kTileFree ? 2
                                                                : 1);
        tc::barriers_ready();
      }
      __syncwarp();
      // the first tiles come while the block gets ready
      for (int t = 0; t < S::kStages && t < nt; ++t) issue(t);
      if constexpr (kKeysPass) load_values(0);
    } else if (warp < kRowWarps) {
      const Chunks c = chunks_of(a.dim, tid, kRowWarps * 32);
      if constexpr (kKeysPass) {
        const T* k = static_cast<const T*>(a.k) + k0 * a.k_row + hk * a.k_head;
        const T* v = static_cast<const T*>(a.v) + k0 * a.v_row + hk * a.v_head;
        load_packed<T, kRows>(c, x1, k, a.k_row, 0, 1, r0, nk);
        load_packed<T, kRows>(c, x2, v, a.v_row, 0, 1, r0, nk);
        // rows that no walked tile fills
        for (int i = each * 8 + tid; i < W * 8; i += kRowWarps * 32)
          for (int s = 0; s < 2 * S::kStages; ++s)
            for (int p = 0; p < kDim / 64; ++p)
              store(y1 + s * S::kTile + p * W * 128 + i * 16, 0, 0);
        // the resident tiles' further columns, and the second half (zeros) of
        // the walked ones'
        if (tid < kRows) {
          const uint2 u = four_units<T>();
          for (int x = 0; x < 2; ++x) {
            const uint32_t to = x ? x2_more : x1_more;
            store(to + tc::narrow_offset(tid, 0), u.x, u.y);
            store(to + tc::narrow_offset(tid, 1), 0, 0);
          }
        }
        if (tid < W)
          for (int s = 0; s < 2 * S::kStages; ++s)
            store(y1_more + s * S::kTileMore + tc::narrow_offset(tid, 1), 0, 0);
      } else {
        // delta = <dout, out>, a share of the row's elements each (of one
        // tile it comes from P and dP instead)
        const int r = min(r0 + (tid & (kRows - 1)), n - 1), qr = r / a.group;
        const int h = hk * a.group + r - qr * a.group;
        const T* o = static_cast<const T*>(a.out) + (q0 + qr) * a.o_row +
                     h * a.o_head;
        const T* d = static_cast<const T*>(a.dout) + (q0 + qr) * a.d_row +
                     h * a.d_head;
        constexpr int kEach = kDim / 8 / S::kShare;
        uint4 u[kEach], v[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int at = ((tid >> 7) + i * S::kShare) * 8;
          u[i] = v[i] = make_uint4(0, 0, 0, 0);
          if (!kOneTile && at < a.dim)
            u[i] = *reinterpret_cast<const uint4*>(o + at);
          if ((!kOneTile || kSizes) && at < a.dim)
            v[i] = *reinterpret_cast<const uint4*>(d + at);
        }
        const long long head = (long long)hk * a.group;
        load_packed<T, kRows>(
            c, x1, static_cast<const T*>(a.q) + q0 * a.q_row + head * a.q_head,
            a.q_row, a.q_head, a.group, r0, n);
        load_packed<T, kRows>(
            c, x2,
            static_cast<const T*>(a.dout) + q0 * a.d_row + head * a.d_head,
            a.d_row, a.d_head, a.group, r0, n);
        float sum = 0.f, square = 0.f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          float x[8], y[8];
          Vec<T>::unpack(u[i], x);
          Vec<T>::unpack(v[i], y);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            sum = fmaf(x[e], y[e], sum);
            if constexpr (kSizes) square = fmaf(y[e], y[e], square);
          }
        }
        part_delta[tid >> 7][tid & (kRows - 1)] = sum;
        if constexpr (kSizes)
          shared.part_size[tid >> 7][tid & (kRows - 1)] = square;
      }
      if constexpr (kSizes && !kKeysPass) {
        for (int i = lane; i < a.value_chunks; i += 32)
          v_size = max(v_size, __ldg(sizes + 2 + i));
        v_size = __reduce_max_sync(kFull, v_size);
      }
      tc::copy_commit();
      tc::copy_wait<0>();
      tc::fence_shared();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    tmem = shared.tmem_at;
  }

  if (warp == kRowWarps + 1) {
    int sent = min(nt, S::kStages);
    for (int t = 0; t < nt; ++t) {
      if (t >= S::kStages && issue(t)) sent = t + 1;
      finish(t);
    }
    // No copy is under way when the block ends, also where a wait ran out.  Rows
    // to be cleared were waited for.
    const bool fine = __all_sync(kFull, ok);
    for (int t = max(sent - S::kStages, 0); t < sent; ++t) {
      const int stage = t % S::kStages;
      uint32_t open[W / 32];
      const bool all = whole(t, open);
      int round = t / S::kStages;
      if (!all && !fine) {
        round = 0;
        for (int u = stage; u < t; u += S::kStages) round += !whole(u, open);
      }
      if (all || !fine)
        tc::barrier_wait(bar((all ? kTileFull : kTileRaw) + stage), round & 1);
    }
  } else if (warp == kRowWarps) {
    for (int t = 0; t < nt; ++t) {
      const int stage = t % S::kStages;
      wait(kTileFull + stage, t / S::kStages);
      if (t > 0) wait(kRead, t - 1);
      tc::fence_after();
      __syncwarp();
      if (tc::elect()) {
        tc::product_by_columns<T, kRows, W, kDim / 16>(
            tmem + S::kS, x1, y1 + stage * S::kTile, steps);
        if constexpr (kKeysPass)
          product_more<T, W>(tmem + S::kS, x1_more,
                             y1_more + stage * S::kTileMore);
        tc::product_by_columns<T, kRows, W, kDim / 16>(
            tmem + S::kDp, x2, y2 + stage * S::kTile, steps);
        if constexpr (kKeysPass)
          product_more<T, W>(tmem + S::kDp, x2_more,
                             y2_more + stage * S::kTileMore);
        tc::commit(bar(kScores));
      }
      __syncwarp();
    }
    // nor is a product
    if (nt > 0) tc::barrier_wait(bar(kScores), (nt - 1) & 1);
  } else if (warp == kRowWarps + 2) {
    for (int t = 0; t < nt; ++t) {
      const int stage = t % S::kStages;
      wait(kWeights, t);
      tc::fence_after();
      __syncwarp();
      if (tc::elect()) {
        tc::product_by_rows<T, W>(tmem + S::kOut1, tmem + S::kDs,
                                  y1 + stage * S::kTile, steps * 16, t > 0);
        if constexpr (kKeysPass)
          tc::product_by_rows<T, W>(tmem + S::kOut2, tmem + S::kP,
                                    y2 + stage * S::kTile, steps * 16, t > 0);
        tc::commit(bar(kOutput));
        tc::commit(bar(kTileFree + stage));
      }
      __syncwarp();
    }
    if (nt > 0) tc::barrier_wait(bar(kOutput), (nt - 1) & 1);
  } else {
    constexpr int kMine = W / S::kShare;  // a thread's columns of its row
    const int part = warp >> 2, group = warp & 3;
    const int r = r0 + group * 32 + lane;
    const bool live = r < own;
    const bool busy = r0 + group * 32 < own;  // the warp holds rows
    const uint32_t mine = tmem + ((uint32_t)group << 21);
    bool open = live;
    float lse2 = -kInf, delta = 0.f;
    int bits = 0;  // the factor that dS carries
    // The scene has one open key, whose P is 1 whatever the scores and its dS
    // 0 (in the keys' pass: which is the warp's).
    bool single = false;
    // what the keys' pass needs of this row
    auto put_values = [&](float minus_delta) {
      const uint2 u = four_parts<T>(lse2 / a.scale_log2e);
      const uint2 v = four_parts<T>(minus_delta);
      a.row_values[((long long)hk * a.n_q + q0) * a.group + r] =
          make_uint4(u.x, u.y, v.x, v.y);
    };
    auto my_word = [&](const uint32_t* words) {  // of this thread's columns
      uint32_t word = words[0];
#pragma unroll
      for (int i = 1; i < W / 32; ++i)
        if (part == i) word = words[i];
      return word;
    };
    if constexpr (kKeysPass) {
      open = live && (!mask || __ldg(mask + r));
      if (__popc(__ballot_sync(kFull, open)) == 1)
        single = single_key(mask, nk);
      if constexpr (kSizes)
        bits = ds_bits<T>(size_exponent(__uint_as_float(__ldg(sizes)),
                                        __uint_as_float(__ldg(sizes + 1))));
    } else if (nt > 0) {
      single = single_key(mask, nk);
      if constexpr (!kOneTile) {
#pragma unroll
        for (int i = 0; i < S::kShare; ++i)
          delta += part_delta[i][group * 32 + lane];
      }
      if (live) {
        const int qr = r / a.group;
        const long long row = q0 + qr;
        const int h = hk * a.group + (r - qr * a.group);
        // a row without keys gets P = 0
        const float x = __ldg(a.lse + row * a.heads + h);
        if (x != -kInf) lse2 = fmaf(x, -kLog2e, (float)p_bits<T>());
        if (!kOneTile && part == 0) put_values(-delta);
      }
      if constexpr (kSizes) {
        float size = 0.f;
#pragma unroll
        for (int i = 0; i < S::kShare; ++i)
          size += shared.part_size[i][group * 32 + lane];
        bits = ds_bits<T>(size_exponent(size, __uint_as_float(v_size)));
        if (part == 0) {
          const unsigned most = __reduce_max_sync(
              kFull, live && size < kInf ? __float_as_uint(size) : 0u);
          if (lane == 0) {
            if (most) atomicMax(sizes, most);
            if (r0 == 0 && group == 0) sizes[1] = v_size;
          }
        }
      }
      delta *= -power_of_two(bits - p_bits<T>());
    }
    const float ds_factor = power_of_two(bits - p_bits<T>());
    __syncwarp();
    const bool all_open = __all_sync(kFull, open);
    const uint64_t scale2 = tc::pair(a.scale_log2e, a.scale_log2e);
    const uint64_t factor2 = tc::pair(ds_factor, ds_factor);
    const uint64_t row_lse2 = tc::pair(lse2, lse2);
    uint64_t row_delta2 = tc::pair(delta, delta);
    if (!busy) {
      for (int t = 0; t < nt; ++t) {
        wait(kScores, t);
        if (lane == 0) tc::barrier_arrive(bar(kRead));
        // no arrival for the next tile before this one's phase is complete
        if (t > 0) wait(kOutput, t - 1);
        if (lane == 0) tc::barrier_arrive(bar(kWeights));
        __syncwarp();
      }
    } else {
      const uint32_t at = mine + part * kMine;
      const uint32_t to = mine + part * (kMine / 2);
      for (int t = 0; t < nt; ++t) {
        uint32_t s[kMine], d[kMine];
        wait(kScores, t);
        __syncwarp();
        tc::fence_after();
        if constexpr (kMine == 32) {
          tc::load32(at + S::kS, s);
          tc::load32(at + S::kDp, d);
        } else {
          tc::load16(at + S::kS, s);
          tc::load16(at + S::kDp, d);
        }
        tc::wait_load();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::barrier_arrive(bar(kRead));
        uint32_t words[W / 32];
        bool some = false;  // keys of the tile are shut or absent
        if constexpr (!kKeysPass) {
          const int first = (begin + t) * W;
          some = mask || first + W > nk;
          if (some) key_words<W>(words, mask, first, nk);
          if constexpr (kOneTile) {
            float sum = 0.f;
            const uint32_t word = some ? my_word(words) : 0xffffffffu;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
              const float w = exp2_fast(
                  fmaf(__uint_as_float(s[i]), a.scale_log2e, lse2));
              if ((word >> i) & 1) sum = fmaf(w, __uint_as_float(d[i]), sum);
            }
            part_delta[part][group * 32 + lane] = sum;
            __syncwarp();
            tc::meet(1 + group, 32 * S::kShare);
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < S::kShare; ++i)
              sum += part_delta[i][group * 32 + lane];
            sum *= power_of_two(-p_bits<T>());
            row_delta2 = tc::pair(-sum * ds_factor, -sum * ds_factor);
            if (live && part == 0) put_values(-sum);
          }
        }
        uint32_t p[kMine / 2], ds[kMine / 2];
#pragma unroll
        for (int i = 0; i < kMine; i += 2) {
          uint64_t x = tc::pair(__uint_as_float(s[i]),
                                __uint_as_float(s[i + 1]));
          uint64_t e = tc::pair(__uint_as_float(d[i]),
                                __uint_as_float(d[i + 1]));
          if constexpr (kKeysPass) {
            x = tc::mul2(x, scale2);
            if constexpr (__is_same(T, __half)) e = tc::mul2(e, factor2);
          } else {
            x = tc::fma2(x, scale2, row_lse2);
            e = tc::fma2(e, factor2, row_delta2);
          }
          float u0, u1, w0, w1;
          tc::unpair(x, &u0, &u1);
          u0 = exp2_fast(u0);
          u1 = exp2_fast(u1);
          tc::unpair(tc::mul2(tc::pair(u0, u1), e), &w0, &w1);
          if constexpr (kKeysPass) p[i / 2] = pack2<T>(u0, u1);
          ds[i / 2] = pack2<T>(w0, w1);
        }
        if constexpr (kKeysPass) {
          if (!all_open) {
#pragma unroll
            for (int i = 0; i < kMine / 2; ++i) {
              p[i] = open ? p[i] : 0u;
              ds[i] = open ? ds[i] : 0u;
            }
          }
        } else {
          if (some) {
            const uint32_t word = my_word(words);
#pragma unroll
            for (int i = 0; i < kMine / 2; ++i) {
              const uint32_t two = word >> (2 * i);
              ds[i] &= ((two & 1) ? 0xffffu : 0u) |
                       ((two & 2) ? 0xffff0000u : 0u);
            }
          }
        }
        // P's and dS's places are free once the last products are complete
        if (t > 0) wait(kOutput, t - 1);
        __syncwarp();
        tc::fence_after();
        if constexpr (kMine == 32) {
          if constexpr (kKeysPass) tc::store16(to + S::kP, p);
          tc::store16(to + S::kDs, ds);
        } else {
          if constexpr (kKeysPass) tc::store8(to + S::kP, p);
          tc::store8(to + S::kDs, ds);
        }
        tc::wait_store();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::barrier_arrive(bar(kWeights));
      }
    }
    if (nt > 0) {
      wait(kOutput, nt - 1);
      __syncwarp();
      tc::fence_after();
    }

    // Results: packed rows of dq, or keys of dk and dv.
    if (busy) {
      long long at;  // element of the first column
      long long parts;
      if constexpr (kKeysPass) {
        at = ((long long)(k0 + r) * a.kv_heads + hk) * a.dim;
        parts = a.n_k * a.kv_heads * a.dim;
      } else {
        const int qr = r / a.group;
        at = ((long long)(q0 + qr) * a.heads + hk * a.group +
              (r - qr * a.group)) * a.dim;
        parts = a.n_q * a.heads * a.dim;
      }
#pragma unroll
      for (int which = 0; which < (kKeysPass ? 2 : 1); ++which) {
        const float f = which    ? power_of_two(-p_bits<T>())
                        : single ? 0.f  // NaN of what is one
                                 : a.scale * power_of_two(-bits);
        T* out = static_cast<T*>(kKeysPass ? (which ? a.dv : a.dk) : a.dq) + at;
        float* sum =
            a.part + ((kKeysPass ? 2 : 1) * split + which) * parts + at;
        for (int i = part * 8; i < a.dim; i += 8 * S::kShare) {
          uint32_t x[8];
          float y[8];
          __syncwarp();
          if (nt > 0) {
            tc::load8(mine + (which ? S::kOut2 : S::kOut1) + i, x);
            tc::wait_load();
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
            y[e] = nt > 0 ? __uint_as_float(x[e]) * f : 0.f;
          if (!live) continue;
          if (a.splits == 1) {
            *reinterpret_cast<uint4*>(out + i) = Vec<T>::pack(y);
          } else {
            float4* o = reinterpret_cast<float4*>(sum + i);
            o[0] = make_float4(y[0], y[1], y[2], y[3]);
            o[1] = make_float4(y[4], y[5], y[6], y[7]);
          }
        }
      }
    }
  }
  if (nt > 0) {
    if (!ok) *a.error = 1;
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == kRowWarps) {
      tc::fence_after();
      tc::tmem_free(tmem, S::kColumns);
    }
  }
}

// kShort (queries' pass): scenes of one tile of keys may be among the others.
// They have code of their own, chosen by the scene, so that a scene's results do
// not depend on the rest of its batch; in one piece with the other it would cost
// longer scenes registers (a training step of 8 x 6,000 rows on 1,500 keys 945 us
// for 920).  It comes first: behind the other it costs 5 rows on 7 keys 22.8 us
// for 20.8, while a scene of 10 rows on 24,000 keys takes 186.8 us for 182.8
// without it.
template <typename T, int kDim, bool kKeysPass, bool kShort>
__global__ void __launch_bounds__(Shape<kDim, kKeysPass>::kThreads,
                                  Shape<kDim, kKeysPass>::kBlocks)
    cross_backward_kernel(const __grid_constant__ CrossArgs a,
                          const __grid_constant__ BackMaps maps) {
  using S = Shape<kDim, kKeysPass>;
  __shared__ Shared<S, kKeysPass> shared;
  unsigned unit = blockIdx.x;
  const int r0 = unit % a.tiles * kRows;
  unit /= a.tiles;
  const int split = unit % a.splits;
  unit /= a.splits;
  const int hk = unit % a.kv_heads;
  const int scene = unit / a.kv_heads;
  const int q0 = __ldg(a.q_seg + scene), k0 = __ldg(a.k_seg + scene);
  const int n = (__ldg(a.q_seg + scene + 1) - q0) * a.group;  // packed rows
  const int nk = __ldg(a.k_seg + scene + 1) - k0;
  if (kShort && nk <= S::kWalk)
    backward_block<T, kDim, kKeysPass, kShort>(a, maps, shared, scene, q0, n, k0,
                                               nk, hk, split, r0);
  else
    backward_block<T, kDim, kKeysPass, false>(a, maps, shared, scene, q0, n, k0,
                                              nk, hk, split, r0);
}

// The largest |v|^2 among the open keys of a chunk, and no |dout|^2 yet.  Maxima
// of bits, whose order is that of the values; what is not finite is left out (it
// makes the results that it reaches NaN whatever the factors).
template <typename T, int kDim>
__global__ void __launch_bounds__(256)
    cross_sizes_kernel(const __grid_constant__ CrossArgs a) {
  constexpr int L = kDim / 8;  // lanes of a row
  __shared__ unsigned tops[8];
  const int hk = blockIdx.y, scene = blockIdx.z;
  const int k0 = __ldg(a.k_seg + scene);
  const int nk = __ldg(a.k_seg + scene + 1) - k0;
  const int first = blockIdx.x * a.value_rows;
  const int rows = min(a.value_rows, nk - first);  // may be negative
  const int chunk = threadIdx.x % L * 8;
  const T* v = static_cast<const T*>(a.v) + ((long long)k0 + first) * a.v_row +
               hk * a.v_head + chunk;
  const unsigned char* mask = a.mask ? a.mask + k0 + first : nullptr;
  float most = 0.f;
#pragma unroll 4
  for (int i0 = 0; i0 < rows; i0 += 256 / L) {
    const int i = i0 + threadIdx.x / L;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (i < rows && chunk < a.dim && (!mask || __ldg(mask + i)))
      u = __ldg(reinterpret_cast<const uint4*>(v + i * a.v_row));
    float x[8], sum = 0.f;
    Vec<T>::unpack(u, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
    for (int o = L / 2; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    if (sum < kInf) most = fmaxf(most, sum);
  }
  const unsigned top = __reduce_max_sync(kFull, __float_as_uint(most));
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x < 32) {
    const unsigned all = __reduce_max_sync(
        kFull, threadIdx.x < 8 ? tops[threadIdx.x] : 0u);
    unsigned* sizes =
        a.sizes + ((long long)scene * a.kv_heads + hk) * (2 + a.value_chunks);
    if (threadIdx.x == 0) {
      sizes[2 + blockIdx.x] = all;
      if (blockIdx.x == 0) sizes[0] = 0;
    }
  }
}

// The parts of a split result added up, four elements a thread.
template <typename T>
__global__ void __launch_bounds__(256)
    cross_sum_kernel(const float* part, long long stride, int splits,
                     long long n, T* out) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float4 s = *reinterpret_cast<const float4*>(part + i);
  for (int k = 1; k < splits; ++k) {
    const float4 x = *reinterpret_cast<const float4*>(part + k * stride + i);
    s.x += x.x;
    s.y += x.y;
    s.z += x.z;
    s.w += x.w;
  }
  *reinterpret_cast<uint2*>(out + i) =
      make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
}

struct Plan {
  long long tiles[2], blocks[2];  // of the keys' pass, of the queries'
  int splits[2];
  long long value_rows, value_chunks;
  long long values, sizes, part;  // bytes
  long long all() const { return values + sizes + part; }
};

Plan backward_plan(const attention_args* a) {
  Plan p;
  const long long rows = a->max_q * (a->heads / a->kv_heads);
  p.tiles[0] = ceil_div(a->max_k, kRows);
  p.tiles[1] = ceil_div(rows, kRows);
  const long long walked[2] = {
      ceil_div(rows, a->dim <= 64 ? Shape<64, true>::kWalk
                                  : Shape<128, true>::kWalk),
      ceil_div(a->max_k, a->dim <= 64 ? Shape<64, false>::kWalk
                                      : Shape<128, false>::kWalk)};
  for (int i = 0; i < 2; ++i) {
    const int room = multiprocessors() * (i && a->dim <= 64 ? 2 : 1);
    p.blocks[i] = p.tiles[i] * a->scenes * a->kv_heads;
    p.splits[i] = split_count(p.blocks[i], walked[i], room);
    p.blocks[i] *= p.splits[i];
  }
  p.values = 16 * a->n_q * a->heads;
  p.value_rows = p.value_chunks = p.sizes = 0;
  if (a->type == kF16 && a->max_k) {
    // at most 128 chunks, which a warp reads at once
    p.value_rows = ceil_div(a->max_k, 128) < 64 ? 64 : ceil_div(a->max_k, 128);
    p.value_chunks = ceil_div(a->max_k, p.value_rows);
    p.sizes =
        ceil_div(a->scenes * a->kv_heads * (2 + p.value_chunks), 4) * 16;
  }
  // the two passes' parts follow one another in the same place
  const long long keys =
      p.splits[0] == 1 ? 0
                       : 8 * p.splits[0] * a->n_k * a->kv_heads * a->dim;
  const long long queries =
      p.splits[1] == 1 ? 0 : 4 * p.splits[1] * a->n_q * a->heads * a->dim;
  p.part = keys > queries ? keys : queries;
  return p;
}

template <typename T, int kDim, bool kKeysPass, bool kShort>
cudaError_t launch_pass(CrossArgs a, const attention_args* in, const Plan& p,
                        cudaStream_t s) {
  using S = Shape<kDim, kKeysPass>;
  a.tiles = (int)p.tiles[kKeysPass ? 0 : 1];
  a.splits = p.splits[kKeysPass ? 0 : 1];
  const long long grid = p.blocks[kKeysPass ? 0 : 1];
  if (grid == 0) return cudaSuccess;
  BackMaps maps = {};
  cudaError_t e = cudaSuccess;
  if (kKeysPass && a.n_q) {
    e = row_map(&maps.y1, in->type, in->q, a.dim, a.heads, a.n_q, a.group,
                S::kWalk / a.group);
    if (!e)
      e = row_map(&maps.y2, in->type, in->dout, a.dim, a.heads, a.n_q, a.group,
                  S::kWalk / a.group);
  } else if (!kKeysPass && a.n_k) {
    e = row_map(&maps.y1, in->type, in->k, a.dim, a.kv_heads, a.n_k, 1,
                S::kWalk);
    if (!e)
      e = row_map(&maps.y2, in->type, in->v, a.dim, a.kv_heads, a.n_k, 1,
                  S::kWalk);
  }
  if (!e)
    e = cudaFuncSetAttribute(cross_backward_kernel<T, kDim, kKeysPass, kShort>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             S::kSmem);
  if (e) return e;
  count_launches(1);
  cross_backward_kernel<T, kDim, kKeysPass, kShort>
      <<<(unsigned)grid, S::kThreads, S::kSmem, s>>>(a, maps);
  if (a.splits > 1) {
    const long long n =
        kKeysPass ? a.n_k * a.kv_heads * a.dim : a.n_q * a.heads * a.dim;
    const unsigned blocks = (unsigned)ceil_div(n, 1024);
    count_launches(kKeysPass ? 2 : 1);
    if (kKeysPass) {
      cross_sum_kernel<T><<<blocks, 256, 0, s>>>(a.part, 2 * n, a.splits, n,
                                                 static_cast<T*>(a.dk));
      cross_sum_kernel<T><<<blocks, 256, 0, s>>>(
          a.part + n, 2 * n, a.splits, n, static_cast<T*>(a.dv));
    } else {
      cross_sum_kernel<T><<<blocks, 256, 0, s>>>(a.part, n, a.splits, n,
                                                 static_cast<T*>(a.dq));
    }
  }
  return cudaGetLastError();
}

// The queries' pass first: it leaves its rows' lse and delta to the keys'.
template <typename T, int kDim>
cudaError_t launch(const CrossArgs& a, const attention_args* in, const Plan& p,
                   cudaStream_t s) {
  if (__is_same(T, __half) && p.sizes) {
    count_launches(1);
    cross_sizes_kernel<T, kDim>
        <<<dim3(a.value_chunks, a.kv_heads, a.scenes), 256, 0, s>>>(a);
  }
  const bool one_long = a.scenes == 1 && a.n_k > Shape<kDim, false>::kWalk;
  const cudaError_t e = one_long
                            ? launch_pass<T, kDim, false, false>(a, in, p, s)
                            : launch_pass<T, kDim, false, true>(a, in, p, s);
  return e ? e : launch_pass<T, kDim, true, false>(a, in, p, s);
}

}  // namespace
}  // namespace gsa

using namespace gsa;

// See include/point_features.h.
GSA_API int64_t cross_attention_grad_workspace(const attention_args* in) {
  if (!cross_sizes(in)) return -2;
  const Plan p = backward_plan(in);
  return p.all();
}

// See include/point_features.h.
GSA_API int cross_attention_grad(const attention_args* in) {
  if (!cross_sizes(in) || !attention_scale(in->scale)) return -2;
  const long long type = in->type;
  if (!in->n_q && !in->n_k) return 0;
  if (!in->q_seg || !in->k_seg || !in->error) return -2;
  if (in->n_q &&
      (!vector_rows(in->q, type) || !vector_rows(in->out, type) ||
       !vector_rows(in->dout, type) || !vector_address(in->dq) || !in->lse))
    return -2;
  if (in->n_k && (!vector_rows(in->k, type) || !vector_rows(in->v, type) ||
                  !vector_address(in->dk) || !vector_address(in->dv)))
    return -2;
  const Plan p = backward_plan(in);
  if (p.blocks[0] > kMaxInt || p.blocks[1] > kMaxInt) return -2;
  if (p.all() && (!vector_address(in->workspace) ||
                  in->workspace_bytes < p.all()))
    return -2;
  CrossArgs a = cross_arguments(in);
  a.out = in->out.data;
  a.dout = in->dout.data;
  a.d_row = in->dout.row;
  a.d_head = in->dout.head;
  char* at = static_cast<char*>(in->workspace);
  a.row_values = reinterpret_cast<uint4*>(at);
  a.sizes = reinterpret_cast<unsigned*>(at + p.values);
  a.value_rows = (int)p.value_rows;
  a.value_chunks = (int)p.value_chunks;
  a.part = reinterpret_cast<float*>(at + p.all() - p.part);
  a.dq = in->dq;
  a.dk = in->dk;
  a.dv = in->dv;
  cudaStream_t s = (cudaStream_t)in->stream;
  if (type == kF16)
    return a.dim <= 64 ? launch<__half, 64>(a, in, p, s)
                       : launch<__half, 128>(a, in, p, s);
  return a.dim <= 64 ? launch<__nv_bfloat16, 64>(a, in, p, s)
                     : launch<__nv_bfloat16, 128>(a, in, p, s);
}
