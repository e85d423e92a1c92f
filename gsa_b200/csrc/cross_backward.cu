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
// A block has eight warps of rows (two threads share a row, half of the walked
// columns each), one that issues products, one that loads walked tiles (TMA;
// rows behind the scene's last and shut keys are cleared).  The scores of the
// next tile are taken as soon as this one's are in registers, so products run
// beside the exponentials; P and dS have columns of their own.
//
// P and dS are rounded to the inputs' type for their products (half a step).
// For fp16, whose smallest normal is 2^-14, P carries a factor of 2^15 (it is
// at most 1) and dS one that grows with the number of keys.
//
// What bounds it, for 128 x 128 scores and a head of 64: 1,024 clocks of
// products in the keys' pass (768 in the queries') beside 1,024 of
// exponentials.
#include "cross.cuh"

namespace gsa {
namespace {

constexpr int kRowWarps = 8;
constexpr int kBackThreads = 32 * (kRowWarps + 2);

template <int kDim, bool kKeysPass>
struct Shape {
  // Rows of a walked tile: 128 where tensor memory has room for their scores.
  static constexpr int kWalk = kDim == 128 && kKeysPass ? 64 : 128;
  static constexpr int kStages = kDim == 128 && !kKeysPass ? 2 : 3;
  static constexpr int kOwn = kRows * kDim * 2;    // bytes of a resident tile
  static constexpr int kTile = kWalk * kDim * 2;   // of a walked one
  static constexpr int kSmem = 1024 + 2 * kOwn + 2 * kStages * kTile;
  static constexpr uint32_t kColumns = 512;
  static constexpr uint32_t kS = 0, kDp = kWalk, kDs = 2 * kWalk;
  static constexpr uint32_t kP = kDs + kWalk / 2;  // keys' pass
  static constexpr uint32_t kOut1 = kKeysPass ? kP + kWalk / 2 : kP;
  static constexpr uint32_t kOut2 = kOut1 + kDim;  // keys' pass: dv
  static constexpr uint32_t kEnd = kKeysPass ? kOut2 + kDim : kOut2;
  static_assert(kEnd <= kColumns, "tensor memory");
  static_assert(kSmem <= 225 * 1024, "shared memory");
};

struct BackMaps {
  CUtensorMap y1, y2;  // walked: queries and dout, or keys and values
};

enum Bar {
  kTileFull = 0,    // [stage] a walked tile and its rows' values are there
  kTileFree = 3,    // [stage] its products are complete
  kTileRaw = 6,     // a tile loaded, rows to be cleared
  kScores = 7,  // S and dP are complete
  kRead = 8,    // S and dP are in registers (a count per warp of rows)
  kWeights = 9,  // P and dS are there (a count per warp of rows)
  kOutput = 10,  // the second products are complete
  kBars = 11
};

// Factors that P and dS carry (2^x).
template <typename T>
__device__ __forceinline__ float p_bits() {
  return __is_same(T, __half) ? 15.f : 0.f;
}
template <typename T>
__device__ __forceinline__ float ds_bits(int keys) {
  if (!__is_same(T, __half)) return 0.f;
  const int b = 31 - __clz(keys | 1) - 10;
  return b > 0 ? (float)b : 0.f;
}

template <typename T, int kDim, bool kKeysPass>
__global__ void __launch_bounds__(kBackThreads, 1)
    cross_backward_kernel(const __grid_constant__ CrossArgs a,
                          const __grid_constant__ BackMaps maps) {
  using S = Shape<kDim, kKeysPass>;
  constexpr int W = S::kWalk;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[kBars];
  __shared__ uint32_t tmem_at;
  // -lse (base 2, less the factor that P carries) and -delta of the walked rows
  __shared__ __align__(16) float row_lse[S::kStages][W];
  __shared__ __align__(16) float row_delta[S::kStages][W];

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
  const uint32_t bar0 = tc::smem_address(bars);
  const int steps = (a.dim + 15) / 16;
  const unsigned char* mask = a.mask ? a.mask + k0 : nullptr;
  bool ok = true;
  uint32_t tmem = 0;
  auto bar = [&](int which) { return bar0 + which * 8; };
  auto wait = [&](int which, int phase) {
    if (ok) ok = tc::barrier_wait(bar0 + which * 8, phase & 1);
  };
  const float bits = ds_bits<T>(nk);
  const float ds_factor = exp2f(bits - p_bits<T>());

  if (nt > 0) {
    if (warp == kRowWarps) {
      tc::tmem_alloc(tc::smem_address(&tmem_at), S::kColumns);
      if (lane == 0) {
        for (int i = 0; i < kBars; ++i)
          tc::barrier_init(bar(i), i == kRead || i == kWeights ? kRowWarps : 1);
        tc::barriers_ready();
      }
      __syncwarp();
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
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                               y1 + s * S::kTile + p * W * 128 + i * 16),
                           "r"(0)
                           : "memory");
      } else {
        const long long head = (long long)hk * a.group;
        load_packed<T, kRows>(
            c, x1, static_cast<const T*>(a.q) + q0 * a.q_row + head * a.q_head,
            a.q_row, a.q_head, a.group, r0, n);
        load_packed<T, kRows>(
            c, x2,
            static_cast<const T*>(a.dout) + q0 * a.d_row + head * a.d_head,
            a.d_row, a.d_head, a.group, r0, n);
      }
      tc::copy_commit();
      tc::copy_wait<0>();
      tc::fence_shared();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    tmem = tmem_at;
  }

  if (warp == kRowWarps + 1) {
    const int panels = a.dim > 64 ? 2 : 1;
    int cleared = 0;
    for (int t = 0; t < nt; ++t) {
      const int stage = t % S::kStages;
      const int at = (begin + t) * each;
      const uint32_t t1 = y1 + stage * S::kTile, t2 = y2 + stage * S::kTile;
      uint32_t open[W / 32];
      bool whole = true;
      if constexpr (kKeysPass) {
        key_words<W>(open, nullptr, 0, min(n - at, each));
        whole = n - at >= each;
      } else {
        key_words<W>(open, mask, at, nk);
#pragma unroll
        for (int i = 0; i < W / 32; ++i) whole &= open[i] == 0xffffffffu;
      }
      float lse[W / 32], delta[W / 32];
      if constexpr (kKeysPass) {
#pragma unroll
        for (int i = 0; i < W / 32; ++i) {
          const int r = at + i * 32 + lane;
          lse[i] = -kInf;  // P = 0: an absent row, or one without keys
          delta[i] = 0.f;
          if (i * 32 + lane < each && r < n) {
            const int qr = r / a.group;
            const long long e = (long long)(q0 + qr) * a.heads +
                                hk * a.group + (r - qr * a.group);
            const float x = __ldg(a.lse + e);
            if (x != -kInf) lse[i] = fmaf(x, -kLog2e, p_bits<T>());
            delta[i] = -a.delta[e] * ds_factor;
          }
        }
      }
      if (t >= S::kStages) wait(kTileFree + stage, t / S::kStages - 1);
      if constexpr (kKeysPass) {
#pragma unroll
        for (int i = 0; i < W / 32; ++i) {
          row_lse[stage][i * 32 + lane] = lse[i];
          row_delta[stage][i * 32 + lane] = delta[i];
        }
      }
      const int full = whole ? kTileFull + stage : kTileRaw;
      __syncwarp();
      if (tc::elect()) {
        tc::barrier_expect(bar(full), 2 * panels * each * 128);
        for (int p = 0; p < panels; ++p) {
          if constexpr (kKeysPass) {
            const int head = hk * a.group, row = q0 + at / a.group;
            tc::copy_box(t1 + p * W * 128, &maps.y1, bar(full), p * 64, head,
                         row);
            tc::copy_box(t2 + p * W * 128, &maps.y2, bar(full), p * 64, head,
                         row);
          } else {
            tc::copy_box(t1 + p * W * 128, &maps.y1, bar(full), p * 64, hk,
                         k0 + at);
            tc::copy_box(t2 + p * W * 128, &maps.y2, bar(full), p * 64, hk,
                         k0 + at);
          }
        }
      }
      if (!whole) {
        wait(kTileRaw, cleared++);
        __syncwarp();
        clear_rows<W>(t1, panels, open);
        clear_rows<W>(t2, panels, open);
        tc::fence_shared();
        __syncwarp();
        if (lane == 0) tc::barrier_arrive(bar(kTileFull + stage));
      }
    }
  } else if (warp == kRowWarps) {
    auto scores = [&](int t) {
      const int stage = t % S::kStages;
      tc::fence_after();
      __syncwarp();
      if (tc::elect()) {
        tc::product_by_columns<T, kRows, W, kDim / 16>(
            tmem + S::kS, x1, y1 + stage * S::kTile, steps);
        tc::product_by_columns<T, kRows, W, kDim / 16>(
            tmem + S::kDp, x2, y2 + stage * S::kTile, steps);
        tc::commit(bar(kScores));
      }
      __syncwarp();
    };
    if (nt > 0) {
      wait(kTileFull, 0);
      scores(0);
    }
    for (int t = 0; t < nt; ++t) {
      const int stage = t % S::kStages;
      if (t + 1 < nt) {
        wait(kTileFull + (t + 1) % S::kStages, (t + 1) / S::kStages);
        wait(kRead, t);
        scores(t + 1);
      }
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
  } else {
    constexpr int kMine = W / 2;  // a thread's columns of its row
    const int half = warp >> 2, group = warp & 3;
    const int in_tile = group * 32 + lane;
    const int r = r0 + in_tile;
    const bool live = r < own;
    const bool busy = r0 + group * 32 < own;  // the warp holds rows
    const uint32_t mine = tmem + ((uint32_t)group << 21);
    bool open = live;
    float lse2 = -kInf, delta = 0.f;
    if constexpr (kKeysPass) {
      open = live && (!mask || __ldg(mask + r));
    } else if (nt > 0) {
      const int qr = live ? r / a.group : 0;
      const int h = hk * a.group + (live ? r - qr * a.group : 0);
      const long long row = q0 + qr;
      if (live) {
        const T* o = static_cast<const T*>(a.out) + row * a.o_row +
                     h * a.o_head;
        const T* d = static_cast<const T*>(a.dout) + row * a.d_row +
                     h * a.d_head;
        for (int i = 0; i < a.dim; i += 8) {
          float x[8], y[8];
          Vec<T>::unpack(*reinterpret_cast<const uint4*>(o + i), x);
          Vec<T>::unpack(*reinterpret_cast<const uint4*>(d + i), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) delta = fmaf(x[e], y[e], delta);
        }
        const long long e = row * a.heads + h;
        if (half == 0) a.delta[e] = delta;
        const float x = __ldg(a.lse + e);
        if (x != -kInf) lse2 = fmaf(x, -kLog2e, p_bits<T>());
      }
      delta *= -ds_factor;
    }
    __syncwarp();
    const bool all_open = __all_sync(kFull, open);
    const uint64_t scale2 = tc::pair(a.scale_log2e, a.scale_log2e);
    const uint64_t factor2 = tc::pair(ds_factor, ds_factor);
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
      for (int t = 0; t < nt; ++t) {
        const int stage = t % S::kStages;
        uint32_t s[kMine], d[kMine];
        if constexpr (kKeysPass) wait(kTileFull + stage, t / S::kStages);
        wait(kScores, t);
        __syncwarp();
        tc::fence_after();
#pragma unroll
        for (int i = 0; i < kMine; i += 32) {
          tc::load32(mine + S::kS + half * kMine + i, s + i);
          tc::load32(mine + S::kDp + half * kMine + i, d + i);
        }
        tc::wait_load();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::barrier_arrive(bar(kRead));
        bool whole = true;
        uint32_t words[W / 32];
        if constexpr (!kKeysPass) {
          const int at = (begin + t) * W;
          if (mask || at + W > nk) {
            key_words<W>(words, mask, at, nk);
            whole = false;
          }
        } else {
          whole = all_open;
        }
        uint32_t p[kMine / 2], ds[kMine / 2];
#pragma unroll
        for (int i = 0; i < kMine; i += 4) {
          uint64_t l[2], e[2];
          if constexpr (kKeysPass) {
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(
                &row_lse[stage][half * kMine + i]);
            const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(
                &row_delta[stage][half * kMine + i]);
            l[0] = x.x;
            l[1] = x.y;
            e[0] = y.x;
            e[1] = y.y;
          } else {
            l[0] = l[1] = tc::pair(lse2, lse2);
            e[0] = e[1] = tc::pair(delta, delta);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int c = i + 2 * j;
            float u0, u1, w0, w1;
            tc::unpair(tc::fma2(tc::pair(__uint_as_float(s[c]),
                                         __uint_as_float(s[c + 1])),
                                scale2, l[j]), &u0, &u1);
            u0 = exp2_fast(u0);
            u1 = exp2_fast(u1);
            tc::unpair(
                tc::mul2(tc::pair(u0, u1),
                         tc::fma2(tc::pair(__uint_as_float(d[c]),
                                           __uint_as_float(d[c + 1])),
                                  factor2, e[j])),
                &w0, &w1);
            if constexpr (kKeysPass) p[c / 2] = pack2<T>(u0, u1);
            ds[c / 2] = pack2<T>(w0, w1);
          }
        }
        if (!whole) {
#pragma unroll
          for (int i = 0; i < kMine / 2; ++i) {
            uint32_t keep;
            if constexpr (kKeysPass) {
              keep = open ? 0xffffffffu : 0u;
              p[i] &= keep;
            } else {
              const uint32_t word =
                  half ? words[W / 64 + i / 16] : words[i / 16];
              const uint32_t two = word >> ((2 * i) & 31);
              keep = ((two & 1) ? 0xffffu : 0u) |
                     ((two & 2) ? 0xffff0000u : 0u);
            }
            ds[i] &= keep;
          }
        }
        // P's and dS's places are free once the last products are complete
        if (t > 0) wait(kOutput, t - 1);
        __syncwarp();
        tc::fence_after();
#pragma unroll
        for (int i = 0; i < kMine / 2; i += 16) {
          if constexpr (kKeysPass)
            tc::store16(mine + S::kP + half * (kMine / 2) + i, p + i);
          tc::store16(mine + S::kDs + half * (kMine / 2) + i, ds + i);
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
        const float f = which ? exp2f(-p_bits<T>()) : a.scale * exp2f(-bits);
        T* out = static_cast<T*>(kKeysPass ? (which ? a.dv : a.dk) : a.dq) + at;
        float* part =
            a.part + ((kKeysPass ? 2 : 1) * split + which) * parts + at;
        for (int i = half * 8; i < a.dim; i += 16) {
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
            float4* o = reinterpret_cast<float4*>(part + i);
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
  long long delta, part;  // bytes
};

Plan backward_plan(const attention_args* a) {
  Plan p;
  const long long rows = a->max_q * (a->heads / a->kv_heads);
  const int room = multiprocessors();
  p.tiles[0] = ceil_div(a->max_k, kRows);
  p.tiles[1] = ceil_div(rows, kRows);
  const long long walked[2] = {ceil_div(rows, a->dim <= 64 ? 128 : 64),
                               ceil_div(a->max_k, 128)};
  for (int i = 0; i < 2; ++i) {
    p.blocks[i] = p.tiles[i] * a->scenes * a->kv_heads;
    p.splits[i] = split_count(p.blocks[i], walked[i], room);
    p.blocks[i] *= p.splits[i];
  }
  p.delta = (a->n_q * a->heads * 4 + 15) / 16 * 16;
  // the two passes' parts follow one another in the same place
  const long long keys =
      p.splits[0] == 1 ? 0
                       : 8 * p.splits[0] * a->n_k * a->kv_heads * a->dim;
  const long long queries =
      p.splits[1] == 1 ? 0 : 4 * p.splits[1] * a->n_q * a->heads * a->dim;
  p.part = keys > queries ? keys : queries;
  return p;
}

template <typename T, int kDim, bool kKeysPass>
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
    e = cudaFuncSetAttribute(cross_backward_kernel<T, kDim, kKeysPass>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                           S::kSmem);
  if (e) return e;
  count_launches(1);
  cross_backward_kernel<T, kDim, kKeysPass>
      <<<(unsigned)grid, kBackThreads, S::kSmem, s>>>(a, maps);
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

// The queries' pass first: it leaves delta to the keys'.
template <typename T>
cudaError_t launch(const CrossArgs& a, const attention_args* in, const Plan& p,
                   cudaStream_t s) {
  cudaError_t e = a.dim <= 64 ? launch_pass<T, 64, false>(a, in, p, s)
                              : launch_pass<T, 128, false>(a, in, p, s);
  if (e) return e;
  return a.dim <= 64 ? launch_pass<T, 64, true>(a, in, p, s)
                     : launch_pass<T, 128, true>(a, in, p, s);
}

}  // namespace
}  // namespace gsa

using namespace gsa;

// See include/point_features.h.
GSA_API int64_t cross_attention_grad_workspace(const attention_args* in) {
  if (!cross_sizes(in)) return -2;
  const Plan p = backward_plan(in);
  return p.delta + p.part;
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
  if (p.delta + p.part && (!vector_address(in->workspace) ||
                           in->workspace_bytes < p.delta + p.part))
    return -2;
  CrossArgs a = cross_arguments(in);
  a.out = in->out.data;
  a.dout = in->dout.data;
  a.d_row = in->dout.row;
  a.d_head = in->dout.head;
  a.delta = static_cast<float*>(in->workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(in->workspace) +
                                    p.delta);
  a.dq = in->dq;
  a.dk = in->dk;
  a.dv = in->dv;
  cudaStream_t s = (cudaStream_t)in->stream;
  return type == kF16 ? launch<__half>(a, in, p, s)
                      : launch<__nv_bfloat16>(a, in, p, s);
}
