// SPDX-License-Identifier: Apache-2.0
// Cross attention between two levels of a hierarchy: the queries of scene i
// read the keys and values of scene i,
//
//   s = scale q k^T,  out = softmax(s) v,  lse = log sum exp s,
//
// over the scene's open keys; a row without any gives 0 and lse = -inf, one
// whose scores are all -inf has no softmax and gives NaN for both.
//
// A block owns 128 packed query rows, a row per thread, and walks the keys in
// tiles of 128.  A fifth warp issues the products (tcgen05), a sixth loads the
// tiles (TMA): one warp for both took longer over a tile than its rows did.
// S = Q K^T comes from tensor memory into registers, the running maximum and
// sum are kept in 32 bits, and P = exp(S - max), rounded to the inputs' type
// for the second product (half a step, 2^-8 for bf16, on weights that are
// summed in 32 bits), goes back to tensor memory, from where O += P V takes
// it.  The maximum that P is taken against may lag the true one by a factor of
// 2^8, so that O is rescaled only when it grew by more.  Value rows of shut or
// absent keys are cleared in shared memory before their product, so that
// whatever lies there takes no part.
//
// What bounds it: a row's chain of waits, softmax and waits again, which only
// another block's work can fill; two blocks share an SM (256 columns of
// tensor memory, at most 97 KB of shared memory each).  Below that lie the
// exponentials (16 a clock on an SM; a quarter are polynomials in the
// multiply-add units) up to a head of 128, where the products take as long.
// 8 x 24,000 queries on 6,000 keys, 4 heads of 128: 2.46 to 2.50 ms replayed from
// a graph (2.18 before the clock falls with the power limit), 2.54 ms as a call,
// 929 TFLOP/s; 8 x 6,000 on 1,500, 8 heads of 64: 242 us replayed, 609 TFLOP/s,
// and 252 us as a call.  Tiles of 64 keys with four blocks on an SM
// took 253 to 274 us and 2.7 to 2.8 ms, two threads per row 268 us and 2.68 ms;
// no polynomials, or a third, 2 to 3 % more.
//
// Where there are too few row tiles to fill the GPU, the keys are split among
// blocks and the parts joined by their lse.
#include "cross.cuh"

namespace gsa {
namespace {

constexpr int kKeys = 128;  // keys of a tile

// Head size up to kDim (64 or 128).  The larger one has room for one tile of
// keys and values in shared memory, and for P in tensor memory only where S
// was: its next scores wait for the product that reads P.
template <int kDim>
struct Shape {
  static constexpr int kStages = kDim == 64 ? 2 : 1;
  static constexpr bool kOverwrite = kDim == 128;
  static constexpr int kQ = kRows * kDim * 2;  // bytes
  static constexpr int kTile = kKeys * kDim * 2;
  static constexpr int kSmem = 1024 + kQ + 2 * kStages * kTile;
  static constexpr uint32_t kColumns = 256;
  static constexpr uint32_t kS = 0, kP = kOverwrite ? 0 : 128,
                            kO = kOverwrite ? 128 : 192;
  static_assert(kO + kDim == kColumns, "tensor memory");
};

struct Maps {
  CUtensorMap q, k, v;
};

enum Bar {
  kKeysFull = 0,    // [stage] the keys are there
  kKeysFree = 2,    // [stage] the scores that read them are complete
  kValuesFull = 4,  // [stage]
  kValuesFree = 6,  // [stage]
  kValuesRaw = 8,   // [stage] values loaded, rows to be cleared
  kScores = 10,     // S is complete
  kScoresRead = 11,  // S is in registers (a count per warp of rows)
  kWeights = 12,    // P is there (a count per warp of rows)
  kOutput = 13,     // O += P V is complete
  kQueries = 14,    // Q is there
  kBars = 15
};

// The largest of three, NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, 2)
    cross_forward_kernel(const __grid_constant__ CrossArgs a,
                         const __grid_constant__ Maps maps) {
  using S = Shape<kDim>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[kBars];
  __shared__ uint32_t tmem_at;

  const int split = a.splits > 1 ? blockIdx.x / a.tiles : 0;
  const int hk = blockIdx.y, scene = blockIdx.z;
  const int each = kRows / a.group * a.group;  // whole query rows
  const int r0 = (blockIdx.x - split * a.tiles) * each;
  const int q0 = __ldg(a.q_seg + scene), k0 = __ldg(a.k_seg + scene);
  const int n = (__ldg(a.q_seg + scene + 1) - q0) * a.group;  // packed rows
  const int nk = __ldg(a.k_seg + scene + 1) - k0;
  if (r0 >= n) return;
  int begin, end;
  share((nk + kKeys - 1) / kKeys, a.splits, split, &begin, &end);
  const int nt = end - begin;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t smem = (tc::smem_address(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_tile = smem, k_tile = smem + S::kQ,
                 v_tile = k_tile + S::kStages * S::kTile;
  const uint32_t bar0 = tc::smem_address(bars);
  const unsigned char* mask = a.mask ? a.mask + k0 : nullptr;
  uint32_t tmem = 0;
  bool ok = true;
  auto bar = [&](int which) { return bar0 + which * 8; };
  auto wait = [&](int which, int phase) {
    if (ok) ok = tc::barrier_wait(bar0 + which * 8, phase & 1);
  };
  // The loading warp: a tile's copies, and what is left to do when they are
  // there.
  const int panels = a.dim > 64 ? 2 : 1;
  int cleared = 0;  // a bit per stage: the phase of its raw barrier
  auto whole = [&](int t, uint32_t* open) {
    key_words<kKeys>(open, mask, (begin + t) * kKeys, nk);
    return (open[0] & open[1] & open[2] & open[3]) == 0xffffffffu;
  };
  auto issue = [&](int t) {
    const int stage = t % S::kStages, round = t / S::kStages;
    const int at = k0 + (begin + t) * kKeys;
    uint32_t open[kKeys / 32];
    const int full = (whole(t, open) ? kValuesFull : kValuesRaw) + stage;
    if (round > 0) wait(kKeysFree + stage, round - 1);
    if (!__all_sync(kFull, ok)) return false;
    if (tc::elect()) {
      tc::barrier_expect(bar(kKeysFull + stage), panels * kKeys * 128);
      for (int p = 0; p < panels; ++p)
        tc::copy_box(k_tile + stage * S::kTile + p * kKeys * 128, &maps.k,
                     bar(kKeysFull + stage), p * 64, hk, at);
    }
    if (round > 0) wait(kValuesFree + stage, round - 1);
    if (!__all_sync(kFull, ok)) return false;
    if (tc::elect()) {
      tc::barrier_expect(bar(full), panels * kKeys * 128);
      for (int p = 0; p < panels; ++p)
        tc::copy_box(v_tile + stage * S::kTile + p * kKeys * 128, &maps.v,
                     bar(full), p * 64, hk, at);
    }
    __syncwarp();
    return true;
  };
  auto finish = [&](int t) {
    const int stage = t % S::kStages;
    uint32_t open[kKeys / 32];
    if (whole(t, open)) return;
    wait(kValuesRaw + stage, cleared >> stage);
    cleared ^= 1 << stage;
    __syncwarp();
    clear_rows<kKeys>(v_tile + stage * S::kTile, panels, open);
    tc::fence_shared();
    __syncwarp();
    if (lane == 0) tc::barrier_arrive(bar(kValuesFull + stage));
  };

  if (nt > 0) {
    if (warp == 4) {
      tc::tmem_alloc(tc::smem_address(&tmem_at), S::kColumns);
    } else if (warp == 5) {
      if (lane == 0) {
        for (int i = 0; i < kBars; ++i)
          tc::barrier_init(bar(i), i == kScoresRead || i == kWeights ? 4 : 1);
        tc::barriers_ready();
      }
      __syncwarp();
      // the first tiles come while the block gets ready.  Rows of Q behind the
      // scene's last hold whatever follows, which no other row sees.
      if (tc::elect()) {
        tc::barrier_expect(bar(kQueries), panels * each * 128);
        for (int p = 0; p < panels; ++p)
          tc::copy_box(q_tile + p * kRows * 128, &maps.q, bar(kQueries), p * 64,
                       hk * a.group, q0 + r0 / a.group);
      }
      __syncwarp();
      for (int t = 0; t < S::kStages && t < nt; ++t) issue(t);
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    tmem = tmem_at;
  }

  if (warp == 5) {
    int sent = min(nt, S::kStages);
    for (int t = 0; t < nt; ++t) {
      if (t >= S::kStages && issue(t)) sent = t + 1;
      finish(t);
    }
    // No copy is under way when the block ends, also where a wait ran out (then
    // a tile's keys may have been the last).  Rows to be cleared were waited for.
    if (nt > 0) {
      const bool fine = __all_sync(kFull, ok);
      tc::barrier_wait(bar(kQueries), 0);
      for (int t = max(sent - S::kStages, 0); t < sent + !fine; ++t) {
        const int stage = t % S::kStages;
        tc::barrier_wait(bar(kKeysFull + stage), t / S::kStages & 1);
        uint32_t open[kKeys / 32];
        const bool all = whole(t, open);
        int round = t / S::kStages;
        if (!all && !fine) {
          round = 0;
          for (int u = stage; u < t; u += S::kStages) round += !whole(u, open);
        }
        if (all || !fine)
          tc::barrier_wait(bar((all ? kValuesFull : kValuesRaw) + stage),
                           round & 1);
      }
    }
  } else if (warp == 4) {
    const int steps = (a.dim + 15) / 16;
    auto scores = [&](int t) {  // its keys are there
      tc::fence_after();
      __syncwarp();
      if (tc::elect()) {
        tc::product_by_columns<T, kRows, kKeys, kDim / 16>(
            tmem + S::kS, q_tile, k_tile + t % S::kStages * S::kTile, steps);
        tc::commit(bar(kScores));
        tc::commit(bar(kKeysFree + t % S::kStages));
      }
      __syncwarp();
    };
    if (nt > 0) {
      wait(kQueries, 0);
      wait(kKeysFull, 0);
      scores(0);
    }
    for (int t = 0; t < nt; ++t) {
      const int stage = t % S::kStages;
      const bool more = t + 1 < nt;
      if (more)
        wait(kKeysFull + (t + 1) % S::kStages, (t + 1) / S::kStages);
      if (!S::kOverwrite && more) {
        wait(kScoresRead, t);
        scores(t + 1);
      }
      wait(kValuesFull + stage, t / S::kStages);
      wait(kWeights, t);
      tc::fence_after();
      __syncwarp();
      if (tc::elect()) {
        tc::product_by_rows<T, kKeys>(tmem + S::kO, tmem + S::kP,
                                      v_tile + stage * S::kTile, steps * 16,
                                      t > 0);
        tc::commit(bar(kOutput));
        tc::commit(bar(kValuesFree + stage));
      }
      __syncwarp();
      if (S::kOverwrite && more) {
        wait(kOutput, t);
        scores(t + 1);
      }
    }
    // nor is a product
    if (nt > 0) tc::barrier_wait(bar(kOutput), (nt - 1) & 1);
  } else {
    const int r = r0 + tid;
    const int rows = min(each, n - r0);
    const bool live = tid < rows;
    const bool busy = warp * 32 < rows;  // the warp holds rows
    const uint32_t mine = tmem + ((uint32_t)warp << 21);  // the warp's rows
    float m = -kInf, l = 0.f;
    bool seen = false;  // an open key
    if (!busy) {
      for (int t = 0; t < nt; ++t) {
        wait(kScores, t);
        if (lane == 0 && !S::kOverwrite) tc::barrier_arrive(bar(kScoresRead));
        // no arrival for the next tile before this one's phase is complete
        if (t > 0) wait(kOutput, t - 1);
        if (lane == 0) tc::barrier_arrive(bar(kWeights));
        __syncwarp();
      }
    } else {
      const uint64_t scale2 = tc::pair(a.scale_log2e, a.scale_log2e);
      for (int t = 0; t < nt; ++t) {
        uint32_t s[kKeys];
        wait(kScores, t);
        __syncwarp();
        tc::fence_after();
#pragma unroll
        for (int i = 0; i < kKeys; i += 32) tc::load32(mine + S::kS + i, s + i);
        tc::wait_load();
        if (!S::kOverwrite) {
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::barrier_arrive(bar(kScoresRead));
        }
        const int at = (begin + t) * kKeys;
        if (mask || at + kKeys > nk) {
          uint32_t open[kKeys / 32];
          key_words<kKeys>(open, mask, at, nk);
#pragma unroll
          for (int w = 0; w < kKeys / 32; ++w) {
            seen |= open[w] != 0;
            if (open[w] != 0xffffffffu) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((open[w] >> i) & 1)) s[w * 32 + i] = 0xff800000u;
            }
          }
        } else {
          seen = true;
        }
        // The maximum, NaN if any score is; an infinite one has no softmax.
        float tops[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          tops[i] = max3(__uint_as_float(s[3 * i]),
                         __uint_as_float(s[3 * i + 1]),
                         __uint_as_float(s[3 * i + 2]));
#pragma unroll
        for (int i = 12; i < kKeys; i += 2)
          tops[(i >> 1) & 3] = max3(tops[(i >> 1) & 3], __uint_as_float(s[i]),
                                    __uint_as_float(s[i + 1]));
        float top = max3(tops[0], tops[1], max3(tops[2], tops[3], tops[3])) *
                    a.scale_log2e;
        if (top == kInf) top = __int_as_float(0x7fffffff);
        float rescale = 1.f;
        if (!(top <= m + 8.f) || m == -kInf) {
          rescale = m == -kInf ? 0.f : exp2_fast(m - top);
          m = top;
          l *= rescale;
        }
        const float shift = m == -kInf ? 0.f : m;
        const uint64_t shift2 = tc::pair(-shift, -shift);
        uint64_t sum[2] = {0, 0};
        // P and its sum, a half at a time; P's place and O are free once the
        // last tile's product is complete, which the first half hides
#pragma unroll
        for (int c = 0; c < kKeys; c += kKeys / 2) {
          uint32_t p[kKeys / 4];
#pragma unroll
          for (int i = 0; i < kKeys / 2; i += 2) {
            const uint64_t x =
                tc::fma2(tc::pair(__uint_as_float(s[c + i]),
                                  __uint_as_float(s[c + i + 1])),
                         scale2, shift2);
            float u0, u1;
            if ((i >> 1) % 4 == 3) {
              exp2_polynomial(x, &u0, &u1);
            } else {
              tc::unpair(x, &u0, &u1);
              u0 = exp2_fast(u0);
              u1 = exp2_fast(u1);
            }
            sum[(i >> 1) & 1] = tc::add2(sum[(i >> 1) & 1], tc::pair(u0, u1));
            p[i / 2] = pack2<T>(u0, u1);
          }
          if (c == 0 && t > 0) {
            wait(kOutput, t - 1);
            __syncwarp();
            tc::fence_after();
            if (__any_sync(kFull, rescale != 1.f)) {
              for (int i = 0; i < a.dim; i += 8) {
                uint32_t o[8];
                tc::load8(mine + S::kO + i, o);
                tc::wait_load();
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  o[e] = __float_as_uint(__uint_as_float(o[e]) * rescale);
                tc::store8(mine + S::kO + i, o);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < kKeys / 4; i += 16)
            tc::store16(mine + S::kP + c / 2 + i, p + i);
        }
        float u0, u1;
        tc::unpair(tc::add2(sum[0], sum[1]), &u0, &u1);
        l += u0 + u1;
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

    if (busy) {
      const int qr = live ? r / a.group : 0;
      const int h = hk * a.group + (live ? r - qr * a.group : 0);
      const long long row = q0 + qr;
      const long long at =
          a.splits == 1 ? row * a.heads + h
                        : ((long long)split * a.n_q + row) * a.heads + h;
      // A part whose scores are all -inf counts for nothing beside others,
      // but a row of nothing else has no softmax (NaN): such a part is told
      // by a finite lse below all others.
      const bool none = !seen || (a.splits > 1 && l == 0.f);
      const float inv = none ? 0.f : 1.f / l;
      if (live) {
        const float lse2 = seen ? m + log2f(l) : -kInf;
        if (a.splits > 1)
          a.part_lse[at] = seen && none ? -3.0e38f : lse2;
        else if (a.lse)
          a.lse[at] =
              seen && l == 0.f ? __int_as_float(0x7fffffff) : lse2 * kLn2;
      }
      if (a.splits == 1) {
        // Through Q's place (its products are complete), so that whole rows
        // are written at a time: chunk c of a row by a lane each.
#pragma unroll
        for (int i = 0; i < kDim; i += 32) {
          uint32_t x[32];
          if (i >= a.dim) break;
          __syncwarp();
          if (seen) {
            tc::load32(mine + S::kO + i, x);
            tc::wait_load();
          }
#pragma unroll
          for (int c = 0; c < 32; c += 8) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              f[e] = none ? 0.f : __uint_as_float(x[c + e]) * inv;
            const uint4 u = Vec<T>::pack(f);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                             q_tile + tc::tile_offset(kRows, tid, (i + c) / 8)),
                         "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w)
                         : "memory");
          }
        }
        __syncwarp();
        constexpr int kChunks = kDim / 8, kAtOnce = 32 / kChunks;
        const int chunk = lane % kChunks;
        if (chunk * 8 < a.dim) {
#pragma unroll 4
          for (int i = lane / kChunks; i < 32; i += kAtOnce) {
            const int w = warp * 32 + i;
            if (w >= rows) break;
            uint4 u;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                         : "r"(q_tile + tc::tile_offset(kRows, w, chunk))
                         : "memory");
            const int p = (r0 + w) / a.group;
            const int head = hk * a.group + (r0 + w - p * a.group);
            *reinterpret_cast<uint4*>(static_cast<T*>(a.o) +
                                      (q0 + p) * a.o_row + head * a.o_head +
                                      chunk * 8) = u;
          }
        }
      } else {
        for (int i = 0; i < a.dim; i += 8) {
          uint32_t x[8];
          float f[8];
          __syncwarp();
          if (seen) {
            tc::load8(mine + S::kO + i, x);
            tc::wait_load();
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
            f[e] = none ? 0.f : __uint_as_float(x[e]) * inv;
          if (!live) continue;
          float4* o = reinterpret_cast<float4*>(a.part + at * a.dim + i);
          o[0] = make_float4(f[0], f[1], f[2], f[3]);
          o[1] = make_float4(f[4], f[5], f[6], f[7]);
        }
      }
    }
  }
  if (nt > 0) {
    if (!ok) *a.error = 1;
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == 4) {
      tc::fence_after();
      tc::tmem_free(tmem, S::kColumns);
    }
  }
}

// The parts of a split row, joined: a block per (row, head), whose warps take
// the parts in turn.
template <typename T>
__global__ void __launch_bounds__(128)
    cross_join_kernel(const __grid_constant__ CrossArgs a) {
  __shared__ float4 sums[4][32];
  __shared__ float weights[4];
  const long long unit = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long step = a.n_q * a.heads;
  float top = -kInf;
  bool nan = false;
  for (int s = lane; s < a.splits; s += 32) {
    const float x = a.part_lse[s * step + unit];
    nan |= x != x;
    top = fmaxf(top, x);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
    top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
  nan = __any_sync(kFull, nan) || (top != -kInf && top <= -3.0e38f);
  float sum = 0.f, f[4] = {0.f, 0.f, 0.f, 0.f};
  const bool mine = lane * 4 < a.dim;
  if (top != -kInf) {
#pragma unroll 4
    for (int s = warp; s < a.splits; s += 4) {
      const float w = exp2_fast(a.part_lse[s * step + unit] - top);
      sum += w;
      if (mine) {
        const float4 x = *reinterpret_cast<const float4*>(
            a.part + (s * step + unit) * a.dim + lane * 4);
        f[0] = fmaf(w, x.x, f[0]);
        f[1] = fmaf(w, x.y, f[1]);
        f[2] = fmaf(w, x.z, f[2]);
        f[3] = fmaf(w, x.w, f[3]);
      }
    }
  }
  sums[warp][lane] = make_float4(f[0], f[1], f[2], f[3]);
  if (lane == 0) weights[warp] = sum;
  __syncthreads();
  if (warp > 0) return;
  sum = (weights[0] + weights[1]) + (weights[2] + weights[3]);
  const float inv = top == -kInf ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      f[i] += reinterpret_cast<const float*>(&sums[w][lane])[i];
    f[i] *= inv;
  }
  if (nan) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __int_as_float(0x7fffffff);
  }
  const long long row = unit / a.heads;
  const int h = (int)(unit - row * a.heads);
  if (mine) {
    T* o = static_cast<T*>(a.o) + row * a.o_row + h * a.o_head + lane * 4;
    *reinterpret_cast<uint2*>(o) =
        make_uint2(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]));
  }
  if (lane == 0 && a.lse)
    a.lse[unit] = nan           ? __int_as_float(0x7fffffff)
                  : top == -kInf ? -kInf
                                 : (top + log2f(sum)) * kLn2;
}

template <typename T, int kDim>
cudaError_t launch(const CrossArgs& a, const Maps& maps, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(
      cross_forward_kernel<T, kDim>,
      cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<kDim>::kSmem);
  if (e) return e;
  count_launches(1);
  const dim3 grid(a.tiles * a.splits, a.kv_heads, a.scenes);
  cross_forward_kernel<T, kDim>
      <<<grid, kThreads, Shape<kDim>::kSmem, s>>>(a, maps);
  if (a.splits > 1) {
    count_launches(1);
    cross_join_kernel<T>
        <<<(unsigned)(a.n_q * a.heads), 128, 0, s>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace

int multiprocessors() {
  int device = 0, n = 0;
  if (cudaGetDevice(&device) ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) ||
      n < 1) {
    cudaGetLastError();
    return 148;
  }
  return n;
}

// How many blocks share a row of work: what takes the least time, in tiles, if
// a block costs five of them to begin and end, `room` blocks run together, and
// parts cost ten more to be joined.
int split_count(long long blocks, long long tiles, int room) {
  if (blocks < 1 || blocks >= 8ll * room) return 1;
  int best = 1;
  long long least = ceil_div(blocks, room) * (tiles + 5);
  for (int n = 2; n <= 128 && 2 * n <= tiles; ++n) {
    const long long t =
        ceil_div(blocks * n, room) * (ceil_div(tiles, n) + 5) + 10;
    if (t < least) {
      least = t;
      best = n;
    }
  }
  return best;
}

bool cross_sizes(const attention_args* a) {
  // a box of packed rows holds at least one query row
  return attention_sizes(a) && a->type != kF32 &&
         a->heads / a->kv_heads <= 64 && a->max_q >= 0 &&
         a->max_q <= a->n_q && a->max_k >= 0 && a->max_k <= a->n_k &&
         a->scenes <= 65535 && a->kv_heads <= 65535 &&  // a grid's limits
         a->max_q * (a->heads / a->kv_heads) < kMaxInt - 2 * kRows &&
         a->max_k < kMaxInt - 2 * kRows;
}

namespace {
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t,
                                void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion,
                                CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000,
                                         cudaEnableDefault, &found) ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return f;
}
}  // namespace

cudaError_t row_map(CUtensorMap* map, long long type, const feature_rows& t,
                    long long dim, long long heads, long long rows,
                    int heads_box, int rows_box) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return cudaErrorNotSupported;
  const cuuint64_t size[3] = {(cuuint64_t)dim, (cuuint64_t)heads,
                              (cuuint64_t)rows};
  // a dimension of one element is never stepped along
  const cuuint64_t step[2] = {
      (cuuint64_t)(heads > 1 ? t.head * 2 : dim * 2),
      (cuuint64_t)(rows > 1 ? t.row * 2 : heads * dim * 2)};
  const cuuint32_t box[3] = {64, (cuuint32_t)heads_box, (cuuint32_t)rows_box};
  const cuuint32_t each[3] = {1, 1, 1};
  const CUresult e = encode(
      map,
      type == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                   : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
      3, const_cast<void*>(t.data), size, step, box, each,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return e == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

CrossArgs cross_arguments(const attention_args* in) {
  CrossArgs a = {};
  a.q = in->q.data;
  a.k = in->k.data;
  a.v = in->v.data;
  a.mask = in->mask;
  a.q_seg = in->q_seg;
  a.k_seg = in->k_seg;
  a.lse = in->lse;
  a.error = in->error;
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
  a.scenes = (int)in->scenes;
  a.heads = (int)in->heads;
  a.kv_heads = (int)in->kv_heads;
  a.group = a.heads / a.kv_heads;
  a.dim = (int)in->dim;
  a.scale = (float)in->scale;
  a.scale_log2e = (float)(in->scale * (double)kLog2e);
  return a;
}

}  // namespace gsa

using namespace gsa;

namespace {

struct ForwardPlan {
  long long tiles, blocks, bytes;
  int splits;
};

ForwardPlan forward_plan(const attention_args* a) {
  ForwardPlan p;
  const long long group = a->heads / a->kv_heads;
  p.tiles = ceil_div(a->max_q * group, kRows / group * group);
  const long long blocks = p.tiles * a->scenes * a->kv_heads;
  p.splits = split_count(blocks, ceil_div(a->max_k, kKeys),
                         2 * multiprocessors());
  p.blocks = blocks * p.splits;
  p.bytes =
      p.splits == 1 ? 0 : 4 * p.splits * a->n_q * a->heads * (a->dim + 1);
  return p;
}

}  // namespace

// See include/point_features.h.
GSA_API int64_t cross_attention_workspace(const attention_args* in) {
  if (!cross_sizes(in)) return -2;
  return forward_plan(in).bytes;
}

// See include/point_features.h.
GSA_API int cross_attention(const attention_args* in) {
  if (!cross_sizes(in) || !attention_scale(in->scale)) return -2;
  if (!in->n_q) return 0;
  if (!vector_rows(in->q, in->type) || !vector_rows(in->out, in->type) ||
      !in->q_seg || !in->k_seg || !in->error)
    return -2;
  if (in->n_k &&
      (!vector_rows(in->k, in->type) || !vector_rows(in->v, in->type)))
    return -2;
  const ForwardPlan p = forward_plan(in);
  if (p.blocks > kMaxInt) return -2;
  if (p.bytes && (!vector_address(in->workspace) ||
                  in->workspace_bytes < p.bytes))
    return -2;
  CrossArgs a = cross_arguments(in);
  a.o = const_cast<void*>(in->out.data);
  a.tiles = (int)p.tiles;
  a.splits = p.splits;
  a.part = static_cast<float*>(in->workspace);
  if (p.splits > 1) a.part_lse = a.part + p.splits * a.n_q * a.heads * a.dim;
  Maps maps = {};
  if (in->n_k) {
    cudaError_t e = row_map(&maps.q, in->type, in->q, a.dim, a.heads, a.n_q,
                            a.group, kRows / a.group);
    if (!e)
      e = row_map(&maps.k, in->type, in->k, a.dim, a.kv_heads, a.n_k,
                            1, kKeys);
    if (!e)
      e = row_map(&maps.v, in->type, in->v, a.dim, a.kv_heads, a.n_k, 1, kKeys);
    if (e) return e;
  }
  cudaStream_t s = (cudaStream_t)in->stream;
  if (in->type == kF16)
    return a.dim <= 64 ? launch<__half, 64>(a, maps, s)
                       : launch<__half, 128>(a, maps, s);
  return a.dim <= 64 ? launch<__nv_bfloat16, 64>(a, maps, s)
                     : launch<__nv_bfloat16, 128>(a, maps, s);
}
