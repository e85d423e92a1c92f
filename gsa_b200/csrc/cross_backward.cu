// SPDX-License-Identifier: Apache-2.0
// Gradients of cross attention.  With P = exp(scale q k^T - lse) and
// delta = rowsum(dout * out):
//
//   dv = P^T dout,  dP = dout v^T,  dS = P * (dP - delta),
//   dq = scale dS k,  dk = scale dS^T q.
//
// Two passes of one kernel, each recomputing P: one block per 128 keys walks
// the queries and keeps dk and dv in tensor memory, one block per 128 packed
// query rows walks the keys and keeps dq.  Seven products instead of five,
// but every sum has one fixed order (no atomics, the same bits each time),
// and nothing but the results is written.  In the keys' pass the products are
// taken transposed (S^T = k q^T), so that P^T and dS^T come out with a key
// per thread and go back to tensor memory as the second products' left side;
// the walked tile serves as the right side of both its products, read by
// columns and by rows, without a transposed copy.
//
// P and dS are rounded to the inputs' type for their products (half a step).
// For fp16, whose smallest normal is 2^-14, P carries a factor of 2^15 (it is
// at most 1) and dS one that grows with the number of keys.
//
// What bounds it: per 128 x 64 tile of the keys' pass 1,024 clocks of products
// at a head of 64 (four of 128 x 64 x 64) against 512 of exponentials.
#include "cross.cuh"

namespace gsa {
namespace {

constexpr int kBlock = 128;
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
template <int kN>
__device__ __forceinline__ void block_words(uint32_t* words,
                                          const unsigned char* mask, int k0,
                                          int n) {
  if (threadIdx.x < kN) {
    const int r = k0 + (int)threadIdx.x;
    const bool open = r < n && (!mask || __ldg(mask + r));
    const uint32_t w = __ballot_sync(kFull, open);
    if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = w;
  }
}
constexpr int kWalk = 64;    // rows of a walked tile
constexpr int kStages = 3;

template <int kDim, bool kKeysPass>
struct Shape {
  static constexpr int kOwn = kRows * kDim * 2;    // bytes of a resident tile
  static constexpr int kTile = kWalk * kDim * 2;   // of a walked one
  static constexpr int kSmem = 1024 + 2 * kOwn + 2 * kStages * kTile;
  // With 256 columns two blocks share an SM (the larger heads' tiles do not
  // fit twice in any case).  The keys' pass then has no columns left for P
  // and dS beside S and dP: they overwrite them, and the next scores wait.
  static constexpr uint32_t kColumns = kDim == 64 ? 256 : 512;
  static constexpr bool kOverwrite = kDim == 64 && kKeysPass;
  static constexpr uint32_t kS = 0, kDp = 64;
  static constexpr uint32_t kDs = kOverwrite ? kDp : 128;
  static constexpr uint32_t kP = kOverwrite ? kS : kDs + kWalk / 2;
  static constexpr uint32_t kOut1 = kOverwrite ? 128 : kKeysPass ? 192 : 160;
  static constexpr uint32_t kOut2 = kOut1 + kDim;  // keys' pass: dv
  static constexpr uint32_t kEnd = kKeysPass ? kOut2 + kDim : kOut2;
  static_assert(kEnd <= kColumns && kP < kEnd, "tensor memory");
  static constexpr int kBlocks = kDim == 64 ? 2 : 1;
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
__global__ void __launch_bounds__(kBlock, Shape<kDim, kKeysPass>::kBlocks)
    cross_backward_kernel(const __grid_constant__ CrossArgs a) {
  using S = Shape<kDim, kKeysPass>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[2];
  __shared__ uint32_t tmem_at;
  __shared__ uint32_t words[4][kWalk / 32];
  __shared__ __align__(16) float row_lse[4][kWalk];
  __shared__ __align__(16) float row_delta[4][kWalk];

  unsigned unit = blockIdx.x;
  const int tile = unit % a.tiles;
  unit /= a.tiles;
  const int split = unit % a.splits;
  unit /= a.splits;
  const int hk = unit % a.kv_heads;
  const int scene = unit / a.kv_heads;
  const int q0 = a.q_seg[scene], k0 = a.k_seg[scene];
  const int n = (a.q_seg[scene + 1] - q0) * a.group;  // packed rows
  const int nk = a.k_seg[scene + 1] - k0;
  const int own = kKeysPass ? nk : n, walked = kKeysPass ? n : nk;
  const int r0 = tile * kRows;
  if (r0 >= own) return;
  int begin, end;
  share((walked + kWalk - 1) / kWalk, a.splits, split, &begin, &end);
  const int nt = end - begin;

  const int tid = threadIdx.x, warp = tid >> 5;
  const uint32_t smem = (tc::smem_address(smem_raw) + 1023u) & ~1023u;
  const uint32_t x1 = smem, x2 = smem + S::kOwn, y1 = x2 + S::kOwn,
                 y2 = y1 + kStages * S::kTile;
  const uint32_t bar_s = tc::smem_address(&bars[0]),
                 bar_a = tc::smem_address(&bars[1]);
  const int steps = (a.dim + 15) / 16;
  const unsigned char* mask = a.mask ? a.mask + k0 : nullptr;

  const int r = r0 + tid;
  const bool live = r < own;
  const bool busy = r0 + warp * 32 < own;
  bool ok = true;
  uint32_t tmem = 0;
  const float bits = ds_bits<T>(nk);
  const float ds_factor = exp2f(bits - p_bits<T>());

  if (nt > 0) {
    if (warp == 0) tc::tmem_alloc(tc::smem_address(&tmem_at), S::kColumns);
    if (tid == 0) {
      tc::barrier_init(bar_s, 1);
      tc::barrier_init(bar_a, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const Chunks c = chunks_of(a.dim, tid, kBlock);
    const T* q = static_cast<const T*>(a.q) + q0 * a.q_row +
                 (long long)hk * a.group * a.q_head;
    const T* d = static_cast<const T*>(a.dout) + q0 * a.d_row +
                 (long long)hk * a.group * a.d_head;
    const T* k = static_cast<const T*>(a.k) + k0 * a.k_row + hk * a.k_head;
    const T* v = static_cast<const T*>(a.v) + k0 * a.v_row + hk * a.v_head;
    // lse (base 2, less the factor that P carries) and delta of a packed row;
    // a row without keys gets P = 0
    auto row_values = [&](int p, float* lse, float* delta) {
      *lse = kInf;
      *delta = 0.f;
      if (p >= n) return;
      const int qr = p / a.group;
      const long long at =
          (long long)(q0 + qr) * a.heads + hk * a.group + (p - qr * a.group);
      const float x = __ldg(a.lse + at);
      if (x != -kInf) *lse = fmaf(x, kLog2e, -p_bits<T>());
      *delta = __ldg(a.delta + at);
    };
    auto load_walked = [&](int t) {
      if (t < nt) {
        const int at = (begin + t) * kWalk;
        const uint32_t t1 = y1 + (t % kStages) * S::kTile,
                       t2 = y2 + (t % kStages) * S::kTile;
        if constexpr (kKeysPass) {
          load_packed<T, kWalk>(c, t1, q, a.q_row, a.q_head, a.group, at, n);
          load_packed<T, kWalk>(c, t2, d, a.d_row, a.d_head, a.group, at, n);
          if (tid < kWalk) {
            float x, y;
            row_values(at + tid, &x, &y);
            row_lse[t & 3][tid] = x;
            row_delta[t & 3][tid] = y * ds_factor;
          }
        } else {
          load_keys<T, kWalk>(c, t1, k, a.k_row, mask, at, nk);
          load_keys<T, kWalk>(c, t2, v, a.v_row, mask, at, nk);
          block_words<kWalk>(words[t & 3], mask, at, nk);
        }
      }
      tc::copy_commit();
    };
    if constexpr (kKeysPass) {
      load_keys<T, kRows>(c, x1, k, a.k_row, mask, r0, nk);
      load_keys<T, kRows>(c, x2, v, a.v_row, mask, r0, nk);
    } else {
      load_packed<T, kRows>(c, x1, q, a.q_row, a.q_head, a.group, r0, n);
      load_packed<T, kRows>(c, x2, d, a.d_row, a.d_head, a.group, r0, n);
    }
    load_walked(0);
    load_walked(1);
    bool open = live;
    float lse2 = kInf, delta = 0.f;
    if constexpr (kKeysPass) {
      open = live && (!mask || __ldg(mask + r));
    } else {
      row_values(r, &lse2, &delta);
      delta *= ds_factor;
    }
    tc::copy_wait<1>();
    tc::fence_shared();
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    tmem = tmem_at;
    auto scores = [&](int t) {
      tc::product_by_columns<T, kRows, kWalk, kDim / 16>(
          tmem + S::kS, x1, y1 + (t % kStages) * S::kTile, steps);
      tc::product_by_columns<T, kRows, kWalk, kDim / 16>(
          tmem + S::kDp, x2, y2 + (t % kStages) * S::kTile, steps);
      tc::commit(bar_s);
    };
    if (tid == 0) scores(0);
    const uint32_t mine = tmem + ((uint32_t)warp << 21);

    for (int t = 0; t < nt; ++t) {
      // the products of tile t - 1 have read their tiles: load tile t + 2
      if (t > 0) {
        ok = ok && tc::barrier_wait(bar_a, (t - 1) & 1);
        tc::fence_after();
      }
      load_walked(t + 2);
      ok = ok && tc::barrier_wait(bar_s, t & 1);
      __syncwarp();
      tc::fence_after();
      if (busy) {
#pragma unroll
        for (int half = 0; half < kWalk; half += 32) {
          uint32_t s[32], e[32], p[16], ds[16];
          tc::load32(mine + S::kS + half, s);
          tc::load32(mine + S::kDp + half, e);
          tc::wait_load();
          const uint32_t w = kKeysPass ? 0u : words[t & 3][half / 32];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float l4[4], d4[4];
            if constexpr (kKeysPass) {
              *reinterpret_cast<float4*>(l4) =
                  *reinterpret_cast<const float4*>(&row_lse[t & 3][half + i]);
              *reinterpret_cast<float4*>(d4) =
                  *reinterpret_cast<const float4*>(
                      &row_delta[t & 3][half + i]);
            }
            float pv[4], dv[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float lj = kKeysPass ? l4[j] : lse2;
              const float dj = kKeysPass ? d4[j] : delta;
              float x = exp2_fast(
                  fmaf(__uint_as_float(s[i + j]), a.scale_log2e, -lj));
              float y = x * fmaf(__uint_as_float(e[i + j]), ds_factor, -dj);
              const bool in = kKeysPass ? open : (w >> (i + j)) & 1;
              pv[j] = in ? x : 0.f;
              dv[j] = in ? y : 0.f;
            }
            p[i / 2] = pack2<T>(pv[0], pv[1]);
            p[i / 2 + 1] = pack2<T>(pv[2], pv[3]);
            ds[i / 2] = pack2<T>(dv[0], dv[1]);
            ds[i / 2 + 1] = pack2<T>(dv[2], dv[3]);
          }
          if constexpr (kKeysPass) tc::store16(mine + S::kP + half / 2, p);
          tc::store16(mine + S::kDs + half / 2, ds);
        }
        tc::wait_store();
      }
      tc::copy_wait<1>();  // tile t + 1 is there
      tc::fence_shared();
      tc::fence_before();
      __syncthreads();
      if (tid == 0) {
        tc::fence_after();
        if (!S::kOverwrite && t + 1 < nt) scores(t + 1);
        const uint32_t t1 = y1 + (t % kStages) * S::kTile,
                       t2 = y2 + (t % kStages) * S::kTile;
        tc::product_by_rows<T, kWalk>(tmem + S::kOut1, tmem + S::kDs, t1,
                                      steps * 16, t > 0);
        if constexpr (kKeysPass)
          tc::product_by_rows<T, kWalk>(tmem + S::kOut2, tmem + S::kP, t2,
                                        steps * 16, t > 0);
        tc::commit(bar_a);
        if (S::kOverwrite && t + 1 < nt) {
          ok = ok && tc::barrier_wait(bar_a, t & 1);
          tc::fence_after();
          scores(t + 1);
        }
      }
    }
    ok = ok && tc::barrier_wait(bar_a, (nt - 1) & 1);
    __syncwarp();
    tc::fence_after();
    tc::copy_wait<0>();
  }

  // Results: packed rows of dq, or keys of dk and dv.
  long long at;  // element of the first column
  long long parts;
  if constexpr (kKeysPass) {
    at = ((long long)(k0 + r) * a.kv_heads + hk) * a.dim;
    parts = a.n_k * a.kv_heads * a.dim;
  } else {
    const int qr = r / a.group;
    at = ((long long)(q0 + qr) * a.heads + hk * a.group + (r - qr * a.group)) *
         a.dim;
    parts = a.n_q * a.heads * a.dim;
  }
  if (busy) {
#pragma unroll
    for (int which = 0; which < (kKeysPass ? 2 : 1); ++which) {
      const float f = which ? exp2f(-p_bits<T>()) : a.scale * exp2f(-bits);
      T* out = static_cast<T*>(kKeysPass ? (which ? a.dv : a.dk) : a.dq) + at;
      float* part =
          a.part + ((kKeysPass ? 2 : 1) * split + which) * parts + at;
      for (int i = 0; i < a.dim; i += 16) {
        uint32_t x[16];
        float y[16];
        if (nt > 0) {
          __syncwarp();
          tc::load16(tmem + ((uint32_t)warp << 21) +
                         (which ? S::kOut2 : S::kOut1) + i, x);
          tc::wait_load();
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
          y[e] = nt > 0 ? __uint_as_float(x[e]) * f : 0.f;
        if (!live) continue;
        if (a.splits == 1) {
          *reinterpret_cast<uint4*>(out + i) = Vec<T>::pack(y);
          if (i + 8 < a.dim)
            *reinterpret_cast<uint4*>(out + i + 8) = Vec<T>::pack(y + 8);
        } else {
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            if (i + e < a.dim)
              *reinterpret_cast<float4*>(part + i + e) =
                  make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
        }
      }
    }
  }
  if (nt > 0) {
    if (!ok && a.error) *a.error = 1;
    tc::fence_before();
    __syncthreads();
    if (warp == 0) {
      tc::fence_after();
      tc::tmem_free(tmem, S::kColumns);
    }
  }
}

// delta = <dout, out> per (row, head): a group of lanes each, 16 bytes a lane.
template <typename T>
__global__ void __launch_bounds__(128)
    cross_delta_kernel(const __grid_constant__ CrossArgs a, int shift) {
  const long long unit = ((long long)blockIdx.x * 128 + threadIdx.x) >> shift;
  const int j = threadIdx.x & ((1 << shift) - 1);
  const bool live = unit < a.n_q * a.heads;
  const long long row = live ? unit / a.heads : 0;
  const int h = live ? (int)(unit - row * a.heads) : 0;
  float sum = 0.f;
  if (live && j * 8 < a.dim) {
    float x[8], y[8];
    Vec<T>::unpack(*reinterpret_cast<const uint4*>(
                       static_cast<const T*>(a.out) + row * a.o_row +
                       h * a.o_head + j * 8), x);
    Vec<T>::unpack(*reinterpret_cast<const uint4*>(
                       static_cast<const T*>(a.dout) + row * a.d_row +
                       h * a.d_head + j * 8), y);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], y[i], sum);
  }
  for (int o = (1 << shift) >> 1; o; o >>= 1)
    sum += __shfl_xor_sync(kFull, sum, o);
  if (live && j == 0) a.delta[unit] = sum;
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
  const int room = multiprocessors() * (a->dim <= 64 ? 2 : 1);
  p.tiles[0] = ceil_div(a->max_k, kRows);
  p.tiles[1] = ceil_div(rows, kRows);
  const long long walked[2] = {ceil_div(rows, kWalk),
                               ceil_div(a->max_k, kWalk)};
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
cudaError_t launch_pass(CrossArgs a, const Plan& p, cudaStream_t s) {
  using S = Shape<kDim, kKeysPass>;
  a.tiles = (int)p.tiles[kKeysPass ? 0 : 1];
  a.splits = p.splits[kKeysPass ? 0 : 1];
  const long long grid = p.blocks[kKeysPass ? 0 : 1];
  if (grid == 0) return cudaSuccess;
  cudaError_t e =
      cudaFuncSetAttribute(cross_backward_kernel<T, kDim, kKeysPass>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                           S::kSmem);
  if (e) return e;
  count_launches(1);
  cross_backward_kernel<T, kDim, kKeysPass>
      <<<(unsigned)grid, kBlock, S::kSmem, s>>>(a);
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

template <typename T>
cudaError_t launch(const CrossArgs& a, const Plan& p, cudaStream_t s) {
  if (a.n_q) {
    int shift = 0;
    while ((8 << shift) < a.dim) ++shift;
    count_launches(1);
    cross_delta_kernel<T>
        <<<(unsigned)ceil_div((a.n_q * a.heads) << shift, 128), 128, 0, s>>>(
            a, shift);
  }
  cudaError_t e = a.dim <= 64 ? launch_pass<T, 64, true>(a, p, s)
                              : launch_pass<T, 128, true>(a, p, s);
  if (e) return e;
  return a.dim <= 64 ? launch_pass<T, 64, false>(a, p, s)
                     : launch_pass<T, 128, false>(a, p, s);
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
  return type == kF16 ? launch<__half>(a, p, s) : launch<__nv_bfloat16>(a, p, s);
}
