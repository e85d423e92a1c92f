// SPDX-License-Identifier: Apache-2.0
// Cross attention between two levels of a hierarchy: the queries of scene i
// read the keys and values of scene i,
//
//   s = scale q k^T,  out = softmax(s) v,  lse = log sum exp s,
//
// over the scene's open keys; a row without any gives 0 and lse = -inf.
//
// A block owns 128 packed query rows and walks the keys in tiles.  Products
// run on tcgen05: S = Q K^T into tensor memory; every thread takes one row of
// it into registers, keeps the running maximum and sum in 32 bits, and writes
// P = exp(S - max), rounded to the inputs' type for the second product (half
// a step, 2^-8 for bf16, on weights that are summed in 32 bits), back to
// tensor memory, from where O += P V takes it.  The maximum that P is taken
// against may lag the true one by a factor of 2^8, so that O is rescaled only
// when it grew by more.
//
// What bounds it: the exponentials (16 a clock on an SM) up to a head of 128
// elements, where the two products take as long.  Tensor memory (256 columns)
// and shared memory (at most 96 KB) leave room for two blocks on an SM, so one
// block's exponentials run beside the other's products.  Where there are too
// few row tiles to fill the GPU, the keys are split among blocks and the
// parts joined by their lse.
#include "cross.cuh"

namespace gsa {
namespace {

// Head size up to kDim (64 or 128); keys per tile.
template <int kDim>
struct Shape {
  static constexpr int kKeys = kDim == 64 ? 128 : 64;
  static constexpr int kQ = kRows * kDim * 2;      // bytes
  static constexpr int kTileBytes = kKeys * kDim * 2;
  static constexpr int kSmem = 1024 + kQ + 4 * kTileBytes;
  static constexpr uint32_t kColumns = 256;
  static constexpr uint32_t kS = 0, kP = kKeys, kO = kKeys + kKeys / 2;
  static_assert(kO + kDim <= 256, "tensor memory");
};

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, 2)
    cross_forward_kernel(const __grid_constant__ CrossArgs a) {
  using S = Shape<kDim>;
  constexpr int kKeys = S::kKeys;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[2];
  __shared__ uint32_t tmem_at;
  __shared__ uint32_t words[4][kKeys / 32];

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
  const int r0 = tile * kRows;
  if (r0 >= n) return;
  int begin, end;
  share((nk + kKeys - 1) / kKeys, a.splits, split, &begin, &end);
  const int nt = end - begin;

  const int tid = threadIdx.x, warp = tid >> 5;
  const uint32_t smem =
      (tc::smem_address(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_tile = smem, k_tile = smem + S::kQ,
                 v_tile = k_tile + 2 * S::kTileBytes;
  const uint32_t bar_s = tc::smem_address(&bars[0]),
                 bar_o = tc::smem_address(&bars[1]);
  const int steps = (a.dim + 15) / 16;

  const int r = r0 + tid;
  const bool live = r < n;
  const bool busy = r0 + warp * 32 < n;  // the warp holds rows
  bool ok = true;
  float m = -kInf, l = 0.f;
  uint32_t seen = 0;
  uint32_t tmem = 0;

  if (nt > 0) {
    if (warp == 0) tc::tmem_alloc(tc::smem_address(&tmem_at), S::kColumns);
    if (tid == 0) {
      tc::barrier_init(bar_s, 1);
      tc::barrier_init(bar_o, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const Chunks c = chunks_of(a.dim);
    const T* q = static_cast<const T*>(a.q) + q0 * a.q_row +
                 (long long)hk * a.group * a.q_head;
    const T* k = static_cast<const T*>(a.k) + k0 * a.k_row + hk * a.k_head;
    const T* v = static_cast<const T*>(a.v) + k0 * a.v_row + hk * a.v_head;
    const unsigned char* mask = a.mask ? a.mask + k0 : nullptr;
    auto load_k = [&](int t) {
      if (t < nt) {
        load_keys<T, kKeys>(c, k_tile + (t & 1) * S::kTileBytes, k, a.k_row,
                            mask, (begin + t) * kKeys, nk);
        key_words<kKeys>(words[t & 3], mask, (begin + t) * kKeys, nk);
      }
      tc::copy_commit();
    };
    auto load_v = [&](int t) {
      if (t < nt)
        load_keys<T, kKeys>(c, v_tile + (t & 1) * S::kTileBytes, v, a.v_row,
                            mask, (begin + t) * kKeys, nk);
      tc::copy_commit();
    };
    load_packed<T, kRows>(c, q_tile, q, a.q_row, a.q_head, a.group, r0, n);
    load_k(0);
    load_k(1);
    load_v(0);
    tc::copy_wait<2>();
    tc::fence_shared();
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    tmem = tmem_at;
    auto scores = [&](int t) {
      tc::product_by_columns<T>(tmem + S::kS, q_tile, kRows,
                                k_tile + (t & 1) * S::kTileBytes, kKeys, kKeys,
                                steps);
      tc::commit(bar_s);
    };
    if (tid == 0) scores(0);
    const uint32_t mine = tmem + ((uint32_t)warp << 21);  // the warp's rows

    for (int t = 0; t < nt; ++t) {
      uint32_t s[kKeys];
      ok = ok && tc::barrier_wait(bar_s, t & 1);
      __syncwarp();
      tc::fence_after();
      if (busy) {
#pragma unroll
        for (int i = 0; i < kKeys; i += 32) tc::load32(mine + S::kS + i, s + i);
        tc::wait_load();
      }
      load_k(t + 2);
      tc::copy_wait<2>();  // the next keys are there
      tc::fence_shared();
      tc::fence_before();
      __syncthreads();
      if (tid == 0 && t + 1 < nt) {
        tc::fence_after();
        scores(t + 1);
      }
      uint32_t p[kKeys / 2];
      float rescale = 1.f;
      if (busy) {
        float top = -kInf;
#pragma unroll
        for (int w = 0; w < kKeys / 32; ++w) {
          const uint32_t open = words[t & 3][w];
          seen |= open;
          if (open != 0xffffffffu) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((open >> i) & 1)) s[w * 32 + i] = 0xff800000u;
          }
        }
#pragma unroll
        for (int i = 0; i < kKeys; ++i) top = fmaxf(top, __uint_as_float(s[i]));
        top *= a.scale_log2e;
        if (top > m + 8.f || m == -kInf) {
          rescale = m == -kInf ? 0.f : exp2_fast(m - top);
          m = top;
          l *= rescale;
        }
        const float shift = m == -kInf ? 0.f : m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kKeys; i += 2) {
          const float x = exp2_fast(
              fmaf(__uint_as_float(s[i]), a.scale_log2e, -shift));
          const float y = exp2_fast(
              fmaf(__uint_as_float(s[i + 1]), a.scale_log2e, -shift));
          sum[i & 2] += x;
          sum[(i & 2) + 1] += y;
          p[i / 2] = pack2<T>(x, y);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      }
      if (t > 0) {
        ok = ok && tc::barrier_wait(bar_o, (t - 1) & 1);
        __syncwarp();
        tc::fence_after();
      }
      load_v(t + 1);
      if (busy) {
        if (t > 0 && __any_sync(kFull, rescale != 1.f)) {
          for (int i = 0; i < steps * 16; i += 16) {
            uint32_t o[16];
            tc::load16(mine + S::kO + i, o);
            tc::wait_load();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e] = __float_as_uint(__uint_as_float(o[e]) * rescale);
            tc::store16(mine + S::kO + i, o);
          }
        }
#pragma unroll
        for (int i = 0; i < kKeys / 2; i += 16)
          tc::store16(mine + S::kP + i, p + i);
        tc::wait_store();
      }
      tc::copy_wait<2>();  // this tile's values are there
      tc::fence_shared();
      tc::fence_before();
      __syncthreads();
      if (tid == 0) {
        tc::fence_after();
        tc::product_by_rows<T>(tmem + S::kO, tmem + S::kP,
                               v_tile + (t & 1) * S::kTileBytes, kKeys,
                               steps * 16, kKeys / 16, t > 0);
        tc::commit(bar_o);
      }
    }
    ok = ok && tc::barrier_wait(bar_o, (nt - 1) & 1);
    __syncwarp();
    tc::fence_after();
    tc::copy_wait<0>();
  }

  const int qr = live ? r / a.group : 0;
  const int h = hk * a.group + (live ? r - qr * a.group : 0);
  const long long row = q0 + qr;
  const float inv = seen ? 1.f / l : 0.f;
  if (a.splits == 1) {
    T* o = static_cast<T*>(a.o) + row * a.o_row + h * a.o_head;
    if (live && a.lse)
      a.lse[row * a.heads + h] = seen ? (m + log2f(l)) * kLn2 : -kInf;
    if (busy) {
      for (int i = 0; i < a.dim; i += 16) {
        uint32_t x[16];
        if (seen) {
          __syncwarp();
          tc::load16(tmem + ((uint32_t)warp << 21) + S::kO + i, x);
          tc::wait_load();
        }
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          f[e] = seen ? __uint_as_float(x[e]) * inv : 0.f;
        if (live) {
          *reinterpret_cast<uint4*>(o + i) = Vec<T>::pack(f);
          if (i + 8 < a.dim)
            *reinterpret_cast<uint4*>(o + i + 8) = Vec<T>::pack(f + 8);
        }
      }
    }
  } else {
    // A part whose scores are all -inf counts for nothing beside others, but
    // a row of nothing else has no softmax (NaN): it is told apart by a
    // finite lse below all others.
    const long long at = ((long long)split * a.n_q + row) * a.heads + h;
    const bool none = !seen || l == 0.f;
    if (live)
      a.part_lse[at] = !seen ? -kInf : l == 0.f ? -3.0e38f : m + log2f(l);
    if (busy) {
      for (int i = 0; i < a.dim; i += 16) {
        uint32_t x[16];
        if (seen) {
          __syncwarp();
          tc::load16(tmem + ((uint32_t)warp << 21) + S::kO + i, x);
          tc::wait_load();
        }
        if (live) {
          float4* o = reinterpret_cast<float4*>(a.part + at * a.dim + i);
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            if (i + e >= a.dim) break;
            float f[4];
#pragma unroll
            for (int d = 0; d < 4; ++d)
              f[d] = none ? 0.f : __uint_as_float(x[e + d]) * inv;
            o[e / 4] = make_float4(f[0], f[1], f[2], f[3]);
          }
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

// The parts of a split row, joined: a warp per (row, head).
template <typename T>
__global__ void __launch_bounds__(128)
    cross_join_kernel(const __grid_constant__ CrossArgs a) {
  const long long unit = ((long long)blockIdx.x * 128 + threadIdx.x) >> 5;
  if (unit >= a.n_q * a.heads) return;
  const int lane = threadIdx.x & 31;
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
    for (int s = 0; s < a.splits; ++s) {
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
    const float inv = 1.f / sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] *= inv;
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
cudaError_t launch(const CrossArgs& a, long long grid, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(
      cross_forward_kernel<T, kDim>,
      cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<kDim>::kSmem);
  if (e) return e;
  count_launches(1);
  cross_forward_kernel<T, kDim>
      <<<(unsigned)grid, kThreads, Shape<kDim>::kSmem, s>>>(a);
  if (a.splits > 1) {
    count_launches(1);
    cross_join_kernel<T>
        <<<(unsigned)ceil_div(a.n_q * a.heads, 4), 128, 0, s>>>(a);
  }
  return cudaGetLastError();
}

int forward_keys(int dim) { return dim <= 64 ? 128 : 64; }

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

// How many blocks share a row of work: as many as still find room on the GPU
// together, each with at least two tiles.
int split_count(long long blocks, long long tiles, int room) {
  if (blocks < 1 || tiles < 4) return 1;
  long long n = room / blocks;
  if (n > tiles / 2) n = tiles / 2;
  return n < 1 ? 1 : (int)n;
}

bool cross_sizes(const attention_args* a) {
  return attention_sizes(a) && a->type != kF32 && a->max_q >= 0 &&
         a->max_q <= a->n_q && a->max_k >= 0 && a->max_k <= a->n_k &&
         a->max_q * (a->heads / a->kv_heads) < kMaxInt - 2 * kRows &&
         a->max_k < kMaxInt - 2 * kRows;
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
  p.tiles = ceil_div(a->max_q * (a->heads / a->kv_heads), kRows);
  const long long blocks = p.tiles * a->scenes * a->kv_heads;
  p.splits = split_count(blocks, ceil_div(a->max_k, forward_keys((int)a->dim)),
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
  cudaStream_t s = (cudaStream_t)in->stream;
  if (in->type == kF16)
    return a.dim <= 64 ? launch<__half, 64>(a, p.blocks, s)
                       : launch<__half, 128>(a, p.blocks, s);
  return a.dim <= 64 ? launch<__nv_bfloat16, 64>(a, p.blocks, s)
                     : launch<__nv_bfloat16, 128>(a, p.blocks, s);
}
