// SPDX-License-Identifier: Apache-2.0
// Rotary positions.  A head's first 2P elements (P = axes * pairs) form P
// pairs; pair p = a * pairs + i turns by the angle
//
//   t = position[a] * turns[i]   (whole turns),
//   (u, v) -> amplitude * (u cos 2 pi t - v sin 2 pi t,
//                          u sin 2 pi t + v cos 2 pi t),
//
// and the transposed turn (the gradient) negates the sine.  Positions are far
// (a million and more along a serialised order), so t and its reduction to
// [-1/2, 1/2] are in 64 bits; sine and cosine of the reduced angle are in 32.
//
// The bound is memory: x read once, y written once.  A head's row is one
// group of lanes, a 16-byte vector each, so that every (row, head) belongs to
// one warp: the pairs' other elements come through the warp's own shared
// memory, and y may be x.  A lane computes the sines of its vector's elements
// once and keeps them over all heads.
#include "features.cuh"

namespace gsa {
namespace {

constexpr int kMaxPairs = 128;

struct RotaryArgs {
  const void* x;
  void* y;
  const void* positions;
  long long rows, x_row, x_head, y_row, y_head, pos_row, pos_axis;
  int heads, dim, axes, pairs;  // pairs per axis
  int heads_each;               // of a block
  float amplitude, sign;        // sign: +1, or -1 for the transposed turn
  double turns[kMaxPairs];      // per axis pair
};

template <typename P>
__device__ __forceinline__ void angle(const RotaryArgs& a, long long row,
                                      int pair, float* c, float* s) {
  const int axis = pair / a.pairs;
  const P* at = static_cast<const P*>(a.positions) + row * a.pos_row +
                axis * a.pos_axis;
  const double t = (double)__ldg(at) * a.turns[pair - axis * a.pairs];
  const float r = (float)(t - rint(t));
  float sn, cs;
  sincospif(2.f * r, &sn, &cs);
  *c = cs * a.amplitude;
  *s = sn * a.amplitude * a.sign;
}

// 4 warps and 4 heads ahead: 558 us of 1.5 M rows of 4 x 64 FP32, the best of many
// replays (8 warps 586, 2 heads 610, 8 heads 751); the median is 594 (5.30 TB/s),
// and calls one after another take 626 (5.03 TB/s).
constexpr int kWarps = 4;
constexpr int kHeadsAhead = 4;
constexpr int kMultiprocessors = 148;  // of a B200

// kInterleaved: pairs (2p, 2p + 1); else (p, p + P).
template <typename T, typename Pos, bool kInterleaved>
__global__ void __launch_bounds__(32 * kWarps)
    rotary_vector_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int V = Vec<T>::V;
  __shared__ uint4 stage[kWarps][kHeadsAhead][32];
  const int lanes = a.dim / V, per_warp = 32 / lanes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = lane / lanes, j = lane - group * lanes;
  const int first = blockIdx.y * a.heads_each;
  const int heads = min(a.heads - first, a.heads_each);
  const long long row =
      ((long long)blockIdx.x * kWarps + warp) * per_warp + group;
  const bool live = group < per_warp && row < a.rows;
  const int half = a.axes * a.pairs, part = 2 * half;
  const T* x = static_cast<const T*>(a.x) + row * a.x_row +
               first * a.x_head + j * V;
  T* y = static_cast<T*>(a.y) + row * a.y_row + first * a.y_head + j * V;
  // the first heads' rows are on their way while the sines are taken
  uint4 u[kHeadsAhead];
  auto load = [&](int h0) {
#pragma unroll
    for (int k = 0; k < kHeadsAhead; ++k)
      if (live && h0 + k < heads)
        u[k] = *reinterpret_cast<const uint4*>(x + (h0 + k) * a.x_head);
  };
  load(0);
  float c[V], s[V];
  if (live) {
    if constexpr (kInterleaved) {
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const int e = j * V + i;
        if (e < part) {
          angle<Pos>(a, row, e >> 1, &c[i], &s[i]);
          c[i + 1] = c[i];
          s[i + 1] = s[i];
          s[i] = -s[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = j * V + i;
        if (e < part) {
          angle<Pos>(a, row, e < half ? e : e - half, &c[i], &s[i]);
          if (e < half) s[i] = -s[i];
        }
      }
    }
  }
  for (int h0 = 0; h0 < heads; h0 += kHeadsAhead) {
    if (h0 > 0) load(h0);
    if constexpr (!kInterleaved) {
#pragma unroll
      for (int k = 0; k < kHeadsAhead; ++k)
        if (live) stage[warp][k][lane] = u[k];
    }
    // Every lane has read its vectors before any is written: y may be x.
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kHeadsAhead; ++k) {
      if (!live || h0 + k >= heads) continue;
      float f[V], g[V];
      Vec<T>::unpack(u[k], f);
      if constexpr (kInterleaved) {
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = f[i ^ 1];
      } else {
        const T* mine =
            reinterpret_cast<const T*>(&stage[warp][k][group * lanes]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = j * V + i;
          const int o = e < half ? e + half : e - half;
          g[i] = e < part ? to_float(mine[o]) : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (j * V + i < part) f[i] = f[i] * c[i] + g[i] * s[i];
      *reinterpret_cast<uint4*>(y + (h0 + k) * a.y_head) = Vec<T>::pack(f);
    }
    __syncwarp();
  }
}

// Rows that do not take 16-byte vectors (odd sizes, strides or addresses): a
// thread per pair, and one per element behind the last pair.
template <typename T, typename Pos>
__global__ void __launch_bounds__(256)
    rotary_element_kernel(const __grid_constant__ RotaryArgs a,
                          int interleaved) {
  const int half = a.axes * a.pairs, rest = a.dim - 2 * half;
  const int width = half + rest;
  const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = t / width;
  const int p = (int)(t - row * width);
  if (row >= a.rows) return;
  const T* x = static_cast<const T*>(a.x) + row * a.x_row;
  T* y = static_cast<T*>(a.y) + row * a.y_row;
  if (p >= half) {
    const int e = p + half;
    for (int h = 0; h < a.heads; ++h) y[h * a.y_head + e] = x[h * a.x_head + e];
    return;
  }
  float c, s;
  angle<Pos>(a, row, p, &c, &s);
  const int first = interleaved ? 2 * p : p;
  const int second = interleaved ? 2 * p + 1 : p + half;
  for (int h = 0; h < a.heads; ++h) {
    const float u = to_float(x[h * a.x_head + first]);
    const float v = to_float(x[h * a.x_head + second]);
    y[h * a.y_head + first] = from_float<T>(u * c - v * s);
    y[h * a.y_head + second] = from_float<T>(v * c + u * s);
  }
}

template <typename T, typename Pos>
cudaError_t launch(RotaryArgs a, int interleaved, cudaStream_t s) {
  constexpr int V = Vec<T>::V;
  const bool vectors =
      a.dim % V == 0 && a.dim / V <= 32 &&
      ((a.x_row | a.x_head | a.y_row | a.y_head) % V) == 0 &&
      (((uintptr_t)a.x | (uintptr_t)a.y) & 15) == 0;
  count_launches(1);
  if (vectors) {
    const int per_block = kWarps * (32 / (a.dim / V));
    dim3 grid((unsigned)ceil_div(a.rows, per_block));
    // Too few rows to fill the GPU: the heads on blocks of their own, which
    // take the sines again (375 rows of 8 heads: 3.9 us instead of 6.4).
    a.heads_each = a.heads;
    if (grid.x < kMultiprocessors) {
      a.heads_each = a.heads < 65536 ? 2 : 64;
      grid.y = (unsigned)ceil_div(a.heads, a.heads_each);
    }
    if (interleaved)
      rotary_vector_kernel<T, Pos, true><<<grid, 32 * kWarps, 0, s>>>(a);
    else
      rotary_vector_kernel<T, Pos, false><<<grid, 32 * kWarps, 0, s>>>(a);
  } else {
    const long long threads = a.rows * (a.dim - a.axes * a.pairs);
    rotary_element_kernel<T, Pos>
        <<<(unsigned)ceil_div(threads, 256), 256, 0, s>>>(a, interleaved);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_for(const RotaryArgs& a, int pos_type, int interleaved,
                       cudaStream_t s) {
  if (pos_type == 0) return launch<T, float>(a, interleaved, s);
  if (pos_type == 1) return launch<T, int>(a, interleaved, s);
  return launch<T, long long>(a, interleaved, s);
}

}  // namespace
}  // namespace gsa

using namespace gsa;

// See include/point_features.h.
GSA_API int rotary_positions(const rotary_args* in) {
  if (!in || in->type < kF32 || in->type > kBF16 || in->rows < 0 ||
      in->rows >= kMaxInt || in->heads < 1 || in->heads >= (1 << 20) ||
      in->dim < 2 || in->dim > 4096 || in->axes < 1 || in->axes > 2048 ||
      in->pairs < 1 || in->pairs > kMaxPairs ||
      2 * in->axes * in->pairs > in->dim || in->pos_type < 0 ||
      in->pos_type > 2 || !in->turns)
    return -2;
  if (!in->rows) return 0;
  if (!in->x.data || !in->y.data || !in->positions) return -2;
  if (in->rows * in->dim / 256 >= kMaxInt) return -2;  // blocks of a launch
  RotaryArgs a = {};
  a.x = in->x.data;
  a.y = const_cast<void*>(in->y.data);
  a.positions = in->positions;
  a.rows = in->rows;
  a.x_row = in->x.row;
  a.x_head = in->x.head;
  a.y_row = in->y.row;
  a.y_head = in->y.head;
  a.pos_row = in->pos_row;
  a.pos_axis = in->pos_axis;
  a.heads = (int)in->heads;
  a.dim = (int)in->dim;
  a.axes = (int)in->axes;
  a.pairs = (int)in->pairs;
  a.amplitude = (float)in->amplitude;
  a.sign = in->transposed ? -1.f : 1.f;
  for (int i = 0; i < a.pairs; ++i) a.turns[i] = in->turns[i];
  cudaStream_t s = (cudaStream_t)in->stream;
  const int pos = (int)in->pos_type, inter = in->interleaved != 0;
  if (in->type == kF32) return launch_for<float>(a, pos, inter, s);
  if (in->type == kF16) return launch_for<__half>(a, pos, inter, s);
  return launch_for<__nv_bfloat16>(a, pos, inter, s);
}
