// Norms of queries and keys for each head with the position rotation, one pass over both:
//   y = x / sqrt(sum_d x_d^2 / D + eps) w   (where the side has weights w; y = x otherwise),
//   (a, b) -> (a cos - b sin, b cos + a sin) for pair i of the token's position, i < half: elements (i, i + half), or (2 i, 2 i + 1)
// of neighbours; elements behind 2 half stay as they are. All of it in 32 bits, rounded once to the output's type. A sum of
// squares past 3.4e38 is infinite there, and the row 0.
//
// head_norm_any_kernel: any D up to 512, half, strides and alignment: a wave per token and head, each lane some pairs of elements.
#pragma once

#include "common.h"
#include "kv_cache.h"

namespace kg_gfx950 {

struct HeadNormSide {
  const void *x, *w;
  void* y;
  long long x_token, x_head, y_token, y_head, w_stride;
  int heads;
  bool wide;  // weights in 32 bits
};
struct HeadNormArgs {
  HeadNormSide side[2];  // queries, keys
  const float *cos, *sin;
  const void* positions;
  long long cos_row, sin_row, cos_stride, sin_stride, position_stride, table;
  int tokens, d, half;
  bool wide_positions, neighbours;
  float eps, inverse_d;
};

__device__ __forceinline__ long long head_norm_position(const HeadNormArgs& a, int t) {
  return a.wide_positions ? static_cast<const long long*>(a.positions)[t * a.position_stride]
                          : (long long)static_cast<const int*>(a.positions)[t * a.position_stride];
}

template <typename T>
__global__ __launch_bounds__(256) void head_norm_any_kernel(HeadNormArgs a) {
  constexpr int kMost = 4;  // pairs of a lane: 512 elements
  const int lane = threadIdx.x & 63;
  const int heads = a.side[0].heads + a.side[1].heads;
  for (long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); item < (long long)a.tokens * heads; item += 4ll * gridDim.x) {
    const int t = (int)(item / heads), h0 = (int)(item - (long long)t * heads);
    const bool keys = h0 >= a.side[0].heads;
    const HeadNormSide& s = a.side[keys];
    const int h = keys ? h0 - a.side[0].heads : h0;
    const long long position = head_norm_position(a, t);
    if (position < 0 || position >= a.table) continue;
    const T* x = static_cast<const T*>(s.x) + t * s.x_token + h * s.x_head;
    T* y = static_cast<T*>(s.y) + t * s.y_token + h * s.y_head;
    // unit u: pair u, or for u >= half the elements 2 u and 2 u + 1
    float e[kMost][2];
    float sum = 0.f;
    auto first = [&](int u) { return u < a.half && !a.neighbours ? u : 2 * u; };
    auto second = [&](int u) { return u < a.half && !a.neighbours ? u + a.half : 2 * u + 1; };
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      const int u = lane + 64 * i;
      e[i][0] = first(u) < a.d ? Elem<T>::load(x + first(u)) : 0.f;
      e[i][1] = second(u) < a.d ? Elem<T>::load(x + second(u)) : 0.f;
      sum += e[i][0] * e[i][0] + e[i][1] * e[i][1];
    }
    if (s.w != nullptr) {
      const float by = __builtin_amdgcn_rsqf(wave_sum(sum) * a.inverse_d + a.eps);
      auto weight = [&](int d) {
        if (d >= a.d) return 0.f;
        return s.wide ? static_cast<const float*>(s.w)[d * s.w_stride] : Elem<T>::load(static_cast<const T*>(s.w) + d * s.w_stride);
      };
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        const int u = lane + 64 * i;
        e[i][0] *= by * weight(first(u));
        e[i][1] *= by * weight(second(u));
      }
    }
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      const int u = lane + 64 * i;
      if (u < a.half) {
        const float c = a.cos[position * a.cos_row + u * a.cos_stride], n = a.sin[position * a.sin_row + u * a.sin_stride];
        const float p = e[i][0], q = e[i][1];
        e[i][0] = p * c - q * n;
        e[i][1] = q * c + p * n;
      }
      if (first(u) < a.d) Elem<T>::store(y + first(u), e[i][0]);
      if (second(u) < a.d) Elem<T>::store(y + second(u), e[i][1]);
    }
  }
}

}  // namespace kg_gfx950
