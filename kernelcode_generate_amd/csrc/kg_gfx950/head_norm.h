// Norms of queries and keys for each head with the position rotation, one pass over both:
//   y = x / sqrt(sum_d x_d^2 / D + eps) w   (where the side has weights w; y = x otherwise),
//   (a, b) -> (a cos - b sin, b cos + a sin) for pair i of the token's position, i < half: elements (i, i + half), or (2 i, 2 i + 1)
// of neighbours; elements behind 2 half stay as they are. All of it in 32 bits, rounded once to the output's type. A sum of
// squares past 3.4e38 is infinite there, and the row 0. A mean square with eps below 2^-100 is taken of 2^100 times the elements, which
// is exact: squares, mean and the inverse root's input (v_rsq_f32 takes subnormal ones for 0) are then normal numbers for elements of any size.
//
// head_norm_kernel: L lanes per head, each with the W elements on both sides of its pairs (2 W side by side of neighbours), so that a
// pair never leaves its lane, and G heads of a token at a time, whose reads are in flight together and whose angles and weights are read
// once; half a multiple of W, an even D of 2 W, rows that start anywhere. Bound by its bytes where there are many: 8192 tokens of 32 and 8
// heads of 128 in bf16 33 us, 4.9 TB/s, in fp32 62, 5.1 TB/s; 64 tokens take 3.3, a launch's 2.3 and one chain of reads.
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

// Of a mean square with eps below kTinyMean, elements are taken kEnlarge times; both products with eps, which is below 2^-100 too, stay in range.
constexpr float kTinyMean = 0x1p-100f, kEnlarge = 0x1p100f;
__device__ __forceinline__ float enlarged_mean(const HeadNormArgs& a, float sum) { return sum * a.inverse_d + a.eps * kEnlarge * kEnlarge; }

// 1 / sqrt(sum of squares / D + eps). squares(): the sum over the head, the same in all of its lanes; enlarge(by): multiplies the elements.
template <typename F, typename G>
__device__ __forceinline__ float head_norm_inverse(const HeadNormArgs& a, F squares, G enlarge) {
  float mean = squares() * a.inverse_d + a.eps;
  if (mean < kTinyMean) {
    enlarge(kEnlarge);
    mean = enlarged_mean(a, squares());
  }
  return __builtin_amdgcn_rsqf(mean);
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
      float mean = wave_sum(sum) * a.inverse_d + a.eps;
      if (mean < kTinyMean) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
          e[i][0] *= kEnlarge, e[i][1] *= kEnlarge;
          sum += e[i][0] * e[i][0] + e[i][1] * e[i][1];
        }
        mean = enlarged_mean(a, wave_sum(sum));
      }
      const float by = __builtin_amdgcn_rsqf(mean);
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

// W elements from any address, in 32 bits, and back.
template <typename T, int W>
struct Elements {
  static constexpr bool kOne = W * sizeof(T) < 4;  // one element of 16 bits
  static constexpr int kDwords = kOne ? 1 : W * sizeof(T) / 4;
  struct __attribute__((packed, aligned(sizeof(T)))) Piece {
    uint32_t w[kDwords];
  };
  static __device__ __forceinline__ void load(const T* p, float (&x)[W]) {
    if constexpr (kOne) {
      x[0] = Elem<T>::load(p);
    } else {
      const Piece q = *reinterpret_cast<const Piece*>(p);
#pragma unroll
      for (int i = 0; i < kDwords; ++i) {
        const uint32_t u = q.w[i];
        if constexpr (sizeof(T) == 4) {
          x[i] = __builtin_bit_cast(float, u);
        } else {
          using H = Half16<typename Eight<T>::Tag>;
          x[2 * i] = H::to_float(u & 0xffffu);
          x[2 * i + 1] = H::to_float(u >> 16);
        }
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&x)[W]) {
    if constexpr (kOne) {
      Elem<T>::store(p, x[0]);
    } else {
      Piece q;
#pragma unroll
      for (int i = 0; i < kDwords; ++i) {
        if constexpr (sizeof(T) == 4) q.w[i] = __builtin_bit_cast(uint32_t, x[i]);
        else q.w[i] = Half16<typename Eight<T>::Tag>::pack2(x[2 * i], x[2 * i + 1]);
      }
      *reinterpret_cast<Piece*>(p) = q;
    }
  }
};

struct HeadNormItems {
  int items, chunks, chunks_q;  // of G heads: of a token, of its queries
  PageDiv by_chunks;
};

// (weights, cos and sin contiguous)
template <typename T, int W, int L, int G>
__global__ __launch_bounds__(256) void head_norm_kernel(HeadNormArgs a, HeadNormItems n) {
  using E = Elements<T, W>;
  const int part = threadIdx.x % L;
  const int item = blockIdx.x * (256 / L) + threadIdx.x / L;
  if (item >= n.items) return;
  const int t = div_page(item, n.by_chunks), c = item - t * n.chunks;
  const long long position = head_norm_position(a, t);
  if (position < 0 || position >= a.table) return;
  const bool keys = c >= n.chunks_q;
  const HeadNormSide& s = a.side[keys];
  const int h0 = (keys ? c - n.chunks_q : c) * G;
  const bool in = 2 * W * part < a.d, turned = in && W * part < a.half;
  // the lane's elements: first .. + W - 1 and second .. + W - 1
  const int first = !in ? 0 : turned && !a.neighbours ? W * part : 2 * W * part;
  const int second = !in ? 0 : turned && !a.neighbours ? a.half + W * part : 2 * W * part + W;
  const T* x = static_cast<const T*>(s.x) + t * s.x_token;
  float p[G][W], q[G][W];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const T* row = x + min(h0 + g, s.heads - 1) * s.x_head;
    E::load(row + first, p[g]);
    E::load(row + second, q[g]);
  }
  float cs[W], sn[W];
  if (turned) {
    Elements<float, W>::load(a.cos + position * a.cos_row + W * part, cs);
    Elements<float, W>::load(a.sin + position * a.sin_row + W * part, sn);
  }
  if (s.w != nullptr) {
    float u[W], v[W];
    if (s.wide) {
      Elements<float, W>::load(static_cast<const float*>(s.w) + first, u);
      Elements<float, W>::load(static_cast<const float*>(s.w) + second, v);
    } else {
      E::load(static_cast<const T*>(s.w) + first, u);
      E::load(static_cast<const T*>(s.w) + second, v);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      auto squares = [&]() {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) sum = __builtin_fmaf(p[g][i], p[g][i], __builtin_fmaf(q[g][i], q[g][i], sum));
        if (!in) sum = 0.f;
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        return sum;
      };
      const float by = head_norm_inverse(a, squares, [&](float f) {
#pragma unroll
        for (int i = 0; i < W; ++i) p[g][i] *= f, q[g][i] *= f;
      });
#pragma unroll
      for (int i = 0; i < W; ++i) p[g][i] *= by * u[i], q[g][i] *= by * v[i];
    }
  }
  if (turned) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (a.neighbours) {
#pragma unroll
        for (int i = 0; i < W; ++i) {  // pair i: elements 2 i and 2 i + 1 of both pieces in a row
          float& e = 2 * i < W ? p[g][2 * i % W] : q[g][2 * i % W];
          float& f = 2 * i + 1 < W ? p[g][(2 * i + 1) % W] : q[g][(2 * i + 1) % W];
          const float r = e * cs[i] - f * sn[i];
          f = f * cs[i] + e * sn[i];
          e = r;
        }
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float r = p[g][i] * cs[i] - q[g][i] * sn[i];
          q[g][i] = q[g][i] * cs[i] + p[g][i] * sn[i];
          p[g][i] = r;
        }
      }
    }
  }
  if (!in) return;
  T* y = static_cast<T*>(s.y) + t * s.y_token;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (h0 + g >= s.heads) continue;
    T* row = y + (h0 + g) * s.y_head;
    E::store(row + first, p[g]);
    E::store(row + second, q[g]);
  }
}

// Whether the kernel above takes the call with pieces of `w` elements; 0 lanes: it does not.
inline int head_norm_lanes(const HeadNormArgs& a, int w) {
  if (a.half % w != 0 || a.d % (2 * w) != 0 || a.d / (2 * w) > 64) return 0;
  for (const HeadNormSide& s : a.side)
    if (s.w != nullptr && s.w_stride != 1) return 0;
  if (a.half > 1 && (a.cos_stride != 1 || a.sin_stride != 1)) return 0;
  int lanes = 4;
  while (lanes * 2 * w < a.d) lanes *= 2;
  return lanes;
}

template <typename T, int W, int G>
bool launch_head_norm(const HeadNormArgs& a, int lanes, hipStream_t stream) {
  HeadNormItems n;
  auto chunks = [](int heads) { return heads / G + (heads % G != 0); };  // (up to 2^31 - 1 heads)
  n.chunks_q = chunks(a.side[0].heads);
  n.chunks = n.chunks_q + chunks(a.side[1].heads);
  const long long items = (long long)a.tokens * n.chunks, blocks = (items + 256 / lanes - 1) / (256 / lanes);
  if (items > 0x7fffff00LL || blocks > (1 << 24) - 1) return false;
  n.items = (int)items;
  n.by_chunks = page_div(n.chunks);
#define KG_HEAD_NORM(L) hipLaunchKernelGGL((head_norm_kernel<T, W, L, G>), dim3((unsigned)blocks), dim3(256), 0, stream, a, n)
  if (lanes == 4) KG_HEAD_NORM(4);
  else if (lanes == 8) KG_HEAD_NORM(8);
  else if (lanes == 16) KG_HEAD_NORM(16);
  else if (lanes == 32) KG_HEAD_NORM(32);
  else if constexpr (W < 8) KG_HEAD_NORM(64);  // (pieces of 8: 512 elements in 32 lanes)
#undef KG_HEAD_NORM
  return true;
}

// False: no form of the kernel takes the call. The widest pieces that the halves allow, and heads at a time that the measurements say, us
// with 1 / 2 / 4: 8 elements, 1600 x 40 x 128 bf16 8.7 / 8.9 / 9.2, 8192 x 40 x 128 35.7 / 34.2 / 36.3; 4 elements, 4000 x 24 x 72 f16 18.9 / 14.1 / 12.5; 2,
// 4000 x 24 x 80 of which 20 turn 16.2 / 12.5 / 11.2; 1, 4000 x 36 x 72 of which 18 turn 30.3 / 20.7 / 16.9 (the kernel of any head 68); few rows 3.3 with any.
template <typename T>
bool launch_head_norm(const HeadNormArgs& a, hipStream_t stream) {
  const long long elements = (long long)a.tokens * (a.side[0].heads + a.side[1].heads) * a.d;
  const bool many = elements >= 1 << 21;
  if (const int lanes = head_norm_lanes(a, 8))
    return elements >= 1 << 24 ? launch_head_norm<T, 8, 2>(a, lanes, stream) : launch_head_norm<T, 8, 1>(a, lanes, stream);
  if (const int lanes = head_norm_lanes(a, 4))
    return many ? launch_head_norm<T, 4, 4>(a, lanes, stream) : launch_head_norm<T, 4, 1>(a, lanes, stream);
  if (const int lanes = head_norm_lanes(a, 2))
    return many ? launch_head_norm<T, 2, 4>(a, lanes, stream) : launch_head_norm<T, 2, 1>(a, lanes, stream);
  if (const int lanes = head_norm_lanes(a, 1))
    return many ? launch_head_norm<T, 1, 4>(a, lanes, stream) : launch_head_norm<T, 1, 1>(a, lanes, stream);
  return false;
}

}  // namespace kg_gfx950
