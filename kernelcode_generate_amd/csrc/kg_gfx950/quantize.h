// Rows in 8-bit integers: s = max|x| fl32(1 / 127), code = x / s as a 32-bit quotient, rounded to the nearest whole number, ties
// to even (0 where s is 0 or not finite: a row with an infinity or NaN keeps that scale, which makes all that is made
// of the row infinite or NaN).
//
// quantize_rows_kernel: a workgroup of kThreads lanes (or a wave of it) per row, which it holds in registers, 8 elements a piece, from
// the one read that there is to the codes; any K up to 8 kPieces kThreads, any alignment (the pieces' loads are of whole
// 16 bytes where the row has them, wherever it starts). quantize_rows_any_kernel reads longer rows twice.
#pragma once

#include <type_traits>

#include "common.h"
#include "kv_cache.h"

namespace kg_gfx950 {

struct QuantizeArgs {
  const void* x;
  int8_t* codes;
  float* scale;
  long long x_row, c_row, scale_stride;
  int rows, k, width;  // width >= k: columns of codes to write, zeros behind k
};

// 8 elements of a row from column c, zeros behind its end.
template <typename T>
__device__ __forceinline__ void load_eight(const T* row, int c, int k, float (&x)[8]) {
  if (c + 8 <= k) {
    if constexpr (std::is_same<T, float>::value) {
      struct __attribute__((packed, aligned(4))) Piece {
        float e[8];
      };
      const Piece p = *reinterpret_cast<const Piece*>(row + c);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p.e[i];
    } else {
      using Tag = typename Eight<T>::Tag;
      struct __attribute__((packed, aligned(2))) Piece {
        u32x4 w;
      };
      const u32x4 w = reinterpret_cast<const Piece*>(row + c)->w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = w[i];
        x[2 * i] = Half16<Tag>::to_float(u & 0xffffu);
        x[2 * i + 1] = Half16<Tag>::to_float(u >> 16);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c + i < k ? Elem<T>::load(row + c + i) : 0.f;
  }
}

// Codes of 8 elements, packed. `inverse`: of a scale within 2^-60..2^60 (scaled_codes), 0 for another one.
__device__ __forceinline__ u32x2 int8_codes(float (&x)[8], float scale) {
  if (!(scale <= 3.4028235e38f)) return u32x2{0u, 0u};
  scaled_codes<int8_t>(x, scale);
  u32x2 w = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i >> 2] |= ((uint32_t)(int)__builtin_rintf(x[i]) & 0xffu) << (8 * (i & 3));
  return w;
}

// 8 codes to columns c .. c + 7 of a row of `width` columns, of which any alignment.
__device__ __forceinline__ void store_codes(int8_t* row, int c, int width, u32x2 w) {
  if (c + 8 <= width) {
    struct __attribute__((packed, aligned(1))) Piece {
      u32x2 w;
    };
    reinterpret_cast<Piece*>(row + c)->w = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < width) row[c + i] = (int8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
}

// kWaves: of a row; a workgroup has 4 / kWaves rows.
template <typename T, int kPieces, int kWaves>
__device__ __forceinline__ void quantize_row(const QuantizeArgs& a, long long row, float* lds) {
  constexpr int kLanes = 64 * kWaves;
  const int part = threadIdx.x % kLanes;
  const bool real = row < a.rows;
  const T* src = static_cast<const T*>(a.x) + (real ? row : 0) * a.x_row;
  float x[kPieces][8];
#pragma unroll
  for (int p = 0; p < kPieces; ++p) load_eight(src, 8 * (part + p * kLanes), real ? a.k : 0, x[p]);
  float top = 0.f;
#pragma unroll
  for (int p = 0; p < kPieces; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = nan_max(top, __builtin_fabsf(x[p][i]));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = nan_max(top, __shfl_xor(top, o, 64));
  if constexpr (kWaves > 1) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = nan_max(top, lds[w]);
  }
  if (!real) return;
  const float scale = top * CacheElem<int8_t>::kInverse;
  if (part == 0) a.scale[row * a.scale_stride] = scale;
  int8_t* dst = a.codes + row * a.c_row;
#pragma unroll
  for (int p = 0; p < kPieces; ++p) {
    const int c = 8 * (part + p * kLanes);
    if (c < a.width) store_codes(dst, c, a.width, int8_codes(x[p], scale));
  }
}

template <typename T, int kPieces, int kWaves>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeArgs a) {
  __shared__ float lds[4];
  quantize_row<T, kPieces, kWaves>(a, (long long)blockIdx.x * (4 / kWaves) + threadIdx.x / (64 * kWaves), lds);
}

template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_any_kernel(QuantizeArgs a) {
  __shared__ float lds[4];
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* src = static_cast<const T*>(a.x) + row * a.x_row;
    float top = 0.f, x[8];
    for (int c = 8 * threadIdx.x; c < a.k; c += 8 * 256) {
      load_eight(src, c, a.k, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = nan_max(top, __builtin_fabsf(x[i]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = nan_max(top, __shfl_xor(top, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
    __syncthreads();
    top = nan_max(nan_max(lds[0], lds[1]), nan_max(lds[2], lds[3]));
    const float scale = top * CacheElem<int8_t>::kInverse;
    if (threadIdx.x == 0) a.scale[row * a.scale_stride] = scale;
    int8_t* dst = a.codes + row * a.c_row;
    for (int c = 8 * threadIdx.x; c < a.width; c += 8 * 256) {
      load_eight(src, c, a.k, x);
      store_codes(dst, c, a.width, int8_codes(x, scale));
    }
  }
}

}  // namespace kg_gfx950
