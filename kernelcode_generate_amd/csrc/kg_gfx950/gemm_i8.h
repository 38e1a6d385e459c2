// Products in 8-bit integers with a scale for each row and channel:
//   out[m, n] = (sum_k x[m, k] w[n, k]) x_scale[m] w_scale[n] + bias[n],
// w one row a channel, so that both operands lie along k. Sums are exact: |x w| <= 2^14, and K <= 131071 of them stay below 2^31.
// They become 32-bit floats (rounded past 2^24), then the two products, the bias, and one rounding to the output's type.
//
// int8_any_kernel: any strides, alignment and K, x in codes or in elements that it quantises itself (quantize.h): a workgroup per row and
// 64 channels, a wave per channel at a time.
#pragma once

#include "common.h"
#include "kv_cache.h"
#include "quantize.h"

namespace kg_gfx950 {

constexpr int kInt8MostK = 131071;

struct Int8Args {
  const void* x;  // codes, or elements to quantise
  const int8_t* w;
  const float *x_scale, *w_scale;
  const void* bias;
  void* out;
  long long x_row, w_row, out_row, x_scale_stride, w_scale_stride, bias_stride;
  int m, n, k;
  bool wide_bias;  // 32 bits
};

template <typename T>
__device__ __forceinline__ float int8_bias(const void* bias, long long stride, bool wide, long long n) {
  if (bias == nullptr) return 0.f;
  return wide ? static_cast<const float*>(bias)[n * stride] : Elem<T>::load(static_cast<const T*>(bias) + n * stride);
}

// X: int8_t (codes) or T
template <typename T, typename X>
__global__ __launch_bounds__(256) void int8_any_kernel(Int8Args a) {
  constexpr bool kCodes = std::is_same<X, int8_t>::value;
  constexpr int kChunk = 8192, kChannels = 16;  // of a wave
  __shared__ int8_t codes[kChunk];
  __shared__ float lds[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int blocks = (int)((a.n + 4ll * kChannels - 1) / (4 * kChannels));  // (up to 2^31 - 1 channels)
  for (long long item = blockIdx.x; item < (long long)a.m * blocks; item += gridDim.x) {
    const int m = (int)(item / blocks), n0 = (int)(item - (long long)m * blocks) * 4 * kChannels + wave * kChannels;
    const X* x = static_cast<const X*>(a.x) + m * a.x_row;
    float scale;
    if constexpr (kCodes) {
      scale = a.x_scale[m * a.x_scale_stride];
    } else {
      float top = 0.f;
      for (int k = tid; k < a.k; k += 256) top = nan_max(top, __builtin_fabsf(Elem<X>::load(x + k)));
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) top = nan_max(top, __shfl_xor(top, o, 64));
      __syncthreads();
      if (lane == 0) lds[wave] = top;
      __syncthreads();
      scale = nan_max(nan_max(lds[0], lds[1]), nan_max(lds[2], lds[3])) * CacheElem<int8_t>::kInverse;
    }
    int acc[kChannels];
#pragma unroll
    for (int i = 0; i < kChannels; ++i) acc[i] = 0;
    for (int k0 = 0; k0 < a.k; k0 += kChunk) {
      const int count = min(kChunk, a.k - k0);
      __syncthreads();
      for (int k = tid; k < count; k += 256) {
        if constexpr (kCodes) codes[k] = x[k0 + k];
        else codes[k] = scale <= 3.4028235e38f ? (int8_t)__builtin_rintf(scaled_code<int8_t>(Elem<X>::load(x + k0 + k), scale)) : (int8_t)0;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kChannels; ++i) {
        if (n0 + i >= a.n) continue;
        const int8_t* w = a.w + (n0 + i) * a.w_row + k0;
        for (int k = lane; k < count; k += 64) acc[i] += (int)codes[k] * (int)w[k];
      }
    }
#pragma unroll
    for (int i = 0; i < kChannels; ++i) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) acc[i] += __shfl_xor(acc[i], o, 64);
      const int n = n0 + i;
      if (lane == 0 && n < a.n)
        Elem<T>::store(static_cast<T*>(a.out) + m * a.out_row + n, (float)acc[i] * scale * a.w_scale[n * a.w_scale_stride] + int8_bias<T>(a.bias, a.bias_stride, a.wide_bias, n));
    }
  }
}

}  // namespace kg_gfx950
