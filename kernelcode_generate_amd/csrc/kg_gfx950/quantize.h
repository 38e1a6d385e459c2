// Rows in 8-bit integers: s = max|x| fl32(1 / 127), code = x / s as a 32-bit quotient, rounded to the nearest whole number, ties
// to even (0 where s is 0 or not finite: a row with an infinity or NaN keeps that scale, which makes all that is made
// of the row infinite or NaN).
//
// quantize_rows_kernel: a row's lanes hold it in registers, 8 elements a piece, from the one read that there is to the codes; rows of 8
// up to 16384 elements, starting anywhere. A wave a row up to 512 elements, four beyond: 4001 rows of 4096 in fp16 9.2 us, 5.3 TB/s, bound by
// their bytes; 4096 rows of 16384 in bf16 36 us, in fp32 68; 16 rows 2.4, a launch's. quantize_rows_any_kernel reads its rows twice, element by
// element: 4096 rows of 28672 in bf16 224 us, 1.6 TB/s, in fp32 281; 16 rows 39.
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

// w >> 8 bytes, of 16 bytes; zeros from 16 on.
__device__ __forceinline__ u32x4 shift_bytes(u32x4 w, int bytes) {
  uint64_t lo = (uint64_t)w[0] | (uint64_t)w[1] << 32, hi = (uint64_t)w[2] | (uint64_t)w[3] << 32;
  if (bytes >= 8) lo = hi, hi = 0;
  const int bits = 8 * (bytes & 7);
  lo = lo >> bits | hi << 1 << (63 - bits);
  hi >>= bits;
  if (bytes >= 16) lo = 0, hi = 0;
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}
// 16 bytes at any address
__device__ __forceinline__ u32x4 load_bytes(const void* p) {
  struct __attribute__((packed, aligned(1))) Piece {
    u32x4 w;
  };
  return reinterpret_cast<const Piece*>(p)->w;
}

// 8 elements of a row as they lie in memory, and in 32 bits.
template <typename T>
struct RawEight {
  using Tag = typename Eight<T>::Tag;
  u32x4 w;
  __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = Half16<Tag>::to_float(w[i] & 0xffffu);
      x[2 * i + 1] = Half16<Tag>::to_float(w[i] >> 16);
    }
  }
};
template <>
struct RawEight<float> {
  float e[8];
  __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = e[i];
  }
};

// 8 elements of a row of k >= 8 from column c, zeros behind its end, without a branch: loads of several pieces are in flight
// together. kWhole: k and c are multiples of 8; otherwise the last 16 bytes of the row are shifted into place.
template <typename T, bool kWhole>
__device__ __forceinline__ RawEight<T> load_eight(const T* row, int c, int k) {
  RawEight<T> x;
  if constexpr (std::is_same<T, float>::value) {
    if constexpr (kWhole) {
      const bool in = c < k;
      const f32x4 a = __builtin_bit_cast(f32x4, load_bytes(row + (in ? c : 0)));
      const f32x4 b = __builtin_bit_cast(f32x4, load_bytes(row + (in ? c : 0) + 4));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x.e[i] = in ? a[i] : 0.f;
        x.e[4 + i] = in ? b[i] : 0.f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = row[min(c + i, k - 1)];
        x.e[i] = c + i < k ? e : 0.f;
      }
    }
  } else {
    const int at = min(c, k - 8);
    x.w = load_bytes(row + at);
    if constexpr (kWhole) x.w = c < k ? x.w : u32x4{0u, 0u, 0u, 0u};
    else x.w = shift_bytes(x.w, 2 * min(c - at, 8));
  }
  return x;
}

template <typename T>
__device__ __forceinline__ float largest_of(const RawEight<T>& raw) {
  float x[8], top = 0.f;
  raw.floats(x);
#pragma unroll
  for (int i = 0; i < 8; ++i) top = nan_max(top, __builtin_fabsf(x[i]));
  return top;
}

// Codes of 8 elements, packed. One branch for all lanes: scales outside 2^-60..2^60 in none of them is the rule.
template <typename T>
__device__ __forceinline__ u32x2 int8_codes(const RawEight<T>& raw, float scale) {
  float x[8];
  raw.floats(x);
  u32x2 w = {0u, 0u};
  if (__builtin_amdgcn_ballot_w64(!(scale >= 0x1p-60f && scale <= 0x1p60f)) == 0) {
    const float inverse = 1.f / scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // x / scale rounded to nearest (scaled_codes); its magnitude is at most 127 by the scale's making and a rounding, which
      // the nearest whole number takes back
      float q = x[i] * inverse;
      q = __builtin_fmaf(__builtin_fmaf(-q, scale, x[i]), inverse, q);
      q = __builtin_fmaf(__builtin_fmaf(-q, scale, x[i]), inverse, q);
      w[i >> 2] |= ((uint32_t)(int)__builtin_rintf(q) & 0xffu) << (8 * (i & 3));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = scale <= 3.4028235e38f ? scaled_code<int8_t>(x[i], scale) : 0.f;
      w[i >> 2] |= ((uint32_t)(int)__builtin_rintf(q) & 0xffu) << (8 * (i & 3));
    }
  }
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

// kWaves waves a row, 4 / kWaves rows a workgroup. Rows of 8 elements and more.
template <typename T, int kPieces, int kWaves, bool kWhole>
__device__ __forceinline__ void quantize_row(const QuantizeArgs& a, long long row, float* lds) {
  constexpr int kLanes = 64 * kWaves;
  const int part = threadIdx.x % kLanes;
  const bool real = row < a.rows;
  const T* src = static_cast<const T*>(a.x) + (real ? row : 0) * a.x_row;
  RawEight<T> raw[kPieces];
#pragma unroll
  for (int p = 0; p < kPieces; ++p) raw[p] = load_eight<T, kWhole>(src, 8 * (part + p * kLanes), a.k);
  float top = 0.f;
#pragma unroll
  for (int p = 0; p < kPieces; ++p) top = nan_max(top, largest_of(raw[p]));
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
    if (c < a.width) store_codes(dst, c, a.width, int8_codes(raw[p], scale));
  }
}

// 16 codes of a row of `count` >= 16 from column k, zeros behind its end, without a branch.
__device__ __forceinline__ u32x4 load_codes(const int8_t* row, int k, int count) {
  const int at = min(k, count - 16);
  return shift_bytes(load_bytes(row + at), min(k - at, 16));
}

// Rows of k >= 16 codes copied into rows of `pitch` bytes, a multiple of 16, zeros behind k: for copies to LDS, which take whole
// 16-byte pieces.
struct PackArgs {
  const int8_t* src;
  int8_t* dst;
  long long ld;
  int pitch, rows, k;
};
__device__ __forceinline__ void pack_rows(const PackArgs& p, long long thread, long long threads) {
  const int pieces = p.pitch / 16;
  for (long long at = thread; at < (long long)p.rows * pieces; at += threads) {
    const int r = (int)(at / pieces), c = 16 * (int)(at - (long long)r * pieces);
    st16(p.dst + (long long)r * p.pitch + c, load_codes(p.src + r * p.ld, c, p.k));
  }
}

// The workgroups behind those of the rows pack: weights beside the rows of one call.
template <typename T, int kPieces, int kWaves, bool kWhole>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeArgs a, PackArgs pack) {
  __shared__ float lds[4];
  const int own = (a.rows + 4 / kWaves - 1) / (4 / kWaves);
  if ((int)blockIdx.x >= own) {
    pack_rows(pack, ((long long)blockIdx.x - own) * 256 + threadIdx.x, 256ll * ((int)gridDim.x - own));
    return;
  }
  quantize_row<T, kPieces, kWaves, kWhole>(a, (long long)blockIdx.x * (4 / kWaves) + threadIdx.x / (64 * kWaves), lds);
}

// Rows of any length, read twice.
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_any_kernel(QuantizeArgs a) {
  __shared__ float lds[4];
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* src = static_cast<const T*>(a.x) + row * a.x_row;
    float top = 0.f;
    for (int c = threadIdx.x; c < a.k; c += 256) top = nan_max(top, __builtin_fabsf(Elem<T>::load(src + c)));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = nan_max(top, __shfl_xor(top, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
    __syncthreads();
    top = nan_max(nan_max(lds[0], lds[1]), nan_max(lds[2], lds[3]));
    const float scale = top * CacheElem<int8_t>::kInverse;
    if (threadIdx.x == 0) a.scale[row * a.scale_stride] = scale;
    int8_t* dst = a.codes + row * a.c_row;
    for (int c = threadIdx.x; c < a.width; c += 256)
      dst[c] = c < a.k && scale <= 3.4028235e38f ? (int8_t)__builtin_rintf(scaled_code<int8_t>(Elem<T>::load(src + c), scale)) : (int8_t)0;
  }
}

}  // namespace kg_gfx950
