// A paged cache of attention keys and values: rows of D elements, one per token and key head, in
// pages of `page_size` tokens ([pages, heads, page_size, D], any strides but the last), held in the
// model's own type or in 8 bits with a 32-bit scale per row ([pages, heads, page_size]).
//
// Written: slot = page page_size + offset; s = max|x| fl32(1 / Q), Q = 448 (e4m3) or 127 (int8);
// code = x / s rounded to the nearest value of the type, ties to even (0 where s is 0). An
// infinity or NaN in a row makes its scale one, and the whole row reads back as NaN. Read back: code s,
// rounded once to the output's type.
//
// kv_store_kernel, kv_load_kernel: rows of whole 16-byte pieces (8 elements a lane), bound by their bytes where there are many:
// 4001 tokens of 8 heads of 128 from fp16 to int8 8.7 us, 2.7 TB/s (28 with a wave per row); four ragged sequences of up to 8192
// back from e4m3 to bf16 34.8 us, 4.1 TB/s (169). 64 tokens take 3.0 us, a launch's. kv_store_any_kernel, kv_load_any_kernel:
// any D and alignment and any number of rows, one wave per row.
#pragma once

#include <type_traits>

#include "common.h"

namespace kg_gfx950 {

// Exact n / d for 0 <= n < 2^31 by one multiplication (Granlund and Montgomery): mult = floor(2^shift / d) + 1
// with shift = 31 + ceil(log2 d), so mult d - 2^shift <= d and the error stays below 1 / d.
struct PageDiv {
  uint64_t mult;
  int shift;
};
inline PageDiv page_div(int d) {
  int s = 0;
  while ((1ll << s) < d) ++s;
  return PageDiv{((1ull << (31 + s)) / (uint64_t)d) + 1, 31 + s};
}
__device__ __forceinline__ int div_page(int n, const PageDiv& p) { return (int)((uint64_t)(uint32_t)n * p.mult >> p.shift); }

// 8-bit cache elements: raw bytes, what they stand for, and the largest magnitude.
struct E4m3 {
  uint8_t bits;
};
template <typename T>
struct CacheElem {
  static constexpr bool kScaled = false;
  static __device__ __forceinline__ float load(const T* p) { return Elem<T>::load(p); }
  static __device__ __forceinline__ void store(T* p, float v) { Elem<T>::store(p, v); }
};
template <>
struct CacheElem<E4m3> {
  static constexpr bool kScaled = true;
  static constexpr float kLargest = 448.f, kInverse = (float)(1.0 / 448.0);
  static __device__ __forceinline__ float load(const E4m3* p) { return __builtin_amdgcn_cvt_f32_fp8((int)p->bits, 0); }
  static __device__ __forceinline__ void store(E4m3* p, float v) {
    p->bits = (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v, 0.f, 0, false) & 0xff);
  }
};
template <>
struct CacheElem<int8_t> {
  static constexpr bool kScaled = true;
  static constexpr float kLargest = 127.f, kInverse = (float)(1.0 / 127.0);
  static __device__ __forceinline__ float load(const int8_t* p) { return (float)*p; }
  static __device__ __forceinline__ void store(int8_t* p, float v) { *p = (int8_t)__builtin_rintf(v); }
};

// x / scale within the type's range; 0 where the scale is 0 or NaN (the scale then makes the row)
template <typename C>
__device__ __forceinline__ float scaled_code(float x, float scale) {
  const float c = scale > 0.f ? x / scale : 0.f;
  // (a NaN, from infinities, passes)
  return c > CacheElem<C>::kLargest ? CacheElem<C>::kLargest : c < -CacheElem<C>::kLargest ? -CacheElem<C>::kLargest : c;
}

__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// One of the two caches with its scales (null: none) and, for a call, the dense rows it is written from
// or read into. Strides in elements; the last axis of rows is contiguous.
struct KvSide {
  void* cache;
  float* scale;
  void* rows;
  long long page, head, row;     // strides of the cache
  long long s_page, s_head, s_row;  // of its scales
  long long r0, r1, r2;          // of the dense rows: store [T, H, D] r0, r1; load [B, H, S, D] r0, r1, r2
};

struct KvStoreArgs {
  KvSide side[2];
  const long long* slots;
  long long slot_stride;
  int tokens, heads, d, page_size;
  long long total_slots;
  PageDiv by_heads;
};

// page and offset of a slot inside the cache
__device__ __forceinline__ void split_slot(long long slot, int page_size, long long* page, int* offset) {
  if (slot <= 0xffffffffll) {  // (a 64-bit division takes some 100 instructions)
    const uint32_t p = (uint32_t)slot / (uint32_t)page_size;
    *page = p;
    *offset = (int)((uint32_t)slot - p * (uint32_t)page_size);
  } else {
    *page = slot / page_size;
    *offset = (int)(slot - *page * page_size);
  }
}

template <typename Src, typename C>
__global__ __launch_bounds__(256) void kv_store_any_kernel(KvStoreArgs a) {
  const int lane = threadIdx.x & 63;
  const long long rows = (long long)a.tokens * a.heads;
  for (long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); item < 2 * rows; item += 4ll * gridDim.x) {
    const KvSide& s = a.side[item >= rows];
    const long long r = item >= rows ? item - rows : item;
    const int t = (int)(r / a.heads), h = (int)(r - (long long)t * a.heads);
    const long long slot = a.slots[t * a.slot_stride];
    if (slot < 0 || slot >= a.total_slots) continue;  // not written
    long long page;
    int offset;
    split_slot(slot, a.page_size, &page, &offset);
    const Src* x = static_cast<const Src*>(s.rows) + t * s.r0 + h * s.r1;
    C* c = static_cast<C*>(s.cache) + page * s.page + h * s.head + offset * s.row;
    if constexpr (CacheElem<C>::kScaled) {
      float top = 0.f;
      for (int d = lane; d < a.d; d += 64) top = nan_max(top, __builtin_fabsf(Elem<Src>::load(x + d)));
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) top = nan_max(top, __shfl_xor(top, o, 64));
      const float scale = top * CacheElem<C>::kInverse;
      for (int d = lane; d < a.d; d += 64) CacheElem<C>::store(c + d, scaled_code<C>(Elem<Src>::load(x + d), scale));
      if (lane == 0) s.scale[page * s.s_page + h * s.s_head + offset * s.s_row] = scale;
    } else {
      for (int d = lane; d < a.d; d += 64) c[d] = x[d];
    }
  }
}

struct KvLoadArgs {
  KvSide side[2];
  const int* table;  // [B, per]
  const int* lens;
  long long table_stride0, table_stride1, len_stride;
  int batch, heads, d, page_size, per, reach;  // reach: rows of the outputs per sequence
  long long pages;
  PageDiv div;
};

template <typename C, typename Dst>
__global__ __launch_bounds__(256) void kv_load_any_kernel(KvLoadArgs a) {
  const int lane = threadIdx.x & 63;
  const long long rows = (long long)a.batch * a.heads * a.reach;
  for (long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); item < 2 * rows; item += 4ll * gridDim.x) {
    const KvSide& s = a.side[item >= rows];
    const long long r = item >= rows ? item - rows : item;
    const int bh = (int)(r / a.reach), i = (int)(r - (long long)bh * a.reach);
    const int b = bh / a.heads, h = bh - b * a.heads;
    if (i >= a.lens[b * a.len_stride]) continue;
    const int p = div_page(i, a.div);
    if (p >= a.per) continue;
    const long long page = a.table[b * a.table_stride0 + p * a.table_stride1];
    if (page < 0 || page >= a.pages) continue;  // no such page: left as it is
    const int offset = i - p * a.page_size;
    const C* c = static_cast<const C*>(s.cache) + page * s.page + h * s.head + offset * s.row;
    Dst* y = static_cast<Dst*>(s.rows) + b * s.r0 + h * s.r1 + i * s.r2;
    if constexpr (CacheElem<C>::kScaled) {
      const float scale = s.scale[page * s.s_page + h * s.s_head + offset * s.s_row];
      for (int d = lane; d < a.d; d += 64) Elem<Dst>::store(y + d, CacheElem<C>::load(c + d) * scale);
    } else {
      for (int d = lane; d < a.d; d += 64) y[d] = c[d];
    }
  }
}

// Eight elements of a row, as a lane of the kernels below holds them.
template <typename T>
struct Eight {  // bf16, f16
  using Tag = typename std::conditional<std::is_same<T, __bf16>::value, Bf16Tag, F16Tag>::type;
  static __device__ __forceinline__ void load(const T* p, float (&x)[8]) {
    const u32x4 w = ld16(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = w[i];
      x[2 * i] = Half16<Tag>::to_float(u & 0xffffu);
      x[2 * i + 1] = Half16<Tag>::to_float(u >> 16);
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&x)[8]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = Half16<Tag>::pack2(x[2 * i], x[2 * i + 1]);
    st16(p, w);
  }
};
template <>
struct Eight<float> {
  static __device__ __forceinline__ void load(const float* p, float (&x)[8]) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  }
  static __device__ __forceinline__ void store(float* p, const float (&x)[8]) {
    *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
  }
};
template <>
struct Eight<E4m3> {
  static __device__ __forceinline__ void load(const E4m3* p, float (&x)[8]) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int u = (int)w[i];
      x[4 * i] = __builtin_amdgcn_cvt_f32_fp8(u, 0);
      x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(u, 1);
      x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(u, 2);
      x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(u, 3);
    }
  }
  static __device__ __forceinline__ void store(E4m3* p, const float (&x)[8]) {
    u32x2 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
      w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], lo, true);
    }
    st8(p, w);
  }
};
template <>
struct Eight<int8_t> {
  static __device__ __forceinline__ void load(const int8_t* p, float (&x)[8]) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)((int)(w[i >> 2] << (24 - 8 * (i & 3))) >> 24);
  }
  static __device__ __forceinline__ void store(int8_t* p, const float (&x)[8]) {
    u32x2 w = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= ((uint32_t)(int)__builtin_rintf(x[i]) & 0xffu) << (8 * (i & 3));
    st8(p, w);
  }
};

// scaled_code of eight elements: x / scale by the scale's inverse, which is rounded, as the quotient is, to nearest: a product within
// 1.5 steps, and two corrections by the exact remainder, of which the second lands on the rounded quotient
// (5 instructions for a division's 11). Quotients under 2^-12, whose remainders may underflow, are codes of 0 either way.
template <typename C>
__device__ __forceinline__ void scaled_codes(float (&x)[8], float scale) {
  if (scale >= 0x1p-60f && scale <= 0x1p60f) {
    const float inverse = 1.f / scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float q = x[i] * inverse;
      q = __builtin_fmaf(__builtin_fmaf(-q, scale, x[i]), inverse, q);
      q = __builtin_fmaf(__builtin_fmaf(-q, scale, x[i]), inverse, q);
      // (the corrections make a zero positive; its sign is the quotient's)
      x[i] = __builtin_copysignf(fminf(fmaxf(q, -CacheElem<C>::kLargest), CacheElem<C>::kLargest), x[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = scaled_code<C>(x[i], scale);
  }
}

// kLanes lanes per row (D <= 8 kLanes), 256 / kLanes rows per workgroup; blockIdx.y: K, V.
template <typename Src, typename C, int kLanes>
__global__ __launch_bounds__(256) void kv_store_kernel(KvStoreArgs a) {
  const KvSide& s = a.side[blockIdx.y];
  const int part = threadIdx.x % kLanes;
  const int r = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (r >= a.tokens * a.heads) return;
  const int t = div_page(r, a.by_heads), h = r - t * a.heads;
  const long long slot = a.slots[t * a.slot_stride];
  const bool in = 8 * part < a.d;
  float x[8];
  const Src* src = static_cast<const Src*>(s.rows) + t * s.r0 + h * s.r1 + (in ? 8 * part : 0);
  Eight<Src>::load(src, x);
  if (slot < 0 || slot >= a.total_slots) return;  // not written
  long long page;
  int offset;
  split_slot(slot, a.page_size, &page, &offset);
  C* c = static_cast<C*>(s.cache) + page * s.page + h * s.head + offset * s.row + 8 * part;
  if constexpr (CacheElem<C>::kScaled) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = nan_max(top, __builtin_fabsf(x[i]));  // (lanes past the row repeat its first elements)
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) top = nan_max(top, __shfl_xor(top, o, 64));
    const float scale = top * CacheElem<C>::kInverse;
    scaled_codes<C>(x, scale);
    if (part == 0) s.scale[page * s.s_page + h * s.s_head + offset * s.s_row] = scale;
  }
  if (in) Eight<C>::store(c, x);
}

// Four rows per lane group, their reads in flight together; blockIdx.x: blocks of rows of a sequence and head.
template <typename C, typename Dst, int kLanes>
__global__ __launch_bounds__(256) void kv_load_kernel(KvLoadArgs a) {
  constexpr int kRows = 256 / kLanes, kTurns = 4;
  const KvSide& s = a.side[blockIdx.z];
  const int part = threadIdx.x % kLanes;
  const int b = blockIdx.y / a.heads, h = blockIdx.y - b * a.heads;
  const int first = blockIdx.x * (kRows * kTurns) + threadIdx.x / kLanes;
  const int len = min(a.lens[b * a.len_stride], a.reach);
  if (blockIdx.x * (kRows * kTurns) >= len) return;
  const bool in = 8 * part < a.d;
  const C* src[kTurns];
  float scale[kTurns];
  bool there[kTurns];
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int i = first + u * kRows, p = div_page(i, a.div);
    there[u] = in && i < len && p < a.per;
    const long long page = there[u] ? a.table[b * a.table_stride0 + p * a.table_stride1] : -1;
    there[u] = page >= 0 && page < a.pages;
    const int offset = i - p * a.page_size;
    src[u] = static_cast<const C*>(s.cache) + (there[u] ? page * s.page + h * s.head + offset * s.row + 8 * part : 0);
    if constexpr (CacheElem<C>::kScaled)
      scale[u] = there[u] ? s.scale[page * s.s_page + h * s.s_head + offset * s.s_row] : 0.f;
  }
  float x[kTurns][8];
#pragma unroll
  for (int u = 0; u < kTurns; ++u) Eight<C>::load(src[u], x[u]);  // (row 0 of page 0 where there is none)
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    if (!there[u]) continue;
    if constexpr (CacheElem<C>::kScaled)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[u][e] *= scale[u];
    Eight<Dst>::store(static_cast<Dst*>(s.rows) + b * s.r0 + h * s.r1 + (long long)(first + u * kRows) * s.r2 + 8 * part, x[u]);
  }
}

}  // namespace kg_gfx950
