// A paged cache of attention keys and values: rows of D elements, one per token and key head, in
// pages of `page_size` tokens ([pages, heads, page_size, D], any strides but the last), held in the
// model's own type or in 8 bits with a 32-bit scale per row ([pages, heads, page_size]).
//
// Written: slot = page page_size + offset; s = max|x| fl32(1 / Q), Q = 448 (e4m3) or 127 (int8);
// code = x / s rounded to the nearest value of the type, ties to even (0 where s is 0). An
// infinity or NaN in a row makes its scale one, and the whole row reads back as NaN. Read back: code s,
// rounded once to the output's type.
//
// kv_store_any_kernel, kv_load_any_kernel: any D and strides, one wave per row.
#pragma once

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
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const long long rows = (long long)a.tokens * a.heads;
  if (item >= 2 * rows) return;
  const KvSide& s = a.side[item >= rows];
  const long long r = item >= rows ? item - rows : item;
  const int t = (int)(r / a.heads), h = (int)(r - (long long)t * a.heads);
  const long long slot = a.slots[t * a.slot_stride];
  if (slot < 0 || slot >= a.total_slots) return;  // not written
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
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const long long rows = (long long)a.batch * a.heads * a.reach;
  if (item >= 2 * rows) return;
  const KvSide& s = a.side[item >= rows];
  const long long r = item >= rows ? item - rows : item;
  const int bh = (int)(r / a.reach), i = (int)(r - (long long)bh * a.reach);
  const int b = bh / a.heads, h = bh - b * a.heads;
  if (i >= a.lens[b * a.len_stride]) return;
  const int p = div_page(i, a.div);
  if (p >= a.per) return;
  const long long page = a.table[b * a.table_stride0 + p * a.table_stride1];
  if (page < 0 || page >= a.pages) return;  // no such page: left as it is
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

}  // namespace kg_gfx950
