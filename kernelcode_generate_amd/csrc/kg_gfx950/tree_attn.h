// Attention of drafted tokens over a paged cache (kv_cache.h): request b has `lens[b]` cached tokens, its
// context, and the drafted tokens starts[b] .. starts[b + 1] - 1 of the batch, whose keys and values
// lie in the cache behind the context. Token j of a request sees its whole context and the drafted
// tokens i whose bit i is set in the token's mask (a tree: itself and its ancestors), or, without masks, i <= j:
//   out[t, h] = sum_i softmax_i(scale q[t, h] . k[i, h / group]) v[i, h / group],
// zeros where nothing is seen. Keys past the page table's reach or on a page that does not exist are
// not seen. Scores, softmax statistics and sums in 32 bits.
//
// tree_attn_any_kernel: any types, D <= 512, page size and strides: one workgroup per token and head.
#pragma once

#include "common.h"
#include "kv_cache.h"

namespace kg_gfx950 {

struct TreeArgs {
  const void *q, *k, *v;
  void* out;
  const float *k_scale, *v_scale;
  const int *table, *lens, *starts;
  const long long* mask;
  long long q_token, q_head, o_token, o_head;
  long long k_page, k_head, k_row, v_page, v_head, v_row;
  long long ks_page, ks_head, ks_row, vs_page, vs_head, vs_row;
  long long table_0, table_1, len_stride, start_stride, mask_0, mask_1;
  int tokens, batch, heads_q, heads, group, d, page_size, per;
  int words;  // of a token's mask; -1: no masks
  long long pages;
  PageDiv div;
  float scale_log2;  // scale log2(e)
};

// A request's first token, number of tokens, context and keys in all, within what the arrays hold.
struct TreeRequest {
  int first, count, context, keys;
};
__device__ __forceinline__ TreeRequest tree_request(const TreeArgs& a, int b) {
  TreeRequest r;
  r.first = max(a.starts[b * a.start_stride], 0);
  r.count = max(min(a.starts[(b + 1) * a.start_stride], a.tokens) - r.first, 0);
  r.context = max(a.lens[b * a.len_stride], 0);
  const long long reach = (long long)a.per * a.page_size, keys = (long long)r.context + r.count;
  r.keys = (int)(keys < reach ? keys : reach);
  return r;
}

// Elements before row `offset` of a page that is there, for strides below 2^32: two multiply-adds (eight multiplications of the
// general product are four cycles each).
__device__ __forceinline__ unsigned long long tree_row(int page, int offset, long long page_stride, long long row_stride) {
  return (unsigned long long)(uint32_t)page * (uint32_t)page_stride + (unsigned long long)(uint32_t)offset * (uint32_t)row_stride;
}

// Whether token j of a request (batch row t) sees the drafted token i >= 0.
__device__ __forceinline__ bool tree_sees(const TreeArgs& a, int t, int j, int i) {
  if (a.words < 0) return i <= j;
  const int w = i >> 6;
  return w < a.words && ((unsigned long long)a.mask[t * a.mask_0 + w * a.mask_1] >> (i & 63) & 1ull) != 0;
}

template <typename T, typename C>
__global__ __launch_bounds__(256) void tree_attn_any_kernel(TreeArgs a) {
  constexpr int kThreads = 256, kMaxD = 512;
  __shared__ float qs[kMaxD];
  __shared__ float ps[kThreads];  // weights of a block of keys, times the values' scales
  __shared__ long long rows[kThreads];
  __shared__ float red[kThreads / 64];
  const int tid = threadIdx.x;
  for (unsigned row = blockIdx.x; row < (unsigned)a.tokens * (unsigned)a.heads_q; row += gridDim.x) {
    const int t = (int)(row / (unsigned)a.heads_q), hq = (int)(row - (unsigned)t * a.heads_q);
    const int h = hq / a.group;

    // the request: the last one that starts at or before t
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.starts[mid * a.start_stride] <= t) lo = mid;
      else hi = mid;
    }
    const TreeRequest r = tree_request(a, lo);
    const int j = t - r.first;
    if (j < 0 || j >= r.count) continue;  // a row of no request

    const T* q = static_cast<const T*>(a.q) + t * a.q_token + hq * a.q_head;
    for (int d = tid; d < a.d; d += kThreads) qs[d] = Elem<T>::load(q + d);  // (read before the last barrier of the row before)
    __syncthreads();

    const C* kc = static_cast<const C*>(a.k) + h * a.k_head;
    const C* vc = static_cast<const C*>(a.v) + h * a.v_head;
    float acc[kMaxD / kThreads] = {0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;
    for (int n0 = 0; n0 < r.keys; n0 += kThreads) {
      const int n = n0 + tid;
      float score = -INFINITY;
      bool seen = n < r.keys && (n < r.context || tree_sees(a, t, j, n - r.context));
      long long v_row = 0;
      float v_scale = 1.f;
      if (seen) {
        const int p = div_page(n, a.div), offset = n - p * a.page_size;
        const long long page = a.table[lo * a.table_0 + p * a.table_1];
        seen = page >= 0 && page < a.pages;
        if (seen) {
          const C* k = kc + page * a.k_page + offset * a.k_row;
          float dot = 0.f;
          for (int d = 0; d < a.d; ++d) dot = __builtin_fmaf(qs[d], CacheElem<C>::load(k + d), dot);
          if constexpr (CacheElem<C>::kScaled) {
            dot *= a.k_scale[page * a.ks_page + h * a.ks_head + offset * a.ks_row];
            v_scale = a.v_scale[page * a.vs_page + h * a.vs_head + offset * a.vs_row];
          }
          score = dot * a.scale_log2;
          v_row = page * a.v_page + offset * a.v_row;
        }
      }
      float top = score;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) top = nan_max(top, __shfl_xor(top, o, 64));
      if ((tid & 63) == 0) red[tid >> 6] = top;
      __syncthreads();
      // a finite lowest maximum: scores of -inf, which infinite inputs give, weigh nothing beside it
      const float m_new = nan_max(nan_max(nan_max(red[0], red[1]), nan_max(red[2], red[3])), nan_max(m_run, -3.0e38f));
      const float p = seen ? __builtin_amdgcn_exp2f(score - m_new) : 0.f;
      __syncthreads();
      float sum = wave_sum(p);
      if ((tid & 63) == 0) red[tid >> 6] = sum;
      ps[tid] = p * v_scale;
      rows[tid] = seen ? v_row : -1;
      __syncthreads();
      sum = red[0] + red[1] + red[2] + red[3];
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      l_run = l_run * alpha + sum;
      m_run = m_new;
      const int keys = min(kThreads, r.keys - n0);
#pragma unroll
      for (int e = 0; e < kMaxD / kThreads; ++e) {
        const int d = tid + e * kThreads;
        if (d >= a.d) continue;
        float o = acc[e] * alpha;
        for (int x = 0; x < keys; ++x)
          if (rows[x] >= 0) o = __builtin_fmaf(ps[x], CacheElem<C>::load(vc + rows[x] + d), o);
        acc[e] = o;
      }
      __syncthreads();
    }
    T* out = static_cast<T*>(a.out) + t * a.o_token + hq * a.o_head;
    for (int e = 0; e < kMaxD / kThreads; ++e) {
      const int d = tid + e * kThreads;
      if (d < a.d) Elem<T>::store(out + d, l_run != 0.f ? acc[e] / l_run : 0.f);
    }
  }
}

}  // namespace kg_gfx950
