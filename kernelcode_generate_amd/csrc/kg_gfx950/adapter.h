// Low-rank adapters beside a shared projection: row m of x with adapter l = index[m] gives
//   out[m] = x[m] W + bias + scale[l] (x[m] A[l]) B[l],    A [L, K, R], B [L, R, N];
// an index outside 0..L-1 is a row without one.
//
// adapter_add_kernel: any types and strides, one workgroup per row: t = scale x A in 32 bits, then
// out += t B, on an output that holds the projection already (matmul's kernels). A 16-bit output is
// so rounded twice, by half a step each time.
#pragma once

#include "common.h"

namespace kg_gfx950 {

struct AdapterArgs {
  const void *x, *w, *bias, *a, *b;
  void* out;
  const int* index;
  const float* scale;  // null: 1
  long long ldx, ldw, ldo, a_l, a_k, b_l, b_r, index_stride, scale_stride;
  int m, n, k, rank, count;
};
constexpr int kAdapterMaxRank = 512;

template <typename T>
__global__ __launch_bounds__(256) void adapter_add_kernel(AdapterArgs p) {
  __shared__ float ts[kAdapterMaxRank];
  __shared__ float xs[256];
  const int tid = threadIdx.x, m = blockIdx.x;
  const int l = p.index[m * p.index_stride];
  if (l < 0 || l >= p.count) return;
  const T* x = static_cast<const T*>(p.x) + m * p.ldx;
  const T* A = static_cast<const T*>(p.a) + l * p.a_l;
  const T* B = static_cast<const T*>(p.b) + l * p.b_l;
  T* out = static_cast<T*>(p.out) + m * p.ldo;
  // ranks of up to 256 share a row's k among 256 / rank groups of threads
  float t[kAdapterMaxRank / 256] = {0.f, 0.f};
  const int groups = p.rank >= 256 ? 1 : 256 / p.rank;
  const int g = tid / (p.rank >= 256 ? 256 : p.rank), r0 = tid - g * (p.rank >= 256 ? 256 : p.rank);
  for (int k0 = 0; k0 < p.k; k0 += 256) {
    __syncthreads();
    xs[tid] = k0 + tid < p.k ? Elem<T>::load(x + k0 + tid) : 0.f;
    __syncthreads();
    const int kn = min(256, p.k - k0);
    if (g < groups)
      for (int k = g; k < kn; k += groups)
#pragma unroll
        for (int e = 0; e < kAdapterMaxRank / 256; ++e)
          if (r0 + 256 * e < p.rank)
            t[e] = __builtin_fmaf(xs[k], Elem<T>::load(A + (k0 + k) * p.a_k + r0 + 256 * e), t[e]);
  }
  for (int r = tid; r < p.rank; r += 256) ts[r] = 0.f;
  // the groups' sums, one group after another: the same order at every call
  for (int s = 0; s < groups; ++s) {
    __syncthreads();
    if (g == s)
#pragma unroll
      for (int e = 0; e < kAdapterMaxRank / 256; ++e)
        if (r0 + 256 * e < p.rank) ts[r0 + 256 * e] += t[e];
  }
  __syncthreads();
  const float scale = p.scale ? p.scale[l * p.scale_stride] : 1.f;
  for (int n = tid; n < p.n; n += 256) {
    float o = 0.f;
    for (int r = 0; r < p.rank; ++r) o = __builtin_fmaf(ts[r], Elem<T>::load(B + r * p.b_r + n), o);
    Elem<T>::store(out + n, Elem<T>::load(out + n) + scale * o);
  }
}

}  // namespace kg_gfx950
