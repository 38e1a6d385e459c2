// Low-rank adapters beside a shared projection: row m of x with adapter l = index[m] gives
//   out[m] = x[m] W + bias + scale[l] (x[m] A[l]) B[l],    A [L, K, R], B [L, R, N];
// an index outside 0..L-1 is a row without one.
//
// 16-bit calls of whole 16-byte rows: adapter_low_kernel writes t = scale x A, rounded to the operands' type as
// a 16-bit layer's output is, to a workspace [M, R]; then the projection's kernels (gemm_skinny.h, gemm_mid.h) take the
// adapters as further k behind their own: the distinct adapters of a tile's rows, one after the other, R values
// each, t's rows in the slots of their adapter and zeros in the others. These products have accumulators of their own: a
// value of B that is not finite, times the zeros of rows that do not use it, would be NaN in them, so where such a sum
// is not finite it is taken again over the row's own adapter alone.
//
// adapter_add_kernel: any types and strides, one workgroup per row: t = scale x A in 32 bits, then
// out += t B, on an output that holds the projection already (matmul's kernels). A 16-bit output is
// so rounded twice, by half a step each time.
#pragma once

#include "common.h"
#include "kv_cache.h"  // PageDiv

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

// The adapters' part of a projection, for its kernels: t [M, rank] 16-bit behind 16 bytes of zeros.
struct AdapterPart {
  const uint16_t *t, *zeros, *b;
  const int* index;
  long long b_l, b_r, index_stride;
  int rank, count;  // rank % 8 == 0
  PageDiv by_pieces;  // division by rank / 8
};
constexpr size_t kAdapterHeader = 256;  // bytes of the workspace before t

// sum_r t[m, r] B[l, r, n], for sums that another row's values have spoilt
template <typename H>
__device__ __forceinline__ float adapter_alone(const AdapterPart& p, int m, int n) {
  const int l = p.index[m * p.index_stride];
  if (l < 0 || l >= p.count) return 0.f;
  const uint16_t *t = p.t + (long long)m * p.rank, *b = p.b + l * p.b_l + n;
  float sum = 0.f;
#pragma unroll 1
  for (int r = 0; r < p.rank; ++r) sum = __builtin_fmaf(H::to_float(t[r]), H::to_float(b[r * p.b_r]), sum);
  return sum;
}

// t = scale x A of 16 rows and up to 64 columns (blockIdx.z) per workgroup: its eight waves share K in steps of
// 32, lanes hold two columns of A by eight k as in gemm_skinny.h, one sum over the waves through LDS. A workgroup takes every
// gridDim.y-th of its rows' distinct adapters and stores the rows that use it: few rows have many adapters
// (gridDim.y workgroups read them at once), many rows few. 16 x 4096, 16 adapters of rank 16: LOW_STEP us; 4096 x 4096 in
// runs: LOW_PROMPTS us, the reading of x.
template <typename Tag>
__global__ __launch_bounds__(512) void adapter_low_kernel(AdapterArgs a, uint16_t* __restrict__ t, uint32_t* __restrict__ zeros) {
  using H = Half16<Tag>;
  constexpr int kWaves = 8, kCols = 64;
  __shared__ float red[kWaves][16][kCols];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int m0 = blockIdx.x * 16, rows = min(a.m - m0, 16), c0 = blockIdx.z * kCols;
  const int cols = min(a.rank - c0, kCols);
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && tid < 4) zeros[tid] = 0;

  int own = -1;  // adapter of row `lane`
  if (lane < rows) own = a.index[(m0 + lane) * a.index_stride];
  if (own >= a.count) own = -1;
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + (m0 + min(l16, rows - 1)) * a.ldx + 8 * lg;
  const int steps = (a.k + 31) / 32;
  unsigned long long left = __builtin_amdgcn_ballot_w64(own >= 0);
  for (int slot = 0; left != 0; ++slot) {
    const int l = __builtin_amdgcn_readlane(own, __builtin_ctzll(left));
    const unsigned long long users = __builtin_amdgcn_ballot_w64(own == l);
    left &= ~users;
    if (slot % gridDim.y != blockIdx.y) continue;
    const uint16_t* A = static_cast<const uint16_t*>(a.a) + l * a.a_l + c0;
    f32x4 acc[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[j][0] = acc[j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = wave; s < steps; s += kWaves) {
      const int k = 32 * s + 8 * lg;  // (K is a multiple of 8)
      const bool in = k < a.k;
      const u32x4 xf = in ? ld16(x + 32 * s) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (32 * j >= cols) break;
        const bool there = in && 32 * j + 2 * l16 < cols;
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          w[e] = there ? *reinterpret_cast<const uint32_t*>(A + (long long)(k + e) * a.a_k + 32 * j + 2 * l16) : 0u;
        u32x4 even, odd;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          even[q] = lo_halves(w[2 * q], w[2 * q + 1]);
          odd[q] = hi_halves(w[2 * q], w[2 * q + 1]);
        }
        acc[j][0] = H::mfma16(xf, even, acc[j][0]);
        acc[j][1] = H::mfma16(xf, odd, acc[j][1]);
      }
    }
    __syncthreads();  // the sums of the adapter before are read
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        red[wave][4 * lg + e][32 * j + 2 * l16] = acc[j][0][e];
        red[wave][4 * lg + e][32 * j + 2 * l16 + 1] = acc[j][1][e];
      }
    __syncthreads();
    const float scale = a.scale ? a.scale[l * a.scale_stride] : 1.f;
    for (int y = tid; y < 16 * kCols / 2; y += 512) {
      const int m = y / (kCols / 2), c = 2 * (y % (kCols / 2));
      if (c >= cols || !(users >> m & 1ull)) continue;
      float v0 = 0.f, v1 = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) v0 += red[w][m][c], v1 += red[w][m][c + 1];
      *reinterpret_cast<uint32_t*>(t + (long long)(m0 + m) * a.rank + c0 + c) = H::pack2(v0 * scale, v1 * scale);
    }
  }
}

}  // namespace kg_gfx950
