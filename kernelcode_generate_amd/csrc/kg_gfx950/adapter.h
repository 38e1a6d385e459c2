// Low-rank adapters beside a shared projection: row m of x with adapter l = index[m] gives
//   out[m] = x[m] W + bias + scale[l] (x[m] A[l]) B[l],    A [L, K, R], B [L, R, N];
// an index outside 0..L-1 is a row without one.
//
// 16-bit calls of whole 16-byte rows: adapter_low_kernel writes t = scale x A, rounded to the operands' type as
// a 16-bit layer's output is, to a workspace [M, R]; then the projection's kernels (gemm_skinny.h, gemm_mid.h, gemm_quad.h)
// take the adapters as further k behind their own: the distinct adapters of a tile's rows, one after the other, R
// values each, t's rows in the slots of their adapter and zeros in the others. A value of B that is not finite, times
// the zeros of rows that do not use it, would be NaN in them: the products run on zeros in place of such values, and
// where there were any each output adds those of its own row's adapter (adapter_nonfinite).
//
// adapter_add_kernel: any types and strides, one workgroup per row: t = scale x A in 32 bits, then
// out += t B, on an output that holds the projection already (matmul's kernels). A 16-bit output is
// so rounded twice, by half a step each time.
#pragma once

#include "common.h"
#include "kv_cache.h"  // PageDiv
#include "lds_dma.h"   // Int

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

// The sum of t[m, r] B[l, r, n] over the B that are not finite, l row m's adapter.
template <typename H>
__device__ __forceinline__ float adapter_nonfinite(const AdapterPart& p, int m, int n) {
  const int l = p.index[m * p.index_stride];
  if (l < 0 || l >= p.count) return 0.f;
  const uint16_t *t = p.t + (long long)m * p.rank, *b = p.b + l * p.b_l + n;
  float sum = 0.f;
#pragma unroll 1
  for (int r = 0; r < p.rank; ++r) {
    const float x = H::to_float(b[r * p.b_r]);
    if (!__builtin_isfinite(x)) sum = __builtin_fmaf(H::to_float(t[r]), x, sum);
  }
  return sum;
}

// The values of B that are not finite, added to outputs that a wave has written: kRows rows from m0, kLanes lanes of 8
// columns from n0 per row, a lane those that it wrote itself. (What is added is not finite, so the output's rounding
// does not matter. In the epilogues' own loops it cost the products their registers.)
template <typename H, int kRows, int kLanes>
__device__ __forceinline__ void adapter_add_nonfinite(const AdapterPart& p, uint16_t* C, long long ldc, int m0, int n0, int M, int N,
                                                      int lane) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const int n = n0 + 8 * (lane % kLanes);
#pragma unroll 1
  for (int r = lane / kLanes; r < kRows; r += 64 / kLanes) {
    const int m = m0 + r;
    if (m >= M || n >= N) continue;
#pragma unroll 1
    for (int u = 0; u < 8; ++u) {
      const float x = adapter_nonfinite<H>(p, m, n + u);
      uint16_t* out = C + (long long)m * ldc + n + u;
      if (x != 0.f) *out = (uint16_t)H::from_float(H::to_float(*out) + x);
    }
  }
}

// The adapters of a tile of kRows rows from m0: row_lds[i] row i's (-1: none), slot_lds[s] the s-th distinct one in the
// order of their first rows. Every wave of the workgroup writes the same. Returns the number of distinct ones.
template <int kRows>
__device__ __forceinline__ int adapter_slots(const AdapterPart& p, int m0, int M, int lane, int* row_lds, int* slot_lds) {
  constexpr int kParts = kRows / 64;
  int own[kParts];
  unsigned long long left[kParts], any = 0;
#pragma unroll
  for (int u = 0; u < kParts; ++u) {
    const int m = m0 + 64 * u + lane;
    own[u] = m < M ? p.index[m * p.index_stride] : -1;
    if (own[u] < 0 || own[u] >= p.count) own[u] = -1;
    row_lds[64 * u + lane] = own[u];
    left[u] = __builtin_amdgcn_ballot_w64(own[u] >= 0);
    any |= left[u];
  }
  int slots = 0;
  while (any != 0) {
    int l = -1;
#pragma unroll
    for (int u = 0; u < kParts; ++u)
      if (l < 0 && left[u] != 0) l = __builtin_amdgcn_readlane(own[u], __builtin_ctzll(left[u]));
    any = 0;
#pragma unroll
    for (int u = 0; u < kParts; ++u) {
      left[u] &= ~__builtin_amdgcn_ballot_w64(own[u] == l);
      any |= left[u];
    }
    slot_lds[slots++] = l;
  }
  return slots;
}

// Where the 16 bytes of a tile's row (t) or of a k-row's columns (B) of an eight-k piece lie; null: zeros.
__device__ __forceinline__ const uint16_t* adapter_t(const AdapterPart& p, int piece, int pieces, int slots, const int* slot_lds, int l,
                                                     int m) {
  const int slot = div_page(piece, p.by_pieces);
  return slot < slots && slot_lds[slot] == l ? p.t + (long long)m * p.rank + 8 * (piece - slot * pieces) : nullptr;
}
__device__ __forceinline__ const uint16_t* adapter_b(const AdapterPart& p, int piece, int pieces, int slots, const int* slot_lds, int k,
                                                     int n) {
  const int slot = div_page(piece, p.by_pieces);
  return slot < slots ? p.b + slot_lds[slot] * p.b_l + (8 * (piece - slot * pieces) + k) * p.b_r + n : nullptr;
}
// 16 bytes of B from there to LDS, zeros in place of what is not finite; `found` gets bits for that.
template <typename H>
__device__ __forceinline__ void adapter_put(u32x4 x, uint32_t to, uint32_t& found) {
#pragma unroll
  for (int q = 0; q < 4; ++q) x[q] = finite_pair<H>(x[q], found);
  *(__attribute__((address_space(3))) u32x4*)(uintptr_t)to = x;
}

// t = scale x A of 16 rows and up to 64 columns (blockIdx.z) per workgroup: its sixteen waves share K in steps of
// 32, lanes hold two columns of A by eight k as in gemm_skinny.h, one sum over the waves through LDS. A workgroup takes every
// gridDim.y-th of its rows' distinct adapters and stores the rows that use it: few rows have many adapters
// (gridDim.y workgroups read them at once), many rows few. 16 x 4096, 16 adapters of rank 16: LOW_STEP us; 4096 x 4096 in
// runs: LOW_PROMPTS us, the reading of x.
constexpr int kAdapterLowThreads = 1024, kAdapterLowCols = 64;
template <typename Tag>
__global__ __launch_bounds__(kAdapterLowThreads) void adapter_low_kernel(AdapterArgs a, uint16_t* __restrict__ t, uint32_t* __restrict__ zeros) {
  using H = Half16<Tag>;
  constexpr int kWaves = kAdapterLowThreads / 64, kCols = kAdapterLowCols;
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
  const int full = a.k / 32;
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
    // columns past the rank repeat the first ones and are dropped
    const uint16_t* a_row = A + (long long)(8 * lg) * a.a_k;
    const int col0 = 2 * l16 < cols ? 2 * l16 : 0, col1 = 32 + 2 * l16 < cols ? 32 + 2 * l16 : 0;
    auto product = [&](u32x4 xf, const uint32_t (&w)[8], int j) __attribute__((always_inline)) {
      u32x4 even, odd;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        even[q] = lo_halves(w[2 * q], w[2 * q + 1]);
        odd[q] = hi_halves(w[2 * q], w[2 * q + 1]);
      }
      acc[j][0] = H::mfma16(xf, even, acc[j][0]);
      acc[j][1] = H::mfma16(xf, odd, acc[j][1]);
    };
    auto loop = [&](auto wide_tag) __attribute__((always_inline)) {
      constexpr bool kWide = decltype(wide_tag)::value != 0;  // more than 32 columns
#pragma unroll 2
      for (int s0 = 2 * wave; s0 < full; s0 += 2 * kWaves) {  // 64 k: whole lines of x
        u32x4 xf[2];
        uint32_t w0[2][8], w1[2][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int s = min(s0 + u, full - 1);
          xf[u] = ld16(x + 32 * s);
          const uint16_t* row = a_row + (long long)(32 * s) * a.a_k;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            w0[u][e] = *reinterpret_cast<const uint32_t*>(row + e * a.a_k + col0);
            if constexpr (kWide) w1[u][e] = *reinterpret_cast<const uint32_t*>(row + e * a.a_k + col1);
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (s0 + u >= full) break;
          product(xf[u], w0[u], 0);
          if constexpr (kWide) product(xf[u], w1[u], 1);
        }
      }
    };
    if (cols > 32) loop(Int<1>{});
    else loop(Int<0>{});
    if (full * 32 < a.k && wave == kWaves - 1) {  // the last K % 32 (a multiple of 8): zeros in both operands
      const bool in = 32 * full + 8 * lg < a.k;
      const u32x4 xf = in ? ld16(x + 32 * full) : u32x4{0, 0, 0, 0};
      uint32_t w0[8], w1[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t* row = a_row + (long long)(32 * full + e) * a.a_k;
        w0[e] = in ? *reinterpret_cast<const uint32_t*>(row + col0) : 0u;
        w1[e] = in ? *reinterpret_cast<const uint32_t*>(row + col1) : 0u;
      }
      product(xf, w0, 0);
      product(xf, w1, 1);
    }
    __syncthreads();  // the sums of the adapter before are read
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f32x2*>(&red[wave][4 * lg + e][32 * j + 2 * l16]) = f32x2{acc[j][0][e], acc[j][1][e]};
    __syncthreads();
    const float scale = a.scale ? a.scale[l * a.scale_stride] : 1.f;
    if (tid < 16 * kCols / 2) {
      const int m = tid / (kCols / 2), c = 2 * (tid % (kCols / 2));
      if (c < cols && (users >> m & 1ull)) {
        f32x2 sum = {0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += *reinterpret_cast<const f32x2*>(&red[w][m][c]);
        *reinterpret_cast<uint32_t*>(t + (long long)(m0 + m) * a.rank + c0 + c) = H::pack2(sum[0] * scale, sum[1] * scale);
      }
    }
  }
}

}  // namespace kg_gfx950
