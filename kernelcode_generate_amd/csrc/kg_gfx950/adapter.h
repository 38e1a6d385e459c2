// Low-rank adapters beside a shared projection: row m of x with adapter l = index[m] gives
//   out[m] = x[m] W + bias + scale[l] (x[m] A[l]) B[l],    A [L, K, R], B [L, R, N];
// an index outside 0..L-1 is a row without one.
//
// 16-bit calls of whole 16-byte rows: adapter_low_kernel writes t = scale x A in 32 bits, as sums over ranges of K, to a
// workspace; then the projection's kernels (gemm_skinny.h, gemm_mid.h, gemm_quad.h, gemm.h) take the adapters as further k
// behind their own: the distinct adapters of a tile's rows, one after the other, R values each, t's rows in the slots of
// their adapter and zeros in the others. A value of B that is not finite, times
// the zeros of rows that do not use it, would be NaN in them: the products run on zeros in place of such values, and
// where there were any each output adds those of its own row's adapter (adapter_nonfinite). For the products t is
// rounded to the operands' type, as the output of a 16-bit layer would be; for fp16, whose range a product of x, A and a scale
// leaves at either end, as a row's t times a power of two (adapter_power): the row's sums are scaled by it before the adapter's
// products, and back after them, both exact. Rows whose t is near 1 take no part in that (4096 x 4096 x 4096 with all rows
// scaled 122 us, so 118, without any of it 115).
//
// adapter_add_kernel: any types and strides, one workgroup per row: t = scale x A in 32 bits, then
// out += t B, on an output that holds the projection already (matmul's kernels). A 16-bit output is
// so rounded twice, by half a step each time; a projection past the type's range is computed again, in 32 bits.
#pragma once

#include <type_traits>

#include "common.h"
#include "kv_cache.h"  // PageDiv
#include "lds_dma.h"   // Int

namespace kg_gfx950 {

struct AdapterArgs {
  const void *x, *w, *bias, *a, *b;
  void* out;
  const int* index;
  const float* scale;  // null: 1
  long long ldx, ldw, ldo, a_l, a_k, b_l, b_r, index_stride, scale_stride, w_n, bias_stride;
  int m, n, k, rank, count;
  bool wide_bias;  // 32 bits, not the operands' type
};
constexpr int kAdapterMaxRank = 512;

template <typename T>
__device__ __forceinline__ float adapter_projection(const AdapterArgs& p, const T* x, int n) {
  const T* w = static_cast<const T*>(p.w) + n * p.w_n;
  float sum = 0.f;
#pragma unroll 1
  for (int k = 0; k < p.k; ++k) sum = __builtin_fmaf(Elem<T>::load(x + k), Elem<T>::load(w + k * p.ldw), sum);
  if (p.bias == nullptr) return sum;
  return sum + (p.wide_bias ? static_cast<const float*>(p.bias)[n * p.bias_stride]
                            : Elem<T>::load(static_cast<const T*>(p.bias) + n * p.bias_stride));
}

template <typename T>
__global__ __launch_bounds__(256) void adapter_add_kernel(AdapterArgs p) {
  __shared__ float ts[kAdapterMaxRank];
  __shared__ float xs[256];
  const int tid = threadIdx.x;
  for (long long m = blockIdx.x; m < p.m; m += gridDim.x) {
    const int l = p.index[m * p.index_stride];
    if (l < 0 || l >= p.count) continue;
    __syncthreads();  // the row before is done with ts
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
      float base = Elem<T>::load(out + n);
      if (sizeof(T) == 2 && !__builtin_isfinite(base)) base = adapter_projection(p, x, n);
      Elem<T>::store(out + n, base + scale * o);
    }
  }
}

// The adapters' part of a projection, for its kernels. sums: t as [splits, M, rank] sums over ranges of K; zeros: 16 bytes of zeros.
struct AdapterPart {
  const float* sums;
  const uint16_t *zeros, *b;
  const int* index;
  long long split_pitch, b_l, b_r, index_stride;  // split_pitch: M rank
  int splits, rank, count;                        // rank % 8 == 0
  PageDiv by_pieces;                              // division by rank / 8
  const float* tops;                              // fp16: [M, top_pitch], the largest of a row's sums in each part of them, or 1 (in range)
  int top_count, top_pitch;                       // adapter_top_pitch(top_count)
};
constexpr int kAdapterLowCols = 64;  // columns of t per workgroup, a part
inline __host__ __device__ int adapter_top_count(int rank, int splits) { return (rank + kAdapterLowCols - 1) / kAdapterLowCols * splits; }
inline __host__ __device__ int adapter_top_pitch(int count) { return (count + 3) / 4 * 4; }
template <typename H>
constexpr bool kAdapterRanged = std::is_same<H, Half16<F16Tag>>::value;
// The power of two for row m's t, from the largest of its sums over ranges of K: 1 where that lies within 2^-3..2^12 (t, of up to 8
// of them, is then below 2^15, and its small values are off by half a subnormal step, 2^-22 of the largest, at most), else what
// brings it to 2^11..2^12. At most 2^60, which the projection's sums bear (of fp16 operands they stay below 2^54); what is smaller then is
// nothing in fp16, times any B. Of infinite sums the least, so that finite ones beside them stay finite.
constexpr float kAdapterSmall = 0x1p-3f, kAdapterLarge = 0x1p12f;
__device__ __forceinline__ float adapter_top(const AdapterPart& p, int m) {
  float top = 0.f;
#pragma unroll 1
  for (int i0 = 0; i0 < p.top_count; i0 += 4) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(p.tops + (long long)m * p.top_pitch + i0);
#pragma unroll
    for (int y = 0; y < 4; ++y) top = i0 + y < p.top_count ? fmaxf(top, v[y]) : top;
  }
  return top;
}
__device__ __forceinline__ float adapter_power(float top) {
  if (top == 0.f || (top >= kAdapterSmall && top < kAdapterLarge)) return 1.f;
  const int exponent = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
  return __builtin_bit_cast(float, (uint32_t)(127 + max(min(11 - exponent, 60), -116)) << 23);
}
__device__ __forceinline__ float inverse_power(float power) {
  return __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, power));
}
// Eight elements of t from `at` on, times their row's power of two, rounded.
constexpr int kAdapterMaxSplits = 8;
template <typename H>
__device__ __forceinline__ u32x4 adapter_t8(const AdapterPart& p, const float* at, float range) {
  f32x4 a = *reinterpret_cast<const f32x4*>(at), b = *reinterpret_cast<const f32x4*>(at + 4);
#pragma unroll
  for (int y = 1; y < kAdapterMaxSplits; ++y) {  // (unrolled: the reads are in flight together)
    if (y >= p.splits) break;
    a += *reinterpret_cast<const f32x4*>(at + y * p.split_pitch);
    b += *reinterpret_cast<const f32x4*>(at + y * p.split_pitch + 4);
  }
  if constexpr (kAdapterRanged<H>) a *= range, b *= range;
  return u32x4{H::pack2(a[0], a[1]), H::pack2(a[2], a[3]), H::pack2(b[0], b[1]), H::pack2(b[2], b[3])};
}
constexpr size_t kAdapterHeader = 256;  // bytes of the workspace before the sums: zeros

// The sum of t[m, r] B[l, r, n] over the B that are not finite, l row m's adapter.
template <typename H>
__device__ __forceinline__ float adapter_nonfinite(const AdapterPart& p, int m, int n) {
  const int l = p.index[m * p.index_stride];
  if (l < 0 || l >= p.count) return 0.f;
  const float* t = p.sums + (long long)m * p.rank;
  const uint16_t* b = p.b + l * p.b_l + n;
  float sum = 0.f;
#pragma unroll 1
  for (int r = 0; r < p.rank; ++r) {
    const float x = H::to_float(b[r * p.b_r]);
    if (__builtin_isfinite(x)) continue;
    float tr = 0.f;
#pragma unroll 1
    for (int y = 0; y < p.splits; ++y) tr += t[y * p.split_pitch + r];
    sum = __builtin_fmaf(tr, x, sum);
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

// The same for the epilogues whose lanes hold 4 columns of a row in each of kM x kN blocks of 16 x 16: outputs
// (pitch ldc) or, before they are summed, fp32 partial sums.
template <typename H, int kM, int kN, typename T>
__device__ __forceinline__ void adapter_add_nonfinite_blocks(const AdapterPart& p, T* C, long long ldc, int m0, int n0, int M, int N,
                                                             int lane) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll 1
  for (int i = 0; i < kM * kN; ++i) {
    const int m = m0 + 16 * (i / kN) + (lane & 15), n = n0 + 16 * (i % kN) + 4 * (lane >> 4);
    if (m >= M || n >= N) continue;
#pragma unroll 1
    for (int u = 0; u < 4; ++u) {
      const float x = adapter_nonfinite<H>(p, m, n + u);
      T* out = C + (long long)m * ldc + n + u;
      if (x == 0.f) continue;
      if constexpr (sizeof(T) == 4) *out += x;
      else *out = (T)H::from_float(H::to_float(*out) + x);
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

// The same and, in fp16, range_lds[i], the power of two of row i (1 without an adapter), and whether there are others than 1.
template <typename H, int kRows>
__device__ __forceinline__ int adapter_slots(const AdapterPart& p, int m0, int M, int lane, int* row_lds, int* slot_lds,
                                             float* range_lds, bool* scaled) {
  if constexpr (kAdapterRanged<H>) {
    float power[kRows / 64];
#pragma unroll
    for (int u = 0; u < kRows / 64; ++u)  // (read ahead of the indexes: a row without an adapter has no value there to keep)
      power[u] = adapter_top(p, min(m0 + 64 * u + lane, M - 1));
    const int slots = adapter_slots<kRows>(p, m0, M, lane, row_lds, slot_lds);
#pragma unroll
    for (int u = 0; u < kRows / 64; ++u) {
      power[u] = row_lds[64 * u + lane] >= 0 ? adapter_power(power[u]) : 1.f;
      range_lds[64 * u + lane] = power[u];
      *scaled = *scaled || __builtin_amdgcn_ballot_w64(power[u] != 1.f) != 0;
    }
    return slots;
  } else {
    return adapter_slots<kRows>(p, m0, M, lane, row_lds, slot_lds);
  }
}

// Where a tile's row of t, or a k-row's columns of B, of an eight-k piece lie; null: zeros.
__device__ __forceinline__ const float* adapter_t(const AdapterPart& p, int piece, int pieces, int slots, const int* slot_lds, int l,
                                                  int m) {
  const int slot = div_page(piece, p.by_pieces);
  return slot < slots && slot_lds[slot] == l ? p.sums + (long long)m * p.rank + 8 * (piece - slot * pieces) : nullptr;
}
__device__ __forceinline__ const uint16_t* adapter_b(const AdapterPart& p, int piece, int pieces, int slots, const int* slot_lds, int k,
                                                     int n) {
  const int slot = div_page(piece, p.by_pieces);
  return slot < slots ? p.b + slot_lds[slot] * p.b_l + (8 * (piece - slot * pieces) + k) * p.b_r + n : nullptr;
}
template <typename H>
__device__ __forceinline__ void adapter_put_t(const AdapterPart& p, const float* from, uint32_t to, float range) {
  u32x4 x = {0, 0, 0, 0};
  if (from) x = adapter_t8<H>(p, from, range);
  *(__attribute__((address_space(3))) u32x4*)(uintptr_t)to = x;
}
// 16 bytes of B from there to LDS, zeros in place of what is not finite; `found` gets bits for that.
template <typename H>
__device__ __forceinline__ void adapter_put(u32x4 x, uint32_t to, uint32_t& found) {
#pragma unroll
  for (int q = 0; q < 4; ++q) x[q] = finite_pair<H>(x[q], found);
  *(__attribute__((address_space(3))) u32x4*)(uintptr_t)to = x;
}

// t = scale x A of 16 rows and up to 64 columns (blockIdx.z) per workgroup, whose four waves share a range of K (blockIdx.x)
// in pieces of 64 and end in one sum through LDS. A step of 32 k is one 16-byte load per lane of x and one of each 16 columns
// of A (rows of k, 32 bytes), which turn through 1 KiB of a wave's own LDS each into MFMA operands (ds_read_b64_tr_b16; rows with
// bit 3 set half a bank row apart); four steps are in flight at once. (Eight, in twice the registers, took 2 us longer; columns loaded
// as pairs straight into operands, eight loads a step, twice as long.) A workgroup takes every gridDim.y-th of its rows' distinct
// adapters and stores the rows that use it: few rows have many adapters (gridDim.y workgroups read them at once), many rows
// few. Few rows also share out K over up to eight workgroups: one CU reads some 16 bytes a clock. 16 x 4096, 16 adapters of
// rank 16: 4-5 us (one workgroup of 16 waves over all of K: 10); 200 x 2048 of rank 64, mixed: 10.6; 4096 x 4096 in runs: 12.6-13.4 us,
// 2.7 TB/s of x.
constexpr int kAdapterLowThreads = 256;
template <typename Tag>
__global__ __launch_bounds__(kAdapterLowThreads) void adapter_low_kernel(AdapterArgs a, uint32_t* __restrict__ zeros,
                                                                          float* __restrict__ sums, int splits,
                                                                          float* __restrict__ tops) {
  using H = Half16<Tag>;
  constexpr int kWaves = kAdapterLowThreads / 64, kCols = kAdapterLowCols;
  static_assert(kAdapterLowThreads == 4 * kCols, "a thread per column and four rows in the sum over the waves");
  __shared__ __attribute__((aligned(16))) float red[kWaves][kCols][16 + 4];
  __shared__ __attribute__((aligned(1024))) char turn[kWaves * 4096];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int split = blockIdx.x % splits, m0 = blockIdx.x / splits * 16, rows = min(a.m - m0, 16), c0 = blockIdx.z * kCols;
  const int cols = min(a.rank - c0, kCols);
  // this range's K, as a product of its own (ranges of whole pieces of 64)
  const int range = ((a.k + 63) / 64 + splits - 1) / splits * 64;
  const int k_begin = split * range, k_end = min(a.k - k_begin, range);
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && tid < 4) zeros[tid] = 0;

  int own = -1;  // adapter of row `lane`
  if (lane < rows) own = a.index[(m0 + lane) * a.index_stride];
  if (own >= a.count) own = -1;
  const uint16_t* x = static_cast<const uint16_t*>(a.x) + (m0 + min(l16, rows - 1)) * a.ldx + k_begin + 8 * lg;
  // this lane's part of 32 rows of 16 columns, and its read addresses (k-rows 8 lg + 0..3, then + 4)
  const int k_row = lane >> 1, half = lane & 1;
  auto turned = [](int k) { return (k * 32) ^ ((k & 8) << 4); };
  const uint32_t turn0 = lds_addr(turn) + wave * 4096;
  const uint32_t put_at = turn0 + turned(k_row) + 16 * half;
  const uint32_t get_at = turn0 + turned(8 * lg + (l16 >> 2)) + 8 * (l16 & 3);
  const int steps = (k_end + 31) / 32;
  unsigned long long left = __builtin_amdgcn_ballot_w64(own >= 0);
  for (int slot = 0; left != 0; ++slot) {
    const int l = __builtin_amdgcn_readlane(own, __builtin_ctzll(left));
    const unsigned long long users = __builtin_amdgcn_ballot_w64(own == l);
    left &= ~users;
    if (slot % gridDim.y != blockIdx.y) continue;
    const float scale = a.scale ? a.scale[l * a.scale_stride] : 1.f;
    const uint16_t* A = static_cast<const uint16_t*>(a.a) + l * a.a_l + c0 + (long long)(k_begin + k_row) * a.a_k;
    f32x4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto loop = [&](auto blocks_tag) __attribute__((always_inline)) {
      constexpr int kBlocks = decltype(blocks_tag)::value;  // of 16 columns
      constexpr int kAhead = 4;                             // steps in flight
      // columns past the rank repeat the first ones and are dropped
      int col[kBlocks];
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) col[j] = 16 * j + 8 * half < cols ? 16 * j + 8 * half : 0;
      // step i of this wave: two consecutive ones of every four pairs, whole 128-byte lines of x
      auto step_of = [&](int i) { return 2 * (wave + kWaves * (i >> 1)) + (i & 1); };
      struct Batch {
        u32x4 x[kAhead], a[kAhead][kBlocks];
      };
      auto load = [&](Batch& to, int i0) __attribute__((always_inline)) {
        if (k_end % 32 == 0) {  // (steps past the last repeat it and are not used)
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            const int k = min(32 * step_of(i0 + u), k_end - 32);
            to.x[u] = ld16(x + k);
#pragma unroll
            for (int j = 0; j < kBlocks; ++j) to.a[u][j] = ld16(A + (long long)k * a.a_k + col[j]);
          }
        } else {  // past K (a multiple of 8): zeros, in both operands
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            const int k = 32 * step_of(i0 + u);
            to.x[u] = k + 8 * lg < k_end ? ld16(x + k) : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < kBlocks; ++j)
              to.a[u][j] = k + k_row < k_end ? ld16(A + (long long)k * a.a_k + col[j]) : u32x4{0, 0, 0, 0};
          }
        }
      };
      auto multiply = [&](const Batch& from, int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (step_of(i0 + u) >= steps) break;
          // (a wave's LDS operations run in order: the reads of the step before are done)
          u32x4 f[kBlocks];
#pragma unroll
          for (int j = 0; j < kBlocks; ++j)
            *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(put_at + 1024 * j) = from.a[u][j];
#pragma unroll
          for (int j = 0; j < kBlocks; ++j) {
            const uint32_t at = get_at + 1024 * j;
            const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)at);
            const s16x4 v1 =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)(at ^ 128));
            const u32x2 lo = __builtin_bit_cast(u32x2, v0), hi = __builtin_bit_cast(u32x2, v1);
            f[j] = u32x4{lo[0], lo[1], hi[0], hi[1]};
          }
#pragma unroll
          for (int j = 0; j < kBlocks; ++j) acc[j] = H::mfma16(from.x[u], f[j], acc[j]);
        }
      };
      if (step_of(0) >= steps) return;
      for (int i0 = 0; step_of(i0) < steps; i0 += kAhead) {
        Batch batch;
        load(batch, i0);
        multiply(batch, i0);
      }
    };
    if (cols > 32) loop(Int<4>{});
    else if (cols > 16) loop(Int<2>{});
    else loop(Int<1>{});
    __syncthreads();  // the sums of the adapter before are read
    // column-major: a lane's four rows in one write
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<f32x4*>(&red[wave][16 * j + l16][4 * lg]) = acc[j];
    __syncthreads();
    const int c = tid % kCols, r0 = 4 * (tid / kCols);  // (a wave has all columns of four rows)
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (c < cols) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) sum += *reinterpret_cast<const f32x4*>(&red[w][c][r0]);
      sum *= scale;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (users >> (r0 + e) & 1ull) sums[((long long)split * a.m + m0 + r0 + e) * a.rank + c0 + c] = sum[e];
    }
    if constexpr (kAdapterRanged<H>) {
      const int top_pitch = adapter_top_pitch(gridDim.z * splits);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float top = __builtin_fabsf(sum[e]);
        const bool large = __builtin_amdgcn_ballot_w64(top >= kAdapterLarge) != 0;  // (a NaN is neither)
        if (large || __builtin_amdgcn_ballot_w64(top >= kAdapterSmall) == 0) {
#pragma unroll 1
          for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        } else {
          top = 1.f;
        }
        if (lane == 0 && (users >> (r0 + e) & 1ull)) tops[(long long)(m0 + r0 + e) * top_pitch + split * gridDim.z + blockIdx.z] = top;
      }
    }
  }
}

}  // namespace kg_gfx950
