// Products in 8-bit integers (gemm_i8.h) of few rows: the weights are the call. A workgroup takes 16 NB channels, its waves equal ranges of
// k; a wave reads 16-byte pieces of the weights' rows straight into operands of v_mfma_i32_16x16x64_i8 (operand A 16 channels x 64 k,
// operand B 16 MB rows), and the waves' sums, whole numbers in any order, meet in LDS once.
//
// int8_few_kernel: rows in codes. int8_few_quantize_kernel: up to 16 rows that it quantises itself, in one launch: each wave holds its range of
// all rows in registers while its weights are on their way, the rows' largest magnitudes meet in LDS, and the codes are made
// where the products need them.
#pragma once

#include "gemm_i8_tiles.h"
#include "quantize.h"

namespace kg_gfx950 {

namespace fewi {
constexpr int kWaves = 16, kThreads = 64 * kWaves;

// 16 codes of a row of `count` >= 16 from column k, zeros behind its end, without a branch.
__device__ __forceinline__ u32x4 load_codes(const int8_t* row, int k, int count) {
  const int at = min(k, count - 16);
  return shift_bytes(load_bytes(row + at), min(k - at, 16));
}

__device__ __forceinline__ i32x4 mfma(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// The waves' sums joined, scaled and written. sums: [kWaves][16 MB rows][16 NB channels + 4]
template <int MB, int NB>
struct Sums {
  static constexpr int kPitch = 16 * NB + 4;  // (a wave's stores of four channels of 16 rows spread over the banks)
  int v[kWaves][16 * MB][kPitch];
};
template <typename T, int MB, int NB>
__device__ __forceinline__ void join(Sums<MB, NB>& sums, const i32x4 (&acc)[MB][NB], const Int8Tiles& g, int n0, const float* scales) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, lg = lane >> 4;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) *reinterpret_cast<i32x4*>(&sums.v[wave][16 * i + l16][16 * j + 4 * lg]) = acc[i][j];
  __syncthreads();
  for (int at = tid; at < 256 * MB * NB; at += kThreads) {
    const int r = at / (16 * NB), c = at % (16 * NB), n = n0 + c;
    if (r >= g.m || n >= g.n) continue;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += sums.v[w][r][c];
    const float xs = scales != nullptr ? scales[r] : g.x_scale[r * g.x_scale_stride];
    float bias = 0.f;
    if (g.bias != nullptr)
      bias = g.wide_bias ? static_cast<const float*>(g.bias)[n * g.bias_stride] : Elem<T>::load(static_cast<const T*>(g.bias) + n * g.bias_stride);
    Elem<T>::store(static_cast<T*>(g.out) + r * g.ldo + n, __builtin_fmaf((float)sum * xs, g.w_scale[n * g.w_scale_stride], bias));
  }
}
}  // namespace fewi

// Rows of k >= 16 codes copied into rows of `pitch` bytes, a multiple of 16, zeros behind k: for copies to LDS, which take whole
// 16-byte pieces.
template <int kUnused = 0>
__global__ __launch_bounds__(256) void int8_pack_kernel(const int8_t* src, long long ld, int8_t* dst, int pitch, int rows, int k) {
  const int pieces = pitch / 16;
  for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < (long long)rows * pieces; at += 256ll * gridDim.x) {
    const int r = (int)(at / pieces), c = 16 * (int)(at - (long long)r * pieces);
    st16(dst + (long long)r * pitch + c, fewi::load_codes(src + r * ld, c, k));
  }
}

// m <= 16 MB
template <typename T, int MB, int NB>
__global__ __launch_bounds__(fewi::kThreads) void int8_few_kernel(Int8Tiles g) {
  using namespace fewi;
  __shared__ __attribute__((aligned(16))) Sums<MB, NB> sums;
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16 * NB;
  const int steps = (g.k + 63) / 64, each = (steps + kWaves - 1) / kWaves;
  const int first = wave * each, last = min(steps, first + each);
  const int8_t *x[MB], *w[NB];
#pragma unroll
  for (int i = 0; i < MB; ++i) x[i] = g.x + (long long)min(16 * i + l16, g.m - 1) * g.ldx;
#pragma unroll
  for (int j = 0; j < NB; ++j) w[j] = g.w + (long long)min(n0 + 16 * j + l16, g.n - 1) * g.ldw;
  i32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  constexpr int kAhead = MB + NB > 4 ? 2 : 4;  // (128 registers a lane)
  auto group = [&](int s, auto whole_tag) __attribute__((always_inline)) {
    constexpr bool kWhole = decltype(whole_tag)::value != 0;
    u32x4 a[kAhead][NB], b[kAhead][MB];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int k = 64 * (s + u) + 16 * lg;
      // (a step behind the wave's last takes codes of 0 for the rows)
#pragma unroll
      for (int j = 0; j < NB; ++j) a[u][j] = kWhole ? load_bytes(w[j] + k) : load_codes(w[j], k, g.k);
#pragma unroll
      for (int i = 0; i < MB; ++i) b[u][i] = kWhole ? load_bytes(x[i] + k) : load_codes(x[i], s + u < last ? k : g.k, g.k);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = mfma(a[u][j], b[u][i], acc[i][j]);
  };
  int s = first;
  for (; s + kAhead <= last && 64 * (s + kAhead) <= g.k; s += kAhead) group(s, Int<1>{});
  for (; s < last; s += kAhead) group(s, Int<0>{});
  join<T>(sums, acc, g, n0, nullptr);
}

// m <= 16; 16 <= k <= 64 kSteps kWaves; x: T, rows of x_row elements. kWhole: k is a multiple of 64.
template <typename T, int kSteps, int NB, bool kWhole>
__global__ __launch_bounds__(fewi::kThreads) void int8_few_quantize_kernel(Int8Tiles g, const T* xt, long long x_row) {
  using namespace fewi;
  __shared__ __attribute__((aligned(16))) Sums<1, NB> sums;
  __shared__ float tops[kWaves][16];
  __shared__ float scales[16];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16 * NB;
  const int steps = (g.k + 63) / 64, each = (steps + kWaves - 1) / kWaves;
  const int first = wave * each, last = min(steps, first + each);
  const T* x = xt + (long long)min(l16, g.m - 1) * x_row;
  RawEight<T> raw[kSteps][2];
#pragma unroll
  for (int u = 0; u < kSteps; ++u) {
    // (steps behind the wave's last: columns behind the row's end, zeros)
    const int k = first + u < last ? 64 * (first + u) + 16 * lg : steps * 64;
    raw[u][0] = load_eight<T, kWhole>(x, k, g.k);
    raw[u][1] = load_eight<T, kWhole>(x, k + 8, g.k);
  }
  u32x4 a[kSteps][NB];
#pragma unroll
  for (int u = 0; u < kSteps; ++u)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int8_t* w = g.w + (long long)min(n0 + 16 * j + l16, g.n - 1) * g.ldw;
      const int k = 64 * (first + u) + 16 * lg;
      a[u][j] = kWhole ? load_bytes(w + (first + u < last ? k : 0)) : load_codes(w, k, g.k);
    }
  float top = 0.f;
#pragma unroll
  for (int u = 0; u < kSteps; ++u)
#pragma unroll
    for (int h = 0; h < 2; ++h) top = nan_max(top, largest_of(raw[u][h]));
  top = nan_max(top, __shfl_xor(top, 16, 64));
  top = nan_max(top, __shfl_xor(top, 32, 64));
  if (lg == 0) tops[wave][l16] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = nan_max(top, tops[w][l16]);
  const float scale = top * CacheElem<int8_t>::kInverse;
  if (tid < 16) scales[tid] = scale;  // (read behind the next barrier)
  i32x4 acc[1][NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) acc[0][j] = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int u = 0; u < kSteps; ++u) {
    const u32x2 lo = int8_codes(raw[u][0], scale), hi = int8_codes(raw[u][1], scale);
    const u32x4 b = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[0][j] = mfma(a[u][j], b, acc[0][j]);
  }
  join<T>(sums, acc, g, n0, scales);
}

}  // namespace kg_gfx950
