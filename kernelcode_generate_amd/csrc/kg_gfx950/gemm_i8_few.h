// Products in 8-bit integers (gemm_i8.h) of up to 32 rows with weights whose rows are no whole 16-byte pieces: the tiles (gemm_i8_tiles.h) would
// need a padded copy of all weights first (16 x 4096 x 4095: 6.5 us against the copy's 9 and 6 more). A workgroup takes 16 channels
// at a time, its waves equal ranges of k; a wave reads 16-byte pieces of the weights' rows, wherever they start, straight into operands of
// v_mfma_i32_16x16x64_i8 (operand A 16 channels x 64 k, operand B 16 MB rows), and the waves' sums, whole numbers in any order, meet in LDS.
#pragma once

#include "gemm_i8_tiles.h"
#include "quantize.h"

namespace kg_gfx950 {

namespace fewi {
constexpr int kWaves = 16, kThreads = 64 * kWaves;

__device__ __forceinline__ i32x4 mfma(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

}  // namespace fewi

// m <= 16 MB. A workgroup's blocks of channels are blockIdx.x, + gridDim.x, ...; kAhead steps of a wave are a group, and the next
// group's reads, of the next block's first where a block ends, are on their way while this one's products and sums are made.
template <typename T, int MB, int NB>
__global__ __launch_bounds__(fewi::kThreads) void int8_few_kernel(Int8Tiles g) {
  using namespace fewi;
  constexpr int kAhead = 4, kPitch = 16 * NB + 4;  // (a wave's stores of four channels of 16 rows spread over the banks)
  constexpr int kOutputs = (256 * MB * NB + kThreads - 1) / kThreads;  // of a thread
  __shared__ __attribute__((aligned(16))) int sums[2][kWaves][16 * MB][kPitch];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = (g.n + 16 * NB - 1) / (16 * NB);
  const int steps = (g.k + 63) / 64, each = (steps + kWaves - 1) / kWaves;
  const int first = wave * each, last = min(steps, first + each);
  const int groups = (each + kAhead - 1) / kAhead;  // of a block, in every wave
  const int8_t* x[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) x[i] = g.x + (long long)min(16 * i + l16, g.m - 1) * g.ldx;
  struct Group {
    u32x4 a[kAhead][NB], b[kAhead][MB];
  };
  auto load = [&](Group& f, int block, int group) __attribute__((always_inline)) {
    const int8_t* w[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) w[j] = g.w + (long long)min(16 * NB * block + 16 * j + l16, g.n - 1) * g.ldw;
    const int s = first + group * kAhead;
    if (s + kAhead <= last && 64 * (s + kAhead) <= g.k) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = 64 * (s + u) + 16 * lg;
#pragma unroll
        for (int j = 0; j < NB; ++j) f.a[u][j] = load_bytes(w[j] + k);
#pragma unroll
        for (int i = 0; i < MB; ++i) f.b[u][i] = load_bytes(x[i] + k);
      }
    } else {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        // (a step behind the wave's last takes codes of 0 for the rows)
        const int k = s + u < last ? 64 * (s + u) + 16 * lg : g.k;
#pragma unroll
        for (int j = 0; j < NB; ++j) f.a[u][j] = load_codes(w[j], k, g.k);
#pragma unroll
        for (int i = 0; i < MB; ++i) f.b[u][i] = load_codes(x[i], k, g.k);
      }
    }
  };
  float xs[kOutputs];
#pragma unroll
  for (int o = 0; o < kOutputs; ++o) xs[o] = g.x_scale[(long long)min((tid + o * kThreads) / (16 * NB), g.m - 1) * g.x_scale_stride];
  i32x4 acc[MB][NB];
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  };
  clear();
  Group even, odd;
  int block = blockIdx.x, group = 0, buffer = 0;
  load(even, block, 0);
  float ws[kOutputs], bias[kOutputs];
  auto turn = [&](const Group& now, Group& next) __attribute__((always_inline)) {
    const bool ends = group + 1 == groups;
    const int next_block = ends ? block + (int)gridDim.x : block, next_group = ends ? 0 : group + 1;
    if (group == 0) {
#pragma unroll
      for (int o = 0; o < kOutputs; ++o) {
        const long long n = min(16 * NB * block + (tid + o * kThreads) % (16 * NB), g.n - 1);
        ws[o] = g.w_scale[n * g.w_scale_stride];
        bias[o] = 0.f;
        if (g.bias != nullptr)
          bias[o] = g.wide_bias ? static_cast<const float*>(g.bias)[n * g.bias_stride] : Elem<T>::load(static_cast<const T*>(g.bias) + n * g.bias_stride);
      }
    }
    if (next_block < blocks) load(next, next_block, next_group);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = mfma(now.a[u][j], now.b[u][i], acc[i][j]);
    if (ends) {
      auto& to = sums[buffer];
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) *reinterpret_cast<i32x4*>(&to[wave][16 * i + l16][16 * j + 4 * lg]) = acc[i][j];
      clear();
      // (a barrier of LDS alone: the next group's reads stay on their way; the block after the next writes here behind the next barrier)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
#pragma unroll
      for (int o = 0; o < kOutputs; ++o) {
        const int at = tid + o * kThreads, r = at / (16 * NB), c = at % (16 * NB), n = 16 * NB * block + c;
        if (at >= 256 * MB * NB || r >= g.m || n >= g.n) continue;
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += to[w][r][c];
        Elem<T>::store(static_cast<T*>(g.out) + r * g.ldo + n, __builtin_fmaf((float)sum * xs[o], ws[o], bias[o]));
      }
      buffer ^= 1;
    }
    block = next_block;
    group = next_group;
  };
  // (two turns, so that a group stays in its registers: a copy would wait for its reads)
  while (block < blocks) {
    turn(even, odd);
    if (block >= blocks) break;
    turn(odd, even);
  }
}

}  // namespace kg_gfx950
