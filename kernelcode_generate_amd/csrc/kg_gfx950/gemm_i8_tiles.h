// gemm_i8_kernel: products in 8-bit integers (gemm_i8.h) in tiles, four waves of 2 x 2, each a (16 NA) x (16 NB) quarter in blocks of
// v_mfma_i32_16x16x64_i8. Both operands lie along k, so both are copied to LDS and read back the same way: rows of 128
// bytes, fragments of 16 bytes (16 k) a lane, which is the form that the instruction takes from both sides. The K loop: a ring of kStages
// slices of 128 k filled by copies straight from memory to LDS, one barrier a slice, and a step's MFMAs (64 k) from registers while the
// next step's fragments are read and a later slice's copies are issued between them. The barrier before a slice's last step finds all its
// fragments read: it publishes the next slice's copies and frees this slice's stage for its refill.
//
// Slices of 128 k: a copy then takes whole 128-byte lines. With 64, each line passes from the L2 twice, and 256 x 256 tiles were bound by
// that (8192^3, 8 % longer with four slices of 64 in the ring than with two of 128). What bounds them now, 8192^3 with codes of a normal
// distribution, 401 to 413 us: power. The products are 524288 cycles of a SIMD, 268 us at the 1.95 GHz to which the clock falls here (on
// registers alone it is 2.0, 4.2 POPS), and 65 % of the cycles that pass (the form with slices of 64 took 419 us, 322 with the
// copies left out, 374 with the reads of LDS left out, in as many cycles as with them). 2.66 to 2.74 POPS; the library's product 2.44. 4096^3 54 us,
// of which 11 are a launch, a ring to fill and the results' way to memory. Small tiles are bound by a slice's chain of barrier, LDS reads and
// products (0.1 us for 32 x 32, 0.2 for 64 x 64), middle ones by what a CU takes into its LDS, some 80 GB/s (20 TB/s where all 256 have a tile).
//
// Copies are buffer loads that land zeros outside the matrices (as fast as plain ones), stores are made inside alone: any M and N. K is a
// multiple of 16 (rows of others are copied into padded ones first).
#pragma once

#include "gemm.h"
#include "gemm_i8.h"
#include "lds_dma.h"

namespace kg_gfx950 {

typedef int i32x4 __attribute__((ext_vector_type(4)));

namespace gemmi {
constexpr int kThreads = 256;
constexpr int kBK = 128, kSteps = kBK / 64;  // k of a slice, its steps
// acc += a b on one 16 x 16 block, the accumulator tied to one register tuple of the accumulation file for the whole kernel (the compiler
// rotates the accumulators of its own form through that file at the loop's edge: 128 x 128 tiles of K = 4096 21.2 us, tied 16.6);
// results are read behind mfma_drain and mfma_order.
__device__ __forceinline__ void mfma(i32x4& acc, u32x4 a, u32x4 b) {
  asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
// more than the instruction's result latency (8 passes) before its result is read
__device__ __forceinline__ void mfma_drain() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }
template <int N>
__device__ __forceinline__ void mfma_order(i32x4 (&a)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+a"(a[i]));
}
// 16-byte chunk c of a row lies at c ^ swizzle(row): the 16 rows of a fragment's read hit distinct banks (256 bytes a cycle)
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }
}  // namespace gemmi

// 16 bytes to any address, past the L2
__device__ __forceinline__ void store_bytes(void* p, u32x4 v) {
  struct __attribute__((packed, aligned(2))) Piece {
    u32x4 w;
  };
  __builtin_nontemporal_store(v, &reinterpret_cast<Piece*>(p)->w);
}

struct Int8Tiles {
  const int8_t *x, *w;
  const float *x_scale, *w_scale;
  const void* bias;
  void* out;
  long long ldx, ldw, ldo, x_scale_stride, w_scale_stride, bias_stride;
  int m, n, k;
  bool wide_bias;
  int chunk;  // of k, a workgroup's (blockIdx.y)
};

// T int: the sums as they are, of one chunk of k: out is [chunks][m][ldo].
template <typename T, int NA, int NB, int kStages>
__global__ __launch_bounds__(gemmi::kThreads, NA * NB > 16 ? 1 : 2) void gemm_i8_kernel(Int8Tiles g) {
  using namespace gemmi;
  constexpr int TM = 32 * NA, TN = 32 * NB;
  constexpr int kRowsPiece = 1024 / kBK;  // rows of a wave's copy
  constexpr int AP = TM / kRowsPiece / 4, BP = TN / kRowsPiece / 4, kPieces = AP + BP;  // copies per wave and slice
  constexpr int kStageA = TM * kBK, kStageB = TN * kBK, kStage = kStageA + kStageB;
  constexpr int kMfmas = NA * NB, kReads = NA + NB;
  static_assert(AP >= 1 && BP >= 1, "pieces");
  static_assert(kStages >= 2, "a ring");
  __shared__ __attribute__((aligned(1024))) char lds[kStages * kStage];
  __shared__ __attribute__((aligned(16))) float xs_lds[TM], ws_lds[TN], bias_lds[TN];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int l16 = lane & 15, lg = lane >> 4;
  const int tiles_n = (g.n + TN - 1) / TN, tiles_m = (g.m + TM - 1) / TM;
  // each XCD takes a contiguous range of tiles in groups of 4 tile rows (few panels per L2)
  const int total = gridDim.x, xcd = blockIdx.x % 8;
  const int logical = xcd * (total / 8) + min(xcd, total % 8) + blockIdx.x / 8;
  constexpr int kGroupM = 4;
  const int group = logical / (kGroupM * tiles_n), first_m = group * kGroupM;
  const int gm = min(tiles_m - first_m, kGroupM), in_group = logical - group * kGroupM * tiles_n;
  const int m0 = (first_m + in_group % gm) * TM, n0 = (in_group / gm) * TN;

  constexpr bool kPartial = std::is_same<T, int>::value;
  const int k0 = kPartial ? blockIdx.y * g.chunk : 0, k_own = kPartial ? min(g.k - k0, g.chunk) : g.k;
  const int count = max((k_own + kBK - 1) / kBK, kStages);  // slices of K, at least a ring of them: zeros behind K

  // ---- memory -> LDS: piece p of a wave is rows (wave AP + p) kRowsPiece + lane / (kBK / 16) ----
  constexpr int kChunks = kBK / 16;
  uint32_t a_off[AP], b_off[BP];
  int chunk_k[2];  // the k of a lane's chunk within the slice, by the parity of the piece's first row / 8
#pragma unroll
  for (int p = 0; p < AP; ++p) {
    const int row = (wave * AP + p) * kRowsPiece + lane / kChunks;
    a_off[p] = (uint32_t)(row * g.ldx + 16 * ((lane % kChunks) ^ swizzle(row)));
    if (m0 + row >= g.m) a_off[p] = kBufOOB;
  }
#pragma unroll
  for (int p = 0; p < BP; ++p) {
    const int row = (wave * BP + p) * kRowsPiece + lane / kChunks;
    b_off[p] = (uint32_t)(row * g.ldw + 16 * ((lane % kChunks) ^ swizzle(row)));
    if (n0 + row >= g.n) b_off[p] = kBufOOB;
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) chunk_k[x] = 16 * ((lane % kChunks) ^ swizzle(x * kRowsPiece + lane / kChunks));
  const char* a_tile = reinterpret_cast<const char*>(g.x) + (long long)m0 * g.ldx + k0;
  const char* b_tile = reinterpret_cast<const char*>(g.w) + (long long)n0 * g.ldw + k0;
  const uint32_t lds0 = lds_addr(lds);
  auto issue_piece = [&](int kt, int stage, int piece) __attribute__((always_inline)) {
    const bool a = piece < AP;
    const int p = a ? piece : piece - AP;
    const char* src = (a ? a_tile : b_tile) + (long long)kt * kBK;
    const uint32_t dst = lds0 + stage * kStage + (a ? (wave * AP + p) * 1024 : kStageA + (wave * BP + p) * 1024);
    const uint32_t off = a ? a_off[a ? p : 0] : b_off[a ? 0 : p];
    const int k = chunk_k[((a ? wave * AP : wave * BP) + p) & 1];
    buf2lds16_s(kt * kBK + k < k_own ? off : kBufOOB, src, dst);
  };

  // ---- fragments of step ks: rows 16 i + lane % 16 of the wave's half, chunk 4 ks + lane / 16 ----
  uint32_t a_rd[kSteps], b_rd[kSteps];
#pragma unroll
  for (int ks = 0; ks < kSteps; ++ks) {
    const int at = 16 * ((4 * ks + lg) ^ swizzle(l16));
    a_rd[ks] = lds0 + (wm * 16 * NA + l16) * kBK + at;
    b_rd[ks] = lds0 + kStageA + (wn * 16 * NB + l16) * kBK + at;
  }
  struct Frags {
    u32x4 a[NA], b[NB];
  };
  // (a step's two addresses by themselves: the blocks' distances are then the instructions' own offsets)
  uint32_t b_at = 0, a_at = 0;
  auto read_from = [&](int stage, int ks) __attribute__((always_inline)) {
    b_at = b_rd[ks] + stage * kStage;
    a_at = a_rd[ks] + stage * kStage;
    asm volatile("" : "+v"(b_at), "+v"(a_at));
  };
  auto read_step = [&](Frags& f, int r) __attribute__((always_inline)) {  // w first
    const uint32_t at = r < NB ? b_at + r * 16 * kBK : a_at + (r - NB) * 16 * kBK;
    const u32x4 v = *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)at;
    if (r < NB) f.b[r < NB ? r : 0] = v;
    else f.a[r < NB ? 0 : r - NB] = v;
  };

  // scales and bias of the tile: read ahead of the K loop, into LDS behind it
  float xs_own = 0.f, ws_own = 0.f, bias_own = 0.f;
  if constexpr (!kPartial) {
    if (tid < TM) xs_own = g.x_scale[(long long)min(m0 + tid, g.m - 1) * g.x_scale_stride];
    if (tid < TN) {
      const long long at = min(n0 + tid, g.n - 1);
      ws_own = g.w_scale[at * g.w_scale_stride];
      bias_own = int8_bias<T>(g.bias, g.bias_stride, g.wide_bias, at);
    }
  }

  i32x4 acc[NA][NB];
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  // (opaque from here on: zeros made again right before the first MFMAs would lack the wait that these need)
#pragma unroll
  for (int i = 0; i < NA; ++i) mfma_order(acc[i]);

  // copies of a slice in its last step, and (kHalves) the others in the next slice's first one
  constexpr bool kHalves = kStages > 2;
  constexpr int kCopies = kHalves ? (kPieces + 1) / 2 : kPieces, kRest = kPieces - kCopies;
#pragma unroll
  for (int i = 0; i < kStages; ++i)
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
      if (i < kStages - 1 || p < kCopies) issue_piece(i, i, p);  // (kHalves: the first slice brings the last one's second half)
  wait_and_barrier<(kStages - 2) * kPieces + kCopies>();  // slice 0 has landed
  Frags fr[2];
  read_from(0, 0);
#pragma unroll
  for (int r = 0; r < kReads; ++r) read_step(fr[0], r);

  // Slice kt, in stage `stage`. kBehind: slices behind it, kStages where there are so many. The refill of its
  // stage (slice kt + kStages) goes into the last step, behind its barrier, with more than two stages half of it into the next
  // slice's first. The last kStages slices are a compile-time group whose waits, reads and copies carry no conditions (with
  // conditions they took about twice a steady one's cycles).
  auto slice = [&](int kt, int stage, auto behind_tag) __attribute__((always_inline)) {
    constexpr int kBehind = decltype(behind_tag)::value;
    constexpr int kYounger = (kBehind < kStages - 1 ? kBehind : kStages - 1) - 1;  // slices behind the next one that are on their way
    const int next = stage + 1 == kStages ? 0 : stage + 1, before = stage == 0 ? kStages - 1 : stage - 1;
    static_for<kSteps>([&](auto step_tag) __attribute__((always_inline)) {
      constexpr int ks = decltype(step_tag)::value;
      constexpr bool kLast = ks == kSteps - 1;
      if constexpr (kLast && kBehind > 0) wait_and_barrier<(kYounger > 0 ? kYounger : 0) * kPieces>();
      if constexpr (!kLast) read_from(stage, 1);
      else if constexpr (kBehind > 0) read_from(next, 0);
      static_for<kMfmas>([&](auto idx_tag) __attribute__((always_inline)) {
        constexpr int idx = decltype(idx_tag)::value;
        constexpr int i = idx / NB, j = idx % NB;
        mfma(acc[i][j], fr[ks].b[j], fr[ks].a[i]);  // blocks of the transpose: a lane's columns lie side by side
        constexpr int r0 = (idx * 2 * kReads + kMfmas - 1) / kMfmas, r1 = ((idx + 1) * 2 * kReads + kMfmas - 1) / kMfmas;
        static_for<(r1 < kReads ? r1 : kReads) - (r0 < kReads ? r0 : kReads)>([&](auto r_tag) __attribute__((always_inline)) {
          constexpr int r = r0 + decltype(r_tag)::value;
          if constexpr (!kLast || kBehind > 0) read_step(fr[ks ^ 1], r);
        });
        constexpr int kOwn = kLast ? kCopies : kRest;
        static_for<kOwn>([&](auto c_tag) __attribute__((always_inline)) {
          constexpr int c = decltype(c_tag)::value;
          if constexpr (idx == (2 * c + 1) * kMfmas / (2 * kOwn)) {
            if constexpr (kLast && kBehind == kStages) issue_piece(kt + kStages, stage, c);
            if constexpr (!kLast && kBehind >= kStages - 1) issue_piece(kt - 1 + kStages, before, kCopies + c);
          }
        });
        __builtin_amdgcn_sched_barrier(0);
      });
    });
  };
  int kt = 0, stage = 0;
  auto step = [&]() __attribute__((always_inline)) { stage = stage + 1 == kStages ? 0 : stage + 1; };
#pragma unroll 1
  for (; kt + kStages < count; ++kt) {
    slice(kt, stage, Int<kStages>{});
    step();
  }
  static_for<kStages>([&](auto u_tag) __attribute__((always_inline)) {
    constexpr int u = decltype(u_tag)::value;
    slice(kt + u, stage, Int<kStages - 1 - u>{});
    step();
  });

  // ---- a lane holds out[16 i + lane % 16][16 j + 4 (lane / 16) .. + 3] of each block (i, j) ----
  mfma_drain();
#pragma unroll
  for (int i = 0; i < NA; ++i) mfma_order(acc[i]);
  if (tid < TM) xs_lds[tid] = xs_own;
  if (tid < TN) ws_lds[tid] = ws_own, bias_lds[tid] = bias_own;
  wait_and_barrier<0>();  // the ring is read
  const int mw = m0 + wm * 16 * NA, nw = n0 + wn * 16 * NB;
  float xs[NA];
#pragma unroll
  for (int i = 0; i < NA; ++i) xs[i] = xs_lds[wm * 16 * NA + 16 * i + l16];
  // Each wave packs P row blocks of its results at a time into a part of the ring that is its own and writes them back as row segments, 16
  // bytes a lane (from the registers as they lie, 32-bit results took 190 us for 8192 x 3304 x 4000 where bf16 ones take 137).
  constexpr int kRow = 16 * NB * (int)sizeof(T), kRowChunks = kRow / 16, kEach = 16 / (int)sizeof(T);  // bytes and chunks of a row, elements of a chunk
  constexpr int P = NA * 16 * kRow <= kStages * kStage / 4 ? NA : NA / 2;
  static_assert(P >= 1 && P * 16 * kRow <= kStages * kStage / 4, "a wave's part of the ring");
  const uint32_t region = lds0 + wave * P * 16 * kRow;
  auto row_swizzle = [](int r) { return kRowChunks == 4 ? (r >> 1) & 3 : r & ((kRowChunks < 16 ? kRowChunks : 16) - 1); };
#pragma unroll
  for (int i0 = 0; i0 < NA; i0 += P) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const f32x4 ws = *reinterpret_cast<const f32x4*>(&ws_lds[wn * 16 * NB + 16 * j + 4 * lg]);
      const f32x4 bv = *reinterpret_cast<const f32x4*>(&bias_lds[wn * 16 * NB + 16 * j + 4 * lg]);
#pragma unroll
      for (int i = i0; i < i0 + P; ++i) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int sum = acc[i][j][e];
          v[e] = kPartial ? __builtin_bit_cast(float, sum) : __builtin_fmaf((float)sum * xs[i], ws[e], bv[e]);
        }
        const int r = 16 * (i - i0) + l16;
        if constexpr (sizeof(T) == 4) {
          const uint32_t at = region + r * kRow + (((4 * j + lg) ^ row_swizzle(r)) * 16);
          *(__attribute__((address_space(3))) f32x4*)(uintptr_t)at = f32x4{v[0], v[1], v[2], v[3]};
        } else {
          using H = Half16<typename Eight<T>::Tag>;
          const uint32_t at = region + r * kRow + (((2 * j + (lg >> 1)) ^ row_swizzle(r)) * 16) + (lg & 1) * 8;
          *(__attribute__((address_space(3))) u32x2*)(uintptr_t)at = u32x2{H::pack2(v[0], v[1]), H::pack2(v[2], v[3])};
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // (a column of blocks at a time: all of them at once are more than the registers hold)
    }
    constexpr int kRowsStore = 64 / kRowChunks;
#pragma unroll
    for (int q = 0; q < (16 * P + kRowsStore - 1) / kRowsStore; ++q) {
      const int r = kRowsStore * q + lane / kRowChunks, c = lane % kRowChunks;
      if (16 * P < kRowsStore && r >= 16 * P) continue;  // (16 x 16 results of 16 bits have 32 chunks)
      const u32x4 v = *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)(region + r * kRow + ((c ^ row_swizzle(r)) * 16));
      const int m = mw + 16 * i0 + r, n = nw + kEach * c;
      if (m >= g.m || n >= g.n) continue;
      T* to = static_cast<T*>(g.out) + ((kPartial ? (long long)blockIdx.y * g.m : 0ll) + m) * g.ldo + n;
      if (n + kEach <= g.n) {
        store_bytes(to, v);
      } else {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          if (n + e >= g.n) continue;
          if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(to)[e] = v[e];
          else reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
  }
}

template <typename T, int NA, int NB, int kStages>
hipError_t launch_gemm_i8(const Int8Tiles& g, hipStream_t stream) {
  constexpr int TM = 32 * NA, TN = 32 * NB;
  const unsigned grid = (unsigned)(((long long)g.m + TM - 1) / TM * (((long long)g.n + TN - 1) / TN));
  const unsigned chunks = std::is_same<T, int>::value ? (unsigned)((g.k + g.chunk - 1) / g.chunk) : 1u;
  hipLaunchKernelGGL((gemm_i8_kernel<T, NA, NB, kStages>), dim3(grid, chunks), dim3(gemmi::kThreads), 0, stream, g);
  return hipGetLastError();
}

// The chunks' sums joined: whole numbers, so the bits are those of one chunk. partial: [chunks][m][ld], ld a multiple of 4; four
// channels a thread.
template <typename T>
__global__ __launch_bounds__(256) void int8_join_kernel(Int8Tiles g, const int* partial, int chunks, int ld) {
  const int at = blockIdx.x * 256 + threadIdx.x, quads = ld / 4;
  const int m = at / quads, n = 4 * (at - m * quads);
  if (m >= g.m) return;
  i32x4 sum = {0, 0, 0, 0};
  const int* from = partial + (long long)m * ld + n;
#pragma unroll 4
  for (int c = 0; c < chunks; ++c) sum += *reinterpret_cast<const i32x4*>(from + (long long)c * g.m * ld);
  const float xs = g.x_scale[m * g.x_scale_stride];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= g.n) continue;
    const float bias = int8_bias<T>(g.bias, g.bias_stride, g.wide_bias, n + e);
    Elem<T>::store(static_cast<T*>(g.out) + m * g.ldo + n + e, __builtin_fmaf((float)sum[e] * xs, g.w_scale[(n + e) * g.w_scale_stride], bias));
  }
}

}  // namespace kg_gfx950
