// Host side of the matrix-core kernels of int8_matmul and of quantize_rows: their forms and launches.
#pragma once

#include "gemm_i8_tiles.h"
#include "quantize.h"

namespace kg_gfx950 {

__global__ __launch_bounds__(256) static void int8_pack_kernel(PackArgs x, PackArgs w) {
  pack_rows(blockIdx.y == 0 ? x : w, (long long)blockIdx.x * 256 + threadIdx.x, 256ll * gridDim.x);
}
inline unsigned pack_blocks(const PackArgs& p) {
  const long long blocks = ((long long)p.rows * (p.pitch / 16) + 255) / 256;
  return (unsigned)(blocks < 4096 ? blocks : 4096);
}
// (either may have no rows)
inline hipError_t launch_int8_pack(const PackArgs& x, const PackArgs& w, hipStream_t stream) {
  const unsigned blocks = pack_blocks(x) > pack_blocks(w) ? pack_blocks(x) : pack_blocks(w);
  if (blocks > 0) hipLaunchKernelGGL(int8_pack_kernel, dim3(blocks, 2), dim3(256), 0, stream, x, w);
  return hipGetLastError();
}

// Rows of 8 to 16384 elements in one pass, others in two; and codes packed beside them.
template <typename T>
hipError_t launch_quantize(const QuantizeArgs& a, const PackArgs& pack, hipStream_t stream) {
  constexpr int kMostBlocks = (1 << 24) - 1;
  const int pieces = (a.width + 2047) / 2048;
#define KG_QUANTIZE(PIECES, WAVES)                                                                                                \
  do {                                                                                                                            \
    const dim3 grid((unsigned)((a.rows + 4 / WAVES - 1) / (4 / WAVES)) + pack_blocks(pack));                                      \
    if (a.k % 8 == 0) hipLaunchKernelGGL((quantize_rows_kernel<T, PIECES, WAVES, true>), grid, dim3(256), 0, stream, a, pack);    \
    else hipLaunchKernelGGL((quantize_rows_kernel<T, PIECES, WAVES, false>), grid, dim3(256), 0, stream, a, pack);                \
  } while (0)
  if (a.k < 8 || pieces > 8 || a.rows > kMostBlocks - 4096) {
    hipLaunchKernelGGL((quantize_rows_any_kernel<T>), dim3((unsigned)(a.rows < kMostBlocks ? a.rows : kMostBlocks)), dim3(256), 0, stream, a);
    return launch_int8_pack(pack, PackArgs{}, stream);
  }
  if (a.width <= 512) KG_QUANTIZE(1, 1);
  else if (pieces == 1) KG_QUANTIZE(1, 4);
  else if (pieces == 2) KG_QUANTIZE(2, 4);
  else if (pieces <= 4) KG_QUANTIZE(4, 4);
  else KG_QUANTIZE(8, 4);
#undef KG_QUANTIZE
  return hipGetLastError();
}

// The tiles of a product by a model of each form's time (ns): a launch, a further round of 256 tiles, a slice of 128 k, and percent more of
// a slice where all CUs have a tile (their clocks go down). Fitted to 350 products of 1..4096 rows, 1024..16384 channels and K of
// 512..11008, of which the one that it picks is 2.9 % above the fastest on average, the measurements' own spread with it. On 165 others of
// 65..640 rows, 4096..14336 channels and K of 4096..14336 it picks what is as fast as the fastest on average, 8 % slower at most (65 rows of K = 8192: 32 x 64
// 19.6, 32 x 32 17.9). us of the forms in
// their order: 4096^3 58 / 66 / 82 / 98 / 113 / - / -; 1000 x 4096 x 4096 44 / 29 / 19.3 / 23 / 31 / - / -; 300 x 4096 x 4096 43 / 27 / 17.5 / 14.0 /
// 14.2 / 16 / 20; 130 x 4096 x 4096 43 / 26 / 17.1 / 13.6 / 10.5 / 11.8 / 13.6; 300 x 11008 x 4096 50 / 31.2 / 33.7 / 35 / 34 / 42 / 54;
// 64 x 4096 x 4096 - / - / - / 12.7 / 9.5 / 8.4 / 6.1; 16 x 11008 x 11008 - / - / - / 43.7 / 33.3 / 32.7 / 30.7. A deeper ring than
// these changes nothing: what a slice of a small tile costs is its own chain of barrier, LDS reads and products.
struct Int8Form {
  int rows, channels, stages, fixed, round, slice, load;
};
constexpr Int8Form kInt8Forms[7] = {{256, 256, 2, 7800, 7600, 1140, 46}, {256, 128, 3, 5500, 4000, 610, 37}, {128, 128, 4, 3900, 1800, 420, 46},
                                    {128, 64, 3, 3350, 220, 290, 15},    {64, 64, 4, 3200, 200, 220, 7},      {32, 64, 4, 3300, 80, 158, 4},
                                    {32, 32, 8, 2800, 140, 98, 6}};
// A product's form and the chunk of k that a workgroup takes. Chunks (two, four or eight, of the three smallest tiles) are for few tiles of
// a long K: a CU takes some 80 GB/s into its LDS, whatever its tile, and has a slice no sooner. Their sums go through the
// workspace, and a second launch joins them: 2700 ns and the sums' way there and back. us without / with: 16 x 500 x 16384 17.6 / 8.8, 16 x 1024 x
// 11008 12.7 / 8.9, 200 x 500 x 16384 18.3 / 12.3; 16 x 4096 x 11008, which the memory bounds, is not split.
struct Int8Plan {
  int form, chunk, chunks;
  long long ld, bytes;  // of the sums: a row's (in elements), all
};
constexpr long long kInt8MostSums = 16ll << 20;
inline Int8Plan int8_plan(long long m, long long n, long long k, bool may_split) {
  Int8Plan best{};
  long long least = 0;
  const long long floor = 2000 + (m + n) * k / 4400;  // operands from memory
  for (int split = 1; split <= (may_split ? 8 : 1); split *= 2) {
    const long long chunk = split == 1 ? k : (k / split + 127) / 128 * 128, chunks = (k + chunk - 1) / chunk, ld = (n + 3) / 4 * 4;
    const long long bytes = split == 1 ? 0 : chunks * m * ld * 4;
    if (split > 1 && (chunks < 2 || bytes > kInt8MostSums || chunk < 1024)) break;
    for (int i = split == 1 ? 0 : 4; i < 7; ++i) {
      const Int8Form& f = kInt8Forms[i];
      const long long tiles = ((m + f.rows - 1) / f.rows) * ((n + f.channels - 1) / f.channels) * chunks, rounds = (tiles + 255) / 256;
      const long long slices = (chunk + 127) / 128 < f.stages ? f.stages : (chunk + 127) / 128;
      long long ns = f.fixed + (rounds - 1) * f.round + rounds * slices * f.slice * (25600 + f.load * (tiles < 256 ? tiles : 256)) / 25600;
      ns = ns > floor ? ns : floor;
      if (split > 1) ns += 2700 + bytes / 2000;
      if (least == 0 || ns < least) {
        least = ns;
        best = Int8Plan{i, (int)chunk, (int)chunks, ld, bytes};
      }
    }
  }
  return best;
}
// MFMA instructions of a product (cost queries).
inline long long int8_tiles_mfma(long long m, long long n, long long k, const Int8Plan& p) {
  const Int8Form& f = kInt8Forms[p.form];
  const long long tiles = ((m + f.rows - 1) / f.rows) * ((n + f.channels - 1) / f.channels);
  long long slices = 0;
  for (int c = 0; c < p.chunks; ++c) {
    const long long own = (k - (long long)c * p.chunk < p.chunk ? k - (long long)c * p.chunk : p.chunk);
    slices += (own + 127) / 128 < f.stages ? f.stages : (own + 127) / 128;
  }
  return tiles * (f.rows / 16) * (f.channels / 16) * 2 * slices;
}
hipError_t launch_int8_chunks(const Int8Tiles& g, int form, hipStream_t stream);
// partial: the workspace of a plan of several chunks
template <typename T>
hipError_t launch_int8_tiles(const Int8Tiles& g, const Int8Plan& p, int* partial, hipStream_t stream) {
  if (p.chunks > 1) {
    Int8Tiles sums = g;
    sums.out = partial;
    sums.ldo = p.ld;
    sums.chunk = p.chunk;
    const hipError_t err = launch_int8_chunks(sums, p.form, stream);
    if (err != hipSuccess) return err;
    const unsigned grid = (unsigned)((g.m * (p.ld / 4) + 255) / 256);
    hipLaunchKernelGGL((int8_join_kernel<T>), dim3(grid), dim3(256), 0, stream, g, partial, p.chunks, (int)p.ld);
    return hipGetLastError();
  }
  switch (p.form) {
    case 0: return launch_gemm_i8<T, 8, 8, 2>(g, stream);
    case 1: return launch_gemm_i8<T, 8, 4, 3>(g, stream);
    case 2: return launch_gemm_i8<T, 4, 4, 4>(g, stream);
    case 3: return launch_gemm_i8<T, 4, 2, 3>(g, stream);
    case 4: return launch_gemm_i8<T, 2, 2, 4>(g, stream);
    case 5: return launch_gemm_i8<T, 1, 2, 4>(g, stream);
    default: return launch_gemm_i8<T, 1, 1, 8>(g, stream);
  }
}

}  // namespace kg_gfx950
