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
// 512..11008, of which the one that it picks is 2.9 % above the fastest on average, the measurements' own spread with it. us of the forms in
// their order: 4096^3 58 / 66 / 82 / 98 / 113 / - / -; 1000 x 4096 x 4096 44 / 29 / 19.3 / 23 / 31 / - / -; 300 x 4096 x 4096 43 / 26 / 17 / 13.1 /
// 13.5 / 15 / 17.3; 64 x 4096 x 4096 - / - / - / 12.7 / 9.5 / 8.4 / 6.1; 16 x 11008 x 11008 - / - / - / 43.7 / 33.3 / 32.7 / 30.7. A deeper ring than
// these changes nothing: what a slice of a small tile costs is its own chain of barrier, LDS reads and products.
struct Int8Form {
  int rows, channels, stages, fixed, round, slice, load;
};
constexpr Int8Form kInt8Forms[7] = {{256, 256, 2, 7800, 7600, 1140, 46}, {256, 128, 3, 5500, 4000, 610, 37}, {128, 128, 4, 3900, 1800, 420, 46},
                                    {128, 64, 3, 3350, 220, 290, 15},    {64, 64, 4, 3200, 200, 220, 7},      {32, 64, 4, 3300, 80, 158, 4},
                                    {32, 32, 8, 2800, 140, 98, 6}};
inline int int8_form(long long m, long long n, long long k) {
  int best = 0;
  long long least = 0;
  for (int i = 0; i < 7; ++i) {
    const Int8Form& f = kInt8Forms[i];
    const long long tiles = ((m + f.rows - 1) / f.rows) * ((n + f.channels - 1) / f.channels), rounds = (tiles + 255) / 256;
    const long long slices = (k + 127) / 128 < f.stages ? f.stages : (k + 127) / 128;
    const long long ns = f.fixed + (rounds - 1) * f.round + rounds * slices * f.slice * (25600 + f.load * (tiles < 256 ? tiles : 256)) / 25600;
    if (i == 0 || ns < least) best = i, least = ns;
  }
  return best;
}
// MFMA instructions of a product (cost queries).
inline long long int8_tiles_mfma(long long m, long long n, long long k) {
  const Int8Form& f = kInt8Forms[int8_form(m, n, k)];
  const long long tiles = ((m + f.rows - 1) / f.rows) * ((n + f.channels - 1) / f.channels), slices = (k + 127) / 128;
  return tiles * (f.rows / 16) * (f.channels / 16) * 2 * (slices < f.stages ? f.stages : slices);
}
template <typename T>
hipError_t launch_int8_tiles(const Int8Tiles& g, int form, hipStream_t stream) {
  switch (form) {
    case 0: return launch_gemm_i8<T, 8, 8, 128, 2>(g, stream);
    case 1: return launch_gemm_i8<T, 8, 4, 128, 3>(g, stream);
    case 2: return launch_gemm_i8<T, 4, 4, 128, 4>(g, stream);
    case 3: return launch_gemm_i8<T, 4, 2, 128, 3>(g, stream);
    case 4: return launch_gemm_i8<T, 2, 2, 128, 4>(g, stream);
    case 5: return launch_gemm_i8<T, 1, 2, 128, 4>(g, stream);
    default: return launch_gemm_i8<T, 1, 1, 128, 8>(g, stream);
  }
}

}  // namespace kg_gfx950
