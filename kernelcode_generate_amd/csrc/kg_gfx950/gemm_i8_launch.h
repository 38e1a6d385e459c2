// Host side of the matrix-core kernels of int8_matmul and of quantize_rows: their forms and launches.
#pragma once

#include "gemm_i8_few.h"
#include "gemm_i8_tiles.h"
#include "quantize.h"

namespace kg_gfx950 {

// Rows of 8 to 16384 elements in one pass, others in two.
template <typename T>
hipError_t launch_quantize(const QuantizeArgs& a, hipStream_t stream) {
  const int pieces = (a.width + 2047) / 2048;
#define KG_QUANTIZE(PIECES, WAVES)                                                                                                \
  do {                                                                                                                            \
    const dim3 grid((unsigned)((a.rows + 4 / WAVES - 1) / (4 / WAVES)));                                                          \
    if (a.k % 8 == 0) hipLaunchKernelGGL((quantize_rows_kernel<T, PIECES, WAVES, true>), grid, dim3(256), 0, stream, a);          \
    else hipLaunchKernelGGL((quantize_rows_kernel<T, PIECES, WAVES, false>), grid, dim3(256), 0, stream, a);                      \
  } while (0)
  if (a.k < 8 || pieces > 8 || a.rows > (1 << 24) - 1)
    hipLaunchKernelGGL((quantize_rows_any_kernel<T>), dim3((unsigned)(a.rows < (1 << 24) - 1 ? a.rows : (1 << 24) - 1)), dim3(256), 0, stream, a);
  else if (a.width <= 512) KG_QUANTIZE(1, 1);
  else if (pieces == 1) KG_QUANTIZE(1, 4);
  else if (pieces == 2) KG_QUANTIZE(2, 4);
  else if (pieces <= 4) KG_QUANTIZE(4, 4);
  else KG_QUANTIZE(8, 4);
#undef KG_QUANTIZE
  return hipGetLastError();
}

// rows: 16, 32 or 64, at least m; channels: 16 or 32 a workgroup
template <typename T>
hipError_t launch_int8_few(const Int8Tiles& g, int rows, int channels, hipStream_t stream) {
  const dim3 grid((unsigned)((g.n + channels - 1) / channels));
#define KG_INT8_FEW(MB, NB) hipLaunchKernelGGL((int8_few_kernel<T, MB, NB>), grid, dim3(fewi::kThreads), 0, stream, g)
  if (channels == 16) {
    if (rows == 16) KG_INT8_FEW(1, 1);
    else if (rows == 32) KG_INT8_FEW(2, 1);
    else KG_INT8_FEW(4, 1);
  } else {
    if (rows == 16) KG_INT8_FEW(1, 2);
    else if (rows == 32) KG_INT8_FEW(2, 2);
    else KG_INT8_FEW(4, 2);
  }
#undef KG_INT8_FEW
  return hipGetLastError();
}

constexpr int kInt8FewQuantizeMostK = 8 * 64 * fewi::kWaves;
template <typename T>
hipError_t launch_int8_few_quantize(const Int8Tiles& g, const void* x, long long x_row, int channels, hipStream_t stream) {
  const dim3 grid((unsigned)((g.n + channels - 1) / channels));
#define KG_INT8_FEW(STEPS, NB)                                                                                              \
  do {                                                                                                                      \
    if (g.k % 64 == 0)                                                                                                      \
      hipLaunchKernelGGL((int8_few_quantize_kernel<T, STEPS, NB, true>), grid, dim3(fewi::kThreads), 0, stream, g,          \
                         static_cast<const T*>(x), x_row);                                                                  \
    else                                                                                                                    \
      hipLaunchKernelGGL((int8_few_quantize_kernel<T, STEPS, NB, false>), grid, dim3(fewi::kThreads), 0, stream, g,         \
                         static_cast<const T*>(x), x_row);                                                                  \
  } while (0)
  if (g.k <= kInt8FewQuantizeMostK / 2) {
    if (channels == 16) KG_INT8_FEW(4, 1);
    else KG_INT8_FEW(4, 2);
  } else {
    if (channels == 16) KG_INT8_FEW(8, 1);
    else KG_INT8_FEW(8, 2);
  }
#undef KG_INT8_FEW
  return hipGetLastError();
}

// tile: rows of a square tile
template <typename T>
hipError_t launch_int8_tiles(const Int8Tiles& g, int tile, hipStream_t stream) {
  if (tile == 256) return launch_gemm_i8<T, 8, 8, 64, 4>(g, stream);
  if (tile == 128) return launch_gemm_i8<T, 4, 4, 128, 4>(g, stream);
  return launch_gemm_i8<T, 2, 2, 128, 4>(g, stream);
}

}  // namespace kg_gfx950
