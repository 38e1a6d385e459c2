// Translation unit of one kernel family of libkg_gfx950.so: the explicit instantiations
// kg_gfx950/instances_int8.h lists for it (compiled in parallel with the other families).
#define KG_INSTANTIATE
#define KG_INSTANTIATE_QUANTIZE
#include "kg_gfx950/instances_int8.h"

namespace kg_gfx950 {

hipError_t launch_int8_chunks(const Int8Tiles& g, int form, hipStream_t stream) {
  if (form == 4) return launch_gemm_i8<int, 2, 2, 4>(g, stream);
  if (form == 5) return launch_gemm_i8<int, 1, 2, 4>(g, stream);
  return launch_gemm_i8<int, 1, 1, 8>(g, stream);
}

}  // namespace kg_gfx950
