// Explicit instantiations of the launchers of int8_matmul and quantize_rows, as instances.h has them of the other families.
#pragma once

#include "gemm_i8_launch.h"

#ifdef KG_INSTANTIATE
#define KG_INSTANCE template
#else
#define KG_INSTANCE extern template
#endif

namespace kg_gfx950 {

#define KG_INT8_INSTANCE(T) KG_INSTANCE hipError_t launch_int8_tiles<T>(const Int8Tiles&, const Int8Plan&, int*, hipStream_t);
#if !defined(KG_INSTANTIATE) || defined(KG_INSTANTIATE_INT8_F32)
KG_INT8_INSTANCE(float)
#endif
#if !defined(KG_INSTANTIATE) || defined(KG_INSTANTIATE_INT8_BF16)
KG_INT8_INSTANCE(__bf16)
#endif
#if !defined(KG_INSTANTIATE) || defined(KG_INSTANTIATE_INT8_F16)
KG_INT8_INSTANCE(_Float16)
#endif
#undef KG_INT8_INSTANCE
#if !defined(KG_INSTANTIATE) || defined(KG_INSTANTIATE_QUANTIZE)
#define KG_QUANTIZE_INSTANCE(T) KG_INSTANCE hipError_t launch_quantize<T>(const QuantizeArgs&, const PackArgs&, hipStream_t);
KG_QUANTIZE_INSTANCE(float)
KG_QUANTIZE_INSTANCE(__bf16)
KG_QUANTIZE_INSTANCE(_Float16)
#undef KG_QUANTIZE_INSTANCE
#endif

}  // namespace kg_gfx950

#undef KG_INSTANCE
