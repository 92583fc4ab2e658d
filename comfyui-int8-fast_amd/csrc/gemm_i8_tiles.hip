// One tile configuration of the int8 GEMM for one output type: the build script compiles this file once for each pair
// (I8F_TU_CFG, I8F_TU_OUT; I8F_TU_GROUPED where the configuration also serves the grouped launch, I8F_TU_ADAPTED where it serves layers
// with adapters, I8F_TU_ADAPTED_ONLY where it serves nothing else).
#include "gemm_i8_impl.hpp"

namespace i8f {
namespace gemm {
#if !I8F_TU_ADAPTED_ONLY
template int launch_cfg<I8F_TU_CFG, I8F_TU_OUT>(GemmArgs &, hipStream_t);
#endif
#if I8F_TU_ADAPTED
template int launch_cfg_adapted<I8F_TU_CFG, I8F_TU_OUT>(AdaptedLayers &, const int8_t *, const float *, int, int, hipStream_t);
#endif
#if I8F_TU_GROUPED
template int launch_cfg_grouped<I8F_TU_CFG, I8F_TU_OUT>(const GemmArgs *, int, hipStream_t);
#endif
}  // namespace gemm
}  // namespace i8f
