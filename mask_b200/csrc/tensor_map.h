// Tensor maps for TMA copies.  The encoder comes from the runtime's driver entry point lookup: the library does not link libcuda.
#pragma once

#include <cuda.h>

namespace mask {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, or nullptr where the driver has none.
EncodeTiledFn encode_tiled_fn();

}  // namespace mask
