// Host side of TMA: the driver's tensor map encoder, looked up at run time so
// that the library links no driver library.
#pragma once
#include <cudaTypedefs.h>

namespace tcu {

// Null when the driver has none (the lookup is in runtime.cu).
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

}  // namespace tcu
