// The attention kernels for a cache of E4M3 codes.
#include "attention_launch.hpp"

namespace iris_amd {
namespace calls {
IRIS_ATTENTION_CALLS(, IRIS_DTYPE_E4M3)
}  // namespace calls
}  // namespace iris_amd
