// The attention kernels for a cache of E5M2 codes.
#include "attention_launch.hpp"

namespace iris_amd {
namespace calls {
IRIS_ATTENTION_CALLS(, IRIS_DTYPE_E5M2)
}  // namespace calls
}  // namespace iris_amd
