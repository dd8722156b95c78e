// Attention over the paged cache, head dimension 128 (the instances of tri_attend_device.h).
#include "tri_attend_device.h"

namespace tri {
hipError_t launch_attend_128(const AttendLaunch& a, hipStream_t s) { return launch_attend_dim<128>(a, s); }
}  // namespace tri
