// Attention over the paged cache: head dimension 64, bf16 queries (the instances of tri_attend_device.h).
#include "tri_attend_device.h"

namespace tri {
hipError_t launch_attend_64_bf16(const AttendLaunch& a, hipStream_t s) { return launch_attend_dim<TRI_KV_BF16, 64>(a, s); }
}  // namespace tri
