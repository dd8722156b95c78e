// Attention over the paged cache: head dimension 256, fp16 queries (the instances of tri_attend_device.h).
#include "tri_attend_device.h"

namespace tri {
hipError_t launch_attend_256_fp16(const AttendLaunch& a, hipStream_t s) { return launch_attend_dim<TRI_KV_FP16, 256>(a, s); }
}  // namespace tri
