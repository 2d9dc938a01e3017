// Host helpers shared by the library's translation units (defined in sinkcache_b200.cu, or
// where the comment says).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <stdint.h>

namespace sinkb200 {

// Counts a successful launch (sink_launch_count) and passes the code on.
cudaError_t counted(cudaError_t err);

// SM count of the current device (cached; <= 0 when there is none) and its index.
int device_sms(int* dev_out);

// cuTensorMapEncodeTiled, looked up once (nullptr when the driver has none).
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

// What sink_debug_fail_next_wait armed, (chunk << 32) | polls, or -1; disarms it.
int64_t take_fail_next_wait();

// One-time set-up of device `dev` for the paged attention (sink_ops.cu); outside captures.
int32_t prepare_paged(int dev);

}  // namespace sinkb200
