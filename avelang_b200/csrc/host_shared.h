// Host-side parts that the library's translation units share; defined in ave_fp4_api.cu.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace avefp4 {

struct HostDevice {
    int sm_count;
    int* status;    // device status word of the bounded waits
};

// All of them return 0 or an error code after setting the calling thread's message.
int host_fail(int code, const char* message);
int host_fail_cuda(cudaError_t e, const char* what);
int host_device(HostDevice* out);      // the current device, after ave_fp4_init

// Tensor map of a matrix of `outer` rows of `inner` bytes, 128-byte swizzle, boxes of 128 bytes x box_rows.
int host_encode_bytes(CUtensorMap* tm, const void* base, uint64_t inner, uint64_t outer, uint64_t stride, uint32_t box_rows, const char* what);

// Attributes of the kernels in ave_dense_api.cu, set once per device by ave_fp4_init.
cudaError_t prepare_dense_kernels();

}  // namespace avefp4
