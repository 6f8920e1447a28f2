// Host helpers shared by the library's translation units (not exported).
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <stdint.h>

#define QLIN_HIDDEN __attribute__((visibility("hidden")))

// The current device: QLIN_OK with its SM count, or why it cannot run the kernels.
QLIN_HIDDEN int qlin_host_device(int* sms);

// cuTensorMapEncodeTiled, resolved once (null: not available).
QLIN_HIDDEN PFN_cuTensorMapEncodeTiled_v12000 qlin_host_encoder();

// Reads (and clears) the error word of the other translation unit's kernels.
QLIN_HIDDEN int qlin_mx_device_error(void* stream, int clear, int* device_status);
