// Decode-side products with 4-bit weights: host entry point.
#pragma once
#include <stddef.h>
#include <stdint.h>
#include <cuda_runtime.h>

#include "../../include/aicas_b200.h"

namespace aicas {

// Launches the kernel for validated parameters on a device with `sms` SMs.
// Returns an AICAS_* status and writes a message into err on failure.
int run_linear_int4(const aicas_linear_int4_params* p, int sms, cudaStream_t stream, unsigned int* dev_err, char* err,
                    size_t errlen);

}  // namespace aicas
