// Paged KV cache (append and decode attention): host entry points.
#pragma once
#include <stddef.h>
#include <stdint.h>
#include <cuda_runtime.h>

#include "../../include/aicas_b200.h"

namespace aicas {

// Each launches its kernel for validated parameters, returns an AICAS_* status
// and writes a message into err on failure.
int run_paged_append(const aicas_paged_append_params* p, cudaStream_t stream, char* err, size_t errlen);

// Bytes of workspace run_paged_decode needs on a device with `sms` SMs, whatever the call.
size_t paged_decode_workspace(int sms);
int run_paged_decode(const aicas_paged_decode_params* p, int sms, void* workspace, cudaStream_t stream,
                     unsigned int* dev_err, char* err, size_t errlen);

}  // namespace aicas
