// Paged KV cache of 4-bit rows, and eviction from a paged cache: host entry points.
#pragma once
#include <stddef.h>
#include <stdint.h>
#include <cuda_runtime.h>

#include "../../include/aicas_b200.h"

namespace aicas {

// Each launches its kernel for validated parameters, returns an AICAS_* status
// and writes a message into err on failure.
int run_paged_append_int4(const aicas_paged_append_int4_params* p, int sms, cudaStream_t stream, char* err, size_t errlen);
int run_paged_read_int4(const aicas_paged_read_int4_params* p, cudaStream_t stream, char* err, size_t errlen);

// Bytes of workspace run_paged_decode_int4 needs on a device with `sms` SMs.
size_t paged_decode_int4_workspace(const aicas_paged_decode_int4_params* p, int sms);
int run_paged_decode_int4(const aicas_paged_decode_int4_params* p, int sms, void* workspace, cudaStream_t stream,
                          char* err, size_t errlen);

int run_paged_weights(const aicas_paged_weights_params* p, int sms, cudaStream_t stream, char* err, size_t errlen);
int run_paged_evict(const aicas_paged_evict_params* p, int sms, cudaStream_t stream, char* err, size_t errlen);

}  // namespace aicas
