// i4d_internal.h -- what the operators' translation unit needs of a context.
#pragma once

#include <cuda_runtime.h>

#include "i4d.h"

namespace i4d_ops {

struct OpContext {
    int device;
    int num_sms;
    cudaStream_t stream;
    unsigned* err;  // device error word of the operators
    unsigned* err_taken;       // host memory that the device can write: what ops_report took out of it
    cudaStream_t err_stream;   // which nothing else uses
    bool* used;                // host: an operator has been enqueued (null: nobody asks)
};

// i4d.cu
OpContext op_context(const i4d_ctx* c);
i4d_status op_fail(i4d_ctx* c, i4d_status st, const char* fmt, ...) __attribute__((format(printf, 3, 4)));

// i4d_ops.cu.  The operators' error word since the last call, with zero put in its place in
// the same step; the caller has waited for the operators that it asks about.
i4d_status ops_report(i4d_ctx* c);

}  // namespace i4d_ops
