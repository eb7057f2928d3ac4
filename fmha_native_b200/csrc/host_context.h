// host_context.h -- per-device host state that the launchers of this library
// share: the device error word read by fmha_fwd_d64_status, the driver's
// tensor-map encoder and the limit of the kernels' bounded waits.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

namespace fmha_host {

// Codes of the paged operators in the device error word.
constexpr int kErrIndex = 0x201;         // index data out of range (FMHA_ERR_INDEX)
constexpr int kErrTimeoutPaged = 0x202;  // a bounded wait ran out (FMHA_ERR_TIMEOUT)

struct Context {
    int device = 0;
    int* err_word = nullptr;
    PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    unsigned long long wait_limit_ns = 0;
};

// The current device's state; its first call on a device sets it up (and
// allocates the error word).  Returns an FMHA_* status.
__attribute__((visibility("hidden"))) int acquire(Context* out);

}  // namespace fmha_host
