// Waiting for the verdict words of calls whose arguments the device checks (see CallCheck).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace kvhip {

// Waits until each of `words` verdict words carries `stamp`; *refused tells whether any of them refuses the call.
hipError_t await_verdict(const int64_t* report, int64_t words, int64_t stamp, hipStream_t stream, bool* refused);

}  // namespace kvhip
