// The bounded waits of the 4-bit cache's attention (k_kv4.cu): their limit, and the error they raise.
#pragma once

#include "enx_internal.cuh"

namespace enx {

cudaError_t kv4_set_spin(uint32_t spins);
// Reads and clears the current device's error word (0: no wait gave up).
cudaError_t kv4_take_error(uint32_t* code);

}  // namespace enx
