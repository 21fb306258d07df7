// The bounded waits of the packed prompt attention (k_packed.cu): their limit, and the error they raise.
#pragma once

#include "enx_internal.cuh"

namespace enx {

cudaError_t packed_set_spin(uint32_t spins);
// Reads and clears the current device's error word (0: no wait gave up).
cudaError_t packed_take_error(uint32_t* code);

}  // namespace enx
