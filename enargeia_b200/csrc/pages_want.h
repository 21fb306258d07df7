// What the rows of one enx_pages_grow call want, in one 64-bit sum: pages in the low 40 bits (copies among
// them) and copies above.  Plain C++, so that the host can check the arithmetic at sizes no table has.
//
// A row's want is cut to one page more than the pool has, and the sum is looked at after every kPgThreads =
// 1024 rows: it is then at most 2^28 + 1024 (2^28 + 1) < 2^40 pages, and at most 2^18 copies.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define ENX_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define ENX_HOST_DEVICE inline
#endif

namespace enx {

constexpr uint32_t kWantShift = 40;

ENX_HOST_DEVICE unsigned long long want_of(bool copy, uint32_t fresh, uint32_t pages) {
    const uint32_t cut = fresh > pages ? pages + 1 : fresh;
    return ((unsigned long long)copy << kWantShift) + cut + copy;
}

ENX_HOST_DEVICE unsigned long long want_pages(unsigned long long sum) { return sum & ((1ull << kWantShift) - 1); }
ENX_HOST_DEVICE uint32_t want_copies(unsigned long long sum) { return (uint32_t)(sum >> kWantShift); }

}  // namespace enx
