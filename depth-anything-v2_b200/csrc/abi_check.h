// Argument checks shared by the C ABI entries that live beside their kernels.
#pragma once

#include "launch.h"

#define DAV2_REQUIRE(cond, msg)                                                                  \
    do {                                                                                         \
        if (!(cond)) return ::dav2cuda::set_error(DAV2CUDA_INVALID_ARGUMENT, msg);               \
    } while (0)

namespace dav2cuda {

template <typename... P>
bool any_null(P... p) {
    return ((p == nullptr) || ...);
}

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Bytes of one element of a `precision` argument (0 f32, 1 bf16, 2 f16).
inline uint32_t element_bytes(uint32_t precision) { return precision == 0 ? 4u : 2u; }

}  // namespace dav2cuda
