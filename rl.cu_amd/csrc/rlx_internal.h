// What the library's translation units share on the host side (not part of the C ABI).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "rlx_adamw.h"

// Every buffer handed to this library is HIP device memory, so all accesses go through
// global-address-space pointers (global_load/global_store rather than flat).
#define RLX_GLOBAL __attribute__((address_space(1)))

// Keeps the text for rlx_last_hip_error() and returns RLX_ERR_HIP.
__attribute__((visibility("hidden"))) int rlx_internal_hip_fail(hipError_t e, const char* what);

#define RLX_HIP(call)                                               \
    do {                                                            \
        hipError_t e_ = (call);                                     \
        if (e_ != hipSuccess) return rlx_internal_hip_fail(e_, #call); \
    } while (0)

inline bool rlx_is_aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
