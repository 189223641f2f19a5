// arg_types.hpp -- sizes and alignment of what the C structs point to.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "tmnn_hip.h"

namespace tmnn_hip {

inline size_t dtype_size(int32_t dtype) { return dtype == TMNN_DTYPE_F32 ? 4 : 2; }

inline bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace tmnn_hip
