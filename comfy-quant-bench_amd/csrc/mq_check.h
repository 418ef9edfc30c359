// Argument checks shared by the extern "C" entry points.
#pragma once

#include <cstdint>

#include "../../include/mq.h"
#include "mq_internal.h"

#define MQ_REQUIRE(cond, ...)        \
    do {                             \
        if (!(cond)) {               \
            set_error(__VA_ARGS__);  \
            return MQ_EINVAL;        \
        }                            \
    } while (0)

namespace mq {

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }
inline int dtype_bytes(int dt) { return dt == MQ_DT_F32 ? 4 : 2; }

}  // namespace mq
