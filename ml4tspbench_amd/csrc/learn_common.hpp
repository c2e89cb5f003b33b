// ml4tspbench_amd/csrc/learn_common.hpp -- element types shared by the learning operators
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "host_util.hpp"

namespace t2o {

// Stored element types.  All arithmetic is in float (or double where said): a value is widened exactly on load and
// rounded once, to nearest even, on store.
using bf16_t = __bf16;
using f16_t = _Float16;

template <typename T>
__device__ __forceinline__ float widen(T x)
{
    return static_cast<float>(x);
}

template <typename T>
__device__ __forceinline__ T narrow(float x)
{
    return static_cast<T>(x);
}

inline int element_size(int dtype)
{
    return dtype == TSP2OPT_DTYPE_F32 ? 4 : (dtype == TSP2OPT_DTYPE_BF16 || dtype == TSP2OPT_DTYPE_F16) ? 2 : 0;
}

#define T2O_BY_DTYPE(dtype, CALL)                                  \
    switch (dtype) {                                               \
        case TSP2OPT_DTYPE_F32: { using E = float; CALL; break; }  \
        case TSP2OPT_DTYPE_BF16: { using E = bf16_t; CALL; break; } \
        default: { using E = f16_t; CALL; break; }                 \
    }

}  // namespace t2o
