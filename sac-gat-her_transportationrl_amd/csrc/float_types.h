// float_types.h -- the element types of the kernels that take float32,
// bfloat16 and float16 alike: eight consecutive elements as float32 and back.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace trx {
namespace {

typedef uint32_t word4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Eight {   // 16 bytes of a two-byte type
    T e[8];
};
template <>
struct Eight<float> {
    float e[8];
};

// eight elements at a 16-byte-aligned address
template <typename T>
__device__ __forceinline__ Eight<T> load8(const T* p) {
    Eight<T> r;
    reinterpret_cast<word4*>(&r)[0] = reinterpret_cast<const word4*>(p)[0];
    if constexpr (sizeof(T) == 4) reinterpret_cast<word4*>(&r)[1] = reinterpret_cast<const word4*>(p)[1];
    return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Eight<T>& r) {
    reinterpret_cast<word4*>(p)[0] = reinterpret_cast<const word4*>(&r)[0];
    if constexpr (sizeof(T) == 4) reinterpret_cast<word4*>(p)[1] = reinterpret_cast<const word4*>(&r)[1];
}

// calls f with a null pointer of the element type that dtype (0 float32, 1
// bfloat16, 2 float16) names
template <typename F>
inline hipError_t by_dtype(int dtype, F&& f) {
    if (dtype == 0) return f(static_cast<float*>(nullptr));
    if (dtype == 1) return f(static_cast<__bf16*>(nullptr));
    return f(static_cast<_Float16*>(nullptr));
}

}  // namespace
}  // namespace trx
