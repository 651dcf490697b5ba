// What the context-free operators on caller-owned device arrays share (layer norm, gated unit, draws): element types,
// wide loads, the guard that puts the caller's device back, wave and workgroup sums in a fixed order.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/gpbo.h"

namespace gpbo_static {

using bf16 = __hip_bfloat16;
using f16 = _Float16;

constexpr int MAX_DEVICES = 64;

__host__ __device__ constexpr int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }
__host__ __device__ constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Makes `device` current and puts the caller's device back on every way out.
struct DeviceGuard {
    int prev = -1;
    bool ok = false;
    explicit DeviceGuard(int device) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        ok = (prev == device) || hipSetDevice(device) == hipSuccess;
        if (prev == device) prev = -1;
    }
    ~DeviceGuard() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

inline int64_t type_bytes(int32_t dtype) {
    switch (dtype) {
        case GPBO_TYPE_F64: return 8;
        case GPBO_TYPE_F32: return 4;
        case GPBO_TYPE_BF16:
        case GPBO_TYPE_F16: return 2;
        default: return 0;
    }
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(f16 v) { return (float)v; }
__device__ __forceinline__ float to_float(bf16 v) {
    return __uint_as_float((uint32_t)__builtin_bit_cast(unsigned short, v) << 16);
}

// Round to nearest, ties to even: the one rounding an output gets.
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ f16 from_float<f16>(float v) { return (f16)v; }
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float v) {
    return __builtin_bit_cast(bf16, (__bf16)v);
}

// 16 bytes of elements; the address needs the element's alignment only (rows of odd length start anywhere: global memory
// takes 16-byte accesses at any address, and the compiler is told no more than that).
template <typename T>
struct Pack {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};
template <typename T>
__device__ __forceinline__ Pack<T> load_pack(const T* p) {
    Pack<T> r;
    __builtin_memcpy(&r, p, 16);
    return r;
}
template <typename T>
__device__ __forceinline__ void store_pack(T* p, const Pack<T>& r) {
    __builtin_memcpy(p, &r, 16);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

}  // namespace gpbo_static
