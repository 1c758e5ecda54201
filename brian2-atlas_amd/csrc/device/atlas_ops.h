// What the operator kernels share: element types, wave reductions, launch and error helpers.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../../include/operators/atlas_ops.h"

namespace atlas_ops {

typedef int64_t i64;
typedef uint64_t u64;
typedef uint16_t bf16_t;
typedef float float4_t __attribute__((ext_vector_type(4)));

inline int fail(char* err, size_t cap, int code, const char* fmt, ...) {
    if (err && cap) {
        va_list args;
        va_start(args, fmt);
        vsnprintf(err, cap, fmt, args);
        va_end(args);
    }
    return code;
}

// The status of the launches just made (no wait).
inline int launched(char* err, size_t cap, const char* what) {
    const hipError_t status = hipGetLastError();
    return status == hipSuccess ? 0 : fail(err, cap, 4, "%s: %s", what, hipGetErrorString(status));
}

constexpr i64 THREADS = (i64)1 << 32;  // a grid's threads along x stay below

inline bool known_type(int type) { return type == ATLAS_OPS_F32 || type == ATLAS_OPS_BF16; }

inline i64 ceil_div(i64 a, i64 b) { return (a + b - 1) / b; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16_t v) { return __uint_as_float((uint32_t)v << 16); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
// Round to nearest even, a NaN stays one: gfx950 converts two values per instruction.
template <>
__device__ __forceinline__ bf16_t from_float<bf16_t>(float v) { return __builtin_bit_cast(bf16_t, (__bf16)v); }

// Sum over groups of LANES neighbouring lanes (16, 32 or 64); every lane gets it.  Within 16 lanes the values
// rotate in the adder's own operand (DPP); only the steps beyond go through the LDS crossbar.
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
    static_assert(LANES == 16 || LANES == 32 || LANES == 64, "whole rows of 16 lanes");
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xF, 0xF, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x124, 0xF, 0xF, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x122, 0xF, 0xF, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x121, 0xF, 0xF, false));
#pragma unroll
    for (int d = 16; d < LANES; d *= 2) v += __shfl_xor(v, d, 64);
    return v;
}

}  // namespace atlas_ops
