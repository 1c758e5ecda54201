// Rows of any width and alignment, read and written 16 bytes a lane, and sums over the lanes of a row.
#pragma once
#include "atlas_ops.h"

namespace atlas_ops {

// A lane's unit of a row: 16 bytes.  Rows need no alignment beyond their element's: gfx950 takes
// unaligned vector accesses, and 2-byte accesses for odd widths would need eight times the
// instructions.
template <typename T>
struct Unit {
    static constexpr int N = 16 / sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Raw { T v[N]; };
    uint64_t low, high;

    // The unit at column `col`, zeros beyond the row's width, with one load and no branch that lanes could
    // take differently: a unit that the row's end cuts is read as the row's last 16 bytes and shifted down.
    __device__ __forceinline__ void load(const T* row, int col, int width) {
        if (width >= N) {
            const int at = min(col, width - N);
            memcpy_in(row + at);
            if (width % N) {
                const int bits = min((col - at) * (int)sizeof(T) * 8, 128);
                const uint64_t up = bits >= 64 ? high >> (bits & 63) : (high << 1) << (63 - (bits & 63));
                low = bits >= 128 ? 0 : bits >= 64 ? up : (low >> bits) | up;
                high = bits >= 64 ? 0 : high >> bits;
            } else if (col >= width) {
                low = high = 0;
            }
        } else {
            T v[N];
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = col + i < width ? row[col + i] : T{};
            memcpy_in(v);
        }
    }
    __device__ __forceinline__ void memcpy_in(const T* p) {
        Raw raw;
        __builtin_memcpy(&raw, p, sizeof(raw));
        __builtin_memcpy(&low, &raw, 8);
        __builtin_memcpy(&high, (const char*)&raw + 8, 8);
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float((uint32_t)((i < 2 ? low : high) >> (i % 2 * 32)));
        else return to_float((bf16_t)((i < 4 ? low : high) >> (i % 4 * 16)));
    }
};

template <typename T, int N = Unit<T>::N>
__device__ __forceinline__ void store_unit(T* p, int left, const float* v) {
    if (left >= N) {
        struct __attribute__((packed, aligned(sizeof(T)))) Raw { T v[N]; } raw;
#pragma unroll
        for (int i = 0; i < N; ++i) raw.v[i] = from_float<T>(v[i]);
        __builtin_memcpy(p, &raw, sizeof(raw));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = from_float<T>(v[i]);
    }
}

// N values of the weight or bias (W is float or T) from column `col`, `fallback` where there is none.
template <typename W, int N>
__device__ __forceinline__ void load_columns(const W* p, int col, int width, float fallback, float* out) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = fallback;
        return;
    }
    constexpr int PER = Unit<W>::N;
    Unit<W> units[N / PER];
#pragma unroll
    for (int u = 0; u < N / PER; ++u) units[u].load(p, col + u * PER, width);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = units[i / PER][i % PER];
}

// A grid of `groups` workgroups for 32 columns each, 1024 threads, of which along x no more than a launch may have; the first
// column of a workgroup of it.
inline dim3 column_grid(i64 groups) {
    const i64 across = groups < THREADS / 1024 ? groups : THREADS / 1024 - 1;
    return dim3((unsigned)across, (unsigned)ceil_div(groups, across));
}
__device__ __forceinline__ i64 first_column() { return (i64)(blockIdx.y * gridDim.x + blockIdx.x) * 32; }

struct Rows {
    const void* data;
    i64 inner, outer_stride, inner_stride;
    template <typename T>
    __device__ __forceinline__ const T* at(i64 r) const {
        const i64 o = inner_stride * (r < inner ? r : r % inner) + (r < inner ? 0 : outer_stride * (r / inner));
        return (const T*)data + o;
    }
};

// Sums of K values over a row's group: LANES lanes of one wave, or (LANES = 256 or 512) the workgroup.
template <int LANES, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* shared) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lane_sum<LANES <= 64 ? LANES : 64>(v[k]);
    if constexpr (LANES > 64) {
        __syncthreads();  // the previous use of `shared` is read
        if (threadIdx.x % 64 == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) shared[LANES / 64 * k + threadIdx.x / 64] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const float* part = shared + LANES / 64 * k;
            v[k] = (part[0] + part[1]) + (part[2] + part[3]);
            if constexpr (LANES == 512) v[k] += (part[4] + part[5]) + (part[6] + part[7]);
        }
    }
}

}  // namespace atlas_ops
