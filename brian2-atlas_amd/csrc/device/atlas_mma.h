// Products of float32 accuracy on bfloat16 MFMA, and what the chunk kernels of sequences share with them.
#pragma once
#include "atlas_ops.h"

namespace atlas_ops {

// A tensor of (batch, time, head) strides with a contiguous last axis.
struct Tensor {
    const void* data;
    i64 batch, time, head;
    template <typename T>
    __device__ __forceinline__ const T* at(i64 b, i64 t, i64 h) const {
        return (const T*)data + b * batch + t * time + h * head;
    }
};

// Products run on bfloat16 MFMA blocks of 16 x 16 with 32 sum indices, at float32's accuracy: a float
// is the sum of three bfloat16 pieces (to 2^-24), a product takes the pieces' products down to that
// size, three where one side is bfloat16 already and six where neither is, summed in float32.  Float32
// MFMA would take 16 times the cycles of one such product.
//
// Lane l gives 8 values of row l % 16 of A, 8 of column l % 16 of B, and receives rows 4 (l / 16) + j of
// column l % 16.  The sum may take its indices in any order that A and B share: here lane group g = l / 16
// holds the indices 4 g + j and 16 + 4 g + j of 32, so that two blocks of results on top of each other are, without
// any exchange, the B operand of a product that sums over their rows, and the A operand of one whose rows
// are their columns.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));

constexpr float4_t ZERO = {0.0f, 0.0f, 0.0f, 0.0f};

// N pieces of 8 values, the largest first.
template <int N>
struct Pieces {
    bf16x8 p[N];
};

// N pieces of 4 values: half an operand.
template <int N>
struct Halves {
    bf16x4 p[N];
};

__device__ __forceinline__ float4_t widen(bf16x4 v) {
    const uint2_t bits = __builtin_bit_cast(uint2_t, v);
    return float4_t{__uint_as_float(bits[0] << 16), __uint_as_float(bits[0] & 0xFFFF0000u),
                    __uint_as_float(bits[1] << 16), __uint_as_float(bits[1] & 0xFFFF0000u)};
}

template <int N>
__device__ __forceinline__ Halves<N> split(float4_t v) {
    Halves<N> h;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        h.p[i] = __builtin_convertvector(v, bf16x4);
        if (i + 1 < N) v -= widen(h.p[i]);
    }
    return h;
}

// split with one instruction for each remainder: a dot product of two pieces with (-1, 0) or (0, -1), exact as the plain
// difference is.  The pieces of an infinity's neighbour in a pair become NaNs too, so both must enter the same sums.
__device__ __forceinline__ Halves<3> split_pairs(float4_t v) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    uint32_t first = 0x0000BF80u, second = 0xBF800000u;
    asm("" : "+s"(first), "+s"(second));  // in registers: written as a constant, the second reads as another pair
    const bf16x2 a = __builtin_bit_cast(bf16x2, first), b = __builtin_bit_cast(bf16x2, second);
    Halves<3> h;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        h.p[i] = __builtin_convertvector(v, bf16x4);
        if (i == 2) break;
        const bf16x2 low = __builtin_shufflevector(h.p[i], h.p[i], 0, 1), high = __builtin_shufflevector(h.p[i], h.p[i], 2, 3);
        v = float4_t{__builtin_amdgcn_fdot2_f32_bf16(low, a, v[0], false), __builtin_amdgcn_fdot2_f32_bf16(low, b, v[1], false),
                     __builtin_amdgcn_fdot2_f32_bf16(high, a, v[2], false), __builtin_amdgcn_fdot2_f32_bf16(high, b, v[3], false)};
    }
    return h;
}

template <int N>
__device__ __forceinline__ Pieces<N> join(const Halves<N>& a, const Halves<N>& b) {
    Pieces<N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.p[i] = __builtin_shufflevector(a.p[i], b.p[i], 0, 1, 2, 3, 4, 5, 6, 7);
    return r;
}

template <int N>
__device__ __forceinline__ Pieces<N> split(float4_t a, float4_t b) {
    return join(split<N>(a), split<N>(b));
}

__device__ __forceinline__ Pieces<3> split_pairs(float4_t a, float4_t b) { return join(split_pairs(a), split_pairs(b)); }

// c + A B: the products of pieces whose order together is below three (below two where no side has
// three), the smallest first.
template <int NA, int NB>
__device__ __forceinline__ float4_t mma(const Pieces<NA>& a, const Pieces<NB>& b, float4_t c) {
    constexpr int ORDERS = NA > NB ? NA : NB;
#pragma unroll
    for (int order = ORDERS - 1; order >= 0; --order)
#pragma unroll
        for (int i = 0; i <= order; ++i)
            if (i < NA && order - i < NB)
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[order - i], c, 0, 0, 0);
    return c;
}

// c[m][n] + A[m] B[n] for a grid of products, as mma: one product of pieces of all of them after the other, since the next
// on the same sum waits for the one before.
template <int NA, int NB, int R, int S>
__device__ __forceinline__ void mma_grid(const Pieces<NA> (&a)[R], const Pieces<NB> (&b)[S], float4_t (&c)[R][S]) {
    constexpr int ORDERS = NA > NB ? NA : NB;
#pragma unroll
    for (int order = ORDERS - 1; order >= 0; --order)
#pragma unroll
        for (int i = 0; i <= order; ++i)
            if (i < NA && order - i < NB)
#pragma unroll
                for (int m = 0; m < R; ++m)
#pragma unroll
                    for (int n = 0; n < S; ++n)
                        c[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m].p[i], b[n].p[order - i], c[m][n], 0, 0, 0);
}

// The same with the first pieces' products in `c` alone, the others in `small`: a sum over many operands is then rounded at its
// full size once for each of them, not once for each product of pieces.
template <int NA, int NB, int R, int S>
__device__ __forceinline__ void mma_grid(const Pieces<NA> (&a)[R], const Pieces<NB> (&b)[S], float4_t (&c)[R][S], float4_t (&small)[R][S]) {
    constexpr int ORDERS = NA > NB ? NA : NB;
#pragma unroll
    for (int order = ORDERS - 1; order >= 0; --order)
#pragma unroll
        for (int i = 0; i <= order; ++i)
            if (i < NA && order - i < NB)
#pragma unroll
                for (int m = 0; m < R; ++m)
#pragma unroll
                    for (int n = 0; n < S; ++n) {
                        float4_t& sum = order ? small[m][n] : c[m][n];
                        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m].p[i], b[n].p[order - i], sum, 0, 0, 0);
                    }
}

// c[m] + A[m] B[m], likewise.
template <int NA, int NB, int R>
__device__ __forceinline__ void mma_each(const Pieces<NA> (&a)[R], const Pieces<NB> (&b)[R], float4_t (&c)[R], float4_t (&small)[R]) {
    constexpr int ORDERS = NA > NB ? NA : NB;
#pragma unroll
    for (int order = ORDERS - 1; order >= 0; --order)
#pragma unroll
        for (int i = 0; i <= order; ++i)
            if (i < NA && order - i < NB)
#pragma unroll
                for (int m = 0; m < R; ++m) {
                    float4_t& sum = order ? small[m] : c[m];
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m].p[i], b[m].p[order - i], sum, 0, 0, 0);
                }
}

// c + A B in two chains, the smaller products apart from the larger: half the latency of mma.
template <int NA, int NB>
__device__ __forceinline__ void mma2(const Pieces<NA>& a, const Pieces<NB>& b, float4_t& large, float4_t& small) {
    constexpr int ORDERS = NA > NB ? NA : NB;
#pragma unroll
    for (int order = ORDERS - 1; order >= 0; --order)
#pragma unroll
        for (int i = 0; i <= order; ++i)
            if (i < NA && order - i < NB) {
                float4_t& c = order == ORDERS - 1 ? small : large;
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[order - i], c, 0, 0, 0);
            }
}

struct Lane {
    int id, col, quad;  // l, l % 16, 4 (l / 16)
    __device__ __forceinline__ Lane() : Lane(threadIdx.x) {}
    __device__ __forceinline__ explicit Lane(uint32_t thread) : id(thread % 64), col(thread % 16), quad(thread % 64 / 16 * 4) {}
};

// Operands in memory: N pieces, 16 bytes per lane each.
template <int N>
__device__ __forceinline__ Pieces<N> fetch(const bf16_t* p, i64 operand, const Lane& l) {
    Pieces<N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.p[i] = *(const bf16x8*)(p + ((operand * N + i) * 64 + l.id) * 8);
    return r;
}

template <int N>
__device__ __forceinline__ void put(bf16_t* p, i64 operand, const Lane& l, const Pieces<N>& v) {
#pragma unroll
    for (int i = 0; i < N; ++i) *(bf16x8*)(p + ((operand * N + i) * 64 + l.id) * 8) = v.p[i];
}

// Half `half` of an operand: its indices 16 half ...
template <int N>
__device__ __forceinline__ void put_half(bf16_t* p, i64 operand, int half, const Lane& l, const Halves<N>& v) {
#pragma unroll
    for (int i = 0; i < N; ++i) *(bf16x4*)(p + ((operand * N + i) * 64 + l.id) * 8 + 4 * half) = v.p[i];
}

// Keeps what stands before it before it.  A scan's loads return in the order of their issue, so one that the
// scheduler moves behind others is waited for together with them.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// Workgroup barrier for LDS alone: loads and stores of global memory stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
    in_order();
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    in_order();
}

}  // namespace atlas_ops
