// Orthogonalised weight updates: the quintic iteration towards the orthogonal factor of a matrix and
// the optimiser step around it.  Part of libatlas_ops_hip.so.
//
//   momentum <- f momentum + gradient,  u = gradient + f momentum (or the momentum itself)
//   X = u / (|u|_F + eps);  repeat: A = X X^T,  X <- a X + (b A + c A A) X
//   weight <- keep weight - rate X
//
// Each step raises the small singular values by a factor of about a, so rounding in X or A grows by
// a^steps (485 at the defaults) in the weakest directions: bfloat16 or float16 products lose them.  Every
// matrix of the iteration is therefore held as two float16 planes, v = (hi + lo / 2048) / 16, 22
// significant bits (the iterates' entries are below 1.5, so hi is normal down to 4e-6, and lo covers
// what is below), in the 4 bytes that a float32 takes.  A product of two such matrices is three
// float16 MFMAs, hi hi + (hi lo + lo hi) / 2048 with float32 sums; the dropped lo lo term is below
// 2^-22.  That is float32's accuracy at 1/3 of the float16 rate instead of the float32 MFMA's 1/16.
//
// Matrices with more rows than columns are transposed while they are split, so that A is the
// smaller of the two Gram matrices.  Both X and its transpose are kept: every product then has both
// operands contiguous along the sum.  A and b A + c A A are symmetric: only the tiles on and above the
// diagonal are computed, and written twice.
#include <algorithm>

#include "device/atlas_ops.h"

namespace atlas_ops {
namespace {

typedef _Float16 half_t;
typedef half_t half8_t __attribute__((ext_vector_type(8)));
typedef half_t half4_t __attribute__((ext_vector_type(4)));

constexpr float SCALE = 16.0f, LOW = 2048.0f;

__device__ __forceinline__ void split(float v, half_t& hi, half_t& lo) {
    const float s = v * SCALE;
    hi = (half_t)s;
    lo = (half_t)((s - (float)hi) * LOW);
}

__device__ __forceinline__ float join(half_t hi, half_t lo) { return ((float)hi + (float)lo * (1.0f / LOW)) * (1.0f / SCALE); }

struct Planes {
    half_t *hi, *lo;
    __device__ __forceinline__ Planes offset(i64 n) const { return {hi + n, lo + n}; }
};

// The matrix to orthogonalise, element (r, c) of batch b, and its momentum where there is one.
struct Source {
    const void* matrix;
    i64 rows, columns, batch_stride, row_stride;
    float* momentum;
    float factor;
    int nesterov;

    template <typename T>
    __device__ __forceinline__ float gradient(i64 b, i64 r, i64 c) const {
        return to_float(((const T*)matrix)[b * batch_stride + r * row_stride + c]);
    }
};

constexpr int PARTIALS = 256;  // blocks per matrix of the norm's sum

// Updates the momentum and adds the squares of u: block (i, b) visits the rows i, i + gridDim.x, ...
// The sum is held in 64 bits, where no square of a float32 overflows or vanishes.
template <typename T>
__global__ void __launch_bounds__(256) ortho_norm(Source s, double* __restrict__ partial) {
    __shared__ double sums[4];
    const i64 b = blockIdx.y, count = s.rows * s.columns;
    double total = 0.0;
    for (i64 e = (i64)blockIdx.x * 256 + threadIdx.x; e < count; e += (i64)gridDim.x * 256) {
        const float g = s.gradient<T>(b, e / s.columns, e % s.columns);
        float u = g;
        if (s.momentum) {
            float* m = s.momentum + b * count + e;
            const float next = s.factor * *m + g;
            *m = next;
            u = s.nesterov ? g + s.factor * next : next;
        }
        total += (double)u * (double)u;
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) total += __shfl_xor(total, d, 64);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = total;
    __syncthreads();
    if (threadIdx.x == 0) partial[b * PARTIALS + blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// X and its transpose as planes, zero beyond the matrix: one 64 x 64 tile of X per workgroup.
template <typename T>
__global__ void __launch_bounds__(256) ortho_split(Source s, int transposed, int parts,
                                                   const double* __restrict__ partial, float eps, i64 mp, i64 np,
                                                   Planes x, Planes xt) {
    __shared__ float tile[64][65];
    __shared__ double sums[4];
    const i64 b = blockIdx.z, count = s.rows * s.columns;
    double total = (int)threadIdx.x < parts ? partial[b * PARTIALS + threadIdx.x] : 0.0;
#pragma unroll
    for (int d = 32; d > 0; d /= 2) total += __shfl_xor(total, d, 64);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = total;
    __syncthreads();
    const double scale = 1.0 / (sqrt((sums[0] + sums[1]) + (sums[2] + sums[3])) + (double)eps);
    // the tile in the matrix's own orientation: (r0, c0) in rows and columns of the source
    const i64 i0 = (i64)blockIdx.y * 64, j0 = (i64)blockIdx.x * 64;
    const i64 r0 = transposed ? j0 : i0, c0 = transposed ? i0 : j0;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    for (int k = wave; k < 64; k += 4) {
        const i64 r = r0 + k, c = c0 + lane;
        float u = 0.0f;
        if (r < s.rows && c < s.columns) {
            u = s.gradient<T>(b, r, c);
            if (s.momentum) {
                const float m = s.momentum[b * count + r * s.columns + c];
                u = s.nesterov ? u + s.factor * m : m;
            }
        }
        tile[k][lane] = (float)((double)u * scale);
    }
    __syncthreads();
    const Planes a = x.offset(b * mp * np), t = xt.offset(b * mp * np);
    for (int k = wave; k < 64; k += 4) {
        half_t hi, lo;
        split(transposed ? tile[lane][k] : tile[k][lane], hi, lo);
        a.hi[(i0 + k) * np + j0 + lane] = hi;
        a.lo[(i0 + k) * np + j0 + lane] = lo;
        split(transposed ? tile[k][lane] : tile[lane][k], hi, lo);
        t.hi[(j0 + k) * mp + i0 + lane] = hi;
        t.lo[(j0 + k) * mp + i0 + lane] = lo;
    }
}

// What becomes of a tile of products P = Left Right^T.
enum Product {
    GRAM,   // symmetric: out = P
    POLY,   // symmetric: out = b in + c P
    APPLY,  // out and its transpose = a in + P
    FINAL   // the result, a in + P, to the caller
};

struct Result {
    i64 rows, columns;
    void* out;      // or NULL:
    float* weight;  // weight <- keep weight - rate X
    int out_type, transposed;
    float keep, rate;
};

constexpr int DEPTH = 32;           // sum indices per stage: one MFMA's depth
constexpr int PITCH = DEPTH + 8;    // of an LDS row in halves: 16 rows' 16-byte reads hit all banks once

// A TILE x TILE tile of Left (rows x depth) Right^T (depth x columns), both planes contiguous along
// the sum.  Four waves, each a quarter tile of 16 x 16 MFMA blocks; the two operands' planes of
// the next 32 sum indices travel through registers while the current ones are multiplied out of LDS.
template <int TILE, Product WHAT>
__global__ void __launch_bounds__(256) ortho_product(Planes left, i64 left_stride, Planes right, i64 right_stride,
                                                     i64 depth, Planes in, Planes out, Planes out_t, i64 rows,
                                                     i64 columns, float direct, float product, Result result) {
    constexpr int F = TILE / 32;       // blocks per wave and side
    constexpr int LOADS = TILE / 64;   // 16-byte loads per thread, plane and stage
    __shared__ __attribute__((aligned(16))) half_t lds[2][4][TILE * PITCH];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, wi = wave / 2, wj = wave % 2;
    const i64 b = blockIdx.z;
    i64 ti, tj;
    if constexpr (WHAT == GRAM || WHAT == POLY) {
        // tile t of the upper triangle: column tj has tj + 1 tiles
        const int t = blockIdx.x;
        int j = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
        while ((j + 1) * (j + 2) / 2 <= t) ++j;
        while (j * (j + 1) / 2 > t) --j;
        tj = j;
        ti = t - j * (j + 1) / 2;
    } else {
        ti = blockIdx.x % (rows / TILE);
        tj = blockIdx.x / (rows / TILE);
    }
    const half_t* sources[4] = {left.hi + b * left_stride + ti * TILE * depth, left.lo + b * left_stride + ti * TILE * depth,
                                right.hi + b * right_stride + tj * TILE * depth,
                                right.lo + b * right_stride + tj * TILE * depth};
    const int lrow = threadIdx.x / 4, lcol = threadIdx.x % 4 * 8;
    half8_t next[4][LOADS];
    auto fetch = [&](i64 k0) {
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
            for (int q = 0; q < LOADS; ++q)
                next[p][q] = *(const half8_t*)(sources[p] + (i64)(lrow + 64 * q) * depth + k0 + lcol);
    };
    auto stage = [&](int buffer) {
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
            for (int q = 0; q < LOADS; ++q) *(half8_t*)&lds[buffer][p][(lrow + 64 * q) * PITCH + lcol] = next[p][q];
    };
    float4_t main[F][F], cross[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) main[i][j] = cross[i][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    fetch(0);
    stage(0);
    __syncthreads();
    const i64 stages = depth / DEPTH;
    for (i64 k = 0; k < stages; ++k) {
        const int buffer = (int)(k & 1);
        if (k + 1 < stages) fetch((k + 1) * DEPTH);
        half8_t a[2][F], c[2][F];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int i = 0; i < F; ++i) {
                a[p][i] = *(const half8_t*)&lds[buffer][p][(wi * (TILE / 2) + 16 * i + lane % 16) * PITCH + lane / 16 * 8];
                c[p][i] = *(const half8_t*)&lds[buffer][2 + p][(wj * (TILE / 2) + 16 * i + lane % 16) * PITCH + lane / 16 * 8];
            }
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) {
                main[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0][i], c[0][j], main[i][j], 0, 0, 0);
                cross[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0][i], c[1][j], cross[i][j], 0, 0, 0);
                cross[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[1][i], c[0][j], cross[i][j], 0, 0, 0);
            }
        // the other buffer was read in the stage before this one, which every wave has left
        if (k + 1 < stages) stage(buffer ^ 1);
        __syncthreads();
    }
    const i64 area = b * rows * columns;
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) {
            // lane: rows r .. r + 3 of column c
            const i64 r = ti * TILE + wi * (TILE / 2) + 16 * i + lane / 16 * 4;
            const i64 c = tj * TILE + wj * (TILE / 2) + 16 * j + lane % 16;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = product * (main[i][j][e] + cross[i][j][e] * (1.0f / LOW)) * (1.0f / (SCALE * SCALE));
            // `in` is read at (c, r .. r + 3): the symmetric matrix, or the transpose of X
            if constexpr (WHAT != GRAM) {
                const half4_t hi = *(const half4_t*)(in.hi + area + c * rows + r), lo = *(const half4_t*)(in.lo + area + c * rows + r);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += direct * join(hi[e], lo[e]);
            }
            if constexpr (WHAT == FINAL) {
                for (int e = 0; e < 4; ++e) {
                    const i64 orow = result.transposed ? c : r + e, ocol = result.transposed ? r + e : c;
                    if (orow >= result.rows || ocol >= result.columns) continue;
                    const i64 at = b * result.rows * result.columns + orow * result.columns + ocol;
                    if (!result.out) result.weight[at] = result.keep * result.weight[at] - result.rate * v[e];
                    else if (result.out_type == ATLAS_OPS_F32) ((float*)result.out)[at] = v[e];
                    else ((bf16_t*)result.out)[at] = from_float<bf16_t>(v[e]);
                }
            } else {
                half4_t hi, lo;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    half_t h, l;
                    split(v[e], h, l);
                    hi[e] = h;
                    lo[e] = l;
                    out.hi[area + (r + e) * columns + c] = h;
                    out.lo[area + (r + e) * columns + c] = l;
                }
                // the mirror image of a symmetric matrix, or the transpose of X
                if (WHAT == APPLY || ti != tj) {
                    *(half4_t*)(out_t.hi + area + c * rows + r) = hi;
                    *(half4_t*)(out_t.lo + area + c * rows + r) = lo;
                }
            }
        }
}

struct Sizes {
    i64 m, n, mp, np;  // m <= n: the sides of X, and padded to whole tiles
    int tile, transposed;
};

Sizes sizes_of(i64 batch, i64 rows, i64 columns) {
    Sizes s{};
    s.transposed = rows > columns;
    s.m = std::min(rows, columns);
    s.n = std::max(rows, columns);
    // tiles of 128 reuse each operand twice as often; below a tile per CU in every product, 64 spread the work
    const i64 t = ceil_div(s.m, 128);
    s.tile = batch * t * (t + 1) / 2 >= 128 ? 128 : 64;
    s.mp = ceil_div(s.m, s.tile) * s.tile;
    s.np = ceil_div(s.n, s.tile) * s.tile;
    return s;
}

struct Buffers {
    double* partial;
    Planes x, xt[2], gram, poly;
    i64 bytes;
};

// Carves the workspace: the partial sums, then two planes for each matrix.
Buffers carve(const Sizes& s, i64 batch, char* base) {
    Buffers w{};
    i64 at = batch * PARTIALS * (i64)sizeof(double);
    w.partial = (double*)base;
    auto planes = [&](i64 count) {
        Planes p{(half_t*)(base + at), (half_t*)(base + at + 2 * batch * count)};
        at += 4 * batch * count;
        return p;
    };
    w.x = planes(s.mp * s.np);
    w.xt[0] = planes(s.mp * s.np);
    w.xt[1] = planes(s.mp * s.np);
    w.gram = planes(s.mp * s.mp);
    w.poly = planes(s.mp * s.mp);
    w.bytes = at;
    return w;
}

template <int TILE>
void iterate(const Sizes& s, const Buffers& w, i64 batch, int steps, const float* k, const Result& result, hipStream_t st) {
    const i64 t = s.mp / TILE, wide = s.mp * s.np, square = s.mp * s.mp;
    const dim3 triangle((unsigned)(t * (t + 1) / 2), 1, (unsigned)batch), whole((unsigned)(t * (s.np / TILE)), 1, (unsigned)batch);
    const Planes none{nullptr, nullptr};
    int from = 0;
    for (int i = 0; i < steps; ++i) {
        ortho_product<TILE, GRAM><<<triangle, 256, 0, st>>>(w.x, wide, w.x, wide, s.np, none, w.gram, w.gram, s.mp, s.mp,
                                                            0.0f, 1.0f, result);
        ortho_product<TILE, POLY><<<triangle, 256, 0, st>>>(w.gram, square, w.gram, square, s.mp, w.gram, w.poly, w.poly,
                                                            s.mp, s.mp, k[1], k[2], result);
        if (i + 1 < steps)
            ortho_product<TILE, APPLY><<<whole, 256, 0, st>>>(w.poly, square, w.xt[from], wide, s.mp, w.xt[from], w.x,
                                                              w.xt[from ^ 1], s.mp, s.np, k[0], 1.0f, result);
        else
            ortho_product<TILE, FINAL><<<whole, 256, 0, st>>>(w.poly, square, w.xt[from], wide, s.mp, w.xt[from], none,
                                                              none, s.mp, s.np, k[0], 1.0f, result);
        from ^= 1;
    }
}

}  // namespace
}  // namespace atlas_ops

using namespace atlas_ops;

extern "C" {

int64_t atlas_ops_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t columns) {
    if (batch < 1 || rows < 1 || columns < 1) return 0;
    return carve(sizes_of(batch, rows, columns), batch, nullptr).bytes;
}

int atlas_ops_orthogonalize(const AtlasOrthogonal* o, void* workspace, void* stream, char* err, size_t cap) {
    try {
        if (!o || !o->matrix || !workspace || (!o->out) == (!o->weight)) return fail(err, cap, 7, "null argument");
        if (o->batch < 1 || o->batch > 65535 || o->rows < 1 || o->columns < 1 || o->rows > (1 << 20) ||
            o->columns > (1 << 20))
            return fail(err, cap, 7, "batch must be 1 to 65535, rows and columns 1 to 2^20");
        if (o->steps < 1 || o->steps > 64) return fail(err, cap, 7, "steps must be 1 to 64");
        if (!known_type(o->type) || (o->out && !known_type(o->out_type))) return fail(err, cap, 7, "unknown type");
        const Sizes s = sizes_of(o->batch, o->rows, o->columns);
        if (s.mp > 16384) return fail(err, cap, 7, "the smaller side must be at most 16384");
        const Buffers w = carve(s, o->batch, (char*)workspace);
        hipStream_t st = (hipStream_t)stream;
        const Source source{o->matrix, o->rows, o->columns, o->batch_stride, o->row_stride, o->momentum, o->factor, o->nesterov};
        // a block of the norm's sum takes 4096 values or more
        const int parts = (int)std::min<i64>(PARTIALS, ceil_div(o->rows * o->columns, 4096));
        const dim3 norm_grid((unsigned)parts, (unsigned)o->batch);
        const dim3 split_grid((unsigned)(s.np / 64), (unsigned)(s.mp / 64), (unsigned)o->batch);
        if (o->type == ATLAS_OPS_F32) {
            ortho_norm<float><<<norm_grid, 256, 0, st>>>(source, w.partial);
            ortho_split<float><<<split_grid, 256, 0, st>>>(source, s.transposed, parts, w.partial, o->eps, s.mp, s.np, w.x, w.xt[0]);
        } else {
            ortho_norm<bf16_t><<<norm_grid, 256, 0, st>>>(source, w.partial);
            ortho_split<bf16_t><<<split_grid, 256, 0, st>>>(source, s.transposed, parts, w.partial, o->eps, s.mp, s.np, w.x, w.xt[0]);
        }
        const Result result{o->rows, o->columns, o->out, o->weight, o->out_type, s.transposed, o->keep, o->rate};
        if (s.tile == 128) iterate<128>(s, w, o->batch, o->steps, o->coefficients, result, st);
        else iterate<64>(s, w, o->batch, o->steps, o->coefficients, result, st);
        return launched(err, cap, "orthogonalize");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

}  // extern "C"
