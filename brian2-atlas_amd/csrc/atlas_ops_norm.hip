// Layer normalisation, forward and backward, with the reduction of the weight's and bias's
// gradients.  Part of libatlas_ops_hip.so.
//
//   z = (x - mean) rstd,  y = z w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (h - mean(h) - z mean(h z)),  h = g w;   dw = sum_rows g z,  db = sum_rows g
//
// Memory bounds all of it: a row is read once into registers, its mean m and then the squares of its
// centred values are summed from there (no cancellation, unlike E[x^2] - mean^2), and the result is
// written.  With the squares goes the sum of the centred values, whose mean r is what rounding left
// out of m: the row is centred by m + r, its variance is mean((x - m)^2) - r^2, and a mean thousands of
// times the deviation costs no accuracy.  The backward pass gets m rounded and finds r again among its
// own sums.  The backward pass reads x and g once: each lane keeps the same columns of
// every row its group visits, so the column sums of dw and db stay in registers over the rows, a
// workgroup adds its groups' sums in LDS and writes one row of partials, and a second kernel adds
// the partials in a fixed order (no atomics: the same bits every time).
#include <algorithm>

#include "device/atlas_ops.h"

namespace atlas_ops {
namespace {

// A lane's unit of a row: 16 bytes.  Rows need no alignment beyond their element's: gfx950 takes
// unaligned vector accesses, and 2-byte accesses for odd widths would need eight times the
// instructions.
template <typename T>
struct Unit {
    static constexpr int N = 16 / sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Raw { T v[N]; };
};

template <typename T, int N = Unit<T>::N>
__device__ __forceinline__ void load_unit(const T* p, i64 left, float* out) {
    if (left >= N) {
        typename Unit<T>::Raw raw;
        __builtin_memcpy(&raw, p, sizeof(raw));
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = to_float(raw.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = i < left ? to_float(p[i]) : 0.0f;
    }
}

template <typename T, int N = Unit<T>::N>
__device__ __forceinline__ void store_unit(T* p, i64 left, const float* v) {
    if (left >= N) {
        typename Unit<T>::Raw raw;
#pragma unroll
        for (int i = 0; i < N; ++i) raw.v[i] = from_float<T>(v[i]);
        __builtin_memcpy(p, &raw, sizeof(raw));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = from_float<T>(v[i]);
    }
}

// N values of the weight or bias from column c: W is float or T.
template <typename W, int N>
__device__ __forceinline__ void load_columns(const W* p, i64 left, float fallback, float* out) {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = p && i < left ? to_float(p[i]) : fallback;
}

struct Rows {
    const void* data;
    i64 inner, outer_stride, inner_stride;
    template <typename T>
    __device__ __forceinline__ const T* at(i64 r) const {
        const i64 o = inner_stride * (r < inner ? r : r % inner) + (r < inner ? 0 : outer_stride * (r / inner));
        return (const T*)data + o;
    }
};

// Sums of K values over a row's group: LANES lanes of one wave, or (LANES = 256) the workgroup.
template <int LANES, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* shared) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lane_sum<LANES <= 64 ? LANES : 64>(v[k]);
    if constexpr (LANES > 64) {
        __syncthreads();  // the previous use of `shared` is read
        if (threadIdx.x % 64 == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) shared[4 * k + threadIdx.x / 64] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = (shared[4 * k] + shared[4 * k + 1]) + (shared[4 * k + 2] + shared[4 * k + 3]);
    }
}

// The residual of the mean and 1 / sqrt(variance + eps) from the means of the centred values and of
// their squares.
struct Spread {
    float residual, rstd;
    __device__ __forceinline__ Spread(float centred, float squares, float eps) : residual(centred) {
        const float variance = squares - centred * centred;
        rstd = 1.0f / sqrtf((variance < 0.0f ? 0.0f : variance) + eps);  // a NaN stays one
    }
};

// One row per group of LANES lanes; lane l holds units l, l + LANES, ... (CH of them).
template <typename T, typename W, int LANES, int CH>
__global__ void __launch_bounds__(256) norm_forward(Rows x, i64 rows, i64 width, const W* __restrict__ weight,
                                                    const W* __restrict__ bias, float eps, T* __restrict__ y,
                                                    float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int N = Unit<T>::N, GROUPS = 256 / LANES;
    __shared__ float shared[12];
    const int lane = threadIdx.x % LANES;
    const i64 row = (i64)blockIdx.x * GROUPS + threadIdx.x / LANES;
    if (LANES <= 64 && row >= rows) return;  // the grid of whole workgroups per row has no spare rows
    const T* src = x.at<T>(row);
    float v[CH][N];
    float sum[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const i64 col = (i64)(lane + c * LANES) * N;
        load_unit<T>(src + col, width - col, v[c]);
#pragma unroll
        for (int i = 0; i < N; ++i) sum[0] += v[c][i];
    }
    group_sum<LANES>(sum, shared);
    const float mean = sum[0] / (float)width;
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const i64 left = width - (i64)(lane + c * LANES) * N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[c][i] -= mean;
            if (i < left) {
                sums[0] += v[c][i];
                sums[1] += v[c][i] * v[c][i];
            }
        }
    }
    group_sum<LANES>(sums, shared);
    const Spread s(sums[0] / (float)width, sums[1] / (float)width, eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const i64 col = (i64)(lane + c * LANES) * N, left = width - col;
        if (left <= 0) continue;
        float w[N], b[N];
        load_columns<W, N>(weight ? weight + col : nullptr, left, 1.0f, w);
        load_columns<W, N>(bias ? bias + col : nullptr, left, 0.0f, b);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = (v[c][i] - s.residual) * s.rstd * w[i] + b[i];
        store_unit<T>(y + row * width + col, left, w);
    }
    if (mean_out && lane == 0) {
        mean_out[row] = mean + s.residual;
        rstd_out[row] = s.rstd;
    }
}

// Rows that do not fit the registers of a workgroup: three reads, the later two from the caches.
template <typename T, typename W>
__global__ void __launch_bounds__(256) norm_forward_long(Rows x, i64 width, const W* __restrict__ weight,
                                                         const W* __restrict__ bias, float eps, T* __restrict__ y,
                                                         float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int N = Unit<T>::N;
    __shared__ float shared[12];
    const i64 row = blockIdx.x;
    const T* src = x.at<T>(row);
    float v[N], sum[1] = {0.0f}, sums[2] = {0.0f, 0.0f};
    for (i64 col = (i64)threadIdx.x * N; col < width; col += 256 * N) {
        load_unit<T>(src + col, width - col, v);
#pragma unroll
        for (int i = 0; i < N; ++i) sum[0] += v[i];
    }
    group_sum<256>(sum, shared);
    const float mean = sum[0] / (float)width;
    for (i64 col = (i64)threadIdx.x * N; col < width; col += 256 * N) {
        load_unit<T>(src + col, width - col, v);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col + i < width) {
                sums[0] += v[i] - mean;
                sums[1] += (v[i] - mean) * (v[i] - mean);
            }
    }
    group_sum<256>(sums, shared);
    const Spread s(sums[0] / (float)width, sums[1] / (float)width, eps);
    for (i64 col = (i64)threadIdx.x * N; col < width; col += 256 * N) {
        float w[N], b[N];
        load_unit<T>(src + col, width - col, v);
        load_columns<W, N>(weight ? weight + col : nullptr, width - col, 1.0f, w);
        load_columns<W, N>(bias ? bias + col : nullptr, width - col, 0.0f, b);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = (v[i] - mean - s.residual) * s.rstd * w[i] + b[i];
        store_unit<T>(y + row * width + col, width - col, w);
    }
    if (mean_out && threadIdx.x == 0) {
        mean_out[row] = mean + s.residual;
        rstd_out[row] = s.rstd;
    }
}

// Group j of the grid visits rows j, j + groups, ...; partials: block b's sums of dw at
// partial[b * 2 * width], of db right after them.
template <typename T, typename W, int LANES, int CH>
__global__ void __launch_bounds__(256) norm_backward(Rows grad, Rows x, i64 rows, i64 width,
                                                     const W* __restrict__ weight, const float* __restrict__ mean_in,
                                                     const float* __restrict__ rstd_in, T* __restrict__ dx,
                                                     float* __restrict__ partial) {
    constexpr int N = Unit<T>::N, GROUPS = 256 / LANES;
    __shared__ float shared[12];
    extern __shared__ float columns[];  // GROUPS > 1: the groups' column sums, one group after the other
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    float w[CH][N], dw[CH][N], db[CH][N];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const i64 col = (i64)(lane + c * LANES) * N;
        load_columns<W, N>(weight ? weight + col : nullptr, width - col, 1.0f, w[c]);
#pragma unroll
        for (int i = 0; i < N; ++i) dw[c][i] = db[c][i] = 0.0f;
    }
    const i64 stride = (i64)gridDim.x * GROUPS;
    for (i64 row = (i64)blockIdx.x * GROUPS + group; row < rows; row += stride) {
        const T *gp = grad.at<T>(row), *xp = x.at<T>(row);
        const float mean = mean_in[row], rstd = rstd_in[row];
        float g[CH][N], z[CH][N];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const i64 col = (i64)(lane + c * LANES) * N, left = width - col;
            load_unit<T>(gp + col, left, g[c]);
            load_unit<T>(xp + col, left, z[c]);
        }
        float sums[3] = {0.0f, 0.0f, 0.0f};  // of h, h z and z
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const i64 left = width - (i64)(lane + c * LANES) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                z[c][i] = i < left ? (z[c][i] - mean) * rstd : 0.0f;
                const float h = g[c][i] * w[c][i];
                sums[0] += h;
                sums[1] += h * z[c][i];
                sums[2] += z[c][i];
            }
        }
        group_sum<LANES>(sums, shared);
        const float residual = sums[2] / (float)width, sum = sums[0] / (float)width;
        const float dot = sums[1] / (float)width - residual * sum;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const i64 col = (i64)(lane + c * LANES) * N, left = width - col;
            if (left <= 0) continue;
            float d[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float centred = z[c][i] - residual;
                dw[c][i] += g[c][i] * centred;
                db[c][i] += g[c][i];
                d[i] = rstd * (g[c][i] * w[c][i] - sum - centred * dot);
            }
            store_unit<T>(dx + row * width + col, left, d);
        }
    }
    if (!partial) return;
    float* out = partial + (i64)blockIdx.x * 2 * width;
    if constexpr (GROUPS > 1) {
        constexpr int SPAN = LANES * CH * N;  // columns a group holds
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            if (half) __syncthreads();
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    columns[group * SPAN + (lane + c * LANES) * N + i] = half ? db[c][i] : dw[c][i];
            __syncthreads();
            for (int col = threadIdx.x; col < SPAN && col < width; col += 256) {
                float total = 0.0f;
#pragma unroll
                for (int k = 0; k < GROUPS; ++k) total += columns[k * SPAN + col];
                out[half * width + col] = total;
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const i64 col = (i64)(lane + c * LANES) * N;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (col + i < width) {
                    out[col + i] = dw[c][i];
                    out[width + col + i] = db[c][i];
                }
        }
    }
}

// Long rows: the two means of every row, dx in a second read; the column sums come from
// norm_columns.
template <typename T, typename W>
__global__ void __launch_bounds__(256) norm_backward_long(Rows grad, Rows x, i64 width, const W* __restrict__ weight,
                                                          const float* __restrict__ mean_in,
                                                          const float* __restrict__ rstd_in, T* __restrict__ dx,
                                                          float* __restrict__ residuals) {
    constexpr int N = Unit<T>::N;
    __shared__ float shared[12];
    const i64 row = blockIdx.x;
    const T *gp = grad.at<T>(row), *xp = x.at<T>(row);
    const float mean = mean_in[row], rstd = rstd_in[row];
    float g[N], z[N], w[N], sums[3] = {0.0f, 0.0f, 0.0f}, sum = 0.0f, dot = 0.0f, residual = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {
        for (i64 col = (i64)threadIdx.x * N; col < width; col += 256 * N) {
            const i64 left = width - col;
            load_unit<T>(gp + col, left, g);
            load_unit<T>(xp + col, left, z);
            load_columns<W, N>(weight ? weight + col : nullptr, left, 1.0f, w);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                z[i] = i < left ? (z[i] - mean) * rstd : 0.0f;
                g[i] *= w[i];
                if (pass) {
                    g[i] = rstd * (g[i] - sum - (z[i] - residual) * dot);
                } else {
                    sums[0] += g[i];
                    sums[1] += g[i] * z[i];
                    sums[2] += z[i];
                }
            }
            if (pass) store_unit<T>(dx + row * width + col, left, g);
        }
        if (!pass) {
            group_sum<256>(sums, shared);
            sum = sums[0] / (float)width;
            residual = sums[2] / (float)width;
            dot = sums[1] / (float)width - residual * sum;
            if (residuals && threadIdx.x == 0) residuals[row] = residual;
        }
    }
}

// Column sums of long rows: block (i, b) adds the rows b, b + blocks, ... of 256 columns.
template <typename T>
__global__ void __launch_bounds__(256) norm_columns(Rows grad, Rows x, i64 rows, i64 width,
                                                    const float* __restrict__ mean_in,
                                                    const float* __restrict__ rstd_in,
                                                    const float* __restrict__ residuals, float* __restrict__ partial) {
    const i64 col = (i64)blockIdx.x * 256 + threadIdx.x;
    if (col >= width) return;
    float dw = 0.0f, db = 0.0f;
#pragma unroll 4
    for (i64 row = blockIdx.y; row < rows; row += gridDim.y) {
        const float g = to_float(grad.at<T>(row)[col]), v = to_float(x.at<T>(row)[col]);
        dw += g * ((v - mean_in[row]) * rstd_in[row] - residuals[row]);
        db += g;
    }
    partial[(i64)blockIdx.y * 2 * width + col] = dw;
    partial[(i64)blockIdx.y * 2 * width + width + col] = db;
}

// Adds the blocks' partials: 32 columns of the 2 x width sums per workgroup, its 32 row groups
// added in LDS in a fixed order.
template <typename W>
__global__ void __launch_bounds__(1024) norm_reduce(i64 blocks, i64 width, const float* __restrict__ partial,
                                                    W* __restrict__ dweight, W* __restrict__ dbias) {
    __shared__ float sums[32][33];
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
    const i64 col = (i64)blockIdx.x * 32 + lane;
    float total = 0.0f;
    if (col < 2 * width) {
#pragma unroll 8
        for (i64 b = group; b < blocks; b += 32) total += partial[b * 2 * width + col];
    }
    sums[group][lane] = total;
    __syncthreads();
    if (group == 0 && col < 2 * width) {
        total = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; ++k) total += sums[k][lane];
        W* out = col < width ? dweight : dbias;
        if (out) out[col < width ? col : col - width] = from_float<W>(total);
    }
}

// The layout of a row by its width: 16 lanes up to 16 units (16 rows per workgroup), a wave up to
// 4 units per lane, a workgroup up to 4 (bfloat16) or 8 (float32) units per lane, else the long kernels.
struct Shape {
    int lanes, chunks;  // chunks 0: long rows
};

Shape shape_of(i64 width, int type) {
    const i64 units = ceil_div(width, type == ATLAS_OPS_F32 ? 4 : 8);
    if (units <= 16) return {16, 1};
    for (int c : {1, 2, 4})
        if (units <= 64 * c) return {64, c};
    for (int c : {2, 4, 8})
        if (units <= 256 * c && (c < 8 || type == ATLAS_OPS_F32)) return {256, c};
    return {256, 0};
}

template <typename F>
void with_shape(Shape s, F&& f) {
    if (s.lanes == 16) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    else if (s.lanes == 64 && s.chunks == 1) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (s.lanes == 64 && s.chunks == 2) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (s.lanes == 64) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    else if (s.chunks == 2) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (s.chunks == 4) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
}

template <typename F>
void with_types(int type, int weight_type, F&& f) {
    if (type == ATLAS_OPS_F32) f(0.0f, 0.0f);
    else if (weight_type == ATLAS_OPS_F32) f(bf16_t{}, 0.0f);
    else f(bf16_t{}, bf16_t{});
}

// Blocks of the backward pass's rows: a few workgroups per CU, so that the partials stay a small
// share of the traffic.
i64 row_blocks(i64 rows, i64 width, int type) {
    const Shape s = shape_of(width, type);
    if (s.chunks == 0) return std::min<i64>(rows, 64);
    return std::min<i64>(ceil_div(rows, 256 / s.lanes), s.lanes == 256 ? 512 : 1024);
}

bool usable(const AtlasRows* r) { return r && r->data && r->inner > 0; }

int check(const AtlasRows* x, i64 rows, i64 width, int type, int weight_type, char* err, size_t cap) {
    if (rows < 0 || rows > 0x7FFFFFFF || width < 1 || width > 0x7FFFFFFF)
        return fail(err, cap, 7, "rows and width must be below 2^31, width positive");
    if (!known_type(type) || !known_type(weight_type) || (type == ATLAS_OPS_F32 && weight_type != ATLAS_OPS_F32))
        return fail(err, cap, 7, "weight must be float32 or have the rows' type");
    if (rows && !usable(x)) return fail(err, cap, 7, "null rows");
    return 0;
}

}  // namespace
}  // namespace atlas_ops

using namespace atlas_ops;

extern "C" {

int atlas_ops_layer_norm(const AtlasRows* x, int64_t rows, int64_t width, int type, const void* weight, const void* bias,
                         int weight_type, float eps, void* y, float* mean, float* rstd, void* stream, char* err,
                         size_t cap) {
    try {
        if (int rc = check(x, rows, width, type, weight_type, err, cap)) return rc;
        if (!rows) return 0;
        if (!y || (mean == nullptr) != (rstd == nullptr)) return fail(err, cap, 7, "null output");
        const Shape shape = shape_of(width, type);
        const Rows in{x->data, x->inner, x->outer_stride, x->inner_stride};
        with_types(type, weight_type, [&](auto t, auto w) {
            using T = decltype(t);
            using W = decltype(w);
            if (shape.chunks == 0) {
                norm_forward_long<T, W><<<dim3((unsigned)rows), 256, 0, (hipStream_t)stream>>>(
                    in, width, (const W*)weight, (const W*)bias, eps, (T*)y, mean, rstd);
                return;
            }
            with_shape(shape, [&](auto lanes, auto chunks) {
                norm_forward<T, W, lanes(), chunks()>
                    <<<dim3((unsigned)ceil_div(rows, 256 / lanes())), 256, 0, (hipStream_t)stream>>>(
                        in, rows, width, (const W*)weight, (const W*)bias, eps, (T*)y, mean, rstd);
            });
        });
        return launched(err, cap, "layer_norm");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

int64_t atlas_ops_layer_norm_workspace(int64_t rows, int64_t width, int type) {
    if (rows < 1 || width < 1 || !known_type(type)) return 0;
    // the partial sums, and of long rows what their means left out
    return (2 * row_blocks(rows, width, type) * width + (shape_of(width, type).chunks ? 0 : rows)) * (i64)sizeof(float);
}

int atlas_ops_layer_norm_backward(const AtlasRows* grad, const AtlasRows* x, int64_t rows, int64_t width, int type,
                                  const void* weight, int weight_type, const float* mean, const float* rstd, void* dx,
                                  void* dweight, void* dbias, float* workspace, void* stream, char* err, size_t cap) {
    try {
        if (int rc = check(x, rows, width, type, weight_type, err, cap)) return rc;
        const bool sums = dweight || dbias;
        if (rows && (!usable(grad) || !mean || !rstd || !dx || (sums && !workspace)))
            return fail(err, cap, 7, "null argument");
        const i64 blocks = rows ? row_blocks(rows, width, type) : 0;
        hipStream_t st = (hipStream_t)stream;
        with_types(type, weight_type, [&](auto t, auto w) {
            using T = decltype(t);
            using W = decltype(w);
            if (rows) {
                const Shape shape = shape_of(width, type);
                const Rows in{x->data, x->inner, x->outer_stride, x->inner_stride};
                const Rows g{grad->data, grad->inner, grad->outer_stride, grad->inner_stride};
                if (shape.chunks == 0) {
                    norm_backward_long<T, W><<<dim3((unsigned)rows), 256, 0, st>>>(g, in, width, (const W*)weight, mean,
                                                                                  rstd, (T*)dx,
                                                                                  sums ? workspace + 2 * blocks * width : nullptr);
                    if (sums)
                        norm_columns<T><<<dim3((unsigned)ceil_div(width, 256), (unsigned)blocks), 256, 0, st>>>(
                            g, in, rows, width, mean, rstd, workspace + 2 * blocks * width, workspace);
                } else {
                    with_shape(shape, [&](auto lanes, auto chunks) {
                        const size_t lds = lanes() < 256 ? 256 * chunks() * Unit<T>::N * sizeof(float) : 0;
                        norm_backward<T, W, lanes(), chunks()><<<dim3((unsigned)blocks), 256, lds, st>>>(
                            g, in, rows, width, (const W*)weight, mean, rstd, (T*)dx, sums ? workspace : nullptr);
                    });
                }
            }
            if (sums)
                norm_reduce<W><<<dim3((unsigned)ceil_div(2 * width, 32)), 1024, 0, st>>>(
                    blocks, width, workspace, (W*)dweight, (W*)dbias);
        });
        return launched(err, cap, "layer_norm_backward");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

}  // extern "C"
