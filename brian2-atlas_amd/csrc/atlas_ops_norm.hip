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

#include "device/atlas_rows.h"

namespace atlas_ops {
namespace {

// The residual of the mean and 1 / sqrt(variance + eps) from the means of the centred values and of
// their squares.
struct Spread {
    float residual, rstd;
    __device__ __forceinline__ Spread(float centred, float squares, float eps) : residual(centred) {
        const float variance = squares - centred * centred;
        rstd = 1.0f / sqrtf((variance < 0.0f ? 0.0f : variance) + eps);  // a NaN stays one
    }
};

// 32768 x 4096 bfloat16 take 135 us, 4.0 TB/s of what is read and written, and 25600 x 256 float32 13.8 us, 3.8 TB/s
// (a large copy: 5.2); 256 x 256, launch and latency, 3.5 us.
//
// One row at a time per group of LANES lanes; lane l holds units l, l + LANES, ... (CH of them), and the same
// columns of the weight and bias for all its rows.
template <typename T, typename W, int LANES, int CH>
__global__ void __launch_bounds__(256) norm_forward(Rows x, i64 rows, int width, const W* __restrict__ weight,
                                                    const W* __restrict__ bias, float eps, T* __restrict__ y,
                                                    float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int N = Unit<T>::N, GROUPS = 256 / LANES;
    __shared__ float shared[12];
    const int lane = threadIdx.x % LANES;
    const i64 first = (i64)blockIdx.x * GROUPS + threadIdx.x / LANES, stride = (i64)gridDim.x * GROUPS;
    if (first >= rows) return;  // never a part of a workgroup that has barriers: its rows are whole workgroups
    float w[CH][N], b[CH][N];
    Unit<T> unit[CH];
    auto fetch = [&](i64 row) {
        const T* src = x.at<T>(row);
#pragma unroll
        for (int c = 0; c < CH; ++c) unit[c].load(src, (lane + c * LANES) * N, width);
    };
    fetch(first);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        load_columns<W, N>(weight, (lane + c * LANES) * N, width, 1.0f, w[c]);
        load_columns<W, N>(bias, (lane + c * LANES) * N, width, 0.0f, b[c]);
    }
    for (i64 row = first; row < rows; row += stride) {
        float v[CH][N];
        float sum[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[c][i] = unit[c][i];
                sum[0] += v[c][i];
            }
        if (row + stride < rows) fetch(row + stride);
        group_sum<LANES>(sum, shared);
        const float mean = sum[0] / (float)width;
        float sums[2] = {0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int left = width - (lane + c * LANES) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[c][i] = i < left ? v[c][i] - mean : 0.0f;
                sums[0] += v[c][i];
                sums[1] += v[c][i] * v[c][i];
            }
        }
        group_sum<LANES>(sums, shared);
        const Spread s(sums[0] / (float)width, sums[1] / (float)width, eps);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (lane + c * LANES) * N, left = width - col;
            if (left <= 0) continue;
            float out[N];
#pragma unroll
            for (int i = 0; i < N; ++i) out[i] = (v[c][i] - s.residual) * s.rstd * w[c][i] + b[c][i];
            store_unit<T>(y + row * width + col, left, out);
        }
        if (mean_out && lane == 0) {
            mean_out[row] = mean + s.residual;
            rstd_out[row] = s.rstd;
        }
    }
}

// Rows that do not fit the registers of a workgroup: three reads, the later two from the caches.
template <typename T, typename W>
__global__ void __launch_bounds__(256) norm_forward_long(Rows x, int width, const W* __restrict__ weight,
                                                         const W* __restrict__ bias, float eps, T* __restrict__ y,
                                                         float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int N = Unit<T>::N;
    __shared__ float shared[12];
    const i64 row = blockIdx.x;
    const T* src = x.at<T>(row);
    Unit<T> v;
    float sum[1] = {0.0f}, sums[2] = {0.0f, 0.0f};
    for (int col = threadIdx.x * N; col < width; col += 256 * N) {
        v.load(src, col, width);
#pragma unroll
        for (int i = 0; i < N; ++i) sum[0] += v[i];
    }
    group_sum<256>(sum, shared);
    const float mean = sum[0] / (float)width;
    for (int col = threadIdx.x * N; col < width; col += 256 * N) {
        v.load(src, col, width);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float centred = col + i < width ? v[i] - mean : 0.0f;
            sums[0] += centred;
            sums[1] += centred * centred;
        }
    }
    group_sum<256>(sums, shared);
    const Spread s(sums[0] / (float)width, sums[1] / (float)width, eps);
    for (int col = threadIdx.x * N; col < width; col += 256 * N) {
        float w[N], b[N];
        v.load(src, col, width);
        load_columns<W, N>(weight, col, width, 1.0f, w);
        load_columns<W, N>(bias, col, width, 0.0f, b);
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
//
// A row's loads wait for the reduction of the row before; three workgroups per CU hide that where their
// registers allow it (32768 x 4096 bfloat16: 298 us with two of 187 registers, 239 with three of 168 although 8 are
// spilled, 19 with a bfloat16 weight; with four, 667).  Now 224 us there, 3.6 TB/s of the two reads and the write; 25600 x 256 float32 18.1.
template <typename T, typename W, int LANES, int CH>
__global__ void __launch_bounds__(256, CH <= 2 ? 3 : 2) norm_backward(Rows grad, Rows x, i64 rows, int width,
                                                     const W* __restrict__ weight, const float* __restrict__ mean_in,
                                                     const float* __restrict__ rstd_in, T* __restrict__ dx,
                                                     float* __restrict__ partial) {
    constexpr int N = Unit<T>::N, GROUPS = 256 / LANES;
    __shared__ float shared[12];
    extern __shared__ float columns[];  // GROUPS > 1: the groups' column sums, one group after the other
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    float w[CH][N], dw[CH][N], db[CH][N];
    Unit<T> gu[CH], xu[CH];
    float mean = 0.0f, rstd = 0.0f;
    auto fetch = [&](i64 row) {
        const T *gp = grad.at<T>(row), *xp = x.at<T>(row);
        mean = mean_in[row], rstd = rstd_in[row];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            gu[c].load(gp, (lane + c * LANES) * N, width);
            xu[c].load(xp, (lane + c * LANES) * N, width);
        }
    };
    const i64 stride = (i64)gridDim.x * GROUPS, first = (i64)blockIdx.x * GROUPS + group;
    if (first < rows) fetch(first);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        load_columns<W, N>(weight, (lane + c * LANES) * N, width, 1.0f, w[c]);
#pragma unroll
        for (int i = 0; i < N; ++i) dw[c][i] = db[c][i] = 0.0f;
    }
    for (i64 row = first; row < rows; row += stride) {
        float g[CH][N], z[CH][N];
        float sums[3] = {0.0f, 0.0f, 0.0f};  // of h, h z and z
        const float scale = rstd;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int left = width - (lane + c * LANES) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                g[c][i] = gu[c][i];
                z[c][i] = i < left ? (xu[c][i] - mean) * scale : 0.0f;
                const float h = g[c][i] * w[c][i];
                sums[0] += h;
                sums[1] += h * z[c][i];
                sums[2] += z[c][i];
            }
        }
        if (row + stride < rows) fetch(row + stride);
        group_sum<LANES>(sums, shared);
        const float residual = sums[2] / (float)width, sum = sums[0] / (float)width;
        const float dot = sums[1] / (float)width - residual * sum;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (lane + c * LANES) * N, left = width - col;
            if (left <= 0) continue;
            float d[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float centred = z[c][i] - residual;
                dw[c][i] += g[c][i] * centred;
                db[c][i] += g[c][i];
                d[i] = scale * (g[c][i] * w[c][i] - sum - centred * dot);
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
            for (int col = threadIdx.x; col < min(SPAN, width); col += 256) {
                float total = 0.0f;
#pragma unroll
                for (int k = 0; k < GROUPS; ++k) total += columns[k * SPAN + col];
                out[half * width + col] = total;
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (lane + c * LANES) * N;
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
__global__ void __launch_bounds__(256) norm_backward_long(Rows grad, Rows x, int width, const W* __restrict__ weight,
                                                          const float* __restrict__ mean_in,
                                                          const float* __restrict__ rstd_in, T* __restrict__ dx,
                                                          float* __restrict__ residuals) {
    constexpr int N = Unit<T>::N;
    __shared__ float shared[12];
    const i64 row = blockIdx.x;
    const T *gp = grad.at<T>(row), *xp = x.at<T>(row);
    const float mean = mean_in[row], rstd = rstd_in[row];
    float sums[3] = {0.0f, 0.0f, 0.0f}, sum = 0.0f, dot = 0.0f, residual = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {
        for (int col = threadIdx.x * N; col < width; col += 256 * N) {
            Unit<T> g, v;
            float w[N];
            g.load(gp, col, width);
            v.load(xp, col, width);
            load_columns<W, N>(weight, col, width, 1.0f, w);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float z = col + i < width ? (v[i] - mean) * rstd : 0.0f, h = g[i] * w[i];
                if (pass) {
                    w[i] = rstd * (h - sum - (z - residual) * dot);
                } else {
                    sums[0] += h;
                    sums[1] += h * z;
                    sums[2] += z;
                }
            }
            if (pass) store_unit<T>(dx + row * width + col, width - col, w);
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
__global__ void __launch_bounds__(256) norm_columns(Rows grad, Rows x, i64 rows, int width,
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
// added in LDS in a fixed order: 6 us after 32768 x 4096, 4 after 25600 x 256, most of it the launch.
template <typename W>
__global__ void __launch_bounds__(1024) norm_reduce(i64 blocks, i64 width, const float* __restrict__ partial,
                                                    W* __restrict__ dweight, W* __restrict__ dbias) {
    __shared__ float sums[32][33];
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
    const i64 col = first_column() + lane;
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

// The layout of a row by its units of 16 bytes.  16 lanes up to 16 units, 16 rows per workgroup (262144 x 64 float32:
// forward 24 us, backward 41, and 79, 108 with a wave each).  A wave up to 4 units per lane forward (32768 x 2048
// bfloat16 69 us, a workgroup 84), up to 2 backward, where a row's registers are twice as many (a workgroup 146 us,
// a wave 209; the bytes take 77, and half the units of that layout, of 512, lie beyond a row of 129 to 256 units).  A
// workgroup up to 4 per lane, backward of bfloat16 up to 2: the registers of more cost the workgroups that hide
// the loads, and reading the rows again from the caches is faster (4 against long: 8192 x 4096 float32 60 to 62 and 152
// to 164 us; 8192 x 8192 bfloat16 71 to 79 and 314 to 228; 8 against long: 4096 x 8192 float32 99 to 77 and 213 to 168).
struct Shape {
    int lanes, chunks;  // chunks 0: long rows
};

Shape shape_of(i64 width, int type, bool backward) {
    const i64 units = ceil_div(width, type == ATLAS_OPS_F32 ? 4 : 8);
    if (units <= 16) return {16, 1};
    for (int c : {1, 2, 4})
        if (units <= 64 * c && !(backward && c == 4)) return {64, c};
    for (int c : {2, 4})
        if (units <= 256 * c && !(backward && c == 4 && type == ATLAS_OPS_BF16)) return {256, c};
    return {256, 0};
}

template <typename T, bool BACKWARD, typename F>
void with_shape(Shape s, F&& f) {
    if (s.lanes == 16) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    else if (s.lanes == 64 && s.chunks == 1) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (s.lanes == 64 && s.chunks == 2) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else if (s.lanes == 64) {
        if constexpr (!BACKWARD) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    } else if (s.chunks == 2) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if constexpr (!BACKWARD || sizeof(T) == 4) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
}

template <typename F>
void with_types(int type, int weight_type, F&& f) {
    if (type == ATLAS_OPS_F32) f(0.0f, 0.0f);
    else if (weight_type == ATLAS_OPS_F32) f(bf16_t{}, 0.0f);
    else f(bf16_t{}, bf16_t{});
}

// Workgroups at most: each keeps its columns' weights for all its rows and fetches its next row ahead.  Forward
// (us, 1024 / 2048 / 8192): 32768 x 4096 bfloat16 137 / 142 / 180, 9973 x 1023 16 / 20 / 19, 25600 x 256
// float32 15 / 16 / 16.
constexpr i64 FORWARD_BLOCKS = 1024, BACKWARD_BLOCKS = 768;

// Blocks of the backward pass's rows; the partials stay a small share of the traffic.
i64 row_blocks(i64 rows, i64 width, int type) {
    const Shape s = shape_of(width, type, true);
    if (s.chunks == 0) return std::min<i64>(rows, 64);
    return std::min<i64>(ceil_div(rows, 256 / s.lanes), BACKWARD_BLOCKS);
}

// A long row is a workgroup of its own.
bool fits(i64 rows, i64 width, int type, bool backward) {
    return shape_of(width, type, backward).chunks > 0 || rows * 256 < THREADS;
}

bool usable(const AtlasRows* r) { return r && r->data && r->inner > 0; }

int check(const AtlasRows* x, i64 rows, i64 width, int type, int weight_type, bool backward, char* err, size_t cap) {
    if (rows < 0 || rows > 0x7FFFFFFF || width < 1 || width > 0x7FFF0000)
        return fail(err, cap, 7, "rows and width must be below 2^31, width positive");
    if (!known_type(type) || !known_type(weight_type) || (type == ATLAS_OPS_F32 && weight_type != ATLAS_OPS_F32))
        return fail(err, cap, 7, "weight must be float32 or have the rows' type");
    if (!fits(rows, width, type, backward))
        return fail(err, cap, 7, "rows of this width must be fewer than 2^24");
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
        if (int rc = check(x, rows, width, type, weight_type, false, err, cap)) return rc;
        if (!rows) return 0;
        if (!y || (mean == nullptr) != (rstd == nullptr)) return fail(err, cap, 7, "null output");
        const Shape shape = shape_of(width, type, false);
        const Rows in{x->data, x->inner, x->outer_stride, x->inner_stride};
        with_types(type, weight_type, [&](auto t, auto w) {
            using T = decltype(t);
            using W = decltype(w);
            if (shape.chunks == 0) {
                norm_forward_long<T, W><<<dim3((unsigned)rows), 256, 0, (hipStream_t)stream>>>(
                    in, (int)width, (const W*)weight, (const W*)bias, eps, (T*)y, mean, rstd);
                return;
            }
            with_shape<T, false>(shape, [&](auto lanes, auto chunks) {
                norm_forward<T, W, lanes(), chunks()>
                    <<<dim3((unsigned)std::min<i64>(ceil_div(rows, 256 / lanes()), FORWARD_BLOCKS)), 256, 0, (hipStream_t)stream>>>(
                        in, rows, (int)width, (const W*)weight, (const W*)bias, eps, (T*)y, mean, rstd);
            });
        });
        return launched(err, cap, "layer_norm");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

int64_t atlas_ops_layer_norm_workspace(int64_t rows, int64_t width, int type) {
    if (rows < 1 || width < 1 || !known_type(type) || !fits(rows, width, type, true)) return 0;
    // the partial sums, and of long rows what their means left out
    return (2 * row_blocks(rows, width, type) * width + (shape_of(width, type, true).chunks ? 0 : rows)) * (i64)sizeof(float);
}

int atlas_ops_layer_norm_backward(const AtlasRows* grad, const AtlasRows* x, int64_t rows, int64_t width, int type,
                                  const void* weight, int weight_type, const float* mean, const float* rstd, void* dx,
                                  void* dweight, void* dbias, float* workspace, void* stream, char* err, size_t cap) {
    try {
        if (int rc = check(x, rows, width, type, weight_type, true, err, cap)) return rc;
        const bool sums = dweight || dbias;
        if (rows && (!usable(grad) || !mean || !rstd || !dx || (sums && !workspace)))
            return fail(err, cap, 7, "null argument");
        const i64 blocks = rows ? row_blocks(rows, width, type) : 0;
        hipStream_t st = (hipStream_t)stream;
        with_types(type, weight_type, [&](auto t, auto w) {
            using T = decltype(t);
            using W = decltype(w);
            if (rows) {
                const Shape shape = shape_of(width, type, true);
                const Rows in{x->data, x->inner, x->outer_stride, x->inner_stride};
                const Rows g{grad->data, grad->inner, grad->outer_stride, grad->inner_stride};
                if (shape.chunks == 0) {
                    norm_backward_long<T, W><<<dim3((unsigned)rows), 256, 0, st>>>(g, in, (int)width, (const W*)weight, mean,
                                                                                  rstd, (T*)dx,
                                                                                  sums ? workspace + 2 * blocks * width : nullptr);
                    if (sums)
                        norm_columns<T><<<dim3((unsigned)ceil_div(width, 256), (unsigned)blocks), 256, 0, st>>>(
                            g, in, rows, (int)width, mean, rstd, workspace + 2 * blocks * width, workspace);
                } else {
                    with_shape<T, true>(shape, [&](auto lanes, auto chunks) {
                        const size_t lds = lanes() < 256 ? 256 * chunks() * Unit<T>::N * sizeof(float) : 0;
                        norm_backward<T, W, lanes(), chunks()><<<dim3((unsigned)blocks), 256, lds, st>>>(
                            g, in, rows, (int)width, (const W*)weight, mean, rstd, (T*)dx, sums ? workspace : nullptr);
                    });
                }
            }
            if (sums)
                norm_reduce<W><<<column_grid(ceil_div(2 * width, 32)), 1024, 0, st>>>(
                    blocks, width, workspace, (W*)dweight, (W*)dbias);
        });
        return launched(err, cap, "layer_norm_backward");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

}  // extern "C"
