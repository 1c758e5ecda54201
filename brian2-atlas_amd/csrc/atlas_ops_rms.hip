// Root-mean-square normalisation of a residual stream, forward (also to 8 bits with a scale by row) and
// backward.  Part of libatlas_ops_hip.so.
//
//   t = x + r (rounded to the rows' type, as the next layer reads it),  z = t rstd,  y = z w,
//   rstd = 1 / sqrt(mean(t^2) + eps)
//   dt = rstd (h - z mean(h z)) + g_t,  h = g w,  which is the gradient of x and of r;   dw = sum_rows g z
//   8 bits: scale = max(max |y| / 448, 2^-126),  value = y / scale as e4m3; infinite where the sum of squares is
//
// Memory bounds all of it.  A row is read once into registers, summed, written; the next row's loads are in
// flight meanwhile.  16384 x 4096 bfloat16 with a residual: forward 94 us (5.7 TB/s over four passes), backward 137 us (3.9: its
// registers leave 12 waves to a CU); 2048 x 4096 to 8 bits 16.7 us.  The backward pass keeps the column sums of dw in registers
// over the rows that a group visits, adds the groups of a workgroup in LDS and writes one row of partial sums per workgroup,
// which a second kernel adds in a fixed order.
#include <algorithm>

#include "device/atlas_rows.h"

namespace atlas_ops {
namespace {

constexpr float LARGEST = 448.0f, SMALLEST_SCALE = 0x1p-126f;  // of e4m3; a zero row's scale

// Of a row of 8 bits.  rstd is 0 where the sum of squares passes float32 and every value is lost: an infinite scale says so.
__device__ __forceinline__ float scale_of(float most, float rstd) {
    return rstd == 0.0f ? INFINITY : fmaxf(most / LARGEST, SMALLEST_SCALE);
}

template <int LANES>
__device__ __forceinline__ float group_max(float v, float* shared) {
#pragma unroll
    for (int d = 1; d < (LANES < 64 ? LANES : 64); d *= 2) v = fmaxf(v, __shfl_xor(v, d, 64));
    if constexpr (LANES > 64) {
        __syncthreads();  // the previous use of `shared` is read
        if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
        __syncthreads();
        v = fmaxf(fmaxf(shared[0], shared[1]), fmaxf(shared[2], shared[3]));
    }
    return v;
}

// N (4 or 8) values as e4m3, rounded to nearest even.
template <int N>
__device__ __forceinline__ void store_8bit(uint8_t* p, int left, const float* v) {
    struct __attribute__((packed, aligned(1))) Raw { uint32_t word[N / 4]; };
    Raw raw;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
        raw.word[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], word, true);
    }
    if (left >= N) {
        __builtin_memcpy(p, &raw, sizeof(raw));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = (uint8_t)(raw.word[i / 4] >> (8 * (i % 4)));
    }
}

// A unit's values with the residual's added and rounded to T.
template <typename T, bool RESIDUAL>
__device__ __forceinline__ void stream_values(const Unit<T>& x, const Unit<T>& r, float* out) {
#pragma unroll
    for (int i = 0; i < Unit<T>::N; ++i) out[i] = RESIDUAL ? to_float(from_float<T>(x[i] + r[i])) : x[i];
}

struct Outputs {
    void* y;         // of the rows' type, or the 8-bit values where scale is not null
    float* scale;    // by row
    void* total;     // null without a residual
    float* rstd;     // may be null
};

// One row at a time per group of LANES lanes; lane l holds units l, l + LANES, ... (CH of them), and the same
// columns of the weight for all its rows.
template <typename T, typename W, int LANES, int CH, bool RESIDUAL>
__global__ void __launch_bounds__(256) rms_forward(Rows x, Rows residual, i64 rows, int width, const W* __restrict__ weight, float eps,
                                                   Outputs out) {
    constexpr int N = Unit<T>::N, GROUPS = 256 / LANES;
    __shared__ float shared[12];
    const int lane = threadIdx.x % LANES;
    const i64 first = (i64)blockIdx.x * GROUPS + threadIdx.x / LANES, stride = (i64)gridDim.x * GROUPS;
    if (first >= rows) return;  // never a part of a workgroup that has barriers: its rows are whole workgroups
    float w[CH][N];
    Unit<T> unit[CH], other[RESIDUAL ? CH : 1];
    auto fetch = [&](i64 row) {
        const T* src = x.at<T>(row);
#pragma unroll
        for (int c = 0; c < CH; ++c) unit[c].load(src, (lane + c * LANES) * N, width);
        if constexpr (RESIDUAL) {
            const T* add = residual.at<T>(row);
#pragma unroll
            for (int c = 0; c < CH; ++c) other[c].load(add, (lane + c * LANES) * N, width);
        }
    };
    fetch(first);
#pragma unroll
    for (int c = 0; c < CH; ++c) load_columns<W, N>(weight, (lane + c * LANES) * N, width, 1.0f, w[c]);
    for (i64 row = first; row < rows; row += stride) {
        float v[CH][N];
        float sum[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            stream_values<T, RESIDUAL>(unit[c], other[RESIDUAL ? c : 0], v[c]);
#pragma unroll
            for (int i = 0; i < N; ++i) sum[0] += v[c][i] * v[c][i];  // zeros beyond the width
        }
        if (row + stride < rows) fetch(row + stride);
        if constexpr (RESIDUAL) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (lane + c * LANES) * N;
                if (col < width) store_unit<T>((T*)out.total + row * width + col, width - col, v[c]);
            }
        }
        group_sum<LANES>(sum, shared);
        const float rstd = 1.0f / sqrtf(sum[0] / (float)width + eps);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < N; ++i) v[c][i] = v[c][i] * rstd * w[c][i];
        if (out.scale) {
            float most = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(v[c][i]));
            const float scale = scale_of(group_max<LANES>(most, shared), rstd), inverse = 1.0f / scale;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (lane + c * LANES) * N;
                if (col >= width) continue;
#pragma unroll
                for (int i = 0; i < N; ++i) v[c][i] *= inverse;
                store_8bit<N>((uint8_t*)out.y + row * width + col, width - col, v[c]);
            }
            if (lane == 0) out.scale[row] = scale;
        } else {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (lane + c * LANES) * N;
                if (col < width) store_unit<T>((T*)out.y + row * width + col, width - col, v[c]);
            }
        }
        if (out.rstd && lane == 0) out.rstd[row] = rstd;
    }
}

// Rows that do not fit the registers of a workgroup: read again from the caches, two or three times.
template <typename T, typename W, bool RESIDUAL>
__global__ void __launch_bounds__(256) rms_forward_long(Rows x, Rows residual, int width, const W* __restrict__ weight, float eps, Outputs out) {
    constexpr int N = Unit<T>::N;
    __shared__ float shared[12];
    const i64 row = blockIdx.x;
    const T *src = x.at<T>(row), *add = RESIDUAL ? residual.at<T>(row) : nullptr;
    auto values = [&](int col, float* v) {
        Unit<T> a, b;
        a.load(src, col, width);
        if constexpr (RESIDUAL) b.load(add, col, width);
        stream_values<T, RESIDUAL>(a, b, v);
    };
    float v[N], w[N], sum[1] = {0.0f};
    for (int col = threadIdx.x * N; col < width; col += 256 * N) {
        values(col, v);
        if constexpr (RESIDUAL) store_unit<T>((T*)out.total + row * width + col, width - col, v);
#pragma unroll
        for (int i = 0; i < N; ++i) sum[0] += v[i] * v[i];
    }
    group_sum<256>(sum, shared);
    const float rstd = 1.0f / sqrtf(sum[0] / (float)width + eps);
    float scale = 1.0f;
    if (out.scale) {
        float most = 0.0f;
        for (int col = threadIdx.x * N; col < width; col += 256 * N) {
            values(col, v);
            load_columns<W, N>(weight, col, width, 1.0f, w);
#pragma unroll
            for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(v[i] * rstd * w[i]));
        }
        scale = scale_of(group_max<256>(most, shared), rstd);
        if (threadIdx.x == 0) out.scale[row] = scale;
    }
    for (int col = threadIdx.x * N; col < width; col += 256 * N) {
        values(col, v);
        load_columns<W, N>(weight, col, width, 1.0f, w);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] * rstd * w[i];
        if (out.scale) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] *= 1.0f / scale;
            store_8bit<N>((uint8_t*)out.y + row * width + col, width - col, v);
        } else {
            store_unit<T>((T*)out.y + row * width + col, width - col, v);
        }
    }
    if (out.rstd && threadIdx.x == 0) out.rstd[row] = rstd;
}

// Group j of the grid visits rows j, j + groups, ...; partials: block b's sums of dw at partial[b * width].
template <typename T, typename W, int LANES, int CH, bool STREAM>
__global__ void __launch_bounds__(LANES > 256 ? LANES : 256, 2) rms_backward(Rows grad, Rows total, Rows grad_total, i64 rows, int width,
                                                       const W* __restrict__ weight, const float* __restrict__ rstd_in,
                                                       T* __restrict__ dx, float* __restrict__ partial) {
    constexpr int N = Unit<T>::N, GROUPS = LANES > 256 ? 1 : 256 / LANES;
    __shared__ float shared[12];
    extern __shared__ float columns[];  // GROUPS > 1: the groups' column sums, one group after the other
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    float w[CH][N], dw[CH][N];
    Unit<T> gu[CH], tu[CH], su[STREAM ? CH : 1];
    float rstd = 0.0f;
    auto fetch = [&](i64 row) {
        const T *gp = grad.at<T>(row), *tp = total.at<T>(row);
        rstd = rstd_in[row];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            gu[c].load(gp, (lane + c * LANES) * N, width);
            tu[c].load(tp, (lane + c * LANES) * N, width);
        }
        if constexpr (STREAM) {
            const T* sp = grad_total.at<T>(row);
#pragma unroll
            for (int c = 0; c < CH; ++c) su[c].load(sp, (lane + c * LANES) * N, width);
        }
    };
    const i64 stride = (i64)gridDim.x * GROUPS, first = (i64)blockIdx.x * GROUPS + group;
    if (first < rows) fetch(first);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        load_columns<W, N>(weight, (lane + c * LANES) * N, width, 1.0f, w[c]);
#pragma unroll
        for (int i = 0; i < N; ++i) dw[c][i] = 0.0f;
    }
    for (i64 row = first; row < rows; row += stride) {
        float h[CH][N], z[CH][N], d[STREAM ? CH : 1][N];
        float sum[1] = {0.0f};
        const float scale = rstd;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                z[c][i] = tu[c][i] * scale;
                dw[c][i] += gu[c][i] * z[c][i];  // zeros beyond the width
                h[c][i] = gu[c][i] * w[c][i];
                sum[0] += h[c][i] * z[c][i];
                if constexpr (STREAM) d[c][i] = su[c][i];
            }
        if (row + stride < rows) fetch(row + stride);
        group_sum<LANES>(sum, shared);
        const float dot = sum[0] / (float)width;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (lane + c * LANES) * N, left = width - col;
            if (left <= 0) continue;
            float g[N];
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = scale * (h[c][i] - z[c][i] * dot) + (STREAM ? d[STREAM ? c : 0][i] : 0.0f);
            store_unit<T>(dx + row * width + col, left, g);
        }
    }
    if (!partial) return;
    float* out = partial + (i64)blockIdx.x * width;
    if constexpr (GROUPS > 1) {
        constexpr int SPAN = LANES * CH * N;  // columns a group holds
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < N; ++i) columns[group * SPAN + (lane + c * LANES) * N + i] = dw[c][i];
        __syncthreads();
        for (int col = threadIdx.x; col < min(SPAN, width); col += 256) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < GROUPS; ++k) sum += columns[k * SPAN + col];
            out[col] = sum;
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (lane + c * LANES) * N;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (col + i < width) out[col + i] = dw[c][i];
        }
    }
}

// Long rows: the mean of every row, dx in a second read; the column sums come from rms_columns.
template <typename T, typename W, bool STREAM>
__global__ void __launch_bounds__(256) rms_backward_long(Rows grad, Rows total, Rows grad_total, int width, const W* __restrict__ weight,
                                                         const float* __restrict__ rstd_in, T* __restrict__ dx) {
    constexpr int N = Unit<T>::N;
    __shared__ float shared[12];
    const i64 row = blockIdx.x;
    const T *gp = grad.at<T>(row), *tp = total.at<T>(row), *sp = STREAM ? grad_total.at<T>(row) : nullptr;
    const float rstd = rstd_in[row];
    float sum[1] = {0.0f}, dot = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {
        for (int col = threadIdx.x * N; col < width; col += 256 * N) {
            Unit<T> g, t, s;
            float w[N];
            g.load(gp, col, width);
            t.load(tp, col, width);
            if constexpr (STREAM) s.load(sp, col, width);
            load_columns<W, N>(weight, col, width, 1.0f, w);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float z = t[i] * rstd, h = g[i] * w[i];
                if (pass) w[i] = rstd * (h - z * dot) + (STREAM ? s[i] : 0.0f);
                else sum[0] += h * z;
            }
            if (pass) store_unit<T>(dx + row * width + col, width - col, w);
        }
        if (!pass) {
            group_sum<256>(sum, shared);
            dot = sum[0] / (float)width;
        }
    }
}

// Column sums of long rows: block (i, b) adds the rows b, b + blocks, ... of 256 columns.
template <typename T>
__global__ void __launch_bounds__(256) rms_columns(Rows grad, Rows total, i64 rows, int width, const float* __restrict__ rstd_in,
                                                   float* __restrict__ partial) {
    const i64 col = (i64)blockIdx.x * 256 + threadIdx.x;
    if (col >= width) return;
    float dw = 0.0f;
#pragma unroll 4
    for (i64 row = blockIdx.y; row < rows; row += gridDim.y)
        dw += to_float(grad.at<T>(row)[col]) * (to_float(total.at<T>(row)[col]) * rstd_in[row]);
    partial[(i64)blockIdx.y * width + col] = dw;
}

// Adds the blocks' partials: 32 columns per workgroup, its 32 row groups added in LDS in a fixed order.
template <typename W>
__global__ void __launch_bounds__(1024) rms_reduce(i64 blocks, i64 width, const float* __restrict__ partial, W* __restrict__ dweight) {
    __shared__ float sums[32][33];
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
    const i64 col = first_column() + lane;
    float total = 0.0f;
    if (col < width) {
#pragma unroll 8
        for (i64 b = group; b < blocks; b += 32) total += partial[b * width + col];
    }
    sums[group][lane] = total;
    __syncthreads();
    if (group == 0 && col < width) {
        total = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; ++k) total += sums[k][lane];
        dweight[col] = from_float<W>(total);
    }
}

// The layout of a row by its units of 16 bytes, as few lanes as hold it in registers: a wider group waits for its sum with less
// to load.  Forward and backward with the layout taken and with the next one:
//   32768 x 64 float32     16 lanes 8.1 and 9.8 us,             64 lanes 13.1 and 18.9
//   32768 x 512 float32    64 lanes of two units 46.8 and 46.3, 256 lanes 55 and 76
//   4096 x 4096 float32    256 lanes of four 54.6 and 62.5,     as long rows 59.5 and 93.7
//   4096 x 8192 bfloat16   backward 512 lanes of two 76 us (four units of 256 lanes spill: 126), as long rows 111
struct Shape {
    int lanes, chunks;  // chunks 0: long rows
};

Shape shape_of(i64 width, int type, bool backward) {
    const i64 units = ceil_div(width, type == ATLAS_OPS_F32 ? 4 : 8);
    if (units <= 16) return {16, 1};
    for (int c : {1, 2})
        if (units <= 64 * c) return {64, c};
    for (int c : {1, 2, 4})
        if (units <= 256 * c) return backward && c == 4 && type == ATLAS_OPS_BF16 ? Shape{512, 2} : Shape{256, c};
    return {256, 0};
}

template <typename T, bool BACKWARD, typename F>
void with_shape(Shape s, F&& f) {
    using std::integral_constant;
    if (s.lanes == 16) f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (s.lanes == 64 && s.chunks == 1) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (s.lanes == 64) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (s.lanes == 256 && s.chunks == 1) f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (s.lanes == 256 && s.chunks == 2) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else if constexpr (BACKWARD && sizeof(T) == 2) f(integral_constant<int, 512>{}, integral_constant<int, 2>{});
    else f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
}

template <typename F>
void with_types(int type, int weight_type, F&& f) {
    if (type == ATLAS_OPS_F32) f(0.0f, 0.0f);
    else if (weight_type == ATLAS_OPS_F32) f(bf16_t{}, 0.0f);
    else f(bf16_t{}, bf16_t{});
}

// Workgroups at most: each keeps its columns' weights for all its rows and fetches its next row ahead.  Forward 1024 are within
// 8 % either way, 4096 up to 18 % slower (4096 x 4096 float32 64 us instead of 54.6).
constexpr i64 FORWARD_BLOCKS = 2048;

// Blocks of the backward pass's rows: as many as its registers let stay on 256 CUs, so that none waits for a second turn.
// 8192 x 4096 bfloat16: 768 in 64 us, 512 in 75, 1024 in 91; of four units 4096 x 4096 float32: 512 in 62.5, 768 in 82.  The
// partials stay a small share of the traffic.
i64 row_blocks(i64 rows, i64 width, int type) {
    const Shape s = shape_of(width, type, true);
    if (s.chunks == 0) return std::min<i64>(rows, 64);
    if (s.lanes == 512) return std::min<i64>(rows, 256);
    return std::min<i64>(ceil_div(rows, 256 / s.lanes), s.chunks == 4 ? 512 : 768);
}

// A long row is a workgroup of its own.
bool fits(i64 rows, i64 width, int type, bool backward) {
    return shape_of(width, type, backward).chunks > 0 || rows * 256 < THREADS;
}

bool usable(const AtlasRows* r) { return r && r->data && r->inner > 0; }

Rows rows_of(const AtlasRows* r) { return r ? Rows{r->data, r->inner, r->outer_stride, r->inner_stride} : Rows{}; }

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

template <typename F>
void with_flag(bool flag, F&& f) {
    if (flag) f(std::true_type{});
    else f(std::false_type{});
}

}  // namespace
}  // namespace atlas_ops

using namespace atlas_ops;

extern "C" {

int atlas_ops_rms_norm(const AtlasRows* x, const AtlasRows* residual, int64_t rows, int64_t width, int type, const void* weight,
                       int weight_type, float eps, void* y, float* scale, void* total, float* rstd, void* stream, char* err, size_t cap) {
    try {
        if (int rc = check(x, rows, width, type, weight_type, false, err, cap)) return rc;
        if (!rows) return 0;
        if (residual && !usable(residual)) return fail(err, cap, 7, "null rows");
        if (!y || (residual != nullptr) != (total != nullptr)) return fail(err, cap, 7, "null output");
        const Shape shape = shape_of(width, type, false);
        const Outputs out{y, scale, total, rstd};
        with_types(type, weight_type, [&](auto t, auto w) {
            using T = decltype(t);
            using W = decltype(w);
            with_flag(residual != nullptr, [&](auto added) {
                if (shape.chunks == 0) {
                    rms_forward_long<T, W, added()><<<dim3((unsigned)rows), 256, 0, (hipStream_t)stream>>>(
                        rows_of(x), rows_of(residual), (int)width, (const W*)weight, eps, out);
                    return;
                }
                with_shape<T, false>(shape, [&](auto lanes, auto chunks) {
                    rms_forward<T, W, lanes(), chunks(), added()>
                        <<<dim3((unsigned)std::min<i64>(ceil_div(rows, 256 / lanes()), FORWARD_BLOCKS)), 256, 0, (hipStream_t)stream>>>(
                            rows_of(x), rows_of(residual), rows, (int)width, (const W*)weight, eps, out);
                });
            });
        });
        return launched(err, cap, "rms_norm");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

int64_t atlas_ops_rms_norm_workspace(int64_t rows, int64_t width, int type) {
    if (rows < 1 || width < 1 || !known_type(type) || !fits(rows, width, type, true)) return 0;
    return row_blocks(rows, width, type) * width * (i64)sizeof(float);
}

int atlas_ops_rms_norm_backward(const AtlasRows* grad, const AtlasRows* total, const AtlasRows* grad_total, int64_t rows, int64_t width,
                                int type, const void* weight, int weight_type, const float* rstd, void* dx, void* dweight,
                                float* workspace, void* stream, char* err, size_t cap) {
    try {
        if (int rc = check(total, rows, width, type, weight_type, true, err, cap)) return rc;
        if (rows && (!usable(grad) || (grad_total && !usable(grad_total)) || !rstd || !dx || (dweight && !workspace)))
            return fail(err, cap, 7, "null argument");
        const i64 blocks = rows ? row_blocks(rows, width, type) : 0;
        hipStream_t st = (hipStream_t)stream;
        with_types(type, weight_type, [&](auto t, auto w) {
            using T = decltype(t);
            using W = decltype(w);
            if (rows)
                with_flag(grad_total != nullptr, [&](auto added) {
                    const Shape shape = shape_of(width, type, true);
                    const Rows g = rows_of(grad), in = rows_of(total), s = rows_of(grad_total);
                    if (shape.chunks == 0) {
                        rms_backward_long<T, W, added()><<<dim3((unsigned)rows), 256, 0, st>>>(g, in, s, (int)width, (const W*)weight,
                                                                                               rstd, (T*)dx);
                        if (dweight)
                            rms_columns<T><<<dim3((unsigned)ceil_div(width, 256), (unsigned)blocks), 256, 0, st>>>(g, in, rows, (int)width,
                                                                                                                   rstd, workspace);
                        return;
                    }
                    with_shape<T, true>(shape, [&](auto lanes, auto chunks) {
                        const size_t lds = lanes() < 256 ? 256 * chunks() * Unit<T>::N * sizeof(float) : 0;
                        rms_backward<T, W, lanes(), chunks(), added()><<<dim3((unsigned)blocks), std::max(256, lanes()), lds, st>>>(
                            g, in, s, rows, (int)width, (const W*)weight, rstd, (T*)dx, dweight ? workspace : nullptr);
                    });
                });
            if (dweight)
                rms_reduce<W><<<column_grid(ceil_div(width, 32)), 1024, 0, st>>>(blocks, width, workspace, (W*)dweight);
        });
        return launched(err, cap, "rms_norm_backward");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

}  // extern "C"
