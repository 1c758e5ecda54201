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
// significant bits (the iterates' entries are below 1.5 with the default coefficients; hi is normal down to
// 4e-6, and lo covers what is below), in the 4 bytes that a float32 takes.  A product of two such matrices is three
// float16 MFMAs, hi hi + (hi lo + lo hi) / 2048 with float32 sums; the dropped lo lo term is below
// 2^-22.  That is float32's accuracy at 1/3 of the float16 rate instead of the float32 MFMA's 1/16.
//
// Matrices with more rows than columns are transposed while they are split, so that A is the
// smaller of the two Gram matrices.  Both X and its transpose are kept: every product then has both
// operands contiguous along the sum.  Planes lie as columns of 32 values, one after the other: what the
// rows of a tile give to a stage of a product is one contiguous piece.  A and b A + c A A are symmetric: only
// the tiles on and above the diagonal are computed, and written twice.
#include <algorithm>
#include <cmath>
#include <type_traits>

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

// Element (r, k) of a plane of `rows` rows.
__device__ __forceinline__ i64 element(i64 rows, int r, int k) { return ((i64)(k / 32) * rows + r) * 32 + k % 32; }

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

constexpr int PARTIALS = 1024;  // blocks per matrix of the norm's sum

// Updates the momentum and adds the squares of u: block (i, b) takes `span` values from i span on, its lanes
// each value 256 after the last (row and column advance with it, without a division).  The sum is held
// in 64 bits, where no square of a float32 overflows or vanishes.  Memory bounds it: 4096 x 2048 with a momentum
// 19.3 us, 5.2 TB/s; 256 x 256 3.6 us.
template <typename T, bool MOMENTUM>
__global__ void __launch_bounds__(256) ortho_norm(Source s, i64 span, double* __restrict__ partial) {
    __shared__ double sums[4];
    const i64 b = blockIdx.y, count = s.rows * s.columns;
    const i64 first = (i64)blockIdx.x * span + threadIdx.x, end = min((i64)(blockIdx.x + 1) * span, count);
    const i64 r0 = first / s.columns, c0 = first % s.columns;
    i64 r = r0, c = c0;
    const i64 step_r = 256 / s.columns, step_c = 256 % s.columns;
    double total = 0.0;
    constexpr int UNROLL = 4;  // loads of so many values before the first is used
    for (i64 e = first; e < end; e += 256 * UNROLL) {
        float g[UNROLL], m[UNROLL];
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const bool any = e + 256 * i < end;  // the others read the block's first value, and count for nothing
            g[i] = s.gradient<T>(b, any ? r : r0, any ? c : c0);
            if constexpr (MOMENTUM) m[i] = s.momentum[b * count + (any ? e + 256 * i : first)];
            r += step_r;
            c += step_c;
            if (c >= s.columns) {
                c -= s.columns;
                ++r;
            }
        }
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            if (e + 256 * i >= end) break;
            float u = g[i];
            if constexpr (MOMENTUM) {
                const float next = s.factor * m[i] + g[i];
                s.momentum[b * count + e + 256 * i] = next;
                u = s.nesterov ? g[i] + s.factor * next : next;
            }
            total += (double)u * (double)u;
        }
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) total += __shfl_xor(total, d, 64);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = total;
    __syncthreads();
    if (threadIdx.x == 0) partial[b * PARTIALS + blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// X and its transpose as planes, zero beyond the matrix: one 64 x 64 tile of X per workgroup, turned in LDS.
// 4096 x 2048 31.7 us, 4.2 TB/s of the source and momentum read and the two matrices' planes written; 256 x 256 6.2 us.
template <typename T>
__global__ void __launch_bounds__(256) ortho_split(Source s, int transposed, int parts,
                                                   const double* __restrict__ partial, float eps, i64 mp, i64 np,
                                                   Planes x, Planes xt) {
    __shared__ float tile[64][65];
    __shared__ double sums[4];
    const i64 b = blockIdx.z, count = s.rows * s.columns;
    // the tile in the matrix's own orientation: (r0, c0) in rows and columns of the source
    const i64 i0 = (i64)blockIdx.y * 64, j0 = (i64)blockIdx.x * 64;
    const i64 r0 = transposed ? j0 : i0, c0 = transposed ? i0 : j0;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    float u[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        // what lies outside is read at the last row and column, and replaced by zero
        const i64 r = min(r0 + wave + 4 * k, s.rows - 1), c = min(c0 + lane, s.columns - 1);
        u[k] = s.gradient<T>(b, r, c);
    }
    if (s.momentum) {
        float m[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const i64 r = min(r0 + wave + 4 * k, s.rows - 1), c = min(c0 + lane, s.columns - 1);
            m[k] = s.momentum[b * count + r * s.columns + c];
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) u[k] = s.nesterov ? u[k] + s.factor * m[k] : m[k];
    }
    double total = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) total += partial[b * PARTIALS + i];
#pragma unroll
    for (int d = 32; d > 0; d /= 2) total += __shfl_xor(total, d, 64);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = total;
    __syncthreads();
    const double scale = 1.0 / (sqrt((sums[0] + sums[1]) + (sums[2] + sums[3])) + (double)eps);
#pragma unroll
    for (int k = 0; k < 16; ++k)
        tile[wave + 4 * k][lane] = r0 + wave + 4 * k < s.rows && c0 + lane < s.columns ? (float)((double)u[k] * scale) : 0.0f;
    __syncthreads();
    const Planes a = x.offset(b * mp * np), t = xt.offset(b * mp * np);
    for (int k = wave; k < 64; k += 4) {
        half_t hi, lo;
        split(transposed ? tile[lane][k] : tile[k][lane], hi, lo);
        const i64 to = element(mp, (int)i0 + k, (int)j0 + lane);
        a.hi[to] = hi;
        a.lo[to] = lo;
        split(transposed ? tile[k][lane] : tile[lane][k], hi, lo);
        const i64 turned = element(np, (int)j0 + k, (int)i0 + lane);
        t.hi[turned] = hi;
        t.lo[turned] = lo;
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

// Workgroup barrier for LDS alone: the loads of a later stage stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// What a product's kernel is given: left rows x depth, right columns x depth.
struct Task {
    Planes left, right;
    i64 left_stride, right_stride;
    Planes in, out, out_t;
    int rows, columns, depth;
    float direct, product;
    float* partial;  // the splits' sums, or NULL
    int splits;
    Result result;
};

// How a product is cut: ROWS x COLUMNS of the result per workgroup, of which each of its WR x WC waves takes
// an equal part in 16 x 16 blocks, DEPTH sum indices per stage.  SPLIT: a triangle's sums may be split.
template <int ROWS_, int COLUMNS_, int WR_, int WC_, int DEPTH_, bool SPLIT_>
struct Cut {
    static constexpr int ROWS = ROWS_, COLUMNS = COLUMNS_, WR = WR_, WC = WC_, DEPTH = DEPTH_;
    static constexpr bool SPLIT = SPLIT_;
    static constexpr int THREADS = 64 * WR * WC, FR = ROWS / WR / 16, FC = COLUMNS / WC / 16;
    // Where 8 halves of a row lie in LDS.  A wave reads 16 rows at 4 neighbouring places each: with the
    // places exchanged by the row they hit every bank equally (padded rows of 80 or 144 bytes take twice the cycles).
    __device__ static __forceinline__ int place(int row, int unit) {
        return row * DEPTH + (unit ^ (DEPTH == 32 ? row / 2 % 4 : row % 8)) * 8;
    }
    static constexpr int RATIO = ROWS / COLUMNS;
    // tiles that reach the upper triangle of n columns of tiles (n a multiple of RATIO)
    static constexpr i64 triangle(i64 n) { return RATIO * (n / RATIO) * (n / RATIO + 1) / 2; }
};

// The tile of workgroup t: of the upper triangle (RATIO neighbouring columns of tiles have as many each) or
// of the whole matrix.
template <typename K, Product WHAT>
__device__ __forceinline__ void tile_of(int t, int rows, int& ti, int& tj) {
    if constexpr (WHAT == GRAM || WHAT == POLY) {
        int q = (int)((sqrtf(8.0f / K::RATIO * (float)t + 1.0f) - 1.0f) * 0.5f);
        while (K::RATIO * (q + 1) * (q + 2) / 2 <= t) ++q;
        while (K::RATIO * q * (q + 1) / 2 > t) --q;
        const int rest = t - K::RATIO * q * (q + 1) / 2;
        tj = K::RATIO * q + rest / (q + 1);
        ti = rest % (q + 1);
    } else {
        ti = t % (rows / K::ROWS);
        tj = t / (rows / K::ROWS);
    }
}

// The four values of `in` that a lane's part of a 16 x 16 block adds, rows r .. r + 3 of column c, read at
// (c, r): `in` is the symmetric matrix or the transpose of X.
struct Direct {
    half4_t hi, lo;
    float weight[4];

    // Where value e of rows r .. of column c belongs in the result; -1 beyond it.
    __device__ static __forceinline__ i64 place(const Result& o, i64 b, int r, int c, int e) {
        const int row = o.transposed ? c : r + e, column = o.transposed ? r + e : c;
        return row < o.rows && column < o.columns ? (b * o.rows + row) * o.columns + column : -1;
    }

    template <Product WHAT>
    __device__ __forceinline__ void load(const Task& t, i64 b, int r, int c) {
        if constexpr (WHAT == FINAL) {
            if (t.result.weight) {
#pragma unroll
                for (int e = 0; e < 4; ++e) weight[e] = t.result.weight[max(place(t.result, b, r, c, e), (i64)0)];
            }
        }
        if constexpr (WHAT != GRAM) {
            const i64 at = b * t.rows * t.columns + element(t.columns, c, r);
            hi = *(const half4_t*)(t.in.hi + at);
            lo = *(const half4_t*)(t.in.lo + at);
        }
    }
};

// What becomes of a lane's four products.
template <Product WHAT>
__device__ __forceinline__ void finish(const Task& t, i64 b, int r, int c, float4_t v, float product, const Direct& in) {
    const i64 area = b * t.rows * t.columns;
    // a symmetric result is written from its upper triangle of blocks, and mirrored
    if constexpr (WHAT == GRAM || WHAT == POLY)
        if (r / 16 > c / 16) return;
    v *= product;
    if constexpr (WHAT != GRAM) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += t.direct * join(in.hi[e], in.lo[e]);
    }
    if constexpr (WHAT == FINAL) {
        const Result& o = t.result;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const i64 at = Direct::place(o, b, r, c, e);
            if (at < 0) continue;
            if (o.weight) o.weight[at] = o.keep * in.weight[e] - o.rate * v[e];
            else if (o.out_type == ATLAS_OPS_F32) ((float*)o.out)[at] = v[e];
            else ((bf16_t*)o.out)[at] = from_float<bf16_t>(v[e]);
        }
    } else {
        half4_t hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            half_t h, l;
            split(v[e], h, l);
            hi[e] = h;
            lo[e] = l;
            const i64 to = area + element(t.rows, r + e, c);
            t.out.hi[to] = h;
            t.out.lo[to] = l;
        }
        // the mirror image of a symmetric matrix, or the transpose of X
        if (WHAT == APPLY || r / 16 != c / 16) {
            const i64 to = area + element(t.columns, c, r);
            *(half4_t*)(t.out_t.hi + to) = hi;
            *(half4_t*)(t.out_t.lo + to) = lo;
        }
    }
}

// 4096 x 2048: (b A + c A A) X 120 us, 859 TFLOP/s of float16 MFMA (a large library product of that type: 1093), bound
// by what an MFMA waits for its operands from LDS; X X^T 67 us and A A 38 us for their triangles, whose 72 tiles are
// split in parts that ortho_join adds in 11 and 13 us.  256 x 256: 5 us each, the way of a few stages from memory
// and the launch.
//
// One tile of Left Right^T.  While a stage is multiplied out of LDS, the next comes from memory into registers,
// and from there into the other buffer.
template <typename K, Product WHAT>
__global__ void __launch_bounds__(K::THREADS) ortho_product(Task t) {
    constexpr int FR = K::FR, FC = K::FC, DEPTH = K::DEPTH, KB = DEPTH / 32;
    constexpr bool SPLIT = K::SPLIT && (WHAT == GRAM || WHAT == POLY);
    constexpr int STEP = K::THREADS / 4, LR = K::ROWS / STEP, LC = K::COLUMNS / STEP;  // rows per round of loads, rounds
    __shared__ __attribute__((aligned(16))) half_t lds[2][2][(K::ROWS + K::COLUMNS) * DEPTH];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, wi = wave / K::WC, wj = wave % K::WC;
    const i64 b = blockIdx.z;
    // read here: the compiler keeps a task's field that it finds behind a branch in LDS, addressed through the
    // dispatch packet in host memory, which every kernel then waits for (up to 7 us)
    const float product = t.product;
    float* const partial = SPLIT ? t.partial : nullptr;
    int ti, tj;
    tile_of<K, WHAT>(blockIdx.x, t.rows, ti, tj);
    // four threads take the 64 bytes of a row
    const int lrow = threadIdx.x / 4, unit = threadIdx.x % 4;
    const i64 left_at = b * t.left_stride + element(t.rows, ti * K::ROWS + lrow, unit * 8);
    const i64 right_at = b * t.right_stride + element(t.columns, tj * K::COLUMNS + lrow, unit * 8);
    const half_t *left_hi = t.left.hi + left_at, *left_lo = t.left.lo + left_at;
    const half_t *right_hi = t.right.hi + right_at, *right_lo = t.right.lo + right_at;
    // the split's part, in columns of 32 sum indices
    const int all = t.depth / 32;
    const int first = SPLIT ? all * (int)blockIdx.y / t.splits : 0, end = SPLIT ? all * ((int)blockIdx.y + 1) / t.splits : all;
    half8_t next_left[2][KB][LR], next_right[2][KB][LC];
    auto fetch = [&](int k) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const i64 at = (i64)min(k + kb, end - 1) * 32;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
#pragma unroll
                for (int q = 0; q < LR; ++q) next_left[p][kb][q] = *(const half8_t*)((p ? left_lo : left_hi) + at * t.rows + STEP * q * 32);
#pragma unroll
                for (int q = 0; q < LC; ++q) next_right[p][kb][q] = *(const half8_t*)((p ? right_lo : right_hi) + at * t.columns + STEP * q * 32);
            }
        }
    };
    auto stage = [&](int buffer) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
#pragma unroll
                for (int q = 0; q < LR; ++q) *(half8_t*)&lds[buffer][p][K::place(lrow + STEP * q, kb * 4 + unit)] = next_left[p][kb][q];
#pragma unroll
                for (int q = 0; q < LC; ++q)
                    *(half8_t*)&lds[buffer][p][K::place(K::ROWS + lrow + STEP * q, kb * 4 + unit)] = next_right[p][kb][q];
            }
    };
    float4_t main[FR][FC], cross[FR][FC];
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int j = 0; j < FC; ++j) main[i][j] = cross[i][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const int row = wi * (FR * 16) + lane % 16, col = K::ROWS + wj * (FC * 16) + lane % 16, group = lane / 16;
    fetch(first);
    stage(0);
    fetch(first + KB);
    lds_barrier();
    int buffer = 0;
    for (int k = first; k < end; k += KB) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            if (KB > 1 && k + kb >= end) break;
            half8_t c[2][FC];
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int j = 0; j < FC; ++j) c[p][j] = *(const half8_t*)&lds[buffer][p][K::place(col + 16 * j, kb * 4 + group)];
#pragma unroll
            for (int i = 0; i < FR; ++i) {
                const half8_t hi = *(const half8_t*)&lds[buffer][0][K::place(row + 16 * i, kb * 4 + group)];
                const half8_t lo = *(const half8_t*)&lds[buffer][1][K::place(row + 16 * i, kb * 4 + group)];
#pragma unroll
                for (int j = 0; j < FC; ++j) {
                    main[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, c[0][j], main[i][j], 0, 0, 0);
                    cross[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, c[1][j], cross[i][j], 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < FC; ++j) cross[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, c[0][j], cross[i][j], 0, 0, 0);
            }
        }
        if (k + KB >= end) break;
        // the other buffer was read in the stage before this one, which every wave has left
        buffer ^= 1;
        stage(buffer);
        fetch(k + 2 * KB);
        lds_barrier();
    }
#pragma unroll
    for (int i = 0; i < FR; ++i) {
        const int r = ti * K::ROWS + wi * (FR * 16) + 16 * i + lane / 16 * 4;
        const int c0 = tj * K::COLUMNS + wj * (FC * 16) + lane % 16;
        Direct in[FC];  // a row of blocks at a time: the stores that follow could touch `in` for all the compiler knows
        if (!partial) {
#pragma unroll
            for (int j = 0; j < FC; ++j) in[j].template load<WHAT>(t, b, r, c0 + 16 * j);
        }
#pragma unroll
        for (int j = 0; j < FC; ++j) {
            const float4_t v = (main[i][j] + cross[i][j] * (1.0f / LOW)) * (1.0f / (SCALE * SCALE));
            if (partial)
                *(float4_t*)(partial + ((((b * t.splits + blockIdx.y) * gridDim.x + blockIdx.x) * (FR * FC) + i * FC + j) *
                                              K::THREADS + threadIdx.x) * 4) = v;
            else
                finish<WHAT>(t, b, r, c0 + 16 * j, v, product, in[j]);
        }
    }
}

// Adds a split product's sums in order; block row i of every wave of a tile per workgroup.
template <typename K, Product WHAT>
__global__ void __launch_bounds__(K::THREADS) ortho_join(Task t) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, wi = wave / K::WC, wj = wave % K::WC, i = blockIdx.y;
    const i64 b = blockIdx.z;
    int ti, tj;
    tile_of<K, WHAT>(blockIdx.x, t.rows, ti, tj);
    const int r = ti * K::ROWS + wi * (K::FR * 16) + 16 * i + lane / 16 * 4, c0 = tj * K::COLUMNS + wj * (K::FC * 16) + lane % 16;
    Direct in[K::FC];
    float4_t v[K::FC];
#pragma unroll
    for (int j = 0; j < K::FC; ++j) {
        in[j].template load<WHAT>(t, b, r, c0 + 16 * j);
        v[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < t.splits; ++s)
            v[j] += *(const float4_t*)(t.partial + ((((b * t.splits + s) * gridDim.x + blockIdx.x) * (K::FR * K::FC) + i * K::FC + j) *
                                                        K::THREADS + threadIdx.x) * 4);
    }
#pragma unroll
    for (int j = 0; j < K::FC; ++j) finish<WHAT>(t, b, r, c0 + 16 * j, v[j], t.product, in[j]);
}

// Tiles of 256 x 128 on eight waves keep the MFMAs fed from LDS (each value read serves 64 products); those of
// 64 x 64, and of 32 x 32 below 192 of these, spread small matrices over the CUs, where a stage's way from memory
// is what takes the time (all five steps, measured side by side, 64 / 32: 256 x 256 107 / 83 us, 768 x 768 218 / 176, 1024 x 1024 273 / 255;
// 32 for up to 400 tiles costs 1536 x 1536 563 instead of 525).
typedef Cut<256, 128, 4, 2, 32, true> Large;
typedef Cut<64, 64, 2, 2, 32, false> Small;
typedef Cut<32, 32, 2, 1, 64, false> Tiny;
constexpr i64 CUS = 256, FEW_TILES = 192;

struct Sizes {
    i64 m, n, mp, np;  // m <= n: the sides of X, and padded to whole tiles
    int large, transposed;
    int gram_splits, poly_splits;
};

int splits_of(i64 batch, i64 mp, i64 depth) {
    // a triangle of few tiles is split along the sum while that fills CUs; a part keeps 512 indices or more
    const i64 tiles = batch * Large::triangle(mp / Large::COLUMNS);
    return (int)std::max<i64>(1, std::min(CUS / tiles, depth / 512));
}

Sizes sizes_of(i64 batch, i64 rows, i64 columns) {
    Sizes s{};
    s.transposed = rows > columns;
    s.m = std::min(rows, columns);
    s.n = std::max(rows, columns);
    // a large tile per CU: below that the small ones win (4 x 1024 x 1024: 549 us against 649, 1536 x 1536: 525
    // against 700, 2048 x 2048: 904 against 896; with one, 2048 x 4096: 1143 us against 1487 with small tiles)
    s.large = batch * ceil_div(s.m, Large::ROWS) * ceil_div(s.n, Large::COLUMNS) >= CUS;
    const i64 side = s.large ? Large::ROWS : Small::ROWS;
    s.mp = ceil_div(s.m, side) * side;
    s.np = ceil_div(s.n, side) * side;
    s.gram_splits = s.large ? splits_of(batch, s.mp, s.np) : 1;
    s.poly_splits = s.large ? splits_of(batch, s.mp, s.mp) : 1;
    return s;
}

struct Buffers {
    double* partial;
    Planes x, xt[2], gram, poly;
    float* sums;
    i64 bytes;
};

// Carves the workspace: the norm's partial sums, two planes for each matrix, the sums of split products.
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
    const i64 splits = std::max(s.gram_splits, s.poly_splits);
    if (splits > 1) {
        w.sums = (float*)(base + at);
        at += batch * splits * Large::triangle(s.mp / Large::COLUMNS) * (Large::ROWS * Large::COLUMNS) * (i64)sizeof(float);
    }
    w.bytes = at;
    return w;
}

// Whether the iteration's matrices stay within what the planes hold (65504 / SCALE = 4094) for every source.  An entry is at
// most the largest singular value, which is |X|_F <= 1 at first.  With s up to `top`: X X^T has s^2, b A + c A A has
// b u + c u^2 with u = s^2, the next X has a s + b s^3 + c s^5; each is largest at an end or where its derivative is zero.
bool within_planes(int steps, const float* k) {
    constexpr double LIMIT = 4000.0;
    const double a = k[0], b = k[1], c = k[2];
    double top = 1.0;
    for (int i = 0; i < steps; ++i) {
        const double end = top * top;
        double poly = 0.0, next = 0.0;
        auto poly_at = [&](double u) {
            if (u >= 0.0 && u <= end) poly = std::max(poly, std::abs(u * (b + c * u)));
        };
        auto next_at = [&](double u) {
            if (u >= 0.0 && u <= end) next = std::max(next, std::abs(std::sqrt(u) * (a + u * (b + c * u))));
        };
        poly_at(end);
        next_at(end);
        if (c != 0.0) {
            poly_at(-b / (2.0 * c));
            const double root = std::sqrt(9.0 * b * b - 20.0 * a * c);  // NaN where there is none: in no range
            next_at((-3.0 * b + root) / (10.0 * c));
            next_at((-3.0 * b - root) / (10.0 * c));
        } else if (b != 0.0) {
            next_at(-a / (3.0 * b));
        }
        // the last X goes to the caller as it is
        if (!(end <= LIMIT && poly <= LIMIT && (i + 1 == steps || next <= LIMIT))) return false;
        top = next;
    }
    return true;
}

// The sizes that the products' grids and the 32-bit numbers of their tiles are made for.
bool in_range(i64 batch, i64 rows, i64 columns) {
    constexpr i64 LONG = 1 << 20, SHORT = 16384;
    return batch >= 1 && batch <= 65535 && rows >= 1 && columns >= 1 && rows <= LONG && columns <= LONG &&
           std::min(rows, columns) <= SHORT;
}

template <typename K, Product WHAT>
i64 tiles_of(const Task& t) {
    return WHAT == GRAM || WHAT == POLY ? K::triangle(t.columns / K::COLUMNS) : (i64)(t.rows / K::ROWS) * (t.columns / K::COLUMNS);
}

template <typename K, Product WHAT>
void multiply(Task t, i64 batch, int splits, float* sums, hipStream_t st) {
    if constexpr (std::is_same_v<K, Small>)
        if (batch * tiles_of<Small, WHAT>(t) < FEW_TILES) return multiply<Tiny, WHAT>(t, batch, 1, nullptr, st);
    const i64 tiles = tiles_of<K, WHAT>(t);
    t.splits = splits;
    t.partial = splits > 1 ? sums : nullptr;
    ortho_product<K, WHAT><<<dim3((unsigned)tiles, (unsigned)splits, (unsigned)batch), K::THREADS, 0, st>>>(t);
    if constexpr (K::SPLIT && (WHAT == GRAM || WHAT == POLY))
        if (splits > 1) ortho_join<K, WHAT><<<dim3((unsigned)tiles, K::FR, (unsigned)batch), K::THREADS, 0, st>>>(t);
}

template <typename K>
void iterate(const Sizes& s, const Buffers& w, i64 batch, int steps, const float* k, const Result& result, hipStream_t st) {
    const i64 wide = s.mp * s.np, square = s.mp * s.mp;
    const Planes none{nullptr, nullptr};
    const int m = (int)s.mp, n = (int)s.np;
    const Task gram{w.x, w.x, wide, wide, none, w.gram, w.gram, m, m, n, 0.0f, 1.0f, nullptr, 1, result};
    const Task poly{w.gram, w.gram, square, square, w.gram, w.poly, w.poly, m, m, m, k[1], k[2], nullptr, 1, result};
    for (int i = 0; i < steps; ++i) {
        const Planes from = w.xt[i % 2], to = w.xt[(i + 1) % 2];
        const Task apply{w.poly, from, square, wide, from, w.x, to, m, n, m, k[0], 1.0f, nullptr, 1, result};
        multiply<K, GRAM>(gram, batch, s.gram_splits, w.sums, st);
        multiply<K, POLY>(poly, batch, s.poly_splits, w.sums, st);
        if (i + 1 < steps) multiply<K, APPLY>(apply, batch, 1, nullptr, st);
        else multiply<K, FINAL>(apply, batch, 1, nullptr, st);
    }
}

}  // namespace
}  // namespace atlas_ops

using namespace atlas_ops;

extern "C" {

int64_t atlas_ops_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t columns) {
    if (!in_range(batch, rows, columns)) return 0;
    return carve(sizes_of(batch, rows, columns), batch, nullptr).bytes;
}

int atlas_ops_orthogonalize(const AtlasOrthogonal* o, void* workspace, void* stream, char* err, size_t cap) {
    try {
        if (!o) return fail(err, cap, 7, "null argument");
        if (!in_range(o->batch, o->rows, o->columns))
            return fail(err, cap, 7, "batch must be 1 to 65535, rows and columns 1 to 2^20 and one of them at most 16384");
        if (!o->matrix || !workspace || (!o->out) == (!o->weight)) return fail(err, cap, 7, "null argument");
        if (o->steps < 1 || o->steps > 64) return fail(err, cap, 7, "steps must be 1 to 64");
        for (const float k : o->coefficients)
            if (!std::isfinite(k)) return fail(err, cap, 7, "the coefficients must be finite");
        if (!within_planes(o->steps, o->coefficients))
            return fail(err, cap, 7, "the coefficients raise the iteration's matrices beyond 4000");
        if (!known_type(o->type) || (o->out && !known_type(o->out_type))) return fail(err, cap, 7, "unknown type");
        const Sizes s = sizes_of(o->batch, o->rows, o->columns);
        const Buffers w = carve(s, o->batch, (char*)workspace);
        hipStream_t st = (hipStream_t)stream;
        const Source source{o->matrix, o->rows, o->columns, o->batch_stride, o->row_stride, o->momentum, o->factor, o->nesterov};
        // a block of the norm's sum takes 1024 values or more, in whole rounds of its lanes
        const i64 span = ceil_div(std::max<i64>(1024, ceil_div(o->rows * o->columns, PARTIALS)), 256) * 256;
        const int parts = (int)ceil_div(o->rows * o->columns, span);
        const dim3 norm_grid((unsigned)parts, (unsigned)o->batch);
        const dim3 split_grid((unsigned)(s.np / 64), (unsigned)(s.mp / 64), (unsigned)o->batch);
        if (o->type == ATLAS_OPS_F32) {
            if (source.momentum) ortho_norm<float, true><<<norm_grid, 256, 0, st>>>(source, span, w.partial);
            else ortho_norm<float, false><<<norm_grid, 256, 0, st>>>(source, span, w.partial);
            ortho_split<float><<<split_grid, 256, 0, st>>>(source, s.transposed, parts, w.partial, o->eps, s.mp, s.np, w.x, w.xt[0]);
        } else {
            if (source.momentum) ortho_norm<bf16_t, true><<<norm_grid, 256, 0, st>>>(source, span, w.partial);
            else ortho_norm<bf16_t, false><<<norm_grid, 256, 0, st>>>(source, span, w.partial);
            ortho_split<bf16_t><<<split_grid, 256, 0, st>>>(source, s.transposed, parts, w.partial, o->eps, s.mp, s.np, w.x, w.xt[0]);
        }
        const Result result{o->rows, o->columns, o->out, o->weight, o->out_type, s.transposed, o->keep, o->rate};
        if (s.large) iterate<Large>(s, w, o->batch, o->steps, o->coefficients, result, st);
        else iterate<Small>(s, w, o->batch, o->steps, o->coefficients, result, st);
        return launched(err, cap, "orthogonalize");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

}  // extern "C"
