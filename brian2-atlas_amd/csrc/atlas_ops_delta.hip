// The gated delta rule: token by token for streaming, in chunks for sequences, and its gradients.
// Part of libatlas_ops_hip.so.
//
// By token: S <- a S, e = v - S^T k, S <- S + beta k e^T, out = scale S^T q.  In a chunk of C = 64 tokens
// that starts from S, with g_i = exp(G_i), G the sum of the log decays up to and with token i, and
// D_ij = exp(G_i - G_j) for j <= i:
//   (I + M B) E = V - g K S        M = strictly lower part of D o K K^T, B = diag(beta)
//   out = scale (g Q S + (lower part of D o Q K^T) B E)
//   S' = g_C S + K^T (rest B E)    rest_i = exp(G_C - G_i)
// so that a chunk costs matrix products and one triangular inverse T = (I + M B)^-1, which no
// state enters: `prepare` inverts for all chunks at once, `scan_forward` carries the states through the
// chunks, and `outputs` takes every chunk's outputs at once.  The columns of S do not touch each other,
// so a wave of the scan owns 16 of them.
//
// Backwards, with P = scale (lower part of D o Q K^T):
//   dV' = P^T dO + rest K dS',  Y = T^T B dV',  dV = Y,  dS = g_C dS' + scale Q^T g dO - K^T g Y
// carries dS through the chunks (`scan_backward`), and from S, dS', E and Y of every chunk `gradients`
// takes, with D1 = scale (lower part of D o dO E^T) and D2 = -(strictly lower part of D o Y E^T):
//   dQ = scale g dO S^T + D1 B K
//   dK = r + B w,   r = -g Y S^T + D2 B K,   w = rest E dS'^T + D1^T Q + D2^T K
//   dbeta_i = k_i . w_i
//   dG_i = q_i . dQ_i + k_i . r_i - beta_i dbeta_i (+ <dS', S'> at the chunk's last token),
// as every factor exp(G_i) comes with q_i or the k_i that reads, and every exp(-G_i) with the k_i that
// writes; dlog_decay sums dG from the token to the chunk's end.
#include <algorithm>

#include "device/atlas_ops.h"

namespace atlas_ops {
namespace {

constexpr int C = 64;         // tokens per chunk
constexpr int CP = C + 4;     // pitch of a C x C matrix in LDS
constexpr float LOWEST = -120.0f;

struct Tensor {
    const void* data;
    i64 batch, time, head;
    template <typename T>
    __device__ __forceinline__ const T* at(i64 b, i64 t, i64 h) const {
        return (const T*)data + b * batch + t * time + h * head;
    }
};

struct Delta {
    Tensor q, k, v, decay, beta;
    const float* state;
    const int32_t* lengths;
    i64 batch, time, heads, value_heads;
    int key, value, group, decay_bf16, beta_bf16;
    i64 chunks, padded;  // padded: value in whole blocks of 16
    float scale;

    __device__ __forceinline__ i64 length(i64 b) const {
        if (!lengths) return time;
        const i64 n = lengths[b];
        return n < 0 ? 0 : n < time ? n : time;
    }
    __device__ __forceinline__ float log_decay(i64 b, i64 t, i64 h) const {
        if (!decay.data) return 0.0f;
        const float g = decay_bf16 ? to_float(*decay.at<bf16_t>(b, t, h)) : *decay.at<float>(b, t, h);
        return g < LOWEST ? LOWEST : g;  // a NaN stays one
    }
    __device__ __forceinline__ float rate(i64 b, i64 t, i64 h) const {
        return beta_bf16 ? to_float(*beta.at<bf16_t>(b, t, h)) : *beta.at<float>(b, t, h);
    }
};

// Four values from column c of a row of `width`, zeros beyond it.  No alignment is needed.
template <typename T>
__device__ __forceinline__ float4_t load4(const T* row, int c, int width) {
    float4_t v;
    if (c + 4 <= width) {
        struct __attribute__((packed, aligned(sizeof(T)))) { T v[4]; } raw;
        __builtin_memcpy(&raw, row + c, sizeof(raw));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_float(raw.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = c + i < width ? to_float(row[c + i]) : 0.0f;
    }
    return v;
}

// ------------------------------------------------------------------ token by token
// A workgroup holds 32 columns of one head's state in registers: row groups of 32 / VEC lanes, each lane
// VEC neighbouring columns of every 8 VEC-th row.  One reduction per token: S^T k and S^T q of the
// decayed state and k . q, as out = scale ((a S)^T q + beta e (k . q)).
constexpr int MAX_KEY = 128;

template <typename T, int VEC>
__global__ void __launch_bounds__(256) step_kernel(Delta d, T* __restrict__ out, float* final_state) {
    constexpr int LANES = 32 / VEC, ROWS = 256 / LANES, PER = MAX_KEY / ROWS;
    __shared__ float sums[2][4][32], dots[2][4];
    const int lane = threadIdx.x % LANES, row = threadIdx.x / LANES, wave = threadIdx.x / 64;
    const i64 b = blockIdx.z, h = blockIdx.y, hk = h / d.group;
    const int col = blockIdx.x * 32 + lane * VEC;
    const i64 base = (b * d.value_heads + h) * d.key * d.value;
    float s[PER][VEC];
#pragma unroll
    for (int r = 0; r < PER; ++r) {
        const int at = row + r * ROWS;
#pragma unroll
        for (int c = 0; c < VEC; ++c) s[r][c] = 0.0f;
        if (d.state && at < d.key && col < d.value) {
            if constexpr (VEC == 4) {  // value is a multiple of 4
                const float4_t v = *(const float4_t*)(d.state + base + (i64)at * d.value + col);
#pragma unroll
                for (int c = 0; c < VEC; ++c) s[r][c] = v[c];
            } else {
                s[r][0] = d.state[base + (i64)at * d.value + col];
            }
        }
    }
    const i64 length = d.length(b);
    for (i64 t = 0; t < d.time; ++t) {
        T* o = out + ((b * d.time + t) * d.value_heads + h) * d.value;
        if (t >= length) {
            if (row == 0)
                for (int c = 0; c < VEC; ++c)
                    if (col + c < d.value) o[col + c] = from_float<T>(0.0f);
            continue;
        }
        const T *qp = d.q.at<T>(b, t, hk), *kp = d.k.at<T>(b, t, hk), *vp = d.v.at<T>(b, t, h);
        const float a = expf(d.log_decay(b, t, h)), rate = d.rate(b, t, h);
        float v[VEC];
#pragma unroll
        for (int c = 0; c < VEC; ++c) v[c] = col + c < d.value ? to_float(vp[col + c]) : 0.0f;
        float kr[PER], qr[PER], ks[VEC], qs[VEC], kq = 0.0f;
#pragma unroll
        for (int c = 0; c < VEC; ++c) ks[c] = qs[c] = 0.0f;
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            const int at = row + r * ROWS;
            kr[r] = at < d.key ? to_float(kp[at]) : 0.0f;
            qr[r] = at < d.key ? to_float(qp[at]) : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            kq += kr[r] * qr[r];
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                s[r][c] *= a;
                ks[c] += s[r][c] * kr[r];
                qs[c] += s[r][c] * qr[r];
            }
        }
#pragma unroll
        for (int step = LANES; step < 64; step *= 2) {
            kq += __shfl_xor(kq, step, 64);
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                ks[c] += __shfl_xor(ks[c], step, 64);
                qs[c] += __shfl_xor(qs[c], step, 64);
            }
        }
        __syncthreads();  // the previous token's sums are read
        if (threadIdx.x % 64 < LANES) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                sums[0][wave][lane * VEC + c] = ks[c];
                sums[1][wave][lane * VEC + c] = qs[c];
            }
            if (lane == 0) dots[0][wave] = kq;
        }
        __syncthreads();
        kq = (dots[0][0] + dots[0][1]) + (dots[0][2] + dots[0][3]);
        float e[VEC];
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
            const int at = lane * VEC + c;
            const float k_sum = (sums[0][0][at] + sums[0][1][at]) + (sums[0][2][at] + sums[0][3][at]);
            const float q_sum = (sums[1][0][at] + sums[1][1][at]) + (sums[1][2][at] + sums[1][3][at]);
            e[c] = rate * (v[c] - k_sum);
            if (row == 0 && col + c < d.value) o[col + c] = from_float<T>(d.scale * (q_sum + e[c] * kq));
        }
#pragma unroll
        for (int r = 0; r < PER; ++r)
#pragma unroll
            for (int c = 0; c < VEC; ++c) s[r][c] += kr[r] * e[c];
    }
#pragma unroll
    for (int r = 0; r < PER; ++r) {
        const int at = row + r * ROWS;
        if (at >= d.key || col >= d.value) continue;
        float* p = final_state + base + (i64)at * d.value + col;
        if constexpr (VEC == 4) {
            float4_t v;
#pragma unroll
            for (int c = 0; c < VEC; ++c) v[c] = s[r][c];
            *(float4_t*)p = v;
        } else {
            *p = s[r][0];
        }
    }
}

// ------------------------------------------------------------------ what the chunk kernels share
// Float32 MFMA blocks of 16 x 16 with 4 sum indices: lane l gives A[l % 16][l / 16] and B[l / 16][l % 16]
// and receives rows 4 (l / 16) + j, column l % 16.  The sum may take its indices in any order that A and B
// share, so a block of results is the B operand of a following product as it is: register j holds
// the indices 4 (l / 16) + j of 16, and A gives the same ones (one 16-byte read of a row).
__device__ __forceinline__ float4_t mfma(float a, float b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// c += A B over 16 sum indices, `a` and `b` in the order above.
__device__ __forceinline__ float4_t mfma16(float4_t a, float4_t b, float4_t c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = mfma(a[j], b[j], c);
    return c;
}

constexpr float4_t ZERO = {0.0f, 0.0f, 0.0f, 0.0f};

struct Lane {
    int col, quad;  // l % 16, 4 (l / 16)
    __device__ __forceinline__ Lane() : col(threadIdx.x % 16), quad(threadIdx.x % 64 / 16 * 4) {}
    // operand from rows: row `col` of the block at `m`, columns quad ..
    __device__ __forceinline__ float4_t row(const float* m, int pitch) const {
        return *(const float4_t*)(m + col * pitch + quad);
    }
    // operand from columns: column `col` of the block at `m`, rows quad ..
    __device__ __forceinline__ float4_t column(const float* m, int pitch) const {
        float4_t v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = m[(quad + j) * pitch + col];
        return v;
    }
};

// A product with a triangular matrix adds zeros times the terms it masks, which a NaN or an infinity
// there turns into NaNs of earlier tokens.  So where a wave finds any among the 64 tokens of its columns
// (one FMA per value says so), it takes them out before the product and marks the rows from the first
// on as NaN after it: a token's fault reaches its own and later tokens only.
struct Faults {
    int first;
    __device__ __forceinline__ Faults(const Lane& l, float4_t (&v)[4]) : first(C) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = fmaf(v[i][e], 0.0f, sum);
        if (__ballot(sum != sum)) {
#pragma unroll
            for (int i = 3; i >= 0; --i)
#pragma unroll
                for (int e = 3; e >= 0; --e)
                    if (!(fabsf(v[i][e]) < INFINITY)) {
                        v[i][e] = 0.0f;
                        first = 16 * i + l.quad + e;
                    }
            first = min(first, __shfl_xor(first, 16, 64));
            first = min(first, __shfl_xor(first, 32, 64));
        }
    }
    __device__ __forceinline__ float mark(int row, float v) const { return row < first ? v : NAN; }
};

// A chunk's decays: the running sums in 64 bits, as differences of large sums lose what a small
// decay adds; kept as a float and its remainder.
struct Gates {
    float sum[C], remainder[C], since[C], rest[C], beta[C];

    // By the workgroup's first wave; the caller synchronises.
    __device__ __forceinline__ void load(const Delta& d, i64 b, i64 h, i64 n, i64 length) {
        if (threadIdx.x >= 64) return;
        const int i = threadIdx.x;
        const i64 t = n * C + i;
        double g = t < length ? (double)d.log_decay(b, t, h) : 0.0;
#pragma unroll
        for (int s = 1; s < 64; s *= 2) {
            const double below = __shfl_up(g, s, 64);
            if (i >= s) g += below;
        }
        const double last = __shfl(g, 63, 64);
        sum[i] = (float)g;
        remainder[i] = (float)(g - (double)sum[i]);
        since[i] = expf((float)g);
        rest[i] = expf((float)(last - g));
        beta[i] = t < length ? d.rate(b, t, h) : 0.0f;
    }
    __device__ __forceinline__ float decay(int i, int j) const {
        return expf((sum[i] - sum[j]) + (remainder[i] - remainder[j]));
    }
};

// A chunk's keys or queries as floats in LDS, zero beyond the key width and the sequence.
template <typename T, int DK>
__device__ __forceinline__ void load_chunk(float* lds, const Tensor& x, i64 b, i64 h, i64 n, i64 length, int width) {
    constexpr int UNITS = DK / 4;
#pragma unroll 4
    for (int u = threadIdx.x; u < C * UNITS; u += 256) {
        const int i = u / UNITS, c = u % UNITS * 4;
        const i64 t = n * C + i;
        float4_t v = ZERO;
        if (t < length && c < width) v = load4(x.at<T>(b, t, h), c, width);
        *(float4_t*)(lds + i * (DK + 4) + c) = v;
    }
}

// Workspace positions of head (b, h), chunk n, in floats.
struct Tape {
    float *inverse, *scores, *errors, *states;
    __device__ __forceinline__ i64 chunk(const Delta& d, i64 b, i64 h, i64 n) const {
        return (b * d.value_heads + h) * d.chunks + n;
    }
};

// ------------------------------------------------------------------ T = (I + M B)^-1 of every chunk
template <typename T, int DK>
__global__ void __launch_bounds__(256) prepare(Delta d, Tape tape) {
    constexpr int P = DK + 4;
    __shared__ __attribute__((aligned(16))) float k[C * P], low[C * CP], inv[C * CP];
    __shared__ Gates gates;
    __shared__ int faulty;  // the first row with a NaN or an infinity; it and those after it become NaN
    const i64 n = blockIdx.x, h = blockIdx.y, b = blockIdx.z, length = d.length(b);
    const int wave = threadIdx.x / 64;
    const Lane l;
    if (threadIdx.x == 0) faulty = C;
    gates.load(d, b, h, n, length);
    load_chunk<T, DK>(k, d.k, b, h / d.group, n, length, d.key);
    for (int e = threadIdx.x; e < C * CP; e += 256) inv[e] = 0.0f;
    __syncthreads();
    for (int j = 0; j <= wave; ++j) {
        float4_t acc = ZERO;
#pragma unroll 8
        for (int f = 0; f < DK / 16; ++f)
            acc = mfma16(l.row(k + 16 * wave * P + 16 * f, P), l.row(k + 16 * j * P + 16 * f, P), acc);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 16 * wave + l.quad + e, c = 16 * j + l.col;
            float v = r > c ? acc[e] * gates.decay(r, c) * gates.beta[c] : 0.0f;
            if (!(fabsf(v) < INFINITY)) {
                atomicMin(&faulty, r);
                v = 0.0f;
            }
            low[r * CP + c] = v;
        }
    }
    __syncthreads();
    // the diagonal blocks' inverses by forward substitution, a column per lane
    if (threadIdx.x % 64 < 16) {
        const float* m = low + 16 * wave * (CP + 1);
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float v = i == l.col ? 1.0f : 0.0f;
#pragma unroll
            for (int j = 0; j < i; ++j) v -= m[i * CP + j] * x[j];
            x[i] = v;
            inv[(16 * wave + i) * CP + 16 * wave + l.col] = v;
        }
    }
    __syncthreads();
    // the inverse of [[a, 0], [m, c]] has -c^-1 m a^-1 below: blocks of 16, then of 32
    if (wave < 2) {
        float* corner = inv + (32 * wave + 16) * CP + 32 * wave;
        const float4_t x = mfma16(l.row(low + (32 * wave + 16) * CP + 32 * wave, CP),
                                  l.column(inv + 32 * wave * (CP + 1), CP), ZERO);
        const float4_t y = mfma16(l.row(corner + 16, CP), x, ZERO);
#pragma unroll
        for (int e = 0; e < 4; ++e) corner[(l.quad + e) * CP + l.col] = -y[e];
    }
    __syncthreads();
    if (wave < 2) {  // column block `wave` of the lower left 32 x 32
        float4_t x[2], y[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = ZERO;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                x[i] = mfma16(l.row(low + (32 + 16 * i) * CP + 16 * j, CP), l.column(inv + 16 * j * CP + 16 * wave, CP), x[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            y[i] = ZERO;
#pragma unroll
            for (int j = 0; j < 2; ++j) y[i] = mfma16(l.row(inv + (32 + 16 * i) * CP + 32 + 16 * j, CP), x[j], y[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) inv[(32 + 16 * i + l.quad + e) * CP + 16 * wave + l.col] = -y[i][e];
        }
    }
    __syncthreads();
    float* to = tape.inverse + tape.chunk(d, b, h, n) * C * C;
    for (int u = threadIdx.x; u < C * C / 4; u += 256) {
        const float4_t row = *(const float4_t*)(inv + u / 16 * CP + u % 16 * 4);
        *(float4_t*)(to + 4 * u) = u / 16 < faulty ? row : float4_t{NAN, NAN, NAN, NAN};
    }
}

// ------------------------------------------------------------------ the states through the chunks
template <typename T, int DK>
__global__ void __launch_bounds__(256) scan_forward(Delta d, Tape tape, float* __restrict__ final_state) {
    constexpr int P = DK + 4, F = DK / 16;
    __shared__ __attribute__((aligned(16))) float k[C * P], inv[C * CP];
    __shared__ Gates gates;
    const i64 h = blockIdx.y, b = blockIdx.z, length = d.length(b);
    const int wave = threadIdx.x / 64;
    const Lane l;
    const int first = blockIdx.x * 64 + 16 * wave, col = first + l.col;
    const bool works = first < d.padded, live = col < d.value;
    float4_t s[F];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 16 * f + l.quad + e;
            s[f][e] = d.state && r < d.key && live
                          ? d.state[((b * d.value_heads + h) * d.key + r) * d.value + col] : 0.0f;
        }
    for (i64 n = 0; n < d.chunks; ++n) {
        const i64 chunk = tape.chunk(d, b, h, n);
        __syncthreads();  // the previous chunk's LDS is read
        gates.load(d, b, h, n, length);
        load_chunk<T, DK>(k, d.k, b, h / d.group, n, length, d.key);
        for (int u = threadIdx.x; u < C * C / 4; u += 256)
            *(float4_t*)(inv + u / 16 * CP + u % 16 * 4) = *(const float4_t*)(tape.inverse + chunk * C * C + 4 * u);
        __syncthreads();
        if (!works) continue;
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                tape.states[(chunk * DK + 16 * f + l.quad + e) * d.padded + col] = s[f][e];
        // R = V - g K S, then E = T R
        float4_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float4_t acc = ZERO;
#pragma unroll
            for (int f = 0; f < F; ++f) acc = mfma16(l.row(k + 16 * i * P + 16 * f, P), s[f], acc);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * i + l.quad + e;
                const i64 t = n * C + row;
                const float v = t < length && live ? to_float(d.v.at<T>(b, t, h)[col]) : 0.0f;
                r[i][e] = v - gates.since[row] * acc[e];
            }
        }
        const Faults faults(l, r);
        float4_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float4_t acc = ZERO;
#pragma unroll
            for (int j = 0; j <= i; ++j) acc = mfma16(l.row(inv + 16 * i * CP + 16 * j, CP), r[j], acc);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * i + l.quad + e;
                acc[e] = faults.mark(row, acc[e]);
                tape.errors[(chunk * C + row) * d.padded + col] = acc[e];
                w[i][e] = acc[e] * gates.rest[row] * gates.beta[row];
            }
        }
        const float fade = gates.since[C - 1];
#pragma unroll
        for (int f = 0; f < F; ++f) {
            s[f] *= fade;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[f] = mfma16(l.column(k + 16 * i * P + 16 * f, P), w[i], s[f]);
        }
    }
    if (!works || !live) return;
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 16 * f + l.quad + e;
            if (r < d.key) final_state[((b * d.value_heads + h) * d.key + r) * d.value + col] = s[f][e];
        }
}

// ------------------------------------------------------------------ every chunk's outputs
template <typename T, int DK>
__global__ void __launch_bounds__(256) outputs(Delta d, Tape tape, T* __restrict__ out) {
    constexpr int P = DK + 4, F = DK / 16;
    __shared__ __attribute__((aligned(16))) float q[C * P], k[C * P], scores[C * CP];
    __shared__ Gates gates;
    const i64 n = blockIdx.x, h = blockIdx.y, b = blockIdx.z, length = d.length(b);
    const i64 chunk = tape.chunk(d, b, h, n);
    const int wave = threadIdx.x / 64;
    const Lane l;
    gates.load(d, b, h, n, length);
    load_chunk<T, DK>(q, d.q, b, h / d.group, n, length, d.key);
    load_chunk<T, DK>(k, d.k, b, h / d.group, n, length, d.key);
    __syncthreads();
    for (int j = 0; j < 4; ++j) {
        float4_t acc = ZERO;
        if (j <= wave) {
#pragma unroll 8
            for (int f = 0; f < F; ++f)
                acc = mfma16(l.row(q + 16 * wave * P + 16 * f, P), l.row(k + 16 * j * P + 16 * f, P), acc);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 16 * wave + l.quad + e, c = 16 * j + l.col;
            const float p = r >= c ? d.scale * acc[e] * gates.decay(r, c) : 0.0f;
            scores[r * CP + c] = p;
            if (tape.scores) tape.scores[chunk * C * C + r * C + c] = p;
        }
    }
    __syncthreads();
    for (int first = 16 * wave; first < d.padded; first += 64) {
        const int col = first + l.col;
        float4_t acc[4] = {ZERO, ZERO, ZERO, ZERO};
#pragma unroll
        for (int f = 0; f < F; ++f) {
            float4_t s;
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = tape.states[(chunk * DK + 16 * f + l.quad + e) * d.padded + col];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = mfma16(l.row(q + 16 * i * P + 16 * f, P), s, acc[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] *= d.scale * gates.since[16 * i + l.quad + e];
        float4_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * j + l.quad + e;
                w[j][e] = gates.beta[row] * tape.errors[(chunk * C + row) * d.padded + col];
            }
        const Faults faults(l, w);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = j; i < 4; ++i) acc[i] = mfma16(l.row(scores + 16 * i * CP + 16 * j, CP), w[j], acc[i]);
        if (col >= d.value) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const i64 t = n * C + 16 * i + l.quad + e;
                if (t < d.time)
                    out[((b * d.time + t) * d.value_heads + h) * d.value + col] =
                        from_float<T>(t < length ? faults.mark(16 * i + l.quad + e, acc[i][e]) : 0.0f);
            }
    }
}

// ------------------------------------------------------------------ the states' gradients backwards
struct Back {
    Tensor grad;              // of out
    const float* grad_state;  // of the final state, or NULL
    float *residuals;         // Y
    float *states;            // dS' of every chunk
};

template <typename T, int DK>
__global__ void __launch_bounds__(256) scan_backward(Delta d, Tape tape, Back back, T* __restrict__ dv,
                                                     float* __restrict__ dstate) {
    constexpr int P = DK + 4, F = DK / 16;
    __shared__ __attribute__((aligned(16))) float k[C * P], q[C * P], inv[C * CP], scores[C * CP];
    __shared__ Gates gates;
    const i64 h = blockIdx.y, b = blockIdx.z, length = d.length(b);
    const int wave = threadIdx.x / 64;
    const Lane l;
    const int first = blockIdx.x * 64 + 16 * wave, col = first + l.col;
    const bool works = first < d.padded, live = col < d.value;
    float4_t s[F];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 16 * f + l.quad + e;
            s[f][e] = back.grad_state && r < d.key && live
                          ? back.grad_state[((b * d.value_heads + h) * d.key + r) * d.value + col] : 0.0f;
        }
    for (i64 n = d.chunks; n-- > 0;) {
        const i64 chunk = tape.chunk(d, b, h, n);
        __syncthreads();
        gates.load(d, b, h, n, length);
        load_chunk<T, DK>(k, d.k, b, h / d.group, n, length, d.key);
        load_chunk<T, DK>(q, d.q, b, h / d.group, n, length, d.key);
        for (int u = threadIdx.x; u < C * C / 4; u += 256) {
            *(float4_t*)(inv + u / 16 * CP + u % 16 * 4) = *(const float4_t*)(tape.inverse + chunk * C * C + 4 * u);
            *(float4_t*)(scores + u / 16 * CP + u % 16 * 4) = *(const float4_t*)(tape.scores + chunk * C * C + 4 * u);
        }
        __syncthreads();
        if (!works) continue;
        float4_t o[4], u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const i64 t = n * C + 16 * i + l.quad + e;
                o[i][e] = t < length && live ? to_float(back.grad.at<T>(b, t, h)[col]) : 0.0f;
            }
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                back.states[(chunk * DK + 16 * f + l.quad + e) * d.padded + col] = s[f][e];
        // B dV' = B (P^T dO + rest K dS')
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float4_t acc = ZERO;
#pragma unroll
            for (int f = 0; f < F; ++f) acc = mfma16(l.row(k + 16 * i * P + 16 * f, P), s[f], acc);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] *= gates.rest[16 * i + l.quad + e];
#pragma unroll
            for (int j = i; j < 4; ++j) acc = mfma16(l.column(scores + 16 * j * CP + 16 * i, CP), o[j], acc);
#pragma unroll
            for (int e = 0; e < 4; ++e) u[i][e] = acc[e] * gates.beta[16 * i + l.quad + e];
        }
        const float fade = gates.since[C - 1];
#pragma unroll
        for (int f = 0; f < F; ++f) s[f] *= fade;
        // Y = T^T B dV', and both products into dS
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float4_t acc = ZERO;
#pragma unroll
            for (int j = i; j < 4; ++j) acc = mfma16(l.column(inv + 16 * j * CP + 16 * i, CP), u[j], acc);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * i + l.quad + e;
                const i64 t = n * C + row;
                back.residuals[(chunk * C + row) * d.padded + col] = acc[e];
                if (t < d.time && live)
                    dv[((b * d.time + t) * d.value_heads + h) * d.value + col] = from_float<T>(t < length ? acc[e] : 0.0f);
                acc[e] *= -gates.since[row];
                o[i][e] *= d.scale * gates.since[row];
            }
#pragma unroll
            for (int f = 0; f < F; ++f) {
                s[f] = mfma16(l.column(k + 16 * i * P + 16 * f, P), acc, s[f]);
                s[f] = mfma16(l.column(q + 16 * i * P + 16 * f, P), o[i], s[f]);
            }
        }
    }
    if (!dstate || !works || !live) return;
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 16 * f + l.quad + e;
            if (r < d.key) dstate[((b * d.value_heads + h) * d.key + r) * d.value + col] = s[f][e];
        }
}

// ------------------------------------------------------------------ every chunk's gradients
// One workgroup per chunk and key head; it visits the value heads that share the key head one after the
// other, so their sums into dq and dk need no atomics.  Wave w holds the tokens 16 w .. 16 w + 15.
template <typename T, int DK>
__global__ void __launch_bounds__(256) gradients(Delta d, Tape tape, Back back, T* __restrict__ dq, T* __restrict__ dk,
                                                 void* __restrict__ ddecay, void* __restrict__ dbeta) {
    constexpr int P = DK + 4, F = DK / 16;
    __shared__ __attribute__((aligned(16))) float q[C * P], k[C * P], d1[C * CP], d2[C * CP];
    __shared__ float line[C], part[4];
    __shared__ Gates gates;
    const i64 n = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, length = d.length(b);
    const int wave = threadIdx.x / 64, token = 16 * wave;
    const Lane l;
    load_chunk<T, DK>(q, d.q, b, hk, n, length, d.key);
    load_chunk<T, DK>(k, d.k, b, hk, n, length, d.key);
    float4_t gq[F], gk[F];
#pragma unroll
    for (int f = 0; f < F; ++f) gq[f] = gk[f] = ZERO;
    for (int member = 0; member < d.group; ++member) {
        const i64 h = hk * d.group + member, chunk = tape.chunk(d, b, h, n);
        __syncthreads();
        gates.load(d, b, h, n, length);
        __syncthreads();
        float4_t reads[F], backs[F], writes[F], oe[4], ye[4];  // dO S^T, Y S^T, E dS'^T, dO E^T, Y E^T
#pragma unroll
        for (int f = 0; f < F; ++f) reads[f] = backs[f] = writes[f] = ZERO;
#pragma unroll
        for (int j = 0; j < 4; ++j) oe[j] = ye[j] = ZERO;
        float carried = 0.0f;  // this wave's share of <dS', S>
        const float* errors = tape.errors + chunk * C * d.padded;
        const float* residuals = back.residuals + chunk * C * d.padded;
        const i64 t = n * C + token + l.col;
        for (int c = 0; c < d.padded; c += 16) {
            float4_t o = ZERO;
            if (t < length) o = load4(back.grad.at<T>(b, t, h), c + l.quad, d.value);
            const float4_t y = *(const float4_t*)(residuals + (token + l.col) * d.padded + c + l.quad);
            const float4_t e = *(const float4_t*)(errors + (token + l.col) * d.padded + c + l.quad);
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const i64 at = (chunk * DK + 16 * f + l.col) * d.padded + c + l.quad;
                const float4_t s = *(const float4_t*)(tape.states + at), ds = *(const float4_t*)(back.states + at);
                reads[f] = mfma16(o, s, reads[f]);
                backs[f] = mfma16(y, s, backs[f]);
                writes[f] = mfma16(e, ds, writes[f]);
                if (f % 4 == wave) carried += (s[0] * ds[0] + s[1] * ds[1]) + (s[2] * ds[2] + s[3] * ds[3]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j > wave) continue;
                const float4_t other = *(const float4_t*)(errors + (16 * j + l.col) * d.padded + c + l.quad);
                oe[j] = mfma16(o, other, oe[j]);
                ye[j] = mfma16(y, other, ye[j]);
            }
        }
        carried = lane_sum<64>(carried);
        if (threadIdx.x % 64 == 0) part[wave] = carried;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = token + l.quad + e, c = 16 * j + l.col;
                const float decay = r >= c ? gates.decay(r, c) : 0.0f;
                d1[r * CP + c] = r >= c ? d.scale * decay * oe[j][e] : 0.0f;
                d2[r * CP + c] = r > c ? -decay * ye[j][e] : 0.0f;
            }
        __syncthreads();
        float4_t written = ZERO;  // per row, k . rest B E dS'^T: its sum and <dS', S> make <dS', S'>
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = token + l.quad + e;
                reads[f][e] *= d.scale * gates.since[r];
                backs[f][e] *= -gates.since[r];
                writes[f][e] *= gates.rest[r];
                written[e] += k[r * P + 16 * f + l.col] * writes[f][e] * gates.beta[r];
            }
        for (int j = 0; j <= wave; ++j) {
            const float4_t a1 = l.row(d1 + token * CP + 16 * j, CP), a2 = l.row(d2 + token * CP + 16 * j, CP);
#pragma unroll
            for (int f = 0; f < F; ++f) {
                float4_t kj = l.column(k + 16 * j * P + 16 * f, P);
#pragma unroll
                for (int e = 0; e < 4; ++e) kj[e] *= gates.beta[16 * j + l.quad + e];
                reads[f] = mfma16(a1, kj, reads[f]);
                backs[f] = mfma16(a2, kj, backs[f]);
            }
        }
        for (int j = wave; j < 4; ++j) {
            const float4_t a1 = l.column(d1 + 16 * j * CP + token, CP), a2 = l.column(d2 + 16 * j * CP + token, CP);
#pragma unroll
            for (int f = 0; f < F; ++f) {
                writes[f] = mfma16(a1, l.column(q + 16 * j * P + 16 * f, P), writes[f]);
                writes[f] = mfma16(a2, l.column(k + 16 * j * P + 16 * f, P), writes[f]);
            }
        }
        float4_t db = ZERO, dg = ZERO;
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = token + l.quad + e;
                const float kv = k[r * P + 16 * f + l.col], qv = q[r * P + 16 * f + l.col];
                db[e] += kv * writes[f][e];
                dg[e] += qv * reads[f][e] + kv * backs[f][e];
                gq[f][e] += reads[f][e];
                gk[f][e] += backs[f][e] + gates.beta[r] * writes[f][e];
            }
        float ends = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = token + l.quad + e;
            db[e] = lane_sum<16>(db[e]);
            dg[e] = lane_sum<16>(dg[e]) - gates.beta[r] * db[e];
            ends += written[e];
            const i64 at = n * C + r;
            if (l.col == 0) {
                line[r] = dg[e];
                if (at < d.time) {
                    const i64 to = (b * d.time + at) * d.value_heads + h;
                    const float v = at < length ? db[e] : 0.0f;
                    if (d.beta_bf16) ((bf16_t*)dbeta)[to] = from_float<bf16_t>(v);
                    else ((float*)dbeta)[to] = v;
                }
            }
        }
        ends = lane_sum<64>(ends);
        if (threadIdx.x % 64 == 0) part[wave] = gates.since[C - 1] * part[wave] + ends;
        __syncthreads();
        if (ddecay && threadIdx.x < 64) {
            const int i = threadIdx.x;
            float v = line[i];
            if (i == C - 1) v += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
            for (int s = 1; s < 64; s *= 2) {
                const float above = __shfl_down(v, s, 64);
                if (i + s < 64) v += above;
            }
            const i64 at = n * C + i;
            if (at < d.time) {
                const i64 to = (b * d.time + at) * d.value_heads + h;
                if (at >= length) v = 0.0f;
                if (d.decay_bf16) ((bf16_t*)ddecay)[to] = from_float<bf16_t>(v);
                else ((float*)ddecay)[to] = v;
            }
        }
    }
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const i64 t = n * C + token + l.quad + e;
            const int c = 16 * f + l.col;
            if (t >= d.time || c >= d.key) continue;
            const i64 to = ((b * d.time + t) * d.heads + hk) * d.key + c;
            dq[to] = from_float<T>(t < length ? gq[f][e] : 0.0f);
            dk[to] = from_float<T>(t < length ? gk[f][e] : 0.0f);
        }
}

// ------------------------------------------------------------------ host
Tensor tensor(const void* p, const int64_t* s) { return Tensor{p, s[0], s[1], s[2]}; }

int check(const AtlasDelta* a, Delta& d, char* err, size_t cap) {
    if (!a) return fail(err, cap, 7, "null argument");
    if (a->batch < 1 || a->time < 1 || a->heads < 1 || a->value_heads < 1 || a->value < 1)
        return fail(err, cap, 7, "every size must be positive");
    if (a->key < 1 || a->key > MAX_KEY) return fail(err, cap, 7, "key must be 1 to %d", MAX_KEY);
    if (a->value_heads % a->heads) return fail(err, cap, 7, "value_heads must be a multiple of heads");
    if (a->batch > 65535 || a->value_heads > 65535 || a->time > 0x7FFFFFFF - C || a->value > (1 << 20))
        return fail(err, cap, 7, "batch and value_heads must be at most 65535, time below 2^31 - 64, value at most 2^20");
    if (!known_type(a->type) || !known_type(a->log_decay_type) || !known_type(a->beta_type))
        return fail(err, cap, 7, "unknown type");
    if (!a->q || !a->k || !a->v || !a->beta) return fail(err, cap, 7, "null argument");
    d = Delta{};
    d.q = tensor(a->q, a->q_stride);
    d.k = tensor(a->k, a->k_stride);
    d.v = tensor(a->v, a->v_stride);
    d.decay = tensor(a->log_decay, a->log_decay_stride);
    d.beta = tensor(a->beta, a->beta_stride);
    d.state = a->state;
    d.lengths = a->lengths;
    d.batch = a->batch, d.time = a->time, d.heads = a->heads, d.value_heads = a->value_heads;
    d.key = (int)a->key, d.value = (int)a->value, d.group = (int)(a->value_heads / a->heads);
    d.decay_bf16 = a->log_decay_type == ATLAS_OPS_BF16, d.beta_bf16 = a->beta_type == ATLAS_OPS_BF16;
    d.chunks = ceil_div(a->time, C);
    d.padded = ceil_div(a->value, 16) * 16;
    d.scale = a->scale;
    return 0;
}

int key_width(const Delta& d) { return d.key <= 64 ? 64 : 128; }

i64 carve(const Delta& d, int train, char* base, Tape* tape) {
    const i64 chunks = d.batch * d.value_heads * d.chunks;
    i64 at = 0;
    auto floats = [&](i64 n) {
        float* p = (float*)(base + at);
        at += n * (i64)sizeof(float);
        return p;
    };
    Tape t{};
    t.inverse = floats(chunks * C * C);
    t.errors = floats(chunks * C * d.padded);
    t.states = floats(chunks * key_width(d) * d.padded);
    if (train) t.scores = floats(chunks * C * C);
    if (tape) *tape = t;
    return at;
}

template <typename F>
void with_kernel(const Delta& d, int type, F&& f) {
    const auto narrow = std::integral_constant<int, 64>{};
    const auto wide = std::integral_constant<int, 128>{};
    if (type == ATLAS_OPS_F32) key_width(d) == 64 ? f(0.0f, narrow) : f(0.0f, wide);
    else key_width(d) == 64 ? f(bf16_t{}, narrow) : f(bf16_t{}, wide);
}

}  // namespace
}  // namespace atlas_ops

using namespace atlas_ops;

extern "C" {

int atlas_ops_delta_step(const AtlasDelta* a, void* out, float* final_state, void* stream, char* err, size_t cap) {
    try {
        Delta d;
        if (int rc = check(a, d, err, cap)) return rc;
        if (!out || !final_state) return fail(err, cap, 7, "null argument");
        const dim3 grid((unsigned)ceil_div(d.value, 32), (unsigned)d.value_heads, (unsigned)d.batch);
        hipStream_t st = (hipStream_t)stream;
        // 16-byte accesses of the state need its rows to start on 16 bytes
        const bool wide = d.value % 4 == 0 && ((uintptr_t)d.state | (uintptr_t)final_state) % 16 == 0;
        if (a->type == ATLAS_OPS_F32) {
            if (wide) step_kernel<float, 4><<<grid, 256, 0, st>>>(d, (float*)out, final_state);
            else step_kernel<float, 1><<<grid, 256, 0, st>>>(d, (float*)out, final_state);
        } else {
            if (wide) step_kernel<bf16_t, 4><<<grid, 256, 0, st>>>(d, (bf16_t*)out, final_state);
            else step_kernel<bf16_t, 1><<<grid, 256, 0, st>>>(d, (bf16_t*)out, final_state);
        }
        return launched(err, cap, "delta_step");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

int64_t atlas_ops_delta_workspace(const AtlasDelta* a, int train) {
    Delta d;
    return check(a, d, nullptr, 0) ? 0 : carve(d, train, nullptr, nullptr);
}

int atlas_ops_delta_forward(const AtlasDelta* a, int train, void* out, float* final_state, void* workspace, void* stream,
                            char* err, size_t cap) {
    try {
        Delta d;
        if (int rc = check(a, d, err, cap)) return rc;
        if (!out || !final_state || !workspace) return fail(err, cap, 7, "null argument");
        Tape tape;
        carve(d, train, (char*)workspace, &tape);
        hipStream_t st = (hipStream_t)stream;
        const dim3 all((unsigned)d.chunks, (unsigned)d.value_heads, (unsigned)d.batch);
        const dim3 columns((unsigned)ceil_div(d.value, 64), (unsigned)d.value_heads, (unsigned)d.batch);
        with_kernel(d, a->type, [&](auto t, auto width) {
            using T = decltype(t);
            prepare<T, width()><<<all, 256, 0, st>>>(d, tape);
            scan_forward<T, width()><<<columns, 256, 0, st>>>(d, tape, final_state);
            outputs<T, width()><<<all, 256, 0, st>>>(d, tape, (T*)out);
        });
        return launched(err, cap, "delta_forward");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

int64_t atlas_ops_delta_backward_workspace(const AtlasDelta* a) {
    Delta d;
    if (check(a, d, nullptr, 0)) return 0;
    return d.batch * d.value_heads * d.chunks * (C + key_width(d)) * d.padded * (i64)sizeof(float);
}

int atlas_ops_delta_backward(const AtlasDelta* a, const void* tape_memory, const void* grad_out,
                             const int64_t* grad_out_stride, const float* grad_state, void* dq, void* dk, void* dv,
                             void* dlog_decay, void* dbeta, float* dstate, void* workspace, void* stream, char* err,
                             size_t cap) {
    try {
        Delta d;
        if (int rc = check(a, d, err, cap)) return rc;
        if (!tape_memory || !grad_out || !grad_out_stride || !dq || !dk || !dv || !dbeta || !workspace)
            return fail(err, cap, 7, "null argument");
        Tape tape;
        carve(d, 1, (char*)tape_memory, &tape);
        float* floats = (float*)workspace;
        const Back back{tensor(grad_out, grad_out_stride), grad_state, floats,
                        floats + d.batch * d.value_heads * d.chunks * C * d.padded};
        hipStream_t st = (hipStream_t)stream;
        const dim3 columns((unsigned)ceil_div(d.value, 64), (unsigned)d.value_heads, (unsigned)d.batch);
        const dim3 all((unsigned)d.chunks, (unsigned)d.heads, (unsigned)d.batch);
        with_kernel(d, a->type, [&](auto t, auto width) {
            using T = decltype(t);
            scan_backward<T, width()><<<columns, 256, 0, st>>>(d, tape, back, (T*)dv, dstate);
            gradients<T, width()><<<all, 256, 0, st>>>(d, tape, back, (T*)dq, (T*)dk, dlog_decay, dbeta);
        });
        return launched(err, cap, "delta_backward");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

}  // extern "C"
