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
// state enters: `prepare` inverts for all chunks at once, and `scan_forward` carries the states through the
// chunks and takes the outputs on the way.  The columns of S do not touch each other: each workgroup of the
// scan has 16 of them.
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
#include <type_traits>

#include "device/atlas_mma.h"

namespace atlas_ops {
namespace {

constexpr int C = 64;         // tokens per chunk
constexpr int CP = C + 4;     // pitch of a C x C matrix in LDS
constexpr float LOWEST = -120.0f;

struct Delta {
    Tensor q, k, v, decay, beta;
    const float* state;
    const int32_t* lengths;
    i64 batch, time, heads, value_heads;
    int key, value, group, decay_bf16, beta_bf16;
    i64 chunks, padded;  // padded: value in whole operands of 32
    float scale;

    __device__ __forceinline__ i64 length(i64 b) const {
        if (!lengths) return time;
        const i64 n = lengths[b];
        return n < 0 ? 0 : n < time ? n : time;
    }
    // A sequence's chunks with a token.  No kernel visits the others: there a product of zeros would turn a NaN or an
    // infinity of the state, which they leave as it is, into NaNs of its column.
    __device__ __forceinline__ i64 used_chunks(i64 b) const { return (length(b) + C - 1) / C; }
    // A gate of either type, with loads that stand behind no branch.
    struct Gate { uint32_t low, high; };
    __device__ static __forceinline__ Gate load(const Tensor& x, int bf16, i64 b, i64 t, i64 h) {
        const uint16_t* p = (const uint16_t*)x.data + ((b * x.batch + t * x.time + h * x.head) << (bf16 ? 0 : 1));
        return {p[0], p[bf16 ? 0 : 1]};
    }
    __device__ static __forceinline__ float value_of(Gate g, int bf16) {
        return __uint_as_float(bf16 ? g.low << 16 : g.high << 16 | g.low);
    }
    __device__ __forceinline__ Gate load_decay(i64 b, i64 t, i64 h) const {
        return load(decay.data ? decay : beta, decay.data ? decay_bf16 : beta_bf16, b, t, h);
    }
    __device__ __forceinline__ Gate load_rate(i64 b, i64 t, i64 h) const { return load(beta, beta_bf16, b, t, h); }
    __device__ __forceinline__ float log_decay(Gate x) const {
        const float g = value_of(x, decay_bf16);
        return !decay.data ? 0.0f : g < LOWEST ? LOWEST : g;  // a NaN stays one
    }
    __device__ __forceinline__ float rate(Gate x) const { return value_of(x, beta_bf16); }
    __device__ __forceinline__ float log_decay(i64 b, i64 t, i64 h) const { return log_decay(load_decay(b, t, h)); }
    __device__ __forceinline__ float rate(i64 b, i64 t, i64 h) const { return rate(load_rate(b, t, h)); }
};

// ------------------------------------------------------------------ token by token
// A workgroup holds 32 columns of one head's state in registers: row groups of 32 / VEC lanes, each lane
// VEC neighbouring columns of every 8 VEC-th row.  One reduction per token: S^T k and S^T q of the
// decayed state and k . q, as out = scale ((a S)^T q + beta e (k . q)).  Memory bounds one token: the state is read
// and written once, 64 x 8 heads of 128 x 128 in 13.4 us, 5.0 TB/s.  More tokens follow one another at 2 to 9 us each.
constexpr int MAX_KEY = 128;

template <typename T, int VEC>
__global__ void __launch_bounds__(256) step_kernel(Delta d, T* __restrict__ out, float* final_state) {
    constexpr int LANES = 32 / VEC, ROWS = 256 / LANES, PER = MAX_KEY / ROWS;
    __shared__ float sums[2][4][32], dots[2][4];
    const int lane = threadIdx.x % LANES, row = threadIdx.x / LANES, wave = threadIdx.x / 64;
    const i64 b = blockIdx.z, h = blockIdx.y, hk = h / d.group;
    const int col = blockIdx.x * 32 + lane * VEC;
    const i64 base = (b * d.value_heads + h) * d.key * d.value;
    // Nothing is loaded behind a branch, or each load would be waited for before the next: rows and columns that
    // do not exist read the last, and their values become zeros.
    T kt[PER], qt[PER], vt[VEC];
    Delta::Gate decay, beta;
    auto fetch = [&](i64 t) {
        const T *qp = d.q.at<T>(b, t, hk), *kp = d.k.at<T>(b, t, hk), *vp = d.v.at<T>(b, t, h);
        decay = d.load_decay(b, t, h), beta = d.load_rate(b, t, h);
#pragma unroll
        for (int c = 0; c < VEC; ++c) vt[c] = vp[min(col + c, (int)d.value - 1)];
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            const int at = min(row + r * ROWS, d.key - 1);
            kt[r] = kp[at];
            qt[r] = qp[at];
        }
    };
    float s[PER][VEC];
    const float* from = (d.state ? d.state : final_state) + base + min(col, (int)d.value - VEC);
#pragma unroll
    for (int r = 0; r < PER; ++r) {
        const float* p = from + (i64)min(row + r * ROWS, d.key - 1) * d.value;
        if constexpr (VEC == 4) {  // value is a multiple of 4
            const float4_t v = *(const float4_t*)p;
#pragma unroll
            for (int c = 0; c < VEC; ++c) s[r][c] = v[c];
        } else {
            s[r][0] = *p;
        }
    }
    fetch(0);
#pragma unroll
    for (int r = 0; r < PER; ++r)
#pragma unroll
        for (int c = 0; c < VEC; ++c) s[r][c] = d.state && row + r * ROWS < d.key && col < d.value ? s[r][c] : 0.0f;
    const i64 length = d.length(b);
    for (i64 t = 0; t < d.time; ++t) {
        T* o = out + ((b * d.time + t) * d.value_heads + h) * d.value;
        if (t >= length) {
            if (row == 0)
                for (int c = 0; c < VEC; ++c)
                    if (col + c < d.value) o[col + c] = from_float<T>(0.0f);
            continue;
        }
        const float a = expf(d.log_decay(decay)), rate = d.rate(beta);
        float v[VEC];
#pragma unroll
        for (int c = 0; c < VEC; ++c) v[c] = col + c < d.value ? to_float(vt[c]) : 0.0f;
        float kr[PER], qr[PER], ks[VEC], qs[VEC], kq = 0.0f;
#pragma unroll
        for (int c = 0; c < VEC; ++c) ks[c] = qs[c] = 0.0f;
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            const int at = row + r * ROWS;
            kr[r] = at < d.key ? to_float(kt[r]) : 0.0f;
            qr[r] = at < d.key ? to_float(qt[r]) : 0.0f;
        }
        if (t + 1 < length) fetch(t + 1);
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
// Loads of the caller's tensors stand behind no branch (there each would be waited for before the next): they go
// to a row and column that exist, and what lies outside is replaced by zero afterwards.
__device__ __forceinline__ i64 existing(i64 t, const Delta& d) { return t < d.time ? t : d.time - 1; }

// 32 columns of a row from column c0, as loaded and as an operand in the order above, zeros beyond the row's
// width.  WIDE: rows of four values or more, read four at a time without alignment; where the row ends among
// them its last four are read and shifted down (a value at a time, prepare took 68 us more for 16384 tokens of 16 heads
// of 128, gradients 19 us more for 2 x 4099).
template <typename T, bool WIDE>
struct Row {
    struct __attribute__((packed, aligned(sizeof(T)))) Four { T v[4]; };
    Four raw[2];

    __device__ __forceinline__ void load(const T* row, int c0, int width, const Lane& l) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int c = c0 + 16 * half + l.quad;
            if constexpr (WIDE) {
                raw[half] = *(const Four*)(row + min(c, width - 4));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) raw[half].v[e] = row[min(c + e, width - 1)];
            }
        }
    }

    template <int N>
    __device__ __forceinline__ Pieces<N> operand(int c0, int width, bool live, const Lane& l) const {
        if constexpr (WIDE && sizeof(T) == 2) {
            uint64_t bits[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int c = c0 + 16 * half + l.quad, gone = c - min(c, width - 4);
                bits[half] = live && gone < 4 ? __builtin_bit_cast(uint64_t, raw[half]) >> (16 * gone) : 0;
            }
            return Pieces<N>{{__builtin_bit_cast(bf16x8, bits)}};
        } else {
            float4_t v[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int c = c0 + 16 * half + l.quad, gone = WIDE ? c - min(c, width - 4) : 0;
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = to_float(raw[half].v[e]);
                if constexpr (WIDE) {
                    const bool one = gone & 1, two = gone & 2;
                    x[0] = one ? x[1] : x[0], x[1] = one ? x[2] : x[1], x[2] = one ? x[3] : x[2];
                    x[0] = two ? x[2] : x[0], x[1] = two ? x[3] : x[1];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) v[half][e] = live && c + e < width ? x[e] : 0.0f;
            }
            return split<N>(v[0], v[1]);
        }
    }
};

// COUNT operands of a row at once.
template <typename T, bool WIDE, int N, int COUNT>
__device__ __forceinline__ void row_operands(Pieces<N> (&out)[COUNT], const T* row, int c0, int width, bool live, const Lane& l) {
    Row<T, WIDE> raw[COUNT];
#pragma unroll
    for (int i = 0; i < COUNT; ++i) raw[i].load(row, c0 + 32 * i, width, l);
#pragma unroll
    for (int i = 0; i < COUNT; ++i) out[i] = raw[i].template operand<N>(c0 + 32 * i, width, live, l);
}

// The values of four tokens from t0 in one column, as loaded and as floats.
template <typename T>
struct Tokens {
    T raw[4];
    __device__ __forceinline__ void load(const Delta& d, const Tensor& x, i64 b, i64 h, i64 t0, int col, int width) {
        const T* p = x.at<T>(b, 0, h) + (col < width ? col : width - 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[e] = p[existing(t0 + e, d) * x.time];
    }
    __device__ __forceinline__ float4_t floats(i64 t0, i64 length, bool live) const {
        float4_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = live && t0 + e < length ? to_float(raw[e]) : 0.0f;
        return v;
    }
};

// Rows quad .. quad + 3 of column l % 16 of a row-major block.
__device__ __forceinline__ float4_t column(const float* m, i64 pitch, const Lane& l) {
    float4_t v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = m[(l.quad + j) * pitch + l.col];
    return v;
}

__device__ __forceinline__ void put_column(float* m, i64 pitch, const Lane& l, float4_t v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) m[(l.quad + j) * pitch + l.col] = v[j];
}

// Matrices of floats between the kernels lie as 16 x 16 blocks of results, 16 bytes per lane: block
// (r, c) of a matrix of `blocks` block columns.
__device__ __forceinline__ float4_t block(const float* m, i64 r, i64 c, i64 blocks, const Lane& l) {
    return *(const float4_t*)(m + ((r * blocks + c) * 64 + l.id) * 4);
}

__device__ __forceinline__ void put_block(float* m, i64 r, i64 c, i64 blocks, const Lane& l, float4_t v) {
    *(float4_t*)(m + ((r * blocks + c) * 64 + l.id) * 4) = v;
}

// A product with a triangular matrix adds zeros times the terms it masks, which a NaN or an infinity
// there turns into NaNs of earlier tokens.  So where a wave finds any among its tokens (one FMA per value
// says so), it takes them out before the product, and the rows from the column's first on are NaN after
// it: a token's fault reaches its own and later tokens only.  Returns the column's first row of the
// `count` blocks at `row`, C if there is none.
template <int COUNT>
__device__ __forceinline__ int take_faults(float4_t (&v)[COUNT], int row, const Lane& l) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = fmaf(v[i][e], 0.0f, sum);
    int first = C;
    if (__ballot(sum != sum)) {
#pragma unroll
        for (int i = COUNT - 1; i >= 0; --i)
#pragma unroll
            for (int e = 3; e >= 0; --e)
                if (!(fabsf(v[i][e]) < INFINITY)) {
                    v[i][e] = 0.0f;
                    first = row + 16 * i + l.quad + e;
                }
        first = min(first, __shfl_xor(first, 16, 64));
        first = min(first, __shfl_xor(first, 32, 64));
    }
    return first;
}

// Of a triangle of 4 x 4 blocks, the operands that are not zero: row block i, 32 sum indices kb.
__device__ __forceinline__ constexpr int lower(int i, int kb) { return i < 2 ? i : 2 * (i - 1) + kb; }
__device__ __forceinline__ constexpr int upper(int i, int kb) { return i < 2 ? 2 * i + kb : i + 2; }
constexpr int TRIANGLE = 6;

// A chunk's decays.  The running sums are taken in 64 bits, as differences of large sums lose what a
// small decay adds, and kept in powers of two as a float and its remainder: exp(G_i - G_j) is then one
// hardware exp2 of an accurate difference.
enum Gate { SUM, REMAINDER, SINCE, REST, RATE, WRITE, GATES };  // WRITE = REST RATE

// The workspace: operands of chunk n of key head (b, hk) or value head (b, h), and what the scans leave.
struct Tape {
    bf16_t *keys, *queries;                  // rows are tokens
    bf16_t *keys_t, *queries_t;              // rows are key indices, sums over tokens
    bf16_t *inverse, *scores;                // T and P
    bf16_t *inverse_t, *scores_t;            // T^T and P^T
    float *gates, *errors, *states;          // E and S in blocks

    __device__ __forceinline__ i64 shared_chunk(const Delta& d, i64 b, i64 hk, i64 n) const {
        return (b * d.heads + hk) * d.chunks + n;
    }
    __device__ __forceinline__ i64 chunk(const Delta& d, i64 b, i64 h, i64 n) const {
        return (b * d.value_heads + h) * d.chunks + n;
    }
    __device__ __forceinline__ const float* gate(i64 chunk, Gate which) const {
        return gates + (chunk * GATES + which) * C;
    }
};

__device__ __forceinline__ float decay(const float* sum, const float* remainder, int i, int j) {
    return __builtin_amdgcn_exp2f((sum[i] - sum[j]) + (remainder[i] - remainder[j]));
}

// ------------------------------------------------------------------ operands and T = (I + M B)^-1
// One workgroup per chunk and key head: the keys (and, to train, queries) as operands, then for each
// value head that shares them the gates, the scores and the inverse, 16 x 16 blocks by forward substitution, joined in
// pairs: the inverse of [[a, 0], [m, c]] has -c^-1 m a^-1 below.  Its steps wait for one another, so what counts is
// how many workgroups a CU holds: 168 registers, three of them with bfloat16 (2 x 4099 tokens of 4 x 4 heads of
// 128: 59 us with three, 82 with two; 16384 of 16 heads 119 us), two by their LDS with float32 (256 x 100 of 4 heads
// of 64: 102 us).
template <typename T, int DK, bool WIDE>
__global__ void __launch_bounds__(256, 3) prepare(Delta d, Tape tape, int train) {
    constexpr int N = sizeof(T) == 2 ? 1 : 3, KB = DK / 32;
    __shared__ __attribute__((aligned(16))) bf16_t rows[4 * KB * N * 512];
    __shared__ __attribute__((aligned(16))) float low[C * CP], inv[C * CP];
    __shared__ __attribute__((aligned(16))) float gates[GATES][C];
    __shared__ int faulty;  // the first row with a NaN or an infinity; it and those after it become NaN
    const i64 n = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, length = d.length(b);
    if (n * C >= length) return;
    const i64 shared = tape.shared_chunk(d, b, hk, n);
    const int wave = threadIdx.x / 64;
    const Lane l;
    bf16_t *keys = tape.keys + shared * (4 * KB * N * 512), *queries = tape.queries + shared * (4 * KB * N * 512);
    // the first wave's gates, a value head ahead
    const i64 gate_time = n * C + l.id;
    float next_decay = 0.0f, next_rate = 0.0f;
    auto fetch_gates = [&](i64 h) {
        next_decay = d.log_decay(b, existing(gate_time, d), h);
        next_rate = d.rate(b, existing(gate_time, d), h);
    };
    fetch_gates(hk * d.group);
    const i64 t = n * C + 16 * wave + l.col;
    Pieces<N> own[KB], query[KB];
    row_operands<T, WIDE, N, KB>(own, d.k.at<T>(b, existing(t, d), hk), 0, d.key, t < length, l);
    row_operands<T, WIDE, N, KB>(query, d.q.at<T>(b, existing(t, d), hk), 0, d.key, t < length, l);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        put<N>(rows, wave * KB + kb, l, own[kb]);
        put<N>(keys, wave * KB + kb, l, own[kb]);
        put<N>(queries, wave * KB + kb, l, query[kb]);
    }
    for (int what = 0; what < 1 + (train != 0); ++what) {
        const Tensor& x = what ? d.q : d.k;
        bf16_t* to = (what ? tape.queries_t : tape.keys_t) + shared * (4 * KB * N * 512);
        Tokens<T> v[KB][2];  // operand u: row block u / 2, tokens 32 (u % 2) ..
#pragma unroll
        for (int i = 0; i < KB; ++i) {
            const int u = wave + 4 * i;
#pragma unroll
            for (int half = 0; half < 2; ++half)
                v[i][half].load(d, x, b, hk, n * C + u % 2 * 32 + half * 16 + l.quad, u / 2 * 16 + l.col, d.key);
        }
#pragma unroll
        for (int i = 0; i < KB; ++i) {
            const int u = wave + 4 * i;
            const i64 t0 = n * C + u % 2 * 32 + l.quad;
            const bool live = u / 2 * 16 + l.col < d.key;
            put<N>(to, u, l, split<N>(v[i][0].floats(t0, length, live), v[i][1].floats(t0 + 16, length, live)));
        }
    }
    __syncthreads();
    float4_t kk[4], kq[4], qk[4];  // K K^T and K Q^T (rows are the earlier tokens: operands of P), Q K^T (of P^T)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        kk[j] = kq[j] = qk[j] = ZERO;
        if (j > wave) continue;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const Pieces<N> other = fetch<N>(rows, j * KB + kb, l);
            kk[j] = mma<N, N>(other, own[kb], kk[j]);
            kq[j] = mma<N, N>(other, query[kb], kq[j]);
            if (train) qk[j] = mma<N, N>(query[kb], other, qk[j]);
        }
    }
    for (int member = 0; member < d.group; ++member) {
        const i64 h = hk * d.group + member, chunk = tape.chunk(d, b, h, n);
        __syncthreads();  // the member before is written out
        if (threadIdx.x == 0) faulty = C;
        if (threadIdx.x < 64) {
            const int i = threadIdx.x;
            double g = gate_time < length ? (double)next_decay * 1.4426950408889634 : 0.0;
            const float own_rate = gate_time < length ? next_rate : 0.0f;
            if (member + 1 < d.group) fetch_gates(h + 1);
#pragma unroll
            for (int s = 1; s < 64; s *= 2) {
                const double below = __shfl_up(g, s, 64);
                if (i >= s) g += below;
            }
            const double last = __shfl(g, 63, 64);
            float v[GATES];
            v[SUM] = (float)g;
            v[REMAINDER] = (float)(g - (double)v[SUM]);
            v[SINCE] = __builtin_amdgcn_exp2f((float)g);
            v[REST] = __builtin_amdgcn_exp2f((float)(last - g));
            v[RATE] = own_rate;
            v[WRITE] = v[REST] * v[RATE];
#pragma unroll
            for (int w = 0; w < GATES; ++w) {
                gates[w][i] = v[w];
                tape.gates[(chunk * GATES + w) * C + i] = v[w];
            }
        }
        for (int e = threadIdx.x; e < C * CP; e += 256) inv[e] = 0.0f;
        __syncthreads();
        {
            float4_t p[4] = {ZERO, ZERO, ZERO, ZERO};
            const int i = 16 * wave + l.col;
            const float sum = gates[SUM][i], remainder = gates[REMAINDER][i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j > wave) continue;
                const int k0 = 16 * j + l.quad;
                const float4_t sums = *(const float4_t*)(gates[SUM] + k0), remainders = *(const float4_t*)(gates[REMAINDER] + k0);
                const float4_t rates = *(const float4_t*)(gates[RATE] + k0);
                float4_t m;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float fade = __builtin_amdgcn_exp2f((sum - sums[e]) + (remainder - remainders[e]));
                    p[j][e] = i >= k0 + e ? d.scale * kq[j][e] * fade : 0.0f;
                    m[e] = i > k0 + e ? kk[j][e] * fade * rates[e] : 0.0f;
                    if (!(fabsf(m[e]) < INFINITY)) {
                        atomicMin(&faulty, i);
                        m[e] = 0.0f;
                    }
                }
                *(float4_t*)(low + i * CP + k0) = m;
            }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
                if (2 * kb <= wave) put<3>(tape.scores + chunk * (TRIANGLE * 3 * 512), lower(wave, kb), l, split<3>(p[2 * kb], p[2 * kb + 1]));
        }
        if (train) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j > (wave | 1)) continue;
                float4_t p;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 16 * wave + l.quad + e, k = 16 * j + l.col;
                    p[e] = i >= k ? d.scale * qk[j][e] * decay(gates[SUM], gates[REMAINDER], i, k) : 0.0f;
                }
                put_half<3>(tape.scores_t + chunk * (TRIANGLE * 3 * 512), upper(j, wave / 2), wave % 2, l, split<3>(p));
            }
        }
        __syncthreads();
        if (l.id < 16) {  // a column per lane
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
        // operands out of LDS: row l % 16 of a block, and the block's columns; indices 16 .. 31 of the sum
        // are zero where a block stands alone
        auto rows_of = [&](const float* m, bool both) {
            const float4_t a = *(const float4_t*)(m + l.col * CP + l.quad);
            return split<3>(a, both ? *(const float4_t*)(m + l.col * CP + 16 + l.quad) : ZERO);
        };
        if (wave < 2) {
            float* corner = inv + (32 * wave + 16) * CP + 32 * wave;
            const float4_t x = mma<3, 3>(rows_of(low + (32 * wave + 16) * CP + 32 * wave, false),
                                         split<3>(column(inv + 32 * wave * (CP + 1), CP, l), ZERO), ZERO);
            const float4_t y = mma<3, 3>(rows_of(corner + 16, false), split<3>(x, ZERO), ZERO);
            put_column(corner, CP, l, -y);
        }
        __syncthreads();
        if (wave < 2) {  // column block `wave` of the lower left 32 x 32
            const float* a = inv + 16 * wave;
            const Pieces<3> above = split<3>(column(a, CP, l), column(a + 16 * CP, CP, l));
            float4_t x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) x[i] = mma<3, 3>(rows_of(low + (32 + 16 * i) * CP, true), above, ZERO);
            const Pieces<3> below = split<3>(x[0], x[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                put_column(inv + (32 + 16 * i) * CP + 16 * wave, CP, l, -mma<3, 3>(rows_of(inv + (32 + 16 * i) * CP + 32, true), below, ZERO));
        }
        __syncthreads();
        const int bad = faulty;
        const float4_t nans = {NAN, NAN, NAN, NAN};
        for (int u = wave; u < TRIANGLE; u += 4) {
            const int i = u < 2 ? u : 1 + u / 2, kb = u < 2 ? 0 : u % 2;
            const float* m = inv + (16 * i + l.col) * CP + 32 * kb + l.quad;
            const bool fine = 16 * i + l.col < bad;
            put<3>(tape.inverse + chunk * (TRIANGLE * 3 * 512), u, l,
                   split<3>(fine ? *(const float4_t*)m : nans, fine ? *(const float4_t*)(m + 16) : nans));
        }
        if (!train) continue;
        for (int u = wave; u < TRIANGLE; u += 4) {
            const int i = u < 4 ? u / 2 : u - 2, kb = u < 4 ? u % 2 : 1;
            const float* m = inv + 32 * kb * CP + 16 * i;
            float4_t v[2] = {column(m, CP, l), column(m + 16 * CP, CP, l)};
            if (bad < C) {
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (32 * kb + 16 * half + l.quad + e >= bad) v[half][e] = NAN;
            }
            put<3>(tape.inverse_t + chunk * (TRIANGLE * 3 * 512), u, l, split<3>(v[0], v[1]));
        }
    }
}

// ------------------------------------------------------------------ the states through the chunks, and the outputs
// A workgroup carries 16 columns of one head's state.  Its first DK / 32 waves hold 32 rows of them each in
// registers and take a chunk in three exchanges through LDS: their partial sums of K S (each then adds those
// of its own tokens), R for T R, and rest B E for the state.  That chain bounds the scan, so a chunk's operands
// are fetched while the chunk before it runs, and as many waves again take the outputs of the chunk before from
// the states and errors that the first leave in LDS: in inference neither goes to memory.
//
// Measured: 16384 tokens of 16 heads of 128, bfloat16, 256 chunks one after the other, 480 us or 1.9 us a chunk (a
// kernel of its own for the outputs: 440 and 178 us, and the states written).  The three exchanges, their MFMA latencies
// and the splits between them make 1.5 us of that; the rest is operands that arrive late and what the outputs take
// of the load path (with queries loaded from the caller's rows, 8 bytes a lane, 577 us; a value at a time, 1207).
// 256 x 100 of 4 heads of 64, float32: 157 us for 4096 workgroups of two chunks, bound by the operands that every 16
// columns read anew from the L2.
//
// Workgroups of one head run on one XCD (they share its operands in the L2): workgroups go to the 8 XCDs
// in turn, so head 8 k + x takes the workgroups with index % 8 = x.
constexpr int XCDS = 8;

struct Place {
    i64 b, h;
    int column;
    bool any;
    __device__ __forceinline__ Place(const Delta& d) {
        const int slices = (int)(d.padded / 16);
        const int slot = (int)blockIdx.x / XCDS, head = slot / slices * XCDS + (int)blockIdx.x % XCDS;
        column = slot % slices * 16;
        any = head < d.batch * d.value_heads;
        b = head / (int)d.value_heads;
        h = head % (int)d.value_heads;
    }
};

template <typename T, int DK, bool TRAIN>
__global__ void __launch_bounds__(DK * 4, 2) scan_forward(Delta d, Tape tape, T* __restrict__ out, float* __restrict__ final_state) {
    constexpr int N = sizeof(T) == 2 ? 1 : 3, WAVES = DK / 32, OWN = 4 / WAVES;
    __shared__ __attribute__((aligned(16))) float part[WAVES][4][64][4];
    __shared__ __attribute__((aligned(16))) bf16_t seen[2 * 3 * 512], written[2 * 3 * 512];
    // of two chunks in turn: S and B E as operands, and the first faulty row of each column
    __shared__ __attribute__((aligned(16))) bf16_t held[2][WAVES * 3 * 512], errors[2][2 * 3 * 512];
    __shared__ int first[4][16], blame[2][4][16];
    const Place at(d);
    if (!at.any) return;
    const i64 b = at.b, h = at.h, length = d.length(b);
    const int wave = threadIdx.x / 64 % WAVES;
    const Lane l;
    const int col = at.column + l.col;
    const bool live = col < d.value;
    const i64 chunk0 = tape.chunk(d, b, h, 0), shared0 = tape.shared_chunk(d, b, h / d.group, 0);
    const i64 chunks = d.used_chunks(b), last = chunks - 1;

    if (threadIdx.x >= 64 * WAVES) {  // the outputs of tokens 16 OWN wave ..
        Pieces<N> q[OWN][WAVES];
        Pieces<3> scores[OWN][2];
        float4_t since[OWN];
        // each is fetched for the next chunk as soon as this one's is used
        auto fetch_queries = [&](i64 n) {
#pragma unroll
            for (int o = 0; o < OWN; ++o)
#pragma unroll
                for (int kb = 0; kb < WAVES; ++kb)
                    q[o][kb] = fetch<N>(tape.queries + (shared0 + n) * (4 * WAVES * N * 512), (wave * OWN + o) * WAVES + kb, l);
        };
        auto fetch_scores = [&](i64 n) {
#pragma unroll
            for (int o = 0; o < OWN; ++o) {
                const int i = wave * OWN + o;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    scores[o][kb] = fetch<3>(tape.scores + (chunk0 + n) * (TRIANGLE * 3 * 512), lower(i, min(kb, i / 2)), l);
                since[o] = *(const float4_t*)(tape.gate(chunk0 + n, SINCE) + 16 * i + l.quad);
            }
        };
        // Chunk n, with `more` a part of it between each two barriers of chunk n + 1; `whole`: all tokens and columns exist.
        // Neither is asked within the loop, as a load or store behind a branch makes later waits wait for all before it.
        auto chunk = [&](i64 n, auto more, auto whole) {
            const int turn = (int)(n & 1);
            float4_t acc[OWN][2];
#pragma unroll
            for (int o = 0; o < OWN; ++o) acc[o][0] = acc[o][1] = ZERO;
#pragma unroll
            for (int kb = 0; kb < WAVES; ++kb) {
                const Pieces<3> s = fetch<3>(held[turn], kb, l);
#pragma unroll
                for (int o = 0; o < OWN; ++o) acc[o][kb % 2] = mma<N, 3>(q[o][kb], s, acc[o][kb % 2]);
            }
            if constexpr (more()) {
                fetch_queries(n + 1);
                in_order();
                lds_barrier();
            }
            const Pieces<3> e[2] = {fetch<3>(errors[turn], 0, l), fetch<3>(errors[turn], 1, l)};
#pragma unroll
            for (int o = 0; o < OWN; ++o) {
                acc[o][0] = (acc[o][0] + acc[o][1]) * since[o] * d.scale;
                acc[o][1] = ZERO;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    if (2 * kb <= wave * OWN + o) acc[o][kb] = mma<3, 3>(scores[o][kb], e[kb], acc[o][kb]);
                acc[o][0] += acc[o][1];
            }
            int fault = C;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) fault = min(fault, blame[turn][w][l.col]);
            if constexpr (more()) {
                fetch_scores(n + 1);
                in_order();
                lds_barrier();
            }
            T* to = out + ((b * d.time + n * C) * d.value_heads + h) * d.value + col;
#pragma unroll
            for (int o = 0; o < OWN; ++o)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = 16 * (wave * OWN + o) + l.quad + j;
                    const i64 t = n * C + row;
                    if (whole() || (t < d.time && live))
                        to[row * d.value_heads * d.value] = from_float<T>(t >= length ? 0.0f : row < fault ? acc[o][0][j] : NAN);
                }
            if constexpr (more()) lds_barrier();
        };
        constexpr std::true_type yes{};
        constexpr std::false_type no{};
        if (chunks > 0) {
            fetch_queries(0);
            fetch_scores(0);
            for (int i = 0; i < 3; ++i) lds_barrier();
            if (at.column + 16 <= d.value)
                for (i64 n = 0; n < last; ++n) chunk(n, yes, yes);
            else
                for (i64 n = 0; n < last; ++n) chunk(n, yes, no);
            chunk(last, no, no);
        }
        if (live)
            for (i64 t = chunks * C + 4 * wave + l.quad / 4; t < d.time; t += 4 * WAVES)
                out[((b * d.time + t) * d.value_heads + h) * d.value + col] = from_float<T>(0.0f);
        return;
    }

    const i64 base = (b * d.value_heads + h) * d.key * d.value + col;
    float4_t s[2];
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 32 * wave + 16 * f + l.quad + e;
            s[f][e] = d.state && r < d.key && live ? d.state[base + (i64)r * d.value] : 0.0f;
        }
    // Chunks ahead that keys are fetched (16384 tokens of 16 heads: two take 65 us less than one); where
    // the operands of one chunk alone fill the registers, each is fetched only after those of the product
    // before it are used (TIGHT; 256 x 100 of 4 heads of 64, float32: 157 us with 45 to 47 registers spilled, otherwise 226
    // with 52 to 64).
    constexpr bool TIGHT = DK == 64 && N == 3;
    constexpr int DEPTH = DK == 128 && N == 1 ? 2 : 1;
    Pieces<N> k[DEPTH][4], kt[DEPTH][2][2];
    Pieces<3> inverse[OWN][2];
    Tokens<T> v[OWN];
    float4_t since[OWN], write[OWN], rate[OWN];
    float fade[DEPTH];
    auto fetch_keys = [&](i64 n, int to) {
#pragma unroll
        for (int i = 0; i < 4; ++i) k[to][i] = fetch<N>(tape.keys + (shared0 + n) * (4 * WAVES * N * 512), i * WAVES + wave, l);
    };
    auto fetch_tokens = [&](i64 n) {
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
            const int i = wave * OWN + o;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
                inverse[o][kb] = fetch<3>(tape.inverse + (chunk0 + n) * (TRIANGLE * 3 * 512), lower(i, min(kb, i / 2)), l);
            since[o] = *(const float4_t*)(tape.gate(chunk0 + n, SINCE) + 16 * i + l.quad);
            write[o] = *(const float4_t*)(tape.gate(chunk0 + n, WRITE) + 16 * i + l.quad);
            rate[o] = *(const float4_t*)(tape.gate(chunk0 + n, RATE) + 16 * i + l.quad);
            v[o].load(d, d.v, b, h, n * C + 16 * i + l.quad, col, d.value);
        }
    };
    auto fetch_writes = [&](i64 n, int to) {
        fade[to] = tape.gate(chunk0 + n, SINCE)[C - 1];
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
                kt[to][f][kb] = fetch<N>(tape.keys_t + (shared0 + n) * (4 * WAVES * N * 512), (2 * wave + f) * 2 + kb, l);
    };
    auto chunk = [&](i64 n, auto slot) {
        const i64 next = min(n + 1, last), later = min(n + DEPTH, last);
        const int turn = (int)(n & 1);
        const Pieces<3> state = split<3>(s[0], s[1]);
        float4_t sums[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[i] = mma<N, 3>(k[slot()][i], state, ZERO);
        put<3>(held[turn], wave, l, state);
#pragma unroll
        for (int i = 0; i < 4; ++i) *(float4_t*)part[wave][i][l.id] = sums[i];
        lds_barrier();
        if constexpr (TIGHT) fetch_writes(n, slot());
        else fetch_keys(later, slot());
        in_order();
        if constexpr (TRAIN) {
#pragma unroll
            for (int f = 0; f < 2; ++f) put_block(tape.states, (chunk0 + n) * (DK / 16) + 2 * wave + f, at.column / 16, d.padded / 16, l, s[f]);
        }
        // R = V - g K S of the wave's own tokens
        float4_t r[OWN];
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
            float4_t sum = *(const float4_t*)part[0][wave * OWN + o][l.id];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) sum += *(const float4_t*)part[w][wave * OWN + o][l.id];
            r[o] = v[o].floats(n * C + 16 * (wave * OWN + o) + l.quad, length, live) - since[o] * sum;
        }
        int fault = take_faults(r, 16 * wave * OWN, l);
        if (l.id < 16) first[wave][l.id] = fault;
#pragma unroll
        for (int o = 0; o < OWN; ++o) put_half<3>(seen, (wave * OWN + o) / 2, (wave * OWN + o) % 2, l, split<3>(r[o]));
        lds_barrier();
        fault = C;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) fault = min(fault, first[w][l.col]);
        float4_t e[OWN];
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
            const int i = wave * OWN + o;
            float4_t large[2] = {ZERO, ZERO}, small[2] = {ZERO, ZERO};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
                if (2 * kb <= i) mma2<3, 3>(inverse[o][kb], fetch<3>(seen, kb, l), large[kb], small[kb]);
            e[o] = (large[0] + large[1]) + (small[0] + small[1]);
#pragma unroll
            for (int j = 0; j < 4; ++j) e[o][j] = 16 * i + l.quad + j < fault ? e[o][j] : NAN;
            put_half<3>(written, i / 2, i % 2, l, split<3>(e[o] * write[o]));
            if constexpr (TRAIN) put_block(tape.errors, (chunk0 + n) * 4 + i, at.column / 16, d.padded / 16, l, e[o]);
            e[o] *= rate[o];
        }
        fault = take_faults(e, 16 * wave * OWN, l);
        if (l.id < 16) blame[turn][wave][l.id] = fault;
#pragma unroll
        for (int o = 0; o < OWN; ++o) put_half<3>(errors[turn], (wave * OWN + o) / 2, (wave * OWN + o) % 2, l, split<3>(e[o]));
#pragma unroll
        for (int f = 0; f < 2; ++f) s[f] *= fade[slot()];
        if constexpr (TIGHT) {
            in_order();
            fetch_keys(next, slot());
        }
        lds_barrier();
        if constexpr (!TIGHT) fetch_tokens(next);
        in_order();
        float4_t other[2] = {ZERO, ZERO};
        const Pieces<3> w[2] = {fetch<3>(written, 0, l), fetch<3>(written, 1, l)};
#pragma unroll
        for (int f = 0; f < 2; ++f) s[f] = mma<N, 3>(kt[slot()][f][0], w[0], s[f]);
#pragma unroll
        for (int f = 0; f < 2; ++f) s[f] += mma<N, 3>(kt[slot()][f][1], w[1], other[f]);
        if constexpr (TIGHT) fetch_tokens(next);
        else fetch_writes(later, slot());
        in_order();
    };
    if (chunks > 0) {
#pragma unroll
        for (int ahead = 0; ahead < DEPTH; ++ahead) {
            fetch_keys(min((i64)ahead, last), ahead);
            if constexpr (!TIGHT) fetch_writes(min((i64)ahead, last), ahead);
        }
        fetch_tokens(0);
        if constexpr (DEPTH == 2) {
            for (i64 n = 0; n < last; n += 2) {
                chunk(n, std::integral_constant<int, 0>{});
                chunk(n + 1, std::integral_constant<int, 1>{});
            }
            if (last % 2 == 0) chunk(last, std::integral_constant<int, 0>{});
        } else {
            for (i64 n = 0; n <= last; ++n) chunk(n, std::integral_constant<int, 0>{});
        }
    }
    if (!live) return;
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 32 * wave + 16 * f + l.quad + e;
            if (r < d.key) final_state[base + (i64)r * d.value] = s[f][e];
        }
}

// ------------------------------------------------------------------ the states' gradients backwards
struct Back {
    Tensor grad;              // of out
    const float* grad_state;  // of the final state, or NULL
    float *residuals;         // Y
    float *states;            // dS' of every chunk
};

// As scan_forward, from the last chunk to the first: the first waves' partial sums of K dS', then B dV' for
// T^T B dV', then Y for the state's gradient.  What needs no state, P^T dO and scale Q^T g dO, the other waves
// leave in LDS a chunk ahead.  2 x 4099 of 16 heads of 128, bfloat16: 193 us, 2.9 us a chunk (262 with one set of waves
// for both); fetching its keys two chunks ahead, as forwards, gains nothing here.  256 x 100 of 4 heads of 64,
// float32: 124 us with two workgroups per CU (254 registers), 160 with one.
template <typename T, int DK>
__global__ void __launch_bounds__(DK * 4, 2) scan_backward(Delta d, Tape tape, Back back, float* __restrict__ dstate) {
    constexpr int N = sizeof(T) == 2 ? 1 : 3, WAVES = DK / 32, OWN = 4 / WAVES;
    __shared__ __attribute__((aligned(16))) float part[WAVES][4][64][4];
    __shared__ __attribute__((aligned(16))) bf16_t seen[2 * 3 * 512], written[2 * 3 * 512];
    __shared__ __attribute__((aligned(16))) float direct[2][4][64][4], reads[2][DK / 16][64][4];  // of two chunks in turn
    const Place at(d);
    if (!at.any) return;
    const i64 b = at.b, h = at.h, length = d.length(b);
    const int wave = threadIdx.x / 64 % WAVES;
    const Lane l;
    const int col = at.column + l.col;
    const bool live = col < d.value;
    const i64 chunk0 = tape.chunk(d, b, h, 0), shared0 = tape.shared_chunk(d, b, h / d.group, 0);
    const i64 chunks = d.used_chunks(b);

    if (threadIdx.x >= 64 * WAVES) {
        if (!chunks) return;
        Tokens<T> go[4];
        float4_t since[4];
        Pieces<N> qt[2][2];
        Pieces<3> scores[OWN][2];
        auto fetch_grads = [&](i64 n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) go[i].load(d, back.grad, b, h, n * C + 16 * i + l.quad, col, d.value);
        };
        auto fetch_scores = [&](i64 n) {
#pragma unroll
            for (int w = 0; w < OWN; ++w)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    scores[w][kb] = fetch<3>(tape.scores_t + (chunk0 + n) * (TRIANGLE * 3 * 512),
                                             upper(wave * OWN + w, max(kb, (wave * OWN + w) / 2)), l);
        };
        auto fetch_queries = [&](i64 n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) since[i] = *(const float4_t*)(tape.gate(chunk0 + n, SINCE) + 16 * i + l.quad);
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    qt[f][kb] = fetch<N>(tape.queries_t + (shared0 + n) * (4 * WAVES * N * 512), (2 * wave + f) * 2 + kb, l);
        };
        fetch_grads(chunks - 1);
        fetch_scores(chunks - 1);
        fetch_queries(chunks - 1);
        // chunk n, but for the last chunk while the first waves are at n + 1
        auto chunk = [&](i64 n, auto beside) {
            const int turn = (int)(n & 1);
            const i64 next = n > 0 ? n - 1 : 0;
            float4_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = go[i].floats(n * C + 16 * i + l.quad, length, live);
            fetch_grads(next);
            in_order();
            const Pieces<N> grads[2] = {split<N>(o[0], o[1]), split<N>(o[2], o[3])};
#pragma unroll
            for (int w = 0; w < OWN; ++w) {
                float4_t acc[2] = {ZERO, ZERO};
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    if (2 * kb + 1 >= wave * OWN + w) acc[kb] = mma<3, N>(scores[w][kb], grads[kb], acc[kb]);
                *(float4_t*)direct[turn][wave * OWN + w][l.id] = acc[0] + acc[1];
            }
            fetch_scores(next);
            in_order();
            if constexpr (beside()) lds_barrier();
            float4_t acc[2] = {ZERO, ZERO};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const Pieces<3> g = split<3>(o[2 * kb] * since[2 * kb] * d.scale, o[2 * kb + 1] * since[2 * kb + 1] * d.scale);
#pragma unroll
                for (int f = 0; f < 2; ++f) acc[f] = mma<N, 3>(qt[f][kb], g, acc[f]);
            }
            fetch_queries(next);
            in_order();
            if constexpr (beside()) lds_barrier();
#pragma unroll
            for (int f = 0; f < 2; ++f) *(float4_t*)reads[turn][2 * wave + f][l.id] = acc[f];
            lds_barrier();
        };
        chunk(chunks - 1, std::false_type{});
        for (i64 n = chunks - 1; n-- > 0;) chunk(n, std::true_type{});
        lds_barrier();  // those of chunk 0
        lds_barrier();
        lds_barrier();
        return;
    }

    const i64 base = (b * d.value_heads + h) * d.key * d.value + col;
    float4_t s[2];
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 32 * wave + 16 * f + l.quad + e;
            s[f][e] = back.grad_state && r < d.key && live ? back.grad_state[base + (i64)r * d.value] : 0.0f;
        }
    Pieces<N> k[4], kt[2][2];
    Pieces<3> inverse[OWN][2];
    float4_t since[OWN], rest[OWN], rate[OWN];
    float fade = 1.0f;
    auto fetch_keys = [&](i64 n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = fetch<N>(tape.keys + (shared0 + n) * (4 * WAVES * N * 512), i * WAVES + wave, l);
    };
    auto fetch_tokens = [&](i64 n) {
#pragma unroll
        for (int w = 0; w < OWN; ++w) {
            const int i = wave * OWN + w;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
                inverse[w][kb] = fetch<3>(tape.inverse_t + (chunk0 + n) * (TRIANGLE * 3 * 512), upper(i, max(kb, i / 2)), l);
            since[w] = *(const float4_t*)(tape.gate(chunk0 + n, SINCE) + 16 * i + l.quad);
            rest[w] = *(const float4_t*)(tape.gate(chunk0 + n, REST) + 16 * i + l.quad);
            rate[w] = *(const float4_t*)(tape.gate(chunk0 + n, RATE) + 16 * i + l.quad);
        }
    };
    auto fetch_writes = [&](i64 n) {
        fade = tape.gate(chunk0 + n, SINCE)[C - 1];
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
                kt[f][kb] = fetch<N>(tape.keys_t + (shared0 + n) * (4 * WAVES * N * 512), (2 * wave + f) * 2 + kb, l);
    };
    if (chunks > 0) {
        fetch_keys(chunks - 1);
        fetch_tokens(chunks - 1);
        fetch_writes(chunks - 1);
        lds_barrier();  // the last chunk's P^T dO and Q^T g dO
    }
    for (i64 n = chunks; n-- > 0;) {
        const i64 next = n > 0 ? n - 1 : 0;
        const int turn = (int)(n & 1);
        const Pieces<3> state = split<3>(s[0], s[1]);
        float4_t sums[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[i] = mma<N, 3>(k[i], state, ZERO);
#pragma unroll
        for (int i = 0; i < 4; ++i) *(float4_t*)part[wave][i][l.id] = sums[i];
        lds_barrier();
        fetch_keys(next);
        in_order();
#pragma unroll
        for (int f = 0; f < 2; ++f) put_block(back.states, (chunk0 + n) * (DK / 16) + 2 * wave + f, at.column / 16, d.padded / 16, l, s[f]);
#pragma unroll
        for (int w = 0; w < OWN; ++w) {
            const int i = wave * OWN + w;
            float4_t sum = *(const float4_t*)part[0][i][l.id];
#pragma unroll
            for (int from = 1; from < WAVES; ++from) sum += *(const float4_t*)part[from][i][l.id];
            put_half<3>(seen, i / 2, i % 2, l, split<3>((*(const float4_t*)direct[turn][i][l.id] + sum * rest[w]) * rate[w]));
        }
        lds_barrier();
        float4_t y[OWN];
#pragma unroll
        for (int w = 0; w < OWN; ++w) {
            const int i = wave * OWN + w;
            float4_t large[2] = {ZERO, ZERO}, small[2] = {ZERO, ZERO};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
                if (2 * kb + 1 >= i) mma2<3, 3>(inverse[w][kb], fetch<3>(seen, kb, l), large[kb], small[kb]);
            y[w] = (large[0] + large[1]) + (small[0] + small[1]);
            put_half<3>(written, i / 2, i % 2, l, split<3>(y[w] * -since[w]));
        }
#pragma unroll
        for (int f = 0; f < 2; ++f) s[f] = s[f] * fade + *(const float4_t*)reads[turn][2 * wave + f][l.id];
        lds_barrier();
        fetch_tokens(next);
        in_order();
        float4_t other[2] = {ZERO, ZERO};
        const Pieces<3> w[2] = {fetch<3>(written, 0, l), fetch<3>(written, 1, l)};
#pragma unroll
        for (int f = 0; f < 2; ++f) s[f] = mma<N, 3>(kt[f][0], w[0], s[f]);
#pragma unroll
        for (int f = 0; f < 2; ++f) s[f] += mma<N, 3>(kt[f][1], w[1], other[f]);
        fetch_writes(next);
        in_order();
#pragma unroll
        for (int o = 0; o < OWN; ++o) put_block(back.residuals, (chunk0 + n) * 4 + wave * OWN + o, at.column / 16, d.padded / 16, l, y[o]);
    }
    if (!dstate || !live) return;
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 32 * wave + 16 * f + l.quad + e;
            if (r < d.key) dstate[base + (i64)r * d.value] = s[f][e];
        }
}

// ------------------------------------------------------------------ every chunk's gradients
// Five of the products sum over the value columns, while the scans leave S, dS', E and Y as blocks whose
// lanes are those columns.  A block's transpose is its product with the identity, which MFMA takes
// exactly for bfloat16 pieces: so 32 columns at a time are split into pieces once for the workgroup, turned,
// and kept in LDS as operands for all its waves.
//
// One workgroup per chunk and key head; it visits the value heads that share the key head one after the
// other, so their sums into dq and dk need no atomics.  Eight waves: wave w holds the tokens 16 (w % 4) ..
// of half w / 4 of the key indices, and its half chooses which of the two C x C products it takes.
//
// Bound by its chain of stages (loads, turns, barrier, products) with one workgroup per CU: 2 x 4099 of 4 x 4 heads of
// 128, bfloat16, 335 us, about 275 TFLOP/s of MFMA, a quarter of the rate; 256 x 100 of 4 heads of 64, float32,
// 167 us.  Of its 244 to 256 registers 40 to 68 are spilled with keys above 64, 16 with bfloat16 values of fewer than four
// columns, else none.  Fetching a stage ahead costs more in registers than it hides (365 and 203 us), and so does half the
// registers for twice the workgroups where keys are 64 wide (285 us).
template <typename T, int DK, bool WIDE>
__global__ void __launch_bounds__(512, 2) gradients(Delta d, Tape tape, Back back, T* __restrict__ dq, T* __restrict__ dk,
                                                 T* __restrict__ dv, void* __restrict__ ddecay, void* __restrict__ dbeta) {
    constexpr int N = sizeof(T) == 2 ? 1 : 3, F = DK / 32;
    constexpr int STATES = DK / 16 * 3 * 512, TOKENS = 4 * 3 * 512;
    // S, dS', E and Y of 32 columns; afterwards D1 and D2
    __shared__ __attribute__((aligned(16))) bf16_t stage[2 * STATES + 2 * TOKENS];
    __shared__ __attribute__((aligned(16))) float gates[GATES][C];
    __shared__ float lines[2][2][C], part[8];
    // dq and dk of the value heads so far, each wave's own blocks
    __shared__ __attribute__((aligned(16))) float sums[DK == 64 ? 1 : 2][DK == 64 ? 4 : 8 * F * 64 * 4];
    float4_t gq[F], gk[F];
    bf16_t *s_stage = stage, *g_stage = stage + STATES, *e_stage = stage + 2 * STATES, *y_stage = e_stage + TOKENS;
    float *d1 = (float*)stage, *d2 = d1 + C * CP;
    static_assert(2 * C * CP * sizeof(float) <= sizeof(stage), "D1 and D2 take the stage's place");
    const i64 n = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, length = d.length(b);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), tb = wave % 4, half = wave / 4, token = 16 * tb, key0 = half * F;
    if (n * C >= length) {  // no gradient reaches an unused token
        const i64 first = b * d.time + n * C, tokens = min((i64)C, d.time - n * C), spread = (i64)d.group * d.value;
        for (i64 e = threadIdx.x; e < tokens * d.key; e += 512) {
            const i64 to = ((first + e / d.key) * d.heads + hk) * d.key + e % d.key;
            dq[to] = dk[to] = from_float<T>(0.0f);
        }
        for (i64 e = threadIdx.x; e < tokens * spread; e += 512)
            dv[(first + e / spread) * d.value_heads * d.value + hk * spread + e % spread] = from_float<T>(0.0f);
        for (i64 e = threadIdx.x; e < tokens * d.group; e += 512) {
            const i64 to = (first + e / d.group) * d.value_heads + hk * d.group + e % d.group;
            if (d.beta_bf16) ((bf16_t*)dbeta)[to] = 0;
            else ((float*)dbeta)[to] = 0.0f;
            if (ddecay && d.decay_bf16) ((bf16_t*)ddecay)[to] = 0;
            else if (ddecay) ((float*)ddecay)[to] = 0.0f;
        }
        return;
    }
    const int columns = (int)(d.padded / 16);
    const Lane l;
    const i64 shared = tape.shared_chunk(d, b, hk, n);
    const bf16_t* keys_t = tape.keys_t + shared * (C * DK * N);
    const bf16_t* queries_t = tape.queries_t + shared * (C * DK * N);
    // the identity as operand: indices 16 half .. of 32 against 16 columns
    bf16x8 unit[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        unit[0][j] = j < 4 && l.quad + j == l.col ? (__bf16)1.0f : (__bf16)0.0f;
        unit[1][j] = j >= 4 && l.quad + j - 4 == l.col ? (__bf16)1.0f : (__bf16)0.0f;
    }
    // blocks (2 pair, c) and (2 pair + 1, c), turned, as half c % 2 of operands 2 pair and 2 pair + 1
    auto turn = [&](bf16_t* to, int pair, int c, float4_t a, float4_t b2) {
        const Pieces<3> pieces = split<3>(a, b2);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            Halves<3> turned;
#pragma unroll
            for (int i = 0; i < 3; ++i)
                turned.p[i] = __builtin_convertvector(__builtin_amdgcn_mfma_f32_16x16x32_bf16(pieces.p[i], unit[which], ZERO, 0, 0, 0), bf16x4);
            put_half<3>(to, 2 * pair + which, c, l, turned);
        }
    };
    for (int member = 0; member < d.group; ++member) {
        const i64 h = hk * d.group + member, chunk = tape.chunk(d, b, h, n);
        float4_t reads[F], backs[F], writes[F], pairs[4];  // dO S^T, Y S^T, E dS'^T, dO E^T or Y E^T
#pragma unroll
        for (int f = 0; f < F; ++f) reads[f] = backs[f] = writes[f] = ZERO;
#pragma unroll
        for (int j = 0; j < 4; ++j) pairs[j] = ZERO;
        float carried = 0.0f;  // this wave's share of <dS', S>
        const i64 t = n * C + token + l.col;
        const T* grad = back.grad.at<T>(b, existing(t, d), h);
        // a stage's blocks: DK / 32 x 2 pairs of S and of dS', 2 x 2 of E and of Y
        constexpr int UNITS = DK / 16;
        float4_t sv[2], gv[2], tv[2];
        Row<T, WIDE> next;
        auto fetch_stage = [&](int c) {
            const int u = wave % UNITS, r = u / 2 * 2;
            const float* tokens = (wave < 4 ? tape.errors : back.residuals);
            const int v = wave % 4, q = v / 2 * 2;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                sv[i] = block(tape.states, chunk * (DK / 16) + r + i, c + u % 2, columns, l);
                gv[i] = block(back.states, chunk * (DK / 16) + r + i, c + u % 2, columns, l);
                tv[i] = block(tokens, chunk * 4 + q + i, c + v % 2, columns, l);
            }
            next.load(grad, 16 * c, d.value, l);
        };
        float gate = 0.0f;
        if (threadIdx.x < GATES * C) gate = tape.gates[chunk * GATES * C + threadIdx.x];
        for (int c = 0; c < columns; c += 2) {
            fetch_stage(c);
            __syncthreads();  // the stage before is read
            if (c == 0 && threadIdx.x < GATES * C) gates[threadIdx.x / C][threadIdx.x % C] = gate;
            if (wave < UNITS) {
                const int u = wave;
                turn(s_stage, u / 2, u % 2, sv[0], sv[1]);
                turn(g_stage, u / 2, u % 2, gv[0], gv[1]);
                const float4_t dot = sv[0] * gv[0] + sv[1] * gv[1];
                carried += (dot[0] + dot[1]) + (dot[2] + dot[3]);
            }
            turn(wave < 4 ? e_stage : y_stage, wave % 4 / 2, wave % 2, tv[0], tv[1]);
            if (wave >= 4) {  // Y is the gradient of v
                const int col = (c + wave % 2) * 16 + l.col;
                if (col < d.value) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const i64 at = n * C + 16 * (wave % 4 / 2 * 2 + i) + l.quad + e;
                            if (at < d.time)
                                dv[((b * d.time + at) * d.value_heads + h) * d.value + col] = from_float<T>(at < length ? tv[i][e] : 0.0f);
                        }
                }
            }
            const Pieces<N> o = next.template operand<N>(16 * c, d.value, t < length, l);
            __syncthreads();
            const Pieces<3> y = fetch<3>(y_stage, tb, l), e = fetch<3>(e_stage, tb, l);
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const Pieces<3> s = fetch<3>(s_stage, key0 + f, l);
                reads[f] = mma<N, 3>(o, s, reads[f]);
                backs[f] = mma<3, 3>(y, s, backs[f]);
                writes[f] = mma<3, 3>(e, fetch<3>(g_stage, key0 + f, l), writes[f]);
                in_order();
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j > tb) continue;
                const Pieces<3> other = fetch<3>(e_stage, j, l);
                pairs[j] = half ? mma<3, 3>(y, other, pairs[j]) : mma<N, 3>(o, other, pairs[j]);
                in_order();
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = token + l.quad + e, c = 16 * j + l.col;
                const float a = r >= c ? decay(gates[SUM], gates[REMAINDER], r, c) : 0.0f;
                if (half) d2[r * CP + c] = r > c ? -a * pairs[j][e] : 0.0f;
                else d1[r * CP + c] = r >= c ? d.scale * a * pairs[j][e] : 0.0f;
            }
        __syncthreads();
        // the wave's own rows of the keys and queries, from the operands that hold them
        auto own = [&](const bf16_t* from, int f) {
            float4_t v = ZERO;
#pragma unroll
            for (int i = N - 1; i >= 0; --i)
                v += widen(*(const bf16x4*)(from + (((i64)(2 * (key0 + f) + tb / 2) * N + i) * 64 + l.id) * 8 + tb % 2 * 4));
            return v;
        };
        const float4_t since = *(const float4_t*)(gates[SINCE] + token + l.quad);
        const float4_t rest = *(const float4_t*)(gates[REST] + token + l.quad);
        const float4_t rate = *(const float4_t*)(gates[RATE] + token + l.quad);
        float4_t written = ZERO;  // k . rest B E dS'^T by row: its sum and g_C <dS', S> make <dS', S'>
#pragma unroll
        for (int f = 0; f < F; ++f) {
            reads[f] *= since * d.scale;
            backs[f] *= -since;
            writes[f] *= rest;
            written += own(keys_t, f) * writes[f] * rate;
        }
#pragma unroll 1
        for (int kb = 0; kb < 2; ++kb) {
            if (2 * kb <= tb) {  // sums over the tokens up to the wave's
                Pieces<3> a[2];
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const float* m = (w ? d2 : d1) + (token + l.col) * CP + 32 * kb + l.quad;
                    const float* by = gates[RATE] + 32 * kb + l.quad;
                    a[w] = split<3>(*(const float4_t*)m * *(const float4_t*)by, *(const float4_t*)(m + 16) * *(const float4_t*)(by + 16));
                }
#pragma unroll
                for (int f = 0; f < F; ++f) {
                    const Pieces<N> k = fetch<N>(keys_t, 2 * (key0 + f) + kb, l);
                    reads[f] = mma<3, N>(a[0], k, reads[f]);
                    backs[f] = mma<3, N>(a[1], k, backs[f]);
                }
            }
            if (2 * kb + 1 >= tb) {  // and over those from the wave's on
                Pieces<3> a[2];
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const float* m = (w ? d2 : d1) + 32 * kb * CP + token;
                    a[w] = split<3>(column(m, CP, l), column(m + 16 * CP, CP, l));
                }
#pragma unroll
                for (int f = 0; f < F; ++f) {
                    writes[f] = mma<3, N>(a[0], fetch<N>(queries_t, 2 * (key0 + f) + kb, l), writes[f]);
                    writes[f] = mma<3, N>(a[1], fetch<N>(keys_t, 2 * (key0 + f) + kb, l), writes[f]);
                }
            }
        }
        float4_t db = ZERO, dg = ZERO;
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const float4_t k = own(keys_t, f), q = own(queries_t, f);
            db += k * writes[f];
            dg += q * reads[f] + k * backs[f];
            backs[f] += rate * writes[f];
        }
        if (d.group > 1) {
#pragma unroll
            for (int f = 0; f < F; ++f) {
                float4_t* sum[2];
                if constexpr (DK == 64) {
                    sum[0] = &gq[f];
                    sum[1] = &gk[f];
                } else {
                    sum[0] = (float4_t*)sums[0] + (wave * F + f) * 64 + l.id;
                    sum[1] = (float4_t*)sums[1] + (wave * F + f) * 64 + l.id;
                }
                if (member > 0) {
                    reads[f] += *sum[0];
                    backs[f] += *sum[1];
                }
                *sum[0] = reads[f];
                *sum[1] = backs[f];
            }
        }
        if (member + 1 == d.group) {
#pragma unroll
            for (int f = 0; f < F; ++f)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const i64 at = n * C + token + l.quad + e;
                    const int c = 16 * (key0 + f) + l.col;
                    if (at >= d.time || c >= d.key) continue;
                    const i64 to = ((b * d.time + at) * d.heads + hk) * d.key + c;
                    dq[to] = from_float<T>(at < length ? reads[f][e] : 0.0f);
                    dk[to] = from_float<T>(at < length ? backs[f][e] : 0.0f);
                }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            db[e] = lane_sum<16>(db[e]);
            dg[e] = lane_sum<16>(dg[e]);
            if (l.col == 0) {
                lines[half][0][token + l.quad + e] = db[e];
                lines[half][1][token + l.quad + e] = dg[e];
            }
        }
        const float ends = lane_sum<64>((written[0] + written[1]) + (written[2] + written[3]) + gates[SINCE][C - 1] * carried);
        if (l.id == 0) part[wave] = ends;
        __syncthreads();
        if (threadIdx.x < 64) {
            const int i = threadIdx.x;
            const i64 at = n * C + i, to = (b * d.time + at) * d.value_heads + h;
            const float rates = lines[0][0][i] + lines[1][0][i];
            float v = lines[0][1][i] + lines[1][1][i] - gates[RATE][i] * rates;
            if (i == C - 1) v += ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
#pragma unroll
            for (int s = 1; s < 64; s *= 2) {
                const float above = __shfl_down(v, s, 64);
                if (i + s < 64) v += above;
            }
            if (at < d.time) {
                const bool live = at < length;
                if (d.beta_bf16) ((bf16_t*)dbeta)[to] = from_float<bf16_t>(live ? rates : 0.0f);
                else ((float*)dbeta)[to] = live ? rates : 0.0f;
                if (ddecay && d.decay_bf16) ((bf16_t*)ddecay)[to] = from_float<bf16_t>(live ? v : 0.0f);
                else if (ddecay) ((float*)ddecay)[to] = live ? v : 0.0f;
            }
        }
    }
}

// ------------------------------------------------------------------ host
Tensor tensor(const void* p, const int64_t* s) { return Tensor{p, s[0], s[1], s[2]}; }

// Keys up to 64 take operands of half the width: 256 x 100 of 4 heads of 64, float32, 545 us, and 894 with those of 128.
int key_width(const Delta& d) { return d.key <= 64 ? 64 : 128; }

// Workgroups of a scan: 16 columns each, whole groups of 8 heads (Place).
i64 scan_groups(const Delta& d) { return ceil_div(d.batch * d.value_heads, XCDS) * XCDS * (d.padded / 16); }

int check(const AtlasDelta* a, Delta& d, char* err, size_t cap, bool in_chunks = true) {
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
    d.padded = ceil_div(a->value, 32) * 32;
    d.scale = a->scale;
    if (in_chunks && scan_groups(d) * 4 * key_width(d) >= THREADS)
        return fail(err, cap, 7, "batch x value_heads x value is out of range");
    if (in_chunks && d.chunks * 512 >= THREADS) return fail(err, cap, 7, "time must be at most 2^29 - 64");
    return 0;
}

// Carves the workspace (256-byte pieces); what only the backward pass reads is there only to train.
i64 carve(const Delta& d, int type, int train, char* base, Tape* tape) {
    const i64 chunks = d.batch * d.value_heads * d.chunks, shared = d.batch * d.heads * d.chunks;
    const i64 pieces = type == ATLAS_OPS_BF16 ? 1 : 3;
    i64 at = 0;
    auto take = [&](auto*& p, i64 bytes, bool wanted = true) {
        p = wanted ? (std::decay_t<decltype(p)>)(base + at) : nullptr;
        if (wanted) at += ceil_div(bytes, 256) * 256;
    };
    Tape t{};
    take(t.keys, shared * C * key_width(d) * pieces * 2);
    take(t.queries, shared * C * key_width(d) * pieces * 2);
    take(t.keys_t, shared * C * key_width(d) * pieces * 2);
    take(t.queries_t, shared * C * key_width(d) * pieces * 2, train);
    take(t.inverse, chunks * TRIANGLE * 3 * 1024);
    take(t.scores, chunks * TRIANGLE * 3 * 1024);
    take(t.inverse_t, chunks * TRIANGLE * 3 * 1024, train);
    take(t.scores_t, chunks * TRIANGLE * 3 * 1024, train);
    take(t.gates, chunks * GATES * C * 4);
    take(t.errors, chunks * C * d.padded * 4, train);
    take(t.states, chunks * key_width(d) * d.padded * 4, train);
    if (tape) *tape = t;
    return at;
}

// Calls f with the element type, the key width's instantiation and whether rows of `width` are wide ones.
template <typename F>
void with_kernel(const Delta& d, int type, int width, F&& f) {
    auto by_width = [&](auto t, auto wide) {
        if (key_width(d) == 64) f(t, std::integral_constant<int, 64>{}, wide);
        else f(t, std::integral_constant<int, 128>{}, wide);
    };
    auto by_rows = [&](auto t) { width >= 4 ? by_width(t, std::true_type{}) : by_width(t, std::false_type{}); };
    if (type == ATLAS_OPS_F32) by_rows(0.0f);
    else by_rows(bf16_t{});
}

dim3 scan_grid(const Delta& d) { return dim3((unsigned)scan_groups(d)); }

}  // namespace
}  // namespace atlas_ops

using namespace atlas_ops;

extern "C" {

int atlas_ops_delta_step(const AtlasDelta* a, void* out, float* final_state, void* stream, char* err, size_t cap) {
    try {
        Delta d;
        if (int rc = check(a, d, err, cap, false)) return rc;
        if (!out || !final_state) return fail(err, cap, 7, "null argument");
        const dim3 grid((unsigned)ceil_div(d.value, 32), (unsigned)d.value_heads, (unsigned)d.batch);
        hipStream_t st = (hipStream_t)stream;
        // 16-byte accesses of the state need its rows to start on 16 bytes (64 x 8 heads of 128 x 128: 13.3 us, with
        // 4-byte ones 15.7)
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
    return check(a, d, nullptr, 0) ? 0 : carve(d, a->type, train, nullptr, nullptr);
}

int atlas_ops_delta_forward(const AtlasDelta* a, int train, void* out, float* final_state, void* workspace, void* stream,
                            char* err, size_t cap) {
    try {
        Delta d;
        if (int rc = check(a, d, err, cap)) return rc;
        if (!out || !final_state || !workspace) return fail(err, cap, 7, "null argument");
        Tape tape;
        carve(d, a->type, train, (char*)workspace, &tape);
        hipStream_t st = (hipStream_t)stream;
        const dim3 keys((unsigned)d.chunks, (unsigned)d.heads, (unsigned)d.batch);
        with_kernel(d, a->type, d.key, [&](auto t, auto width, auto wide) {
            using T = decltype(t);
            prepare<T, width(), wide() || width() == 128><<<keys, 256, 0, st>>>(d, tape, train);  // keys that wide fill four values
            if (train) scan_forward<T, width(), true><<<scan_grid(d), 4 * width(), 0, st>>>(d, tape, (T*)out, final_state);
            else scan_forward<T, width(), false><<<scan_grid(d), 4 * width(), 0, st>>>(d, tape, (T*)out, final_state);
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
        carve(d, a->type, 1, (char*)tape_memory, &tape);
        float* floats = (float*)workspace;
        const Back back{tensor(grad_out, grad_out_stride), grad_state, floats,
                        floats + d.batch * d.value_heads * d.chunks * C * d.padded};
        hipStream_t st = (hipStream_t)stream;
        const dim3 all((unsigned)d.chunks, (unsigned)d.heads, (unsigned)d.batch);
        with_kernel(d, a->type, d.value, [&](auto t, auto width, auto wide) {
            using T = decltype(t);
            scan_backward<T, width()><<<scan_grid(d), 4 * width(), 0, st>>>(d, tape, back, dstate);
            gradients<T, width(), wide()><<<all, 512, 0, st>>>(d, tape, back, (T*)dq, (T*)dk, (T*)dv, dlog_decay, dbeta);
        });
        return launched(err, cap, "delta_backward");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

}  // extern "C"
