// Linear attention with a decay by head: token by token for streaming, in chunks for sequences, and its
// gradients.  Part of libatlas_ops_hip.so.
//
// By token: S <- a S + k v^T, out = scale S^T q: Hebb's rule with forgetting.  In a chunk that starts from S,
// with G_i the sum of the log decays up to and with token i and g = exp(G):
//   out_i = scale (g_i S^T q_i + sum_{j <= i} exp(G_i - G_j) (q_i . k_j) v_j)
//   S'    = g_C S + sum_j exp(G_C - G_j) k_j v_j^T
// One kernel, `scan`, does this for three tensors (queries, keys, values), forwards or backwards in time, and
// the gradients are three more runs of it, at once.  With T_t the gradient of the state after token t,
//   T_t = a_{t+1} T_{t+1} + scale q_t dO_t^T   is the same recurrence backwards, and
//   dQ_t = scale S_t dO_t       forwards:  queries dO, keys v, values k (the state S^T)
//   dV_t = T_t^T k_t            backwards: queries k,  keys q, values dO
//   dK_t = T_t v_t              backwards: queries v,  keys dO, values q (the state T^T)
// The gradient of log a_t is L_t = <T_t, a_t S_{t-1}> with L_t = L_{t+1} + q_t . dQ_t - k_t . dK_t.  These dots cancel: with
// keys nearly orthogonal their parts are far larger than their sum.  So what a chunk's own tokens add, W_ij =
// scale exp(G_i - G_j) (dO_i . v_j) (q_i . k_j) for j < i, is taken pair by pair, as sums over rows less sums over columns
// (the dQ run has the first three factors and takes the fourth beside them), only what comes through the states is taken as
// dots, and every ANCHOR chunks L starts anew from the states themselves.  `decay_gradients` sums in 64 bits.
//
// Few sequences are split along time: `scan` first takes the sums of segments from an empty state, `join_states`
// carries the states through them, and every segment then runs from its own.
#include <algorithm>
#include <type_traits>

#include "device/atlas_mma.h"
#include "device/atlas_rows.h"

namespace atlas_ops {
namespace {

constexpr int MAX_WIDTH = 128;
constexpr i64 MAX_STRIDE = 1 << 24;  // from token to token: a chunk's offsets stay below 2^32 bytes
// Log decays are held from below, since differences of infinite sums are none.  No growth that float32 holds (e^88) brings back
// what this has emptied, and 64 of them still leave a chunk's sums, as a float and its remainder, to 2^-28.
constexpr float LOWEST = -16384.0f;

// Log decays of (batch, time, value head), of any strides.
struct Decays {
    Tensor x;
    int bf16;
    struct Raw { uint32_t low, high; };  // apart: joined they would be waited for at once
    // with a load that stands behind no branch (of `other` where there are no decays)
    __device__ __forceinline__ Raw load(const void* other, i64 b, i64 t, i64 h) const {
        const uint16_t* p = x.data ? (const uint16_t*)x.data + ((b * x.batch + t * x.time + h * x.head) << (bf16 ? 0 : 1)) : (const uint16_t*)other;
        return {p[0], p[x.data && !bf16 ? 1 : 0]};
    }
    __device__ __forceinline__ float value(Raw r) const {
        const float g = __uint_as_float(bf16 ? r.low << 16 : r.high << 16 | r.low);
        return !x.data ? 0.0f : g < LOWEST ? LOWEST : g;  // a NaN stays one
    }
};

__device__ __forceinline__ i64 length_of(const int32_t* lengths, i64 time, i64 b) {
    if (!lengths) return time;
    const i64 n = lengths[b];
    return n < 0 ? 0 : n < time ? n : time;
}

// ------------------------------------------------------------------ token by token
// 16 bytes in one access wherever a caller's floats start: a state need not lie on 16 bytes, and gfx950 takes any.
typedef float4_t float4_any_t __attribute__((aligned(4)));

struct Step {
    Tensor q, k, v;
    Decays decay;
    const float* state;
    const int32_t* lengths;
    i64 time;
    int value_heads, group, key, value;
    float scale;
};

// A workgroup holds 32 columns of one head's state in registers: row groups of 32 / VEC lanes, each lane VEC
// neighbouring columns of every 8 VEC-th row.  One reduction per token: S^T q of the new state.  Memory bounds one
// token: the state is read and written once, 64 streams of 8 heads of 128 x 128 in 11.5 us (5.9 TB/s).
template <typename T, int VEC>
__global__ void __launch_bounds__(256) step_kernel(Step d, T* __restrict__ out, float* final_state) {
    constexpr int LANES = 32 / VEC, ROWS = 256 / LANES, PER = MAX_WIDTH / ROWS;
    __shared__ float sums[2][4][32];
    const int lane = threadIdx.x % LANES, row = threadIdx.x / LANES, wave = threadIdx.x / 64;
    const i64 b = blockIdx.z, h = blockIdx.y, hk = h / d.group;
    const int col = blockIdx.x * 32 + lane * VEC;
    const i64 base = (b * d.value_heads + h) * d.key * d.value;
    // Nothing is loaded behind a branch, or each load would be waited for before the next: rows and columns that
    // do not exist read the last, and their values become zeros.
    T kt[PER], qt[PER], vt[VEC];
    Decays::Raw raw;
    auto fetch = [&](i64 t) {
        const T *qp = d.q.at<T>(b, t, hk), *kp = d.k.at<T>(b, t, hk), *vp = d.v.at<T>(b, t, h);
        raw = d.decay.load(qp, b, t, h);
#pragma unroll
        for (int c = 0; c < VEC; ++c) vt[c] = vp[min(col + c, d.value - 1)];
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            const int at = min(row + r * ROWS, d.key - 1);
            kt[r] = kp[at];
            qt[r] = qp[at];
        }
    };
    float s[PER][VEC];
    const float* from = (d.state ? d.state : final_state) + base + min(col, d.value - VEC);
#pragma unroll
    for (int r = 0; r < PER; ++r) {
        const float* p = from + (i64)min(row + r * ROWS, d.key - 1) * d.value;
        if constexpr (VEC == 4) {  // value is a multiple of 4
            const float4_t v = *(const float4_any_t*)p;
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
    const i64 length = length_of(d.lengths, d.time, b);
    for (i64 t = 0; t < d.time; ++t) {
        T* o = out + ((b * d.time + t) * d.value_heads + h) * d.value;
        if (t >= length) {
            if (row == 0)
                for (int c = 0; c < VEC; ++c)
                    if (col + c < d.value) o[col + c] = from_float<T>(0.0f);
            continue;
        }
        const float a = expf(d.decay.value(raw));
        float v[VEC], kr[PER], qr[PER], qs[VEC];
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
            v[c] = col + c < d.value ? to_float(vt[c]) : 0.0f;
            qs[c] = 0.0f;
        }
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            const int at = row + r * ROWS;
            kr[r] = at < d.key ? to_float(kt[r]) : 0.0f;
            qr[r] = at < d.key ? to_float(qt[r]) : 0.0f;
        }
        if (t + 1 < length) fetch(t + 1);
#pragma unroll
        for (int r = 0; r < PER; ++r)
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                s[r][c] = a * s[r][c] + kr[r] * v[c];
                qs[c] += s[r][c] * qr[r];
            }
#pragma unroll
        for (int step = LANES; step < 64; step *= 2)
#pragma unroll
            for (int c = 0; c < VEC; ++c) qs[c] += __shfl_xor(qs[c], step, 64);
        const int turn = t & 1;  // the sums of the token before are read until the next barrier
        if (threadIdx.x % 64 < LANES) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) sums[turn][wave][lane * VEC + c] = qs[c];
        }
        __syncthreads();
        if (row == 0) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                const int at = lane * VEC + c;
                const float sum = (sums[turn][0][at] + sums[turn][1][at]) + (sums[turn][2][at] + sums[turn][3][at]);
                if (col + c < d.value) o[col + c] = from_float<T>(d.scale * sum);
            }
        }
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
            *(float4_any_t*)p = v;
        } else {
            *p = s[r][0];
        }
    }
}

// ------------------------------------------------------------------ chunks
// One of the three tensors of a scan: value head h reads head h / group.
struct Role {
    Tensor x;
    int group, width;
};

struct Scan {
    Role q, k, v;                  // q and k of one width, v of the outputs'
    Decays decay;
    const int32_t* lengths;
    i64 time;
    int value_heads, chunks, per, segments;  // per: chunks of a segment
    int first;                     // the segment of blockIdx.x = 0
    int backwards;                 // in time: row r of a chunk is its token C - 1 - r, which decays by the token behind
    float write, read;             // factors of k v^T and of the outputs
    // the states at the segments' starts, [batch, value head, segment] (or without segments), of q's x v's widths,
    // or `turned`; null: zeros
    const float* start;
    int start_segments, turned;
    // outputs (null to take the segments' sums only)
    void* out;                     // (batch, time, value_heads, v's width) contiguous
    int out_f32;                   // float32 whatever T is
    float *final_state, *copy;     // after the last segment; backwards also decayed by the first token; may be null
    float *sums, *decays;          // [batch, value head, segment]: a segment's state from zeros, and its whole decay
    Role dot;                      // what dots and pairs multiply with
    float* dots;                   // [batch, value head, time] or null: dots with what the states answer
    float* pairs;                  // [batch, value head, time] or null: by token, sums of W over its row less over its column
    float* anchors;                // [batch, value head, anchor] or null: the states there, key by value
};

// Runs of equal widths in one launch: blockIdx.x counts the segments of one after the other.
struct Runs {
    Scan run[3];
    int segments;  // of a run
};

// Anchors lie behind every ANCHOR-th chunk but the last: an error of the dots reaches as far back.  Training on 16384 tokens of 8
// heads of 128: 4, 8 or 16 take 388, 383 or 375 us.
constexpr int ANCHOR = 8;
__host__ __device__ inline i64 anchors_of(i64 chunks) { return (chunks - 1) / ANCHOR; }

template <typename T>
struct Cut {
    static constexpr int N = sizeof(T) == 2 ? 1 : 3;    // bfloat16 pieces of a value
    static constexpr int C = sizeof(T) == 2 ? 64 : 32;  // tokens per chunk
};

// Four values of column l % 16, rows quad .. quad + 3 from `at`, the address of row quad + l % 16 / 4, columns 4 (l % 4) ..:
// the hardware turns 4 x 16 blocks for 16 lanes each.
__device__ __forceinline__ bf16x4 turned_read(const bf16_t* at) {
    typedef __attribute__((address_space(3))) bf16x4 lds;
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds*)(at));
}

__device__ __forceinline__ bf16x8 both(bf16x4 a, bf16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// Whether any of eight values is a NaN or an infinity: its exponent's bits are all ones.
__device__ __forceinline__ bool beyond(bf16x8 v) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    const uint4_t bits = __builtin_bit_cast(uint4_t, v);
    u16x2 most = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, bits[i] & 0x7FFF7FFFu));
    return max(most[0], most[1]) >= 0x7F80;
}
__device__ __forceinline__ bool beyond(float4_t a, float4_t b) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max(max(most, __float_as_uint(a[i]) & 0x7FFFFFFFu), __float_as_uint(b[i]) & 0x7FFFFFFFu);
    return most >= 0x7F800000u;
}

// Four values of a row of `width` from column c0, zeros beyond it.
template <typename T>
struct Four { T v[4]; };

template <bool WHOLE, typename T>
__device__ __forceinline__ Four<T> four(const T* row, int c0, int width) {
    Four<T> x;
    if constexpr (WHOLE) {
        struct __attribute__((packed, aligned(sizeof(T)))) Packed { T v[4]; } raw = *(const Packed*)(row + (c0 < width ? c0 : 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) x.v[e] = c0 < width ? raw.v[e] : T{};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x.v[e] = c0 + e < width ? row[c0 + e] : T{};
    }
    return x;
}

// A thread's share of a chunk's rows, C tokens of up to W values: units of 16 bytes in every STEP-th token.  The loads stand
// behind no branch: what is no unit of the row or not of a live token reads the chunk's first and becomes zero.  Without
// WHOLE units the one that the row's end cuts is read as the row's last 16 bytes and shifted down when it is placed.
template <typename T, int W, int THREADS, int C, bool WHOLE>
struct Share {
    static constexpr int E = Unit<T>::N, ACROSS = W / E, STEP = THREADS / ACROSS, COUNT = C / STEP;
    static_assert(C % STEP == 0, "every thread has the same number of units");
    Unit<T> unit[COUNT];

    __device__ __forceinline__ static int token(uint32_t thread) { return thread / ACROSS; }
    __device__ __forceinline__ static int column(uint32_t thread) { return thread % ACROSS * E; }
    // live: tokens of the chunk that are
    __device__ __forceinline__ void load(uint32_t thread, const T* chunk, int stride, int width, int live) {
        const int column = Share::column(thread);
#pragma unroll
        for (int u = 0; u < COUNT; ++u) {
            const int t = token(thread) + u * STEP;
            if constexpr (WHOLE) {
                unit[u].memcpy_in(chunk + (uint32_t)(t < live && column < width ? t * stride + column : 0));
            } else {
                unit[u].load(chunk + (uint32_t)(t < live ? t * stride : 0), column, width);
            }
        }
    }
    // all: every unit is one of the row and of a live token
    __device__ __forceinline__ Unit<T> value(uint32_t thread, int u, int width, int live, bool all) const {
        Unit<T> x = unit[u];
        if (all) return x;
        const bool some = token(thread) + u * STEP < live && column(thread) < width;
        x.low = some ? x.low : 0;
        x.high = some ? x.high : 0;
        return x;
    }
};

// The thread's number, from which nothing can be computed ahead of a loop: what is kept for every turn there costs
// registers that the state needs.
__device__ __forceinline__ uint32_t thread_here() {
    uint32_t thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    return thread;
}

// Workgroup: one segment of one value head.  Wave w holds the state's columns of its NB blocks of 16 in
// registers, all DK rows.  NB = 2: block n of the wave has columns 32 w + 8 i + 4 n + j (i, j < 4) at lanes 4 i + j, so
// that a lane's results are eight neighbours; NB = 1: 16 w + l.  The tiles lie in LDS token by token, in the order of the
// recurrence; operands whose sums go over tokens are turned as they are read.  WHOLE: both widths are whole units of 16
// bytes.
//
// Products are to 24 bits: a float32 operand is the sum of three bfloat16 pieces (six matrix instructions for a product), the
// state and the decayed scores are so in either type.  16384 tokens of 16 heads of 128 bfloat16 in 32 segments: 105 us, 512
// workgroups at two to a CU, which 253 registers and 75 KB of LDS allow alike; 256 x 100 tokens of 4 heads of 64 float32: 49 us,
// their three gradients 145, three to a CU by 135 registers and 44 KB.  Vector instructions take 48 % of the first's time, LDS 37 %,
// matrix instructions 29 %, of the others 45 to 57 %, 41 to 47 % and 18 to 21 %: what bounds it is the chain of a chunk's stages with 8
// to 12 waves on a CU.
template <typename T, int DK, int NB, bool OUT, bool WHOLE>
__global__ void __launch_bounds__(256, 2) scan(Runs) {
    // the launch's argument, where it lies: an index into a copy would need memory
    const auto* runs = (const __attribute__((address_space(4))) Runs*)__builtin_amdgcn_kernarg_segment_ptr();
    const int which = blockIdx.x / runs->segments;
    const Scan d = ((const Runs*)runs)->run[which];
    constexpr int N = Cut<T>::N, C = Cut<T>::C, QB = C / 16, KB = C / 32, WAVES = 4, THREADS = 64 * WAVES, DV = 16 * NB * WAVES;
    constexpr int PITCH = DK + 8, VPITCH = DV + (sizeof(T) == 2 ? 8 : 4);
    constexpr int BLOCKS = QB * (QB + 1) / 2, OPERANDS = QB == 4 ? 6 : 2;  // of scores that are not zero: 16 x 16, 16 queries x 32 keys
    __shared__ __attribute__((aligned(16))) bf16_t qs[OUT ? N * C * PITCH : 8], ks[N * C * PITCH];
    __shared__ __attribute__((aligned(16))) T vs[C * VPITCH];
    __shared__ __attribute__((aligned(16))) bf16_t scores[OUT ? OPERANDS * 3 * 512 : 8];
    // of two chunks in turn: G as a float and its remainder, the factors of what the state answers and of what is written to it
    __shared__ __attribute__((aligned(16))) float gate_sum[2][C], gate_rest[2][C], since[2][C], rest[2][C], decays[2];
    __shared__ float dot_part[OUT ? WAVES : 1][C], pair_rows[OUT ? BLOCKS : 1][16];
    __shared__ __attribute__((aligned(16))) float pair_columns[OUT ? BLOCKS : 1][16];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int segment = d.first + blockIdx.x - which * runs->segments;
    const i64 h = blockIdx.y, b = blockIdx.z, head = b * d.value_heads + h;
    const i64 length = length_of(d.lengths, d.time, b);
    const int low = segment * d.per, high = min(low + d.per, d.chunks);
    const int used = (int)((length + C - 1) / C);  // chunks with a token
    const int inner = d.q.width, outer = d.v.width;
    const T *qp = d.q.x.at<T>(b, 0, h / d.q.group), *kp = d.k.x.at<T>(b, 0, h / d.k.group), *vp = d.v.x.at<T>(b, 0, h / d.v.group);
    auto cell = [&](const Lane& l, int n) { return 16 * NB * wave + 4 * NB * (l.col / 4) + l.col % 4 + 4 * n; };

    // the state: block r of rows 16 r .., block n of columns
    float4_t s[DK / 16][NB];
#pragma unroll
    for (int r = 0; r < DK / 16; ++r)
#pragma unroll
        for (int n = 0; n < NB; ++n) s[r][n] = ZERO;
    if (OUT && d.start) {
        const float* from = d.start + (d.start_segments ? head * d.segments + segment : head) * inner * outer;
        const int down = d.turned ? 1 : outer, across = d.turned ? inner : 1;
        const Lane l(thread_here());
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int column = cell(l, n), at = min(column, outer - 1) * across;
#pragma unroll
            for (int r = 0; r < DK / 16; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[r][n][j] = from[(uint32_t)(min(16 * r + l.quad + j, inner - 1) * down + at)];
#pragma unroll
            for (int r = 0; r < DK / 16; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[r][n][j] = 16 * r + l.quad + j < inner && column < outer ? s[r][n][j] : 0.0f;
        }
    }
    if constexpr (OUT)  // halves of operands above the diagonal stay zero
        for (int i = threadIdx.x; i < OPERANDS * 3 * 512 / 2; i += THREADS) ((uint32_t*)scores)[i] = 0;

    Share<T, DK, THREADS, C, WHOLE> qu, ku;
    Share<T, DV, THREADS, C, WHOLE> vu;
    Decays::Raw raw;
    // row r of a tile is the chunk's token r, backwards C - 1 - r
    auto token = [&](int row) { return d.backwards ? C - 1 - row : row; };
    auto fetch = [&](int chunk, int which) {  // a part at a time: the loads of one after the other would hold the wave up
        const i64 t0 = (i64)chunk * C;
        const int live = (int)min((i64)C, length - t0);
        const uint32_t thread = thread_here();
        if (which & 1) {
            raw = d.decay.load(qp, b, min(t0 + token(thread % C) + d.backwards, d.time - 1), h);
            if constexpr (OUT) qu.load(thread, qp + t0 * d.q.x.time, (int)d.q.x.time, inner, live);
        }
        if (which & 2) ku.load(thread, kp + t0 * d.k.x.time, (int)d.k.x.time, inner, live);
        if (which & 4) vu.load(thread, vp + t0 * d.v.x.time, (int)d.v.x.time, outer, live);
    };
    // a unit as the N planes of a tile
    auto place = [&](bf16_t* tile, const Unit<T>& u, int row, int col) {
        bf16_t* p = tile + row * PITCH + col;
        if constexpr (N == 1) {
            ((u64*)p)[0] = u.low;
            ((u64*)p)[1] = u.high;
        } else {
            const Halves<3> parts = split<3>(float4_t{u[0], u[1], u[2], u[3]});
#pragma unroll
            for (int i = 0; i < 3; ++i) *(bf16x4*)(p + i * C * PITCH) = parts.p[i];
        }
    };
    // operand of a block of 16 rows of a tile, 32 columns from c0
    auto rows_operand = [&](const Lane& l, const bf16_t* tile, int block, int c0) {
        Pieces<N> r;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bf16_t* p = tile + i * C * PITCH + (16 * block + l.col) * PITCH + c0 + l.quad;
            r.p[i] = both(*(const bf16x4*)p, *(const bf16x4*)(p + 16));
        }
        return r;
    };
    // the values as an operand of block n's columns, sums over 32 tokens: as bfloat16, and as floats
    auto value_raw = [&](const Lane& l, int kb, int n) {
        const bf16_t* p = (const bf16_t*)vs + (32 * kb + l.quad + l.col / 4) * VPITCH + 16 * NB * wave + 4 * NB * (l.col % 4) + 4 * n;
        return Halves<2>{turned_read(p), turned_read(p + 16 * VPITCH)};
    };
    auto value_floats = [&](const Lane& l, int kb, int n, float4_t (&x)[2]) {
        if constexpr (N == 1) {
            const Halves<2> v = value_raw(l, kb, n);
            x[0] = widen(v.p[0]), x[1] = widen(v.p[1]);
        } else {
            const float* p = (const float*)vs + (32 * kb + l.quad) * VPITCH + cell(l, n);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[0][j] = p[j * VPITCH], x[1][j] = p[(16 + j) * VPITCH];
        }
    };

    // a chunk's decays, in powers of two, by the last wave, which has the fewest scores
    double whole = 0.0;  // log decay of the segment's chunks, in that wave
    auto gates = [&](int chunk, int turn) {
        const int lane = thread_here() % 64, row = lane % C;
        const i64 t = (i64)chunk * C + token(row) + d.backwards;
        double sum = t < length ? (double)d.decay.value(raw) * 1.4426950408889634 : 0.0;
#pragma unroll
        for (int k = 1; k < C; k *= 2) {
            const double before = __shfl_up(sum, k, C);
            if (row >= k) sum += before;
        }
        const double total = __shfl(sum, C - 1, 64);
        if (lane < C) {
            gate_sum[turn][row] = (float)sum;
            gate_rest[turn][row] = (float)(sum - (double)(float)sum);
            since[turn][row] = __builtin_amdgcn_exp2f((float)sum) * d.read;
            rest[turn][row] = __builtin_amdgcn_exp2f((float)(total - sum)) * d.write;
        }
        if (lane == 0) decays[turn] = __builtin_amdgcn_exp2f((float)total);
        whole += total;
    };

    auto anchor = [&](int chunk) {  // the state there
        const Lane l(thread_here());
        float* p = d.anchors + (head * anchors_of(d.chunks) + (chunk + 1) / ANCHOR - 1) * inner * outer;
        const int down = d.turned ? 1 : outer, across = d.turned ? inner : 1;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int r = 0; r < DK / 16; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = 16 * r + l.quad + j, column = cell(l, n);
                    if (row < inner && column < outer) p[(uint32_t)(row * down + column * across)] = s[r][n][j];
                }
        in_order();
    };

    const int steps = high - low;
    if (low < used) {
        const int first = d.backwards ? min(high, used) - 1 : low;
        fetch(first, 7);
        if (wave == WAVES - 1) gates(first, (d.backwards ? high - 1 - first : 0) & 1);
    }
    for (int step = 0; step < steps; ++step) {
        const int chunk = d.backwards ? high - 1 - step : low + step;
        const i64 t0 = (i64)chunk * C;
        if (chunk >= used) {  // no token: zeros
            if constexpr (OUT) {
                const int rows = (int)min((i64)C, d.time - t0);
                for (int at = threadIdx.x; at < rows * outer; at += THREADS) {
                    const i64 o = ((b * d.time + t0 + at / outer) * d.value_heads + h) * outer + at % outer;
                    if (d.out_f32) ((float*)d.out)[o] = 0.0f;
                    else ((T*)d.out)[o] = from_float<T>(0.0f);
                }
                if (d.dots && (int)threadIdx.x < rows) d.dots[head * d.time + t0 + threadIdx.x] = 0.0f;
                if (d.pairs && (int)threadIdx.x < rows) d.pairs[head * d.time + t0 + threadIdx.x] = 0.0f;
            }
            continue;
        }
        const int live = (int)min((i64)C, length - t0);
        const uint32_t thread = thread_here();
        const Lane l(thread);
        const bool anchored = OUT && d.anchors && (chunk + 1) % ANCHOR == 0 && chunk + 1 < used;
        if (anchored && d.backwards) anchor(chunk);
        // ---- the chunk into LDS
        const bool all_q = live == C && inner == DK, all_v = live == C && outer == DV;
        const int turn = step & 1;
#pragma unroll
        for (int u = 0; u < ku.COUNT; ++u) {
            const int row = token(ku.token(thread) + u * ku.STEP);
            if constexpr (OUT) place(qs, qu.value(thread, u, inner, live, all_q), row, qu.column(thread));
            place(ks, ku.value(thread, u, inner, live, all_q), row, ku.column(thread));
        }
#pragma unroll
        for (int u = 0; u < vu.COUNT; ++u) {
            const Unit<T> x = vu.value(thread, u, outer, live, all_v);
            u64* p = (u64*)(vs + token(vu.token(thread) + u * vu.STEP) * VPITCH + vu.column(thread));
            p[0] = x.low;
            p[1] = x.high;
        }
        lds_barrier();
        const int next = d.backwards ? chunk - 1 : chunk + 1;
        const bool more = d.backwards ? next >= low : next < min(high, used);
        if (more) fetch(next, OUT ? 1 : 7);
        in_order();

        if constexpr (OUT) {
            // ---- decayed scores, turned: rows are keys, columns queries
            constexpr int OWN = (BLOCKS + WAVES - 1) / WAVES;  // blocks of a wave, all in flight; what lies beyond the last is not kept
            float4_t p[OWN], p_small[OWN];
            int qbs[OWN], kjs[OWN];
#pragma unroll
            for (int m = 0; m < OWN; ++m) {
                const int block = min(wave + WAVES * m, BLOCKS - 1);
                qbs[m] = block >= 6 ? 3 : block >= 3 ? 2 : block >= 1 ? 1 : 0;
                kjs[m] = block - qbs[m] * (qbs[m] + 1) / 2;
                p[m] = p_small[m] = ZERO;
            }
            Pieces<N> kn[2][OWN], qn[2][OWN];
            auto read = [&](int c) {
#pragma unroll
                for (int m = 0; m < OWN; ++m) {
                    kn[c & 1][m] = rows_operand(l, ks, kjs[m], 32 * c);
                    qn[c & 1][m] = rows_operand(l, qs, qbs[m], 32 * c);
                }
                in_order();
            };
            read(0);
#pragma unroll
            for (int c = 0; c < DK / 32; ++c) {
                if (c + 1 < DK / 32) read(c + 1);
                mma_each(kn[c & 1], qn[c & 1], p, p_small);
                in_order();
            }
            if constexpr (N > 1)
#pragma unroll
                for (int m = 0; m < OWN; ++m) p[m] += p_small[m];
            const float factor = d.write * d.read;
#pragma unroll
            for (int m = 0; m < OWN; ++m) {
                const int qb = qbs[m], kj = kjs[m], i = 16 * qb + l.col, at = 16 * kj + l.quad;
                const float sum = gate_sum[turn][i], remainder = gate_rest[turn][i];
                const float4_t sums = *(const float4_t*)(gate_sum[turn] + at), remainders = *(const float4_t*)(gate_rest[turn] + at);
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // both selects: a masked decay may be infinite, a masked score anything
                    const float decay = __builtin_amdgcn_exp2f(at + j <= i ? (sum - sums[j]) + (remainder - remainders[j]) : 0.0f);
                    float x = p[m][j] * decay * factor;
                    asm("" : "+v"(x));  // a select, not a branch
                    p[m][j] = at + j <= i ? x : 0.0f;
                }
                const int operand = QB == 4 ? (qb < 2 ? qb : 2 * (qb - 1) + kj / 2) : qb;
                const Halves<3> parts = split_pairs(p[m]);
                if (wave + WAVES * m < BLOCKS) put_half<3>(scores, operand, kj % 2, l, parts);
            }
            if (d.pairs) {
                // ---- W: the scores times the dots of the other two tensors, a row of `dot` (the queries') and one of the values
#pragma unroll
                for (int m = 0; m < OWN; ++m) {
                    const int qb = qbs[m], kj = kjs[m], t = token(16 * qb + l.col);
                    const T* row = d.dot.x.at<T>(b, t0 + (t < live ? t : 0), h / d.dot.group);
                    const T* key = vs + (16 * kj + l.col) * VPITCH;
                    float4_t w[1] = {ZERO}, w_small[1] = {ZERO};
#pragma unroll
                    for (int c = 0; c < DV / 32; ++c) {
                        const int c0 = 32 * c + l.quad;
                        Pieces<N> a[1], x[1];
                        if constexpr (N == 1) {
                            a[0].p[0] = both(*(const bf16x4*)(key + c0), *(const bf16x4*)(key + c0 + 16));
                            x[0].p[0] = both(__builtin_bit_cast(bf16x4, four<WHOLE>(row, c0, outer)), __builtin_bit_cast(bf16x4, four<WHOLE>(row, c0 + 16, outer)));
                        } else {
                            a[0] = split<3>(*(const float4_t*)(key + c0), *(const float4_t*)(key + c0 + 16));
                            x[0] = split<3>(__builtin_bit_cast(float4_t, four<WHOLE>(row, c0, outer)), __builtin_bit_cast(float4_t, four<WHOLE>(row, c0 + 16, outer)));
                        }
                        mma_each(a, x, w, w_small);
                    }
                    if constexpr (N > 1) w[0] += w_small[0];
                    const int i = 16 * qb + l.col, at = 16 * kj + l.quad;
                    float sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        w[0][j] = at + j < i && t < live ? w[0][j] * p[m][j] : 0.0f;
                        sum += w[0][j];
                    }
                    sum += __shfl_xor(sum, 16, 64);
                    sum += __shfl_xor(sum, 32, 64);
                    float4_t down;
#pragma unroll
                    for (int j = 0; j < 4; ++j) down[j] = lane_sum<16>(w[0][j]);
                    const int block = wave + WAVES * m;
                    if (block < BLOCKS && l.quad == 0) pair_rows[block][l.col] = sum;
                    if (block < BLOCKS && l.col == 0) *(float4_t*)(pair_columns[block] + l.quad) = down;
                }
                in_order();
            }
            if (more) fetch(next, 2);
            in_order();
            // ---- what the state answers: rows are columns of the values, columns are queries
            float4_t o[NB][QB], o_small[N > 1 ? NB : 1][N > 1 ? QB : 1];
#pragma unroll
            for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    o[n][qb] = ZERO;
                    if constexpr (N > 1) o_small[n][qb] = ZERO;
                }
            Pieces<N> q[2][QB];
            auto read_queries = [&](int c) {
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) q[c & 1][qb] = rows_operand(l, qs, qb, 32 * c);
                in_order();
            };
            read_queries(0);
#pragma unroll
            for (int c = 0; c < DK / 32; ++c) {
                Pieces<3> state[NB];
#pragma unroll
                for (int n = 0; n < NB; ++n) state[n] = split_pairs(s[2 * c][n], s[2 * c + 1][n]);
                if (c + 1 < DK / 32) read_queries(c + 1);
                if constexpr (N > 1) mma_grid(state, q[c & 1], o, o_small);
                else mma_grid(state, q[c & 1], o);
                in_order();
            }
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                const float g = since[turn][16 * qb + l.col];
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    if constexpr (N > 1) o[n][qb] += o_small[n][qb];
                    o[n][qb] *= g;
                }
            }
            constexpr bool FULL = WHOLE && (sizeof(T) == 2 || NB == 1);  // a lane's 4 NB neighbouring columns are there or none
            const int c0 = 16 * NB * wave + NB * l.quad, left = outer - c0;
            if (d.dots) {
                const T* x0 = d.dot.x.at<T>(b, t0, h / d.dot.group) + (left > 0 ? c0 : 0);
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) {
                    const int t = token(16 * qb + l.col);
                    const T* x = x0 + (t < live && left > 0 ? (uint32_t)(t * (int)d.dot.x.time) : 0u);
                    struct __attribute__((packed, aligned(sizeof(T)))) Few { T v[4 * NB]; } few;
                    if constexpr (FULL) {
                        few = *(const Few*)x;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4 * NB; ++e) few.v[e] = x[min(e, max(left - 1, 0))];
                    }
                    float dot = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4 * NB; ++e) dot += FULL || e < left ? o[e / 4][qb][e % 4] * to_float(few.v[e]) : 0.0f;
                    dot = t < live && left > 0 ? dot : 0.0f;
                    dot += __shfl_xor(dot, 16, 64);
                    dot += __shfl_xor(dot, 32, 64);
                    if (l.quad == 0) dot_part[wave][16 * qb + l.col] = dot;
                }
            }
            lds_barrier();  // the scores are there
            if (more) fetch(next, 4);
            in_order();
            // ---- the chunk's own tokens.  A NaN or an infinity among the values would reach the tokens before it through
            // zeros of the scores: it is taken out, and the rows from its column's first on are NaN afterwards
            constexpr int PAIRS = QB == 4 ? 3 : 1;  // (32 keys, two blocks of queries) that are not zero: (0, 0), (0, 2), (1, 2)
            Pieces<3> pn[2][2];
            auto read_scores = [&](int pair) {
#pragma unroll
                for (int i = 0; i < 2; ++i) pn[pair & 1][i] = atlas_ops::fetch<3>(scores, pair == 0 ? i : 2 * (i + 1) + pair - 1, l);
                in_order();
            };
            int worst[NB];
            bool any = false;
#pragma unroll
            for (int n = 0; n < NB; ++n) worst[n] = C;
            read_scores(0);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                Pieces<N> value[NB];
                float4_t x[NB][2];
                bool faulty = false;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    if constexpr (N == 1) {
                        const Halves<2> v = value_raw(l, kb, n);
                        value[n].p[0] = both(v.p[0], v.p[1]);
                        faulty |= beyond(value[n].p[0]);
                    } else {
                        value_floats(l, kb, n, x[n]);
                        faulty |= beyond(x[n][0], x[n][1]);
                    }
                }
                if (__ballot(faulty)) {
                    any = true;
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        value_floats(l, kb, n, x[n]);
#pragma unroll
                        for (int e = 7; e >= 0; --e)
                            if (!(fabsf(x[n][e / 4][e % 4]) < INFINITY)) {
                                x[n][e / 4][e % 4] = 0.0f;
                                worst[n] = min(worst[n], 32 * kb + 16 * (e / 4) + l.quad + e % 4);
                            }
                        if constexpr (N == 1) value[n] = split<1>(x[n][0], x[n][1]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NB; ++n)
                    if constexpr (N == 3) value[n] = split_pairs(x[n][0], x[n][1]);
#pragma unroll
                for (int pair = kb == 0 ? 0 : 2; pair < (kb == 0 ? min(2, PAIRS) : 3); ++pair) {
                    if (pair + 1 < PAIRS) read_scores(pair + 1);
                    const int q0 = pair == 0 ? 0 : 2;
                    float4_t sums[NB][2];
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) sums[n][i] = o[n][q0 + i];
                    mma_grid(value, pn[pair & 1], sums);
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) o[n][q0 + i] = sums[n][i];
                    in_order();
                }
            }
            if (any) {
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    worst[n] = min(worst[n], __shfl_xor(worst[n], 16, 64));
                    worst[n] = min(worst[n], __shfl_xor(worst[n], 32, 64));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int first = __shfl(worst[n], l.quad + j, 64);  // of the results' row
#pragma unroll
                        for (int qb = 0; qb < QB; ++qb)
                            if (16 * qb + l.col >= first) o[n][qb][j] = NAN;
                    }
                }
            }
            if (live < C) {
#pragma unroll
                for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                    for (int n = 0; n < NB; ++n)
                        if (token(16 * qb + l.col) >= live) o[n][qb] = ZERO;
            }
            // ---- a lane's 4 NB neighbouring columns of one token
            const i64 out0 = ((b * d.time + t0) * d.value_heads + h) * outer + c0;
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                const int t = token(16 * qb + l.col);
                float row[4 * NB];
#pragma unroll
                for (int e = 0; e < 4 * NB; ++e) row[e] = o[e / 4][qb][e % 4];
                if (t0 + t < d.time && left > 0) {
                    const i64 at = out0 + (uint32_t)(t * d.value_heads * outer);
                    if (d.out_f32) store_unit<float, 4 * NB>((float*)d.out + at, FULL ? 4 * NB : left, row);
                    else store_unit<T, 4 * NB>((T*)d.out + at, FULL ? 4 * NB : left, row);
                }
            }
            in_order();
        }

        // ---- the state behind the chunk; of float32 the chunk's share is summed alone, and the state rounded once
        const float decayed = decays[turn];
        if constexpr (KB > 1)
#pragma unroll
            for (int r = 0; r < DK / 16; ++r)
#pragma unroll
                for (int n = 0; n < NB; ++n) s[r][n] *= decayed;
        constexpr int R = N == 1 ? 4 : 2, GROUPS = DK / 16 / R;  // blocks of rows at a time
        Pieces<N> kt[2][R];
        auto read_keys = [&](int at) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const bf16_t* p = ks + i * C * PITCH + (32 * (at / GROUPS) + l.quad + l.col / 4) * PITCH + 16 * (at % GROUPS * R + r) + 4 * (l.col % 4);
                    kt[at & 1][r].p[i] = both(turned_read(p), turned_read(p + 16 * PITCH));
                }
            in_order();
        };
        read_keys(0);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            Pieces<3> written[NB];
            const float4_t first = *(const float4_t*)(rest[turn] + 32 * kb + l.quad), second = *(const float4_t*)(rest[turn] + 32 * kb + 16 + l.quad);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float4_t x[2];
                value_floats(l, kb, n, x);
                written[n] = split_pairs(x[0] * first, x[1] * second);
            }
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const int at = kb * GROUPS + g, r0 = g * R;
                if (at + 1 < KB * GROUPS) read_keys(at + 1);
                float4_t sums[R][NB];
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int n = 0; n < NB; ++n) sums[r][n] = KB > 1 ? s[r0 + r][n] : ZERO;
                mma_grid(kt[at & 1], written, sums);
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int n = 0; n < NB; ++n) s[r0 + r][n] = KB > 1 ? sums[r][n] : decayed * s[r0 + r][n] + sums[r][n];
                in_order();
            }
        }
        if (anchored && !d.backwards) anchor(chunk);
        if (more && wave == WAVES - 1) gates(next, turn ^ 1);
        lds_barrier();  // the tiles are read, the dots written
        if constexpr (OUT) {
            if (d.dots && thread < C && t0 + token(thread) < d.time) {
                const i64 at = head * d.time + t0 + token(thread);
                float dot = 0.0f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) dot += dot_part[w][thread];
                d.dots[at] = dot;
                if (d.pairs) {
                    const int block = thread / 16, in = thread % 16;
                    float sum = 0.0f;
#pragma unroll
                    for (int k = 0; k < QB; ++k) {
                        if (k <= block) sum += pair_rows[block * (block + 1) / 2 + k][in];
                        if (k >= block) sum -= pair_columns[k * (k + 1) / 2 + block][in];
                    }
                    d.pairs[at] = sum;
                }
            }
        }
    }

    // ---- the state behind the segment
    float *to = nullptr, *copy = nullptr;
    float factor = 1.0f;
    if constexpr (OUT) {
        if (segment != (d.backwards ? 0 : d.segments - 1)) return;
        if (d.final_state) to = d.final_state + head * inner * outer;
        if (d.copy) copy = d.copy + head * inner * outer;
        if (d.backwards && length > 0) factor = expf(d.decay.value(d.decay.load(qp, b, 0, h)));
    } else {
        to = d.sums + (head * d.segments + segment) * inner * outer;
        if (threadIdx.x == THREADS - 1) d.decays[head * d.segments + segment] = (float)exp2(whole);
    }
    if (!to) return;
    const Lane l(thread_here());
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int column = cell(l, n);
#pragma unroll
        for (int r = 0; r < DK / 16; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = 16 * r + l.quad + j;
                if (row >= inner || column >= outer) continue;
                to[row * outer + column] = factor * s[r][n][j];
                if (copy) copy[row * outer + column] = factor * s[r][n][j];
            }
    }
}

// Turns the segments' sums into the states at their starts, in place.  backwards: the last segment's start is `start`.  Memory
// bounds it: 16 heads x 32 segments of 128 x 128 in 17 us (3.9 TB/s), 32 x 16 of 128 x 96 in 8.7.
__global__ void __launch_bounds__(256) join_states(float* sums, const float* decays, const float* start, i64 cells, int segments, int backwards) {
    const i64 cell = (i64)blockIdx.x * 256 + threadIdx.x, head = blockIdx.y;
    if (cell >= cells) return;
    float carry = start ? start[head * cells + cell] : 0.0f;
#pragma unroll 4
    for (int i = 0; i < segments; ++i) {
        const int segment = backwards ? segments - 1 - i : i;
        float* p = sums + (head * segments + segment) * cells + cell;
        const float own = i + 1 < segments ? *p : 0.0f, decay = i + 1 < segments ? decays[head * segments + segment] : 0.0f;
        *p = carry;
        carry = decay * carry + own;
    }
}

// ------------------------------------------------------------------ gradients of the decays
// A workgroup takes the tokens between two anchors: L behind its last token, then back through its tokens.  A launch's chain of
// loads and barriers, 9 us for 1024 sequences of 100 tokens, 12 for 32 of 4099.
struct DecayGradients {
    Decays decay;
    const void* other;                      // memory that may be read where there are no decays
    const int32_t* lengths;
    i64 time, tokens, cells, anchors;       // tokens between anchors; cells of a state
    int value_heads;
    const float *last, *grad_state;         // S after the sequence and its gradient, which may be null
    const float *states, *behind;           // S and T at the anchors
    const float *dq, *dk, *pairs;           // [batch, value head, time]
    void* out;                              // (batch, time, value heads) of the decays' type, or null:
    float* sums;                            // [batch, interval, value head] sums over the interval's tokens
};

__global__ void __launch_bounds__(256) decay_gradients(DecayGradients d) {
    __shared__ double parts[2][4];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, interval = blockIdx.x;
    const i64 h = blockIdx.y, b = blockIdx.z, head = b * d.value_heads + h;
    const i64 length = length_of(d.lengths, d.time, b), first = interval * d.tokens, end = min(first + d.tokens, d.time);
    double carry = 0.0;
    const bool anchored = end < length;
    if (anchored || (d.grad_state && first < length)) {  // <S, T>
        const float* state = anchored ? d.states + (head * d.anchors + interval) * d.cells : d.last + head * d.cells;
        const float* grad = anchored ? d.behind + (head * d.anchors + interval) * d.cells : d.grad_state + head * d.cells;
        double sums[8] = {};
        for (i64 i = threadIdx.x; i < d.cells; i += 8 * 256) {
            float x[8], y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const i64 at = min(i + 256 * k, d.cells - 1);
                x[k] = state[at], y[k] = grad[at];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + 256 * k < d.cells) sums[k] += (double)x[k] * (double)y[k];
        }
        carry = ((sums[0] + sums[1]) + (sums[2] + sums[3])) + ((sums[4] + sums[5]) + (sums[6] + sums[7]));
#pragma unroll
        for (int k = 32; k; k /= 2) carry += __shfl_xor(carry, k, 64);
        if (lane == 0) parts[0][wave] = carry;
        __syncthreads();
        carry = (parts[0][0] + parts[0][1]) + (parts[0][2] + parts[0][3]);
        if (anchored) carry *= exp((double)d.decay.value(d.decay.load(d.other, b, end, h)));
    }
    double sum = 0.0;
    int turn = 1;
    for (i64 base = end; base > first; base -= 256, turn ^= 1) {
        const i64 t = base - 1 - threadIdx.x;
        const bool live = t >= first && t < length;
        const i64 at = head * d.time + (live ? t : first);
        double x = live ? (double)d.dq[at] - (double)d.dk[at] + (double)d.pairs[at] : 0.0;
#pragma unroll
        for (int k = 1; k < 64; k *= 2) {
            const double before = __shfl_up(x, k, 64);
            if (lane >= k) x += before;
        }
        if (lane == 63) parts[turn][wave] = x;
        __syncthreads();
        for (int w = 0; w < wave; ++w) x += parts[turn][w];
        x += carry;
        carry += (parts[turn][0] + parts[turn][1]) + (parts[turn][2] + parts[turn][3]);
        if (live) sum += x;
        if (d.out && t >= first) {
            const i64 o = (b * d.time + t) * d.value_heads + h;
            const float value = live ? (float)x : 0.0f;
            if (d.decay.bf16) ((bf16_t*)d.out)[o] = from_float<bf16_t>(value);
            else ((float*)d.out)[o] = value;
        }
    }
    if (!d.sums) return;
#pragma unroll
    for (int k = 32; k; k /= 2) sum += __shfl_xor(sum, k, 64);
    __syncthreads();  // the last tiles' parts are read
    if (lane == 0) parts[0][wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
        d.sums[(b * gridDim.x + interval) * d.value_heads + h] = (float)((parts[0][0] + parts[0][1]) + (parts[0][2] + parts[0][3]));
}

// Sums over rows of (rows, columns): the gradient of a decay that all sequences share.
__global__ void __launch_bounds__(256) head_sums(const float* __restrict__ sums, i64 rows, int columns, int bf16, void* out) {
    __shared__ double parts[4];
    const int column = blockIdx.x;
    double sum = 0.0;
    for (i64 r = threadIdx.x; r < rows; r += 256) sum += (double)sums[r * columns + column];
#pragma unroll
    for (int k = 32; k; k /= 2) sum += __shfl_xor(sum, k, 64);
    if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    const float total = (float)((parts[0] + parts[1]) + (parts[2] + parts[3]));
    if (bf16) ((bf16_t*)out)[column] = from_float<bf16_t>(total);
    else ((float*)out)[column] = total;
}

// Heads of q and k that `group` value heads share: the sums of their gradients, q's and behind them k's (blockIdx.y), whose
// rows are (head, value head of it, width).  32 lanes take a row's VEC neighbours each; memory bounds it, 134 MB in 22 us.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) group_sums(const float* __restrict__ parts, i64 rows, int width, int group, T* dq, T* dk) {
    struct Packed { float v[VEC]; };
    T* out = blockIdx.y ? dk : dq;
    parts += blockIdx.y * rows * group * width;
    for (i64 row = (i64)blockIdx.x * 8 + threadIdx.x / 32; row < rows; row += (i64)gridDim.x * 8)
        for (int c = threadIdx.x % 32 * VEC; c < width; c += 32 * VEC) {
            const float* p = parts + row * group * width + c;
            float sum[VEC] = {};
#pragma unroll 4
            for (int g = 0; g < group; ++g, p += width) {
                const Packed x = *(const Packed*)p;
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum[e] += x.v[e];
            }
            store_unit<T, VEC>(out + row * width + c, VEC, sum);
        }
}

// ------------------------------------------------------------------ plans
template <typename F>
void with_type(int type, F&& f) {
    if (type == ATLAS_OPS_F32) f(0.0f);
    else f(bf16_t{});
}

int chunk_of(int type) { return type == ATLAS_OPS_F32 ? Cut<float>::C : Cut<bf16_t>::C; }

// Segments: as many as give every CU its two workgroups.  Every chunk that is split off passes the state twice, and two
// launches come before: segments of one chunk are for few of them, and fewer than three segments are none.  (Training on)
// 16384 tokens of 8 heads of 128 bfloat16: 512 workgroups 383 us, 256 385, 1024 497; 16 x 2048 of 8 of 64, forward, 75, 104 and
// 76.  Segments of one chunk: 500 tokens of 8 heads of 64 float32 (128 of them) 19 us, of two 21.5; 8000 of 4 of 128 bfloat16
// (500) 72, of two 54.  Two segments: 32 x 300 of 8 of 128 72 us, one 51; 32 x 2048 of 8 of 64 129, one 140, in training 535
// and 497; 64 tokens of 4 heads of 64 float32 14.4 and 11.7.
struct Plan {
    i64 chunks, heads;  // of a sequence; batch x value heads
    int per, segments;
    i64 state;          // floats of a state
};

Plan plan_of(const AtlasDelta& d) {
    Plan p{};
    p.chunks = ceil_div(d.time, chunk_of(d.type));
    p.heads = d.batch * d.value_heads;
    p.state = d.key * d.value;
    p.per = (int)ceil_div(p.chunks, std::max<i64>(1, 512 / p.heads));
    if (p.per == 1 && p.heads * p.chunks > 256) p.per = 2;
    p.segments = (int)ceil_div(p.chunks, p.per);
    if (p.segments < 3) p.segments = 1, p.per = (int)p.chunks;
    return p;
}

// The workspace of a forward pass, which a backward pass takes as its tape: the states at the segments' starts, the
// decays of segments, and for a tape the final state.
i64 forward_floats(const AtlasDelta& d, bool train) {
    const Plan p = plan_of(d);
    const i64 starts = p.segments > 1 ? p.heads * p.segments * (p.state + 1) : 0;
    return starts + (train ? p.heads * p.state : 0);
}

// Of a backward pass: T behind the segments and their decays, S and T at the anchors, the dots of dQ and dK and the pairs' sums,
// sums of shared decays, float32 gradients of shared heads.  Without a gradient of decays the middle is empty.
struct Back {
    i64 decays, states, anchors, dots, sums, dq, dk, all;
};

Back back_of(const AtlasDelta& d) {
    const Plan p = plan_of(d);
    const bool decays = d.log_decay;
    Back o{};
    o.decays = p.segments > 1 ? p.heads * p.segments * p.state : 0;
    o.states = o.decays + (p.segments > 1 ? p.heads * p.segments : 0);
    o.anchors = o.states + (decays ? p.heads * anchors_of(p.chunks) * p.state : 0);
    o.dots = o.anchors + (decays ? p.heads * anchors_of(p.chunks) * p.state : 0);
    o.sums = o.dots + (decays ? 3 * p.heads * d.time : 0);
    o.dq = o.sums + (decays ? p.heads * ceil_div(p.chunks, ANCHOR) : 0);
    const i64 shared = d.value_heads > d.heads ? p.heads * d.time * d.key : 0;
    o.dk = o.dq + shared;
    o.all = o.dk + shared;
    return o;
}

// The narrowest kernel that holds both widths: 64 x 64 float32, training on 8 x 1000 tokens of 8 heads, 148 us, in the one for
// 128 x 128 274.  Whole units of 16 bytes where both widths have them: 16384 tokens of 8 heads of 128 bfloat16, forward 106 us
// and training 383, without that knowledge 127 and 584.
template <bool OUT>
void launch_scan(const Scan* scans, int count, int type, i64 batch, int segments, hipStream_t st) {
    Runs runs{};
    std::copy(scans, scans + count, runs.run);
    runs.segments = segments;
    const Scan& s = scans[0];
    const dim3 grid((unsigned)(segments * count), (unsigned)s.value_heads, (unsigned)batch);
    with_type(type, [&](auto t) {
        using T = decltype(t);
        constexpr int E = Unit<T>::N;
        auto widths = [&](auto whole) {
            if (s.q.width <= 64 && s.v.width <= 64) scan<T, 64, 1, OUT, whole()><<<grid, 256, 0, st>>>(runs);
            else if (s.q.width <= 64) scan<T, 64, 2, OUT, whole()><<<grid, 256, 0, st>>>(runs);
            else if (s.v.width <= 64) scan<T, 128, 1, OUT, whole()><<<grid, 256, 0, st>>>(runs);
            else scan<T, 128, 2, OUT, whole()><<<grid, 256, 0, st>>>(runs);
        };
        if (s.q.width % E || s.v.width % E) widths(std::false_type{});
        else widths(std::true_type{});
    });
}

Tensor tensor_of(const void* data, const int64_t* stride) { return {data, stride[0], stride[1], stride[2]}; }

int check(const AtlasDelta* d, bool chunks, char* err, size_t cap) {
    if (!d) return fail(err, cap, 7, "null problem");
    if (d->batch < 1 || d->time < 1 || d->heads < 1 || d->value_heads < 1 || d->value < 1)
        return fail(err, cap, 7, "every size must be positive");
    if (d->key < 1 || d->key > MAX_WIDTH || d->value > MAX_WIDTH) return fail(err, cap, 7, "key and value must be 1 to %d", MAX_WIDTH);
    if (d->value_heads % d->heads) return fail(err, cap, 7, "value_heads must be a multiple of heads");
    if (d->batch > 65535 || d->value_heads > 65535) return fail(err, cap, 7, "at most 65535 sequences and value heads");
    if (d->time > ((i64)1 << 29)) return fail(err, cap, 7, "time must be at most 2^29");
    for (const int64_t* stride : {d->q_stride, d->k_stride, d->v_stride})
        if (chunks && (stride[1] < 0 || stride[1] > MAX_STRIDE)) return fail(err, cap, 7, "tokens must be at most 2^24 elements apart");
    if (chunks && d->batch * d->value_heads > 65535 * 512) return fail(err, cap, 7, "batch x value_heads must be below 2^25");
    if (!known_type(d->type) || !known_type(d->log_decay_type)) return fail(err, cap, 7, "unknown type");
    if (!d->q || !d->k || !d->v) return fail(err, cap, 7, "null tensor");
    return 0;
}

Decays decays_of(const AtlasDelta& d) {
    return {tensor_of(d.log_decay, d.log_decay_stride), d.log_decay_type == ATLAS_OPS_BF16};
}

Scan scan_of(const AtlasDelta& d, const Plan& p) {
    Scan s{};
    s.decay = decays_of(d);
    s.lengths = d.lengths;
    s.time = d.time;
    s.value_heads = (int)d.value_heads;
    s.chunks = (int)p.chunks;
    s.per = p.per;
    s.segments = p.segments;
    s.write = s.read = 1.0f;
    return s;
}

}  // namespace
}  // namespace atlas_ops

using namespace atlas_ops;

extern "C" {

int atlas_ops_linear_step(const AtlasDelta* d, void* out, float* final_state, void* stream, char* err, size_t cap) {
    try {
        if (int rc = check(d, false, err, cap)) return rc;
        if (!out || !final_state) return fail(err, cap, 7, "null output");
        const Step s{tensor_of(d->q, d->q_stride), tensor_of(d->k, d->k_stride), tensor_of(d->v, d->v_stride), decays_of(*d), d->state,
                     d->lengths, d->time, (int)d->value_heads, (int)(d->value_heads / d->heads), (int)d->key, (int)d->value, d->scale};
        const dim3 grid((unsigned)ceil_div(d->value, 32), (unsigned)d->value_heads, (unsigned)d->batch);
        with_type(d->type, [&](auto t) {
            using T = decltype(t);
            if (d->value % 4 == 0) step_kernel<T, 4><<<grid, 256, 0, (hipStream_t)stream>>>(s, (T*)out, final_state);
            else step_kernel<T, 1><<<grid, 256, 0, (hipStream_t)stream>>>(s, (T*)out, final_state);
        });
        return launched(err, cap, "linear_step");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

int64_t atlas_ops_linear_workspace(const AtlasDelta* d, int train) {
    char ignored[1];
    if (check(d, true, ignored, 1)) return 0;
    return 4 * forward_floats(*d, train != 0) + 16;  // never 0
}

int atlas_ops_linear_forward(const AtlasDelta* d, int train, void* out, float* final_state, void* workspace, void* stream, char* err,
                             size_t cap) {
    try {
        if (int rc = check(d, true, err, cap)) return rc;
        if (!out || !final_state || !workspace) return fail(err, cap, 7, "null output or workspace");
        const Plan p = plan_of(*d);
        hipStream_t st = (hipStream_t)stream;
        const int group = (int)(d->value_heads / d->heads);
        Scan s = scan_of(*d, p);
        s.q = {tensor_of(d->q, d->q_stride), group, (int)d->key};
        s.k = {tensor_of(d->k, d->k_stride), group, (int)d->key};
        s.v = {tensor_of(d->v, d->v_stride), 1, (int)d->value};
        s.read = d->scale;
        s.start = d->state;
        float* starts = (float*)workspace;
        float* last = starts + (p.segments > 1 ? p.heads * p.segments * (p.state + 1) : 0);
        if (p.segments > 1) {
            s.sums = starts;
            s.decays = starts + p.heads * p.segments * p.state;
            launch_scan<false>(&s, 1, d->type, d->batch, p.segments - 1, st);
            for (i64 b = 0; b < p.heads; b += 65535)
                join_states<<<dim3((unsigned)ceil_div(p.state, 256), (unsigned)std::min<i64>(p.heads - b, 65535)), 256, 0, st>>>(
                    starts + b * p.segments * p.state, s.decays + b * p.segments, d->state ? d->state + b * p.state : nullptr, p.state, p.segments, 0);
            s.start = starts;
            s.start_segments = 1;
        }
        s.out = out;
        s.final_state = final_state;
        s.copy = train ? last : nullptr;
        launch_scan<true>(&s, 1, d->type, d->batch, p.segments, st);
        return launched(err, cap, "linear_forward");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

int64_t atlas_ops_linear_backward_workspace(const AtlasDelta* d) {
    char ignored[1];
    if (check(d, true, ignored, 1)) return 0;
    return 4 * back_of(*d).all + 16;  // never 0
}

int atlas_ops_linear_backward(const AtlasDelta* d, const void* tape, const void* grad_out, const int64_t* grad_out_stride,
                              const float* grad_state, void* dq, void* dk, void* dv, void* dlog_decay, int shared_decay, float* dstate,
                              void* workspace, void* stream, char* err, size_t cap) {
    try {
        if (int rc = check(d, true, err, cap)) return rc;
        if (!tape || !grad_out || !grad_out_stride || !dq || !dk || !dv || !workspace) return fail(err, cap, 7, "null argument");
        if (grad_out_stride[1] < 0 || grad_out_stride[1] > MAX_STRIDE) return fail(err, cap, 7, "tokens must be at most 2^24 elements apart");
        if (dlog_decay && !d->log_decay) return fail(err, cap, 7, "a gradient of decays that were not given");
        const Plan p = plan_of(*d);
        const Back at = back_of(*d);
        hipStream_t st = (hipStream_t)stream;
        const int group = (int)(d->value_heads / d->heads);
        float* base = (float*)workspace;
        const float* starts = (const float*)tape;
        const float* last = starts + (p.segments > 1 ? p.heads * p.segments * (p.state + 1) : 0);
        const Role q{tensor_of(d->q, d->q_stride), group, (int)d->key}, k{tensor_of(d->k, d->k_stride), group, (int)d->key},
            v{tensor_of(d->v, d->v_stride), 1, (int)d->value}, go{tensor_of(grad_out, grad_out_stride), 1, (int)d->value};
        float *dots_q = base + at.dots, *dots_k = dots_q + p.heads * d->time, *pairs = dots_k + p.heads * d->time;
        // T behind the segments
        Scan s = scan_of(*d, p);
        s.backwards = 1;
        s.write = d->scale;
        s.q = k, s.k = q, s.v = go;
        s.start = grad_state;
        if (p.segments > 1) {
            s.sums = base;
            s.decays = base + at.decays;
            s.first = 1;
            launch_scan<false>(&s, 1, d->type, d->batch, p.segments - 1, st);
            s.first = 0;
            for (i64 b = 0; b < p.heads; b += 65535)
                join_states<<<dim3((unsigned)ceil_div(p.state, 256), (unsigned)std::min<i64>(p.heads - b, 65535)), 256, 0, st>>>(
                    s.sums + b * p.segments * p.state, s.decays + b * p.segments, grad_state ? grad_state + b * p.state : nullptr, p.state,
                    p.segments, 1);
            s.start = s.sums;
            s.start_segments = 1;
        }
        Scan runs[3] = {s, scan_of(*d, p), s};
        // dV, backwards
        Scan& v_run = runs[0];
        v_run.out = dv;
        v_run.final_state = dstate;
        v_run.anchors = dlog_decay ? base + at.anchors : nullptr;
        // dQ, forwards
        Scan& q_run = runs[1];
        q_run.q = go, q_run.k = v, q_run.v = k;
        q_run.read = d->scale;
        q_run.start = p.segments > 1 ? starts : d->state;
        q_run.start_segments = p.segments > 1;
        q_run.turned = 1;
        q_run.out = group > 1 ? (void*)(base + at.dq) : dq;
        q_run.out_f32 = group > 1;
        q_run.dot = q;
        q_run.dots = dlog_decay ? dots_q : nullptr;
        q_run.pairs = dlog_decay ? pairs : nullptr;
        q_run.anchors = dlog_decay ? base + at.states : nullptr;
        // dK, backwards
        Scan& k_run = runs[2];
        k_run.q = v, k_run.k = go, k_run.v = q;
        k_run.turned = 1;
        k_run.out = group > 1 ? (void*)(base + at.dk) : dk;
        k_run.out_f32 = group > 1;
        k_run.dot = k;
        k_run.dots = dlog_decay ? dots_k : nullptr;
        // in one launch where one kernel holds the widths both ways round: 2 x 300 tokens of 4 heads of 64 float32 train in 43 us,
        // with a launch for each run in 59; 16384 of 8 of 128 bfloat16 in 383 and 384
        const int together = (d->key <= 64) == (d->value <= 64) ? 3 : 1;
        launch_scan<true>(runs, together, d->type, d->batch, p.segments, st);
        if (together == 1) launch_scan<true>(runs + 1, 2, d->type, d->batch, p.segments, st);
        if (group > 1) {
            const i64 rows = d->batch * d->time * d->heads;
            with_type(d->type, [&](auto t) {
                using T = decltype(t);
                const dim3 grid((unsigned)std::min<i64>(ceil_div(rows, 8), 4096), 2);
                auto* sums = d->key % 4 == 0 ? group_sums<T, 4> : group_sums<T, 1>;
                sums<<<grid, 256, 0, st>>>(base + at.dq, rows, (int)d->key, group, (T*)dq, (T*)dk);
            });
        }
        if (dlog_decay) {
            DecayGradients g{};
            g.decay = decays_of(*d);
            g.other = d->q;
            g.lengths = d->lengths;
            g.time = d->time;
            g.tokens = (i64)ANCHOR * chunk_of(d->type);
            g.cells = p.state;
            g.anchors = anchors_of(p.chunks);
            g.value_heads = (int)d->value_heads;
            g.last = last;
            g.grad_state = grad_state;
            g.states = base + at.states;
            g.behind = base + at.anchors;
            g.dq = dots_q;
            g.dk = dots_k;
            g.pairs = pairs;
            g.out = shared_decay ? nullptr : dlog_decay;
            g.sums = shared_decay ? base + at.sums : nullptr;
            const i64 intervals = ceil_div(p.chunks, ANCHOR);
            decay_gradients<<<dim3((unsigned)intervals, (unsigned)d->value_heads, (unsigned)d->batch), 256, 0, st>>>(g);
            if (shared_decay)
                head_sums<<<dim3((unsigned)d->value_heads), 256, 0, st>>>(g.sums, d->batch * intervals, (int)d->value_heads,
                                                                         d->log_decay_type == ATLAS_OPS_BF16, dlog_decay);
        }
        return launched(err, cap, "linear_backward");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

}  // extern "C"
