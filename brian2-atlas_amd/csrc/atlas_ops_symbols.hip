// The embedding of symbols with its gradient by sorted tokens, and dropout from the simulator's counter
// generator.  Part of libatlas_ops_hip.so.
//
//   out_i = scale table[token_i]            (zeros where the token is no row of the table)
//   dtable_r = scale sum of grad_i over the i with token_i = r
//   y_i = residual_i + (draw_i >= p 2^32 ? x_i / (1 - p) : 0)
//
// The gradient's sums are taken in an order that the tokens alone set.  Few symbols are looked for by every row's
// workgroup.  Else a stable radix sort of (token, place), which starts beside the clearing of the table, brings each row's
// places together; tiles of sorted places are summed in registers, a run of one row within a tile goes straight to the
// table, and runs that cross tiles leave partial sums, which a last kernel adds from the first tile to the last.  Atomics
// count and list, none of them adds values: the same bits every time.
//
// Memory bounds the large ones: 32752 symbols of 50000 rows of 1024 bfloat16 values looked up in 28 us (4.8 TB/s); their
// gradient in 70: the first counts with the clearing 19 (5.4 TB/s), placing 13.7 and 9, sums 19, crossing rows 8.5.  Dropout of
// 12289 x 4099 bfloat16 values with a residual 59 us (5.1 TB/s).
#include <algorithm>
#include <type_traits>

#include "device/atlas_rows.h"

namespace atlas_ops {
namespace {

// ------------------------------------------------------------------ lookup
struct Tokens {
    const void* data;
    int wide;  // 64-bit
    i64 count;
    __device__ __forceinline__ i64 at(i64 i) const { return wide ? ((const i64*)data)[i] : ((const int32_t*)data)[i]; }
};

// A group of LANES lanes copies the rows of TOGETHER tokens at a time, all their loads in flight: 2, 4 or 8 take 29, 30 or
// 31 us for 32752 x 1024 bfloat16 of 50000 rows.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) embed_forward(const T* __restrict__ table, i64 rows, int width, i64 row_stride, Tokens tokens,
                                                     float scale, T* __restrict__ out) {
    constexpr int N = Unit<T>::N, GROUPS = 256 / LANES, TOGETHER = 2;
    const int lane = threadIdx.x % LANES;
    const i64 stride = (i64)gridDim.x * GROUPS * TOGETHER;
    for (i64 i = ((i64)blockIdx.x * GROUPS + threadIdx.x / LANES) * TOGETHER; i < tokens.count; i += stride) {
        i64 row[TOGETHER];
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k) row[k] = tokens.at(min(i + k, tokens.count - 1));
        for (int col = lane * N; col < width; col += LANES * N) {
            Unit<T> unit[TOGETHER];
#pragma unroll
            for (int k = 0; k < TOGETHER; ++k) unit[k].load(table + (row[k] < 0 || row[k] >= rows ? 0 : row[k]) * row_stride, col, width);
#pragma unroll
            for (int k = 0; k < TOGETHER; ++k) {
                if (i + k >= tokens.count) break;
                float v[N];
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = row[k] < 0 || row[k] >= rows ? 0.0f : scale * unit[k][e];
                store_unit<T>(out + (i + k) * width + col, width - col, v);
            }
        }
    }
}

// ------------------------------------------------------------------ the stable sort
// Digits of up to 11 bits, the lowest first.  A tile's workgroup needs the digits' counts of the tiles before it: it adds
// them up itself where there are few tiles, else a kernel between scans them (8 tiles, whole gradient: 64 us without that
// kernel and 68 with it; 32 tiles of two digits 66 and 61; 128 tiles 112 and 110).  The first counts are a kernel's of their
// own, which clears the table beside; those of a later pass are taken where the keys are placed before it.
constexpr int SORT_TILE = 1024, MAX_BITS = 11, SCANNED = 32;

struct Sort {
    i64 count, tiles;
    int rows, shift, bits;  // the key of a token that is no row is `rows`: it sorts behind them
    __device__ __forceinline__ uint32_t key_of(i64 token) const { return token < 0 || token >= rows ? (uint32_t)rows : (uint32_t)token; }
    __device__ __forceinline__ uint32_t digit(uint32_t key) const { return (key >> shift) & ((1u << bits) - 1); }
};

// The first digit's counts by tile (blocks below `tiles`); the other blocks clear two ranges of memory meanwhile.
__global__ void __launch_bounds__(256) sort_count(Sort s, Tokens tokens, uint32_t* __restrict__ counts, char* __restrict__ clear, i64 size,
                                                  char* __restrict__ clear_too, i64 size_too) {
    if (blockIdx.x >= s.tiles) {
        struct __attribute__((packed, aligned(1))) Sixteen { uint32_t word[4]; };
        const i64 stride = ((i64)gridDim.x - s.tiles) * 256 * 16, first = ((blockIdx.x - s.tiles) * 256 + threadIdx.x) * 16;
        for (i64 at = first; at < size; at += stride) {
            if (at + 16 <= size) {
                *(Sixteen*)(clear + at) = Sixteen{};
            } else {
                for (i64 b = at; b < size; ++b) clear[b] = 0;
            }
        }
        for (i64 at = first; at < size_too; at += stride) *(Sixteen*)(clear_too + at) = Sixteen{};  // a multiple of 16
        return;
    }
    __shared__ uint32_t bins[1 << MAX_BITS];
    const int all = 1 << s.bits;
    for (int b = threadIdx.x; b < all; b += 256) bins[b] = 0;
    i64 token[SORT_TILE / 256];
    const i64 start = (i64)blockIdx.x * SORT_TILE;
#pragma unroll
    for (int e = 0; e < SORT_TILE / 256; ++e) token[e] = tokens.at(min(start + e * 256 + threadIdx.x, s.count - 1));
    __syncthreads();
#pragma unroll
    for (int e = 0; e < SORT_TILE / 256; ++e)
        if (start + e * 256 + threadIdx.x < s.count) atomicAdd(&bins[s.digit(s.key_of(token[e]))], 1u);
    __syncthreads();
    for (int b = threadIdx.x; b < all; b += 256) counts[(i64)blockIdx.x * all + b] = bins[b];
}

// Many tiles: each digit's counts become the counts of the tiles before, and their total goes behind them.
__global__ void __launch_bounds__(256) sort_scan(Sort s, uint32_t* __restrict__ counts) {
    const int all = 1 << s.bits, bin = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x % 64;
    if (bin >= all) return;
    uint32_t before = 0;
    for (i64 base = 0; base < s.tiles; base += 64) {
        const i64 tile = base + lane;
        const uint32_t own = tile < s.tiles ? counts[tile * all + bin] : 0;
        uint32_t sum = own;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t other = __shfl_up(sum, d, 64);
            if (lane >= d) sum += other;
        }
        if (tile < s.tiles) counts[tile * all + bin] = before + sum - own;
        before += __shfl(sum, 63, 64);
    }
    if (lane == 0) counts[s.tiles * all + bin] = before;
}

// Places every key of a tile behind those with smaller digits, of earlier tiles and, in the tile, of earlier
// waves and lanes.  A wave takes 64 neighbouring keys at a time; ballots over the digit's bits find the lanes
// with the same digit.  next_counts: those of the next digit by the tile of the new place, or null.
template <bool FIRST, bool PREFIXED>
__global__ void __launch_bounds__(256) sort_scatter(Sort s, Tokens tokens, const uint32_t* __restrict__ keys,
                                                    const uint32_t* __restrict__ places, const uint32_t* __restrict__ counts,
                                                    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ places_out,
                                                    uint32_t* __restrict__ next_counts) {
    constexpr int WAVE_KEYS = SORT_TILE / 4, ROUNDS = WAVE_KEYS / 64, PER = (1 << MAX_BITS) / 256;
    __shared__ uint32_t next[4][1 << MAX_BITS];
    __shared__ uint32_t wave_sums[4];
    const int all = 1 << s.bits, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const i64 tile = blockIdx.x, start = tile * SORT_TILE + wave * WAVE_KEYS;
    uint32_t key[ROUNDS], from[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const i64 i = min(start + r * 64 + lane, s.count - 1);
        key[r] = FIRST ? s.key_of(tokens.at(i)) : keys[i];
        from[r] = FIRST ? (uint32_t)i : places[i];
    }
    // each thread: a run of neighbouring digits, their totals and what the tiles before have of them
    const int per = (all + 255) / 256, b0 = (int)threadIdx.x * per;
    uint32_t total[PER], before[PER], own = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) total[k] = before[k] = 0;
    if constexpr (PREFIXED) {
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (k < per && b0 + k < all) {
                total[k] = counts[s.tiles * all + b0 + k];
                before[k] = counts[tile * all + b0 + k];
            }
    } else {
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (k < per && b0 + k < all) {
                for (int t0 = 0; t0 < (int)s.tiles; t0 += 16) {
                    uint32_t c[16];
#pragma unroll
                    for (int t = 0; t < 16; ++t) c[t] = counts[min(t0 + t, (int)s.tiles - 1) * all + b0 + k];
#pragma unroll
                    for (int t = 0; t < 16; ++t) {
                        total[k] += t0 + t < (int)s.tiles ? c[t] : 0;
                        before[k] += t0 + t < (int)tile ? c[t] : 0;
                    }
                }
            }
    }
    for (int b = threadIdx.x; b < 4 * all; b += 256) next[b / all][b % all] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (start + r * 64 + lane < s.count) atomicAdd(&next[wave][s.digit(key[r])], 1u);
#pragma unroll
    for (int k = 0; k < PER; ++k) own += total[k];
    uint32_t sum = own;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t other = __shfl_up(sum, d, 64);
        if (lane >= d) sum += other;
    }
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();  // the waves' counts and sums are complete
    uint32_t at = sum - own;
    for (int w = 0; w < wave; ++w) at += wave_sums[w];
#pragma unroll
    for (int k = 0; k < PER; ++k)
        if (k < per && b0 + k < all) {
            uint32_t place = at + before[k];
            for (int w = 0; w < 4; ++w) {
                const uint32_t c = next[w][b0 + k];
                next[w][b0 + k] = place;
                place += c;
            }
            at += total[k];
        }
    __syncthreads();
    volatile uint32_t* mine = next[wave];  // only this wave reads and writes it from here on, in program order
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool live = start + r * 64 + lane < s.count;
        const uint32_t digit = s.digit(key[r]);
        u64 same = __ballot(live);
        for (int b = 0; b < s.bits; ++b) {
            const bool bit = digit >> b & 1;
            const u64 ones = __ballot(live && bit);
            same &= bit ? ones : ~ones;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1)), many = __popcll(same);
        uint32_t place = 0;
        if (live) place = mine[digit] + rank;
        __builtin_amdgcn_wave_barrier();
        if (live && rank == many - 1) mine[digit] = place + 1;
        __builtin_amdgcn_wave_barrier();
        if (live) {
            keys_out[place] = key[r];
            places_out[place] = from[r];
        }
        if (next_counts) {
            // equal keys, which neighbour each other now, are counted together where they lie in one tile
            const uint32_t after = key[r] >> (s.shift + s.bits) & (all - 1);
            for (int b = 0; b < s.bits; ++b) {
                const bool bit = after >> b & 1;
                const u64 ones = __ballot(live && bit);
                same &= bit ? ones : ~ones;
            }
            const uint32_t to = place / SORT_TILE;
            const u64 here = same & __ballot(to == (uint32_t)__shfl((int)to, live ? __builtin_ctzll(same) : 0, 64));
            uint32_t* p = next_counts + (i64)to * all + after;
            if (live && here == same) {
                if (lane == __builtin_ctzll(same)) atomicAdd(p, (uint32_t)__popcll(same));
            } else if (live) {
                atomicAdd(p, 1u);
            }
        }
    }
}

// ------------------------------------------------------------------ the sums
// A tile's first run is a part of an earlier tile's row where the key before the tile is the same, its last
// run of a later one's where the key behind is.  Partial sums: slot 0 of a tile for a run that comes from before,
// slot 1 for one that starts here and goes on: it goes on a list, of rows that end within SHORT tiles or of longer ones,
// whose order does not matter, and the tile where it ends is noted by row.  32768 symbols of 1024 bfloat16 values by Zipf's law,
// whole gradient: with 16 tiles 66 us, with 4 tiles 100, with 64 tiles 76.
constexpr int SHORT = 16;

struct Crossing {
    struct Start { uint32_t tile, row; };
    uint32_t *counts, *ends;
    Start* starts[2];
};

template <typename T, typename O, int LANES, int SUM_TILE>
__global__ void __launch_bounds__(256) embed_sum(Rows grad, int width, i64 count, int rows, const uint32_t* __restrict__ keys,
                                                 const uint32_t* __restrict__ places, float scale, O* __restrict__ table,
                                                 float* __restrict__ partial, Crossing crossing) {
    constexpr int N = Unit<T>::N, GROUPS = 256 / LANES, TOGETHER = 8;
    __shared__ uint32_t key[GROUPS][SUM_TILE + 2], place[GROUPS][SUM_TILE];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const i64 tile = (i64)blockIdx.x * GROUPS + group, first = tile * SUM_TILE;
    const int n = first < count ? (int)min((i64)SUM_TILE, count - first) : 0;
    for (int e = lane; e < SUM_TILE + 2; e += LANES) {
        const i64 i = first + e - 1;
        key[group][e] = i >= 0 && i < count ? keys[i] : 0xFFFFFFFFu;  // no row
    }
    for (int e = lane; e < n; e += LANES) place[group][e] = places[first + e];
    __syncthreads();
    const int col = (blockIdx.y * LANES + lane) * N, left = width - col;
    if (left <= 0) return;
    const uint32_t* k = key[group] + 1;
    float sum[N];
    int begun = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
    for (int e0 = 0; e0 < n; e0 += TOGETHER) {
        Unit<T> unit[TOGETHER];
#pragma unroll
        for (int j = 0; j < TOGETHER; ++j) unit[j].load(grad.at<T>(place[group][min(e0 + j, n - 1)]), col, width);
#pragma unroll
        for (int j = 0; j < TOGETHER; ++j) {
            const int e = e0 + j;
            if (e >= n || k[e] >= (uint32_t)rows) break;
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] += unit[j][i];
            if (e + 1 < n && k[e + 1] == k[e]) continue;
            const bool from = begun == 0 && k[-1] == k[e], on = e + 1 == n && k[e + 1] == k[e];
            if (from || on) {
                store_unit<float, N>(partial + (2 * tile + (from ? 0 : 1)) * width + col, left, sum);
                if (blockIdx.y == 0 && lane == 0) {
                    if (!on) crossing.ends[k[e]] = (uint32_t)tile;
                    if (!from) {
                        const i64 far = first + (i64)SUM_TILE * SHORT;
                        const int list = far < count && keys[far] == k[e];
                        crossing.starts[list][atomicAdd(crossing.counts + list, 1u)] = {(uint32_t)tile, k[e]};
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] *= scale;
                store_unit<O, N>(table + (i64)k[e] * width + col, left, sum);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] = 0.0f;
            begun = e + 1;
        }
    }
}

// A row's partial sums: those of its tiles from `from` to `to`, in order; slot 1 in its first, 0 behind.
template <int N>
__device__ __forceinline__ void add_partials(const float* __restrict__ partial, i64 tile, i64 from, i64 to, int col, int width, float (&sum)[N]) {
    for (i64 j0 = from; j0 < to; j0 += 8) {
        float v[8][N];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const i64 j = min(j0 + k, to - 1);
            load_columns<float, N>(partial + (2 * j + (j == tile)) * width, col, width, 0.0f, v[k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (j0 + k < to)
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += v[k][i];
    }
}

// The rows that cross tiles, 64 columns per workgroup.  One half of the workgroups takes the list of long ones, each group of
// 16 lanes a part of a row's tiles in order, then the groups in order; in the other half each group takes short rows of
// its own.

template <typename O>
__global__ void __launch_bounds__(1024) embed_join(int width, float scale, O* __restrict__ table, const float* __restrict__ partial,
                                                   Crossing crossing) {
    constexpr int LANES = 16, N = 4, GROUPS = 1024 / LANES;
    __shared__ float sums[GROUPS][LANES * N + 1];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const int col0 = blockIdx.y * LANES * N, col = col0 + lane * N, left = width - col;
    const int half = gridDim.x / 2;
    const bool is_long = (int)blockIdx.x < half;
    const i64 rows = crossing.counts[is_long];
    for (i64 i = is_long ? blockIdx.x : (blockIdx.x - half) * GROUPS + group; i < rows; i += is_long ? half : half * GROUPS) {
        const Crossing::Start start = crossing.starts[is_long][i];
        const i64 tile = start.tile, end = (i64)crossing.ends[start.row] + 1;
        O* out = table + (i64)start.row * width;
        float sum[N];
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0.0f;
        if (!is_long) {
            if (left <= 0) continue;
            add_partials<N>(partial, tile, tile, end, col, width, sum);
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] *= scale;
            store_unit<O, N>(out + col, left, sum);
            continue;
        }
        const i64 per = (end - tile + GROUPS - 1) / GROUPS, from = tile + group * per;
        if (left > 0) add_partials<N>(partial, tile, from, min(end, from + per), col, width, sum);
        __syncthreads();  // the sums of the row before are read
#pragma unroll
        for (int e = 0; e < N; ++e) sums[group][lane * N + e] = sum[e];
        __syncthreads();
        if (threadIdx.x < LANES * N && col0 + (int)threadIdx.x < width) {
            float total = 0.0f;
#pragma unroll 16
            for (int g = 0; g < GROUPS; ++g) total += sums[g][threadIdx.x];
            out[col0 + threadIdx.x] = from_float<O>(scale * total);
        }
    }
}

// ------------------------------------------------------------------ few symbols
// A workgroup for each row and 8 units of its columns: it finds the row's places among all tokens, in their order, 128 groups of
// 8 lanes add a part of them each, and the groups are added in a fixed order.  One launch; what bounds it is its chain of
// tokens, places, gradients and two sums: 12288 symbols of 32 rows of 128 float32 values 12 us with cold caches, 9 with warm
// ones.  TURNS: tokens of a lane; with 2 rather than 16 turns 2000 tokens take 6.5 us instead of 8.6.
constexpr int FEW_TOKENS = 16384;

template <typename T, typename O, int TURNS>
__global__ void __launch_bounds__(1024) embed_few(Rows grad, int width, Tokens tokens, float scale, O* __restrict__ table) {
    constexpr int N = Unit<T>::N, LANES = 8, GROUPS = 1024 / LANES, WAVES = 16, TOGETHER = 8;
    __shared__ uint16_t list[TURNS * 1024];
    __shared__ int found[WAVES];
    __shared__ float sums[WAVES][LANES * N];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const i64 row = blockIdx.x;
    const int count = (int)tokens.count, turns = (count + 1023) / 1024, first = wave * turns * 64 + lane;
    i64 token[TURNS];
#pragma unroll
    for (int k = 0; k < TURNS; ++k) token[k] = tokens.at(min(first + k * 64, count - 1));
    u64 met[TURNS];
    int own = 0;
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        met[k] = __ballot(k < turns && first + k * 64 < count && token[k] == row);
        own += __popcll(met[k]);
    }
    if (lane == 0) found[wave] = own;
    __syncthreads();
    int at = 0, n = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        at += w < wave ? found[w] : 0;
        n += found[w];
    }
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        if (met[k] >> lane & 1) list[at + __popcll(met[k] & ((1ull << lane) - 1))] = (uint16_t)(first + k * 64);
        at += __popcll(met[k]);
    }
    __syncthreads();
    const int group = threadIdx.x / LANES, from = n * group / GROUPS, to = n * (group + 1) / GROUPS;
    const int col0 = blockIdx.y * LANES * N, col = col0 + threadIdx.x % LANES * N;
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
    for (int e0 = from; e0 < to; e0 += TOGETHER) {
        Unit<T> unit[TOGETHER];
#pragma unroll
        for (int j = 0; j < TOGETHER; ++j) unit[j].load(grad.at<T>(list[min(e0 + j, to - 1)]), col, width);
#pragma unroll
        for (int j = 0; j < TOGETHER; ++j)
            if (e0 + j < to)
#pragma unroll
                for (int i = 0; i < N; ++i) sum[i] += unit[j][i];
    }
#pragma unroll
    for (int k = LANES; k < 64; k *= 2)
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] += __shfl_xor(sum[i], k, 64);
    if (lane < LANES)
#pragma unroll
        for (int i = 0; i < N; ++i) sums[wave][lane * N + i] = sum[i];
    __syncthreads();
    if (threadIdx.x < LANES * N && col0 + (int)threadIdx.x < width) {
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) total += sums[w][threadIdx.x];
        table[row * width + col0 + threadIdx.x] = from_float<O>(scale * total);
    }
}

struct Plan {
    Sort sort;
    int passes, lanes, sum_tile;  // sorted places that a group sums
    i64 tiles, counts, lists_at, keys_at, partial_at, bytes;  // tiles of the sums; bytes of a pass's counts; offsets into the workspace
};

// The longest tiles, of 32, 16 or 8 places, that give the chip this many lanes, else 8.  Whole gradient with 32, 16 and 8:
// 65536 x 512 float32 (32 taken) 84, 98 and 85 us; 32752 x 1024 bfloat16 (16 taken) 70, 69 and 75, by Zipf's law 53, 54 and 66;
// 16384 x 512 float32 (8 taken) 43 with 32 and 38.5 with 8.
constexpr i64 SUM_LANES = 250000;  // about a thousand to a CU

// embed_few takes few symbols: its workgroups all find a place at once, and no row has very many places unless nearly all
// symbols are one.  Whole gradient by it and by sorting: 12288 x 128 float32 of 32 rows 9 and 19 us, by Zipf's law 13 and 23;
// 16000 x 256 of 16 rows by Zipf's law 25 and 24; 16000 x 128 of one row 41 and 31; 16000 x 128 of 500 rows (2000 workgroups)
// 52 and 28, 2000 x 128 of 400 rows (1600) 28 and 23.
i64 few_slices(i64 width, int type) { return ceil_div(width, 8 * (type == ATLAS_OPS_F32 ? 4 : 8)); }
constexpr i64 FEW_BLOCKS = 512;
bool is_few(i64 count, i64 rows, i64 width, int type) {
    return count && count <= std::min<i64>(FEW_TOKENS, std::max<i64>(4096, 1024 * rows)) && rows * few_slices(width, type) <= FEW_BLOCKS;
}

// What both the workspace and the launch go by.  grad's type sets the lanes: as few as hold a row's units.
Plan plan_of(i64 count, i64 rows, i64 width, int type) {
    Plan p{};
    int bits = 1;
    while (rows >> bits) ++bits;
    p.passes = (bits + MAX_BITS - 1) / MAX_BITS;
    p.sort = Sort{count, ceil_div(count, SORT_TILE), (int)rows, 0, (bits + p.passes - 1) / p.passes};
    const i64 units = ceil_div(width, type == ATLAS_OPS_F32 ? 4 : 8);
    p.lanes = 16;
    while (p.lanes < units && p.lanes < 256) p.lanes *= 2;
    const i64 slices = ceil_div(units, p.lanes);
    p.sum_tile = 32;
    while (p.sum_tile > 8 && ceil_div(count, p.sum_tile) * slices * p.lanes < SUM_LANES) p.sum_tile /= 2;
    p.tiles = ceil_div(count, p.sum_tile);
    p.counts = ((p.sort.tiles + 1) * 4 << p.sort.bits) + 15 & ~(i64)15;
    p.lists_at = p.counts * p.passes + 16;  // 16 bytes for the lists' counts, before the second pass's
    p.keys_at = p.lists_at + 16 * p.tiles + 4 * rows;
    p.partial_at = (p.keys_at + 16 * count + 15) / 16 * 16;
    p.bytes = p.partial_at + p.tiles * 2 * width * 4;
    return p;
}

template <typename F>
void with_lanes(int lanes, F&& f) {
    using std::integral_constant;
    if (lanes == 16) f(integral_constant<int, 16>{});
    else if (lanes == 32) f(integral_constant<int, 32>{});
    else if (lanes == 64) f(integral_constant<int, 64>{});
    else if (lanes == 128) f(integral_constant<int, 128>{});
    else f(integral_constant<int, 256>{});
}

template <typename F>
void with_type(int type, F&& f) {
    if (type == ATLAS_OPS_F32) f(0.0f);
    else f(bf16_t{});
}

// ------------------------------------------------------------------ dropout
// The simulator's generator: splitmix64's finaliser of seed ^ stream C1 ^ tick C2 ^ draw C3 (executor.rs:190-222).
// Values 2 n and 2 n + 1 take the low and the high 32 bits of draw n.
constexpr u64 STREAM = 0x9e3779b97f4a7c15ull, TICK = 0xd1b54a32d192ed03ull, INDEX = 0x94d049bb133111ebull;

__device__ __forceinline__ u64 finalise(u64 v) {
    v = (v ^ (v >> 30)) * 0xbf58476d1ce4e5b9ull;
    v = (v ^ (v >> 27)) * 0x94d049bb133111ebull;
    return v ^ (v >> 31);
}

// y may be x or residual: a thread reads its values before it writes them, and no other reads them.
template <typename T, bool RESIDUAL>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, const T* residual, i64 count, uint32_t threshold, float factor, u64 base,
                                                      u64 tick, const i64* tick_at, T* y) {
    constexpr int N = Unit<T>::N;
    if (tick_at) tick = (u64)*tick_at;
    base ^= tick * TICK;
    const i64 stride = (i64)gridDim.x * 256 * N;
    for (i64 at = ((i64)blockIdx.x * 256 + threadIdx.x) * N; at < count; at += stride) {
        const int left = (int)min((i64)N, count - at);
        Unit<T> v, r;
        v.load(x + at, 0, left);
        if constexpr (RESIDUAL) r.load(residual + at, 0, left);
        u64 index = (u64)(at / 2) * INDEX;
        float out[N];
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const u64 draw = finalise(base ^ index);
            index += INDEX;
            out[i] = (uint32_t)draw >= threshold ? v[i] * factor : 0.0f;
            out[i + 1] = (uint32_t)(draw >> 32) >= threshold ? v[i + 1] * factor : 0.0f;
            if constexpr (RESIDUAL) out[i] += r[i], out[i + 1] += r[i + 1];
        }
        store_unit<T>(y + at, left, out);
    }
}

}  // namespace
}  // namespace atlas_ops

using namespace atlas_ops;

extern "C" {

int atlas_ops_embedding(const void* table, int64_t rows, int64_t width, int64_t row_stride, int type, const void* tokens, int wide,
                        int64_t count, float scale, void* out, void* stream, char* err, size_t cap) {
    try {
        if (!known_type(type)) return fail(err, cap, 7, "unknown type");
        if (rows < 1 || width < 1 || width > 0x7FFF0000 || count < 0) return fail(err, cap, 7, "rows and width must be positive, width below 2^31");
        if (!count) return 0;
        if (!table || !tokens || !out) return fail(err, cap, 7, "null argument");
        const int lanes = plan_of(1, 1, width, type).lanes;
        const i64 blocks = std::min<i64>(ceil_div(count, 2 * (256 / lanes)), 1 << 20);
        with_type(type, [&](auto t) {
            using T = decltype(t);
            with_lanes(lanes, [&](auto l) {
                embed_forward<T, l()><<<dim3((unsigned)blocks), 256, 0, (hipStream_t)stream>>>(
                    (const T*)table, rows, (int)width, row_stride, Tokens{tokens, wide, count}, scale, (T*)out);
            });
        });
        return launched(err, cap, "embedding");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

// Sizes that the sort and the sums' grids take.
static bool embedding_fits(i64 count, i64 rows, i64 width) {
    return count >= 0 && count <= (1 << 27) && rows >= 1 && rows < 0x7FFFFFFF && width >= 1 && width <= (1 << 20);
}

int64_t atlas_ops_embedding_workspace(int64_t count, int64_t rows, int64_t width, int type) {
    if (!embedding_fits(count, rows, width) || !known_type(type)) return 0;
    return is_few(count, rows, width, type) ? 16 : plan_of(count, rows, width, type).bytes;
}

int atlas_ops_embedding_backward(const AtlasRows* grad, const void* tokens, int wide, int64_t count, int64_t rows, int64_t width, int type,
                                 int table_type, float scale, void* dtable, void* workspace, void* stream, char* err, size_t cap) {
    try {
        if (!known_type(type) || !known_type(table_type)) return fail(err, cap, 7, "unknown type");
        if (!embedding_fits(count, rows, width)) return fail(err, cap, 7, "at most 2^27 tokens, rows below 2^31 - 1, width up to 2^20, both positive");
        if (!dtable || (count && (!grad || !grad->data || grad->inner < 1 || !tokens || !workspace)))
            return fail(err, cap, 7, "null argument");
        hipStream_t st = (hipStream_t)stream;
        if (is_few(count, rows, width, type)) {
            const Rows g{grad->data, grad->inner, grad->outer_stride, grad->inner_stride};
            const dim3 grid((unsigned)rows, (unsigned)few_slices(width, type));
            with_type(type, [&](auto t) {
                with_type(table_type, [&](auto o) {
                    using O = decltype(o);
                    auto* few = count <= 2048 ? embed_few<decltype(t), O, 2> : embed_few<decltype(t), O, FEW_TOKENS / 1024>;
                    few<<<grid, 1024, 0, st>>>(g, (int)width, Tokens{tokens, wide, count}, scale, (O*)dtable);
                });
            });
            return launched(err, cap, "embedding_backward");
        }
        Plan p = plan_of(count, rows, width, type);
        const i64 size = rows * width * (table_type == ATLAS_OPS_F32 ? 4 : 2);
        const i64 clearing = std::min<i64>(ceil_div(size, 256 * 16 * 4), 2048);
        const Tokens list{tokens, wide, count};
        char* base = (char*)workspace;
        uint32_t *counts = (uint32_t*)base, *keys[2], *places[2];
        for (int i = 0; i < 2; ++i) {
            keys[i] = (uint32_t*)(base + p.keys_at) + 2 * i * count;
            places[i] = keys[i] + count;
        }
        const unsigned tiles = (unsigned)p.sort.tiles;
        sort_count<<<dim3((unsigned)(tiles + clearing)), 256, 0, st>>>(p.sort, list, counts, (char*)dtable, size, base + p.counts,
                                                                      count ? 16 + p.counts * (p.passes - 1) : 0);
        if (!count) return launched(err, cap, "embedding_backward");
        for (int pass = 0; pass < p.passes; ++pass, p.sort.shift += p.sort.bits) {
            const uint32_t *k = keys[(pass + 1) % 2], *v = places[(pass + 1) % 2];
            uint32_t *ko = keys[pass % 2], *vo = places[pass % 2];
            uint32_t* after = pass + 1 < p.passes ? (uint32_t*)(base + 16 + (pass + 1) * p.counts) : nullptr;
            const bool scanned = p.sort.tiles > SCANNED;
            if (scanned) sort_scan<<<dim3((unsigned)ceil_div(1 << p.sort.bits, 4)), 256, 0, st>>>(p.sort, counts);
            if (pass == 0 && scanned) sort_scatter<true, true><<<dim3(tiles), 256, 0, st>>>(p.sort, list, k, v, counts, ko, vo, after);
            else if (pass == 0) sort_scatter<true, false><<<dim3(tiles), 256, 0, st>>>(p.sort, list, k, v, counts, ko, vo, after);
            else if (scanned) sort_scatter<false, true><<<dim3(tiles), 256, 0, st>>>(p.sort, list, k, v, counts, ko, vo, after);
            else sort_scatter<false, false><<<dim3(tiles), 256, 0, st>>>(p.sort, list, k, v, counts, ko, vo, after);
            counts = after;
        }
        const uint32_t *sorted = keys[(p.passes + 1) % 2], *order = places[(p.passes + 1) % 2];
        float* partial = (float*)(base + p.partial_at);
        Crossing::Start* lists = (Crossing::Start*)(base + p.lists_at);
        const Crossing crossing{(uint32_t*)(base + p.counts), (uint32_t*)(lists + 2 * p.tiles), {lists, lists + p.tiles}};
        const Rows g{grad->data, grad->inner, grad->outer_stride, grad->inner_stride};
        with_type(type, [&](auto t) {
            using T = decltype(t);
            constexpr int N = Unit<T>::N;
            with_type(table_type, [&](auto o) {
                using O = decltype(o);
                with_lanes(p.lanes, [&](auto l) {
                    const unsigned slices = (unsigned)ceil_div(width, l() * N);
                    const dim3 grid((unsigned)ceil_div(p.tiles, 256 / l()), slices);
                    auto* sum = p.sum_tile == 32 ? embed_sum<T, O, l(), 32> : p.sum_tile == 16 ? embed_sum<T, O, l(), 16> : embed_sum<T, O, l(), 8>;
                    sum<<<grid, 256, 0, st>>>(g, (int)width, count, (int)rows, sorted, order, scale, (O*)dtable, partial, crossing);
                });
                if (p.tiles > 1) {  // a workgroup to a CU, as its registers allow
                    const i64 slices = ceil_div(width, 64);
                    embed_join<O><<<dim3((unsigned)std::max<i64>(256 / slices & ~(i64)1, 2), (unsigned)slices), 1024, 0, st>>>(
                        (int)width, scale, (O*)dtable, partial, crossing);
                }
            });
        });
        return launched(err, cap, "embedding_backward");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

int atlas_ops_dropout(const void* x, const void* residual, int64_t count, int type, double probability, uint64_t seed, uint64_t counter_stream,
                      uint64_t tick, const int64_t* tick_at, void* y, void* stream, char* err, size_t cap) {
    try {
        if (!known_type(type)) return fail(err, cap, 7, "unknown type");
        if (!(probability >= 0.0 && probability < 1.0)) return fail(err, cap, 7, "probability must be 0 or more and below 1");
        if (count < 0) return fail(err, cap, 7, "count must not be negative");
        if (!count) return 0;
        if (!x || !y) return fail(err, cap, 7, "null argument");
        const double share = probability * 4294967296.0;
        const uint32_t threshold = share >= 4294967295.0 ? 0xFFFFFFFFu : (uint32_t)(share + 0.5);
        const float factor = (float)(1.0 / (1.0 - probability));
        const u64 base = seed ^ counter_stream * STREAM;
        with_type(type, [&](auto t) {
            using T = decltype(t);
            const i64 blocks = std::min<i64>(ceil_div(count, 256 * Unit<T>::N), 4096);
            if (residual)
                dropout_kernel<T, true><<<dim3((unsigned)blocks), 256, 0, (hipStream_t)stream>>>(
                    (const T*)x, (const T*)residual, count, threshold, factor, base, tick, tick_at, (T*)y);
            else
                dropout_kernel<T, false><<<dim3((unsigned)blocks), 256, 0, (hipStream_t)stream>>>(
                    (const T*)x, nullptr, count, threshold, factor, base, tick, tick_at, (T*)y);
        });
        return launched(err, cap, "dropout");
    } catch (...) {
        return fail(err, cap, 7, "host exception");
    }
}

}  // extern "C"
