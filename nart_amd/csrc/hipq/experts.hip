// A layer of experts with 4-bit weights (hipq_w4_experts_*): every token's best experts from its scores, their gated products, the second product of
// each and the weighted sum.  gfx950 only.
//
//   y[t] = sum over the chosen e of share[t][e] * down_e (act(gate_e x[t]) * up_e x[t])
//
// A pair is a token and one of its experts.  Choosing and numbering: a wave finds a token's experts (the largest of its scores, `top` times); one work-group then
// counts the pairs of each expert and numbers them, an expert's side by side.  Behind that few tokens take streams of weights, more the tiles of w4_tile.h, whose blocks of
// rows then have an expert each.  The hidden rows between the products are rounded to 16 bits, as the matrix unit takes them.  The tiles' second product leaves float32 sums,
// of which a last kernel adds a token's, each times its share.
//
// What bounds them, with the launches' own times in us: one token of two of 8 experts of 4096 x 14336 26 + 16, its 183 MB of weights at 4.4 TB/s of the 5.1 that a copy reaches;
// of six of 64 of 2048 x 1408 8.6 + 6.8, two launches' beginnings and ends; 24 tokens of those, groups of 64 with zero points, 7 + 33 + 24 + 5, 209 MB at 3.7 TB/s.  2048 tokens of
// four of 32 of 4096 x 2048 5 + 8 + 8 + 304 + 6 + 188 + 24: 1.02 PFLOP/s of the products, with the rows that fill up the blocks (a fifth), as w4_tile_kernel reaches without experts.  333 tokens of three of 13 of 1056 x 1120 4 + 4 + 21 + 14 + 5:
// vector instructions of groups of 32 with zero points, on a chip that is filled once.
#include <cmath>
#include <new>

#include "overlap.h"
#include "w4_tile.h"

namespace hipq {

constexpr int MOST_EXPERTS = 1024, MOST_TOP = 16;

struct RouteArgs {
    const void *logits;
    int64_t stride;
    int type, M, experts, top, sigmoid, normalize, block_rows;
    int32_t *chosen; // [M][top]: the expert, -1: none
    float *share;    // [M][top]
    int32_t *place;  // [M][top]: the pair's number, -1: none
    int32_t *row;    // [pairs]: its token
    W4Block *block;
    int32_t *count;  // of blocks
    float *placed_share; // [pairs]: by number, or nullptr
    int most_blocks;
};

// the largest of a wave's numbers, within groups of 16 lanes by turning them round
__device__ static __forceinline__ uint32_t largest_of(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x122, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x121, 0xf, 0xf, true));
    const uint32_t a = max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
    return max(a, max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
}

struct Choice {
    int expert; // -1: none
    float share;
};
// A token's experts, lane s has the s-th; its scores over the lanes of a wave: lane l has those of experts l, l + 64, ..., EACH of them
template <int EACH>
__device__ static __forceinline__ void load_scores(const RouteArgs &a, int t, int lane, uint32_t (&raw)[EACH]) // as they are: nothing waits for them here
{
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int64_t at = t * a.stride + min(i * 64 + lane, a.experts - 1);
        if (a.type == HIPQ_REAL_F32)
            raw[i] = ((const uint32_t *)a.logits)[at];
        else
            raw[i] = ((const uint16_t *)a.logits)[at];
    }
}

template <int EACH>
__device__ static __forceinline__ Choice choose(const RouteArgs &a, const uint32_t (&raw)[EACH], int lane)
{
    uint32_t key[EACH]; // in the order of the scores; 0: never taken
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const float x = a.type == HIPQ_REAL_F32 ? __builtin_bit_cast(float, raw[i]) : a.type == HIPQ_REAL_F16 ? Real16<HIPQ_REAL_F16>::low(raw[i]) : Real16<HIPQ_REAL_BF16>::low(raw[i]);
        const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f); // -0 is 0
        key[i] = i * 64 + lane >= a.experts || !(x > -__builtin_inff()) ? 0 : u & 0x80000000u ? ~u : u | 0x80000000u;
    }
    auto largest = [&] {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++)
            most = max(most, key[i]);
        return largest_of(most);
    };
    auto score = [](uint32_t k) { return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k); };
    const uint32_t most = largest();
    const float top_score = most ? score(most) : 0.0f;
    // e^(x - m); of infinite scores each counts as much, and nothing else does
    auto weight = [&](float v) { return v == top_score ? 1.0f : exp2_fast((v - top_score) * 1.4426950408889634f); };
    float all = 0;
    if (!a.sigmoid && !a.normalize) {
#pragma unroll
        for (int i = 0; i < EACH; i++)
            if (key[i])
                all += weight(score(key[i]));
#pragma unroll
        for (int o = 1; o < 64; o *= 2)
            all += __shfl_xor(all, o);
    }
    // 1 / (1 + e^-x), and where shares are divided by their sum, e^-r times that with r = min(0, the largest): not 0 however small they are
    const float low = a.normalize ? fminf(top_score, 0.0f) : 0.0f, lift = exp2_fast(low * 1.4426950408889634f);
    int mine = -1; // lane s: the s-th expert
    float share = 0, sum = 0;
    for (int s = 0; s < a.top; s++) {
        const uint32_t best = s == 0 ? most : largest();
        if (best == 0)
            break;
        int e = -1; // the lowest of those that have it
#pragma unroll
        for (int i = EACH - 1; i >= 0; i--) {
            const uint64_t equal = __ballot(key[i] == best);
            e = equal ? i * 64 + __builtin_ctzll(equal) : e;
        }
#pragma unroll
        for (int i = 0; i < EACH; i++)
            if (i * 64 + lane == e)
                key[i] = 0;
        const float v = score(best), w = a.sigmoid ? 1.0f / (lift + exp2_fast((low - v) * 1.4426950408889634f)) : weight(v);
        sum += w;
        if (lane == s)
            mine = e, share = w;
    }
    return {mine, mine < 0 ? 0.0f : share / (a.normalize ? sum : a.sigmoid ? 1.0f : all)};
}

template <int EACH>
__global__ __launch_bounds__(256) void experts_choose_kernel(const RouteArgs a)
{
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (t >= a.M)
        return;
    uint32_t raw[EACH];
    load_scores<EACH>(a, (int)t, lane, raw);
    const Choice own = choose<EACH>(a, raw, lane);
    if (lane < a.top)
        a.chosen[t * a.top + lane] = own.expert, a.share[t * a.top + lane] = own.share;
}

// an expert's pairs and blocks of rows, by thread, and those before it; lists the blocks, and returns where the expert's pairs begin
__device__ static __forceinline__ int list_blocks(const RouteArgs &a, int pairs_of, int *scan)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, blocks_of = (pairs_of + a.block_rows - 1) / a.block_rows;
    int first = pairs_of, base = blocks_of;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int u = __shfl_up(first, o), v = __shfl_up(base, o);
        first += lane >= o ? u : 0, base += lane >= o ? v : 0;
    }
    if (lane == 63)
        scan[wave] = first, scan[16 + wave] = base;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; w++)
        first += w < wave ? scan[w] : 0, base += w < wave ? scan[16 + w] : 0;
    if (tid == 1023)
        *a.count = base;
    first -= pairs_of, base -= blocks_of;
#pragma unroll 1
    for (int i = 0; i < blocks_of; i++)
        a.block[base + i] = W4Block{tid, first + i * a.block_rows, min(first + pairs_of, first + (i + 1) * a.block_rows), base, blocks_of};
    return first;
}

// the lanes with the same expert
__device__ static __forceinline__ uint64_t same_expert(int e, int experts)
{
    uint64_t lanes = __ballot(e >= 0);
#pragma unroll 1
    for (int bit = 0; experts > 1 << bit; bit++) {
        const uint64_t set = __ballot((e >> bit) & 1);
        lanes &= (e >> bit) & 1 ? set : ~set;
    }
    return lanes;
}

// Few tokens: chooses their experts and numbers the pairs, by expert and then by token: a row's block, and with it the order of its sums, is the same every time.  Each of 16
// waves has a contiguous part of the pairs, and goes through it 64 at a time twice: to count each expert's, and to number them from where the waves before it end.
constexpr int CHOOSE_TOKENS = 128;
template <int EACH>
__global__ __launch_bounds__(1024) void experts_route_kernel(const RouteArgs a)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    int32_t *const counts = (int32_t *)lds; // [wave][expert]
    __shared__ int32_t scan[32], chosen[CHOOSE_TOKENS * MOST_TOP];
    __shared__ float share[CHOOSE_TOKENS * MOST_TOP];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr bool AHEAD = EACH <= 4; // more than that are too many registers
    uint32_t raw[EACH], next[EACH];
    if (wave < a.M)
        load_scores<EACH>(a, wave, lane, next);
#pragma unroll 1
    for (int t = wave; t < a.M; t += 16) {
#pragma unroll
        for (int i = 0; i < EACH; i++)
            raw[i] = next[i];
        if (AHEAD && t + 16 < a.M)
            load_scores<EACH>(a, t + 16, lane, next);
        const Choice own = choose<EACH>(a, raw, lane);
        if (!AHEAD && t + 16 < a.M)
            load_scores<EACH>(a, t + 16, lane, next);
        if (lane < a.top)
            chosen[t * a.top + lane] = own.expert, share[t * a.top + lane] = a.share[t * a.top + lane] = own.share;
    }
    for (int i = tid; i < 16 * a.experts; i += 1024)
        counts[i] = 0;
    __syncthreads();
    const int pairs = a.M * a.top, part = (pairs + 1023) / 1024 * 64, from = wave * part, to = min(pairs, from + part);
#pragma unroll 1
    for (int p = from + lane; p - lane < to; p += 64)
        if (p < to && chosen[p] >= 0)
            atomicAdd(&counts[wave * a.experts + chosen[p]], 1);
    __syncthreads();
    int n[16], all = 0;
    if (tid < a.experts) {
#pragma unroll
        for (int w = 0; w < 16; w++)
            n[w] = counts[w * a.experts + tid];
#pragma unroll
        for (int w = 0; w < 16; w++)
            all += n[w];
    }
    int at = list_blocks(a, all, scan);
    if (tid < a.experts)
#pragma unroll
        for (int w = 0; w < 16; w++) {
            counts[w * a.experts + tid] = at;
            at += n[w];
        }
    __syncthreads();
#pragma unroll 1
    for (int p = from + lane; p - lane < to; p += 64) {
        const int e = p < to ? chosen[p] : -1;
        const uint64_t lanes = same_expert(e, a.experts);
        int place = -1;
        if (e >= 0) {
            place = counts[wave * a.experts + e] + __builtin_popcountll(lanes & ((1ull << lane) - 1));
            a.row[place] = p / a.top;
            if (a.placed_share)
                a.placed_share[place] = share[p];
        }
        if (p < to)
            a.place[p] = place;
        if (e >= 0 && lane == __builtin_ctzll(lanes)) // in order behind the reads above: a wave's LDS accesses are
            counts[wave * a.experts + e] += __builtin_popcountll(lanes);
    }
}

// More tokens, whose experts are chosen (7.5 us of 8192 pairs: a round of eight loads and LDS additions that return): a pair's place among its expert's is the one that it gets first.  Which row of a block it then is does not show in its result, and
// neither does the block: all blocks of an expert's rows go through k from the same place on.
__global__ __launch_bounds__(1024) void experts_number_kernel(const RouteArgs a)
{
    __shared__ int32_t counts[MOST_EXPERTS], scan[32];
    const int tid = threadIdx.x, pairs = a.M * a.top;
    constexpr int STEPS = 8; // on their way at once; the first stay in registers, others' places wait in memory
    int e[STEPS], place[STEPS];
    counts[tid] = 0;
    __syncthreads();
#pragma unroll 1
    for (int p0 = tid + (pairs - 1) / (1024 * STEPS) * (1024 * STEPS); p0 >= 0; p0 -= 1024 * STEPS) { // the first last
#pragma unroll
        for (int k = 0; k < STEPS; k++)
            e[k] = p0 + 1024 * k < pairs ? a.chosen[p0 + 1024 * k] : -1;
#pragma unroll
        for (int k = 0; k < STEPS; k++)
            place[k] = e[k] >= 0 ? atomicAdd(&counts[e[k]], 1) : 0;
        if (p0 >= 1024 * STEPS)
#pragma unroll
            for (int k = 0; k < STEPS; k++)
                if (p0 + 1024 * k < pairs)
                    a.place[p0 + 1024 * k] = place[k];
    }
    __syncthreads();
    const int first = list_blocks(a, tid < a.experts ? counts[tid] : 0, scan);
    __syncthreads();
    counts[tid] = first;
    __syncthreads();
#pragma unroll 1
    for (int p0 = tid; p0 < pairs; p0 += 1024 * STEPS) {
        if (p0 >= 1024 * STEPS)
#pragma unroll
            for (int k = 0; k < STEPS; k++) {
                const int p = p0 + 1024 * k;
                e[k] = p < pairs ? a.chosen[p] : -1, place[k] = p < pairs ? a.place[p] : 0;
            }
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
            const int p = p0 + 1024 * k;
            if (p < pairs) {
                if (e[k] >= 0)
                    place[k] += counts[e[k]], a.row[place[k]] = p / a.top;
                a.place[p] = e[k] >= 0 ? place[k] : -1;
            }
        }
    }
}

// four neighbouring results, the first `left` of them
template <int TYPE>
__device__ static __forceinline__ void put4(uint16_t *to, const f32x4 &v, int left)
{
    if (left >= 4 && (uintptr_t)to % 8 == 0)
        *(u32x2 *)to = u32x2{Real16<TYPE>::pack(v[0], v[1]), Real16<TYPE>::pack(v[2], v[3])};
    else
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < left)
                to[e] = rounded<TYPE>(v[e]);
}

// y[t] = sum of a token's pairs, four values a thread and a token a work-group, whose pairs' numbers then are the same for all; four pairs on their way at once.  2048 tokens of four
// pairs of 4096 values: 151 MB in 23.5 us, 6.4 TB/s, some from the caches (with a division for each thread, one pair at a time and 2-byte stores 33).
template <int TYPE>
__global__ __launch_bounds__(256) void experts_join_kernel(const RouteArgs a, const float *part, int splits, int64_t pairs, int columns, uint16_t *y, int64_t y_stride, int N, int stretches)
{
    const int t = blockIdx.x / stretches, n = ((int)(blockIdx.x - t * stretches) * 256 + (int)threadIdx.x) * 4;
    if (n >= N)
        return;
    f32x4 v = {0, 0, 0, 0};
    for (int s = 0; s < a.top; s += 4) {
        int p[4];
        float share[4];
        f32x4 u[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            p[k] = s + k < a.top ? a.place[(int64_t)t * a.top + s + k] : -1;
            share[k] = s + k < a.top ? a.share[(int64_t)t * a.top + s + k] : 0;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            u[k] = f32x4{0, 0, 0, 0};
            if (p[k] >= 0)
                u[k] = *(const f32x4 *)(part + (int64_t)p[k] * columns + n);
        }
        for (int i = 1; i < splits; i++)
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (p[k] >= 0)
                    u[k] += *(const f32x4 *)(part + (i * pairs + p[k]) * columns + n);
#pragma unroll
        for (int k = 0; k < 4; k++)
            v += share[k] * u[k];
    }
    put4<TYPE>(y + t * y_stride + n, v, N - n);
}

// ---- few tokens: streams of weights --------------------------------------------------------------------------------------------------
// An expert has some rows, so the time is what it takes to read the chosen experts' weights, and to begin with it: they go straight into registers, several blocks
// of k ahead, and no wave waits for another before its end.  A block has up to ROWS rows.  Of 4 rows 128 k are one load, lane c + 16 j of which has row c % 4 and k = 32 (c / 4) +
// 8 j + 0..7, and turning it round within 16 lanes brings the next operand's to lanes 0..3; of 16 rows they are four loads, more than the weights are.
constexpr int FEW_TOKENS = 64, FEW_PAIRS = FEW_TOKENS * MOST_TOP;

template <int N>
__device__ static __forceinline__ u32x4 turned(const u32x4 &v)
{
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = v[i];
        o[i] = (uint32_t)__builtin_amdgcn_mov_dpp((int)w, 0x120 + N, 0xf, 0xf, true);
    }
    return o;
}

// Blocks of 128 k of NT tiles and of ROWS rows, DEPTH of them on their way (w4_stream_kernel's arithmetic)
template <int TYPE, int GPB, bool ZEROS, int ROWS, int NT, int DEPTH>
struct Stream {
    using R = Real16<TYPE>;
    static constexpr int PIECES = ROWS == 4 ? 1 : 4;
    u32x4 w[DEPTH][NT], x[DEPTH][PIECES];
    Scales<TYPE, GPB, ZEROS> s[DEPTH][NT];
    f32x4 total[NT];
    Spread<TYPE> spread;
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
            total[nt] = f32x4{0, 0, 0, 0};
    }
    // the row that a lane reads, and where in it
    static __device__ __forceinline__ int row_of(int c) { return ROWS == 4 ? c % 4 : c; }
    static __device__ __forceinline__ int k_of(int c, int j) { return 8 * j + (ROWS == 4 ? c / 4 * 32 : 0); }
    // q, scales: an array's; row: the lane's row of x, k_of elements into it
    __device__ __forceinline__ void load(int d, const W4Args &a, const uint8_t *q, const uint8_t *scales, const uint16_t *row, int tile, int kb, int lane)
    {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            w[d][nt] = *(const u32x4 *)(q + weights_at(tile + nt, kb, a.blocks) * 1024 + lane * 16);
            s[d][nt].load(scales + (scales_at(tile + nt, kb, a.blocks) + (lane & 15)) * s[d][nt].BYTES);
        }
#pragma unroll
        for (int t = 0; t < PIECES; t++) {
            x[d][t] = u32x4{0, 0, 0, 0};
            if (kb * 128 + (ROWS == 4 ? (lane & 15) / 4 : t) * 32 < a.K)
                x[d][t] = *(const u32x4 *)(row + kb * 128 + t * 32);
        }
    }
    __device__ __forceinline__ void multiply(int d)
    {
        const u32x4 minus_one = {Nibbles<TYPE>::MINUS_ONE, Nibbles<TYPE>::MINUS_ONE, Nibbles<TYPE>::MINUS_ONE, Nibbles<TYPE>::MINUS_ONE};
        u32x4 a[4];
        if constexpr (ROWS == 4)
            a[0] = x[d][0], a[1] = turned<12>(x[d][0]), a[2] = turned<8>(x[d][0]), a[3] = turned<4>(x[d][0]);
        else
#pragma unroll
            for (int t = 0; t < 4; t++)
                a[t] = x[d][t % PIECES];
#pragma unroll
        for (int g = 0; g < GPB; g++) {
            f32x4 less = {0, 0, 0, 0}; // minus the sums of x, in every column
#pragma unroll
            for (int t = g * 4 / GPB; t < (g + 1) * 4 / GPB; t++)
                less = R::mfma(a[t], minus_one, less);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                f32x4 sum = less * s[d][nt].offset(g);
#pragma unroll
                for (int t = g * 4 / GPB; t < (g + 1) * 4 / GPB; t++)
                    sum = R::mfma(a[t], spread(w[d][nt][t]), sum);
                const float scale = s[d][nt].scale(g);
#pragma unroll
                for (int r = 0; r < 4; r++)
                    total[nt][r] = __builtin_fmaf(scale, sum[r], total[nt][r]);
            }
        }
    }
};

struct FewArgs {
    RouteArgs r;
    W4Args a; // x and y: of the launch
    size_t q_bytes, s_bytes; // of an expert
    int groups;              // work-groups of a block of rows
    float *part;             // [split][token][column] of the second launch, where work-groups share a tile
};

// The hidden rows: a work-group has a tile of the gate and its one of the other projection, for a block of rows, and four waves take the blocks of k in turn, two
// ahead each: little for one wave, but many are there.  us of the whole layer with 2 and 4 tiles, 4 and 8 waves, 2 and 3 or 4 blocks: one token through 2 of 8 experts of 4096 x 14336
// 47.5; 48.1 with 4 tiles; 48.1 with 8 waves; 50.0 with 4 blocks; 54 with 4 tiles and 3 blocks; 16 tokens through 6 of 64 of 2048 x 1408 51.8, 52.5, 55.1, 53.2, 56.5.
// Of up to four tokens, whose experts have a block each, every work-group chooses them itself (EACH > 0) rather than wait for a launch that does: a wave a token, and blocks in the
// order in which their experts come first.  One more work-group leaves the list for the second product.  us of the layer with and without, 1, 2 and 4 tokens through 2 of 8 experts of
// 4096 x 14336 50 and 52, 51 and 53, 77 and 78, 6 of 64 of 2048 x 1408 15.3 and 19.2, 20.6 and 23.8, 29.2 and 30.9, 8 of 128 of 2048 x 768 14.1 and 17.7 (1), 26.2 and 28.3 (4), 16 of 256 of
// 1024 x 256 22.8 and 22.7 (4).
template <int TYPE, int GPB, bool ZEROS, int ROWS, int EACH>
__global__ __launch_bounds__(256) void experts_few_up_kernel(const FewArgs f)
{
    constexpr int WAVES = 4, NT = 2, DEPTH = 2;
    using S = Stream<TYPE, GPB, ZEROS, ROWS, NT, DEPTH>;
    __shared__ f32x4 red[WAVES][NT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, j = lane >> 4;
    const W4Args &a = f.a;
    // the first work-group leaves the list
    const int item = (int)blockIdx.x - (EACH > 0), block = item / f.groups, tile0 = (item - block * f.groups) * NT;
    int first, rows, expert;
    const uint16_t *row = a.x + S::k_of(c, j);
    if constexpr (EACH > 0) {
        static_assert(ROWS == 4 && WAVES == 4, "a block for an expert, a wave for a token");
        __shared__ int32_t chosen[64];
        __shared__ float share[64];
        const int top = f.r.top;
        int e = -1, leader = 64; // of the pair that a lane is: its expert, and that expert's first pair
        float part = 0;
        if (f.r.M == 1) {
            uint32_t raw[EACH];
            load_scores<EACH>(f.r, 0, lane, raw);
            const Choice own = choose<EACH>(f.r, raw, lane);
            e = own.expert, part = own.share, leader = e >= 0 ? lane : 64;
        } else {
            if (wave < f.r.M) {
                uint32_t raw[EACH];
                load_scores<EACH>(f.r, wave, lane, raw);
                const Choice own = choose<EACH>(f.r, raw, lane);
                if (lane < top)
                    chosen[wave * top + lane] = own.expert, share[wave * top + lane] = own.share;
            }
            __syncthreads();
            if (lane < f.r.M * top)
                e = chosen[lane], part = share[lane];
            const uint64_t same = same_expert(e, f.r.experts);
            leader = e >= 0 ? __builtin_ctzll(same) : 64;
        }
        const uint64_t leaders = __ballot(leader == lane);
        if (item < 0) { // block by block
            if (wave > 0)
                return;
            int base = 0, number = 0;
#pragma unroll 1
            for (uint64_t left = leaders; left; left &= left - 1, number++) {
                const int of = __builtin_ctzll(left);
                const uint64_t pairs = __ballot(leader == of);
                if (leader == of) {
                    const int place = base + __builtin_popcountll(pairs & ((1ull << lane) - 1));
                    f.r.row[place] = lane / top, f.r.placed_share[place] = part;
                }
                if (lane == of)
                    f.r.block[number] = W4Block{e, base, base + __builtin_popcountll(pairs), 0, 0};
                base += __builtin_popcountll(pairs);
            }
            if (lane == 0)
                *f.r.count = number;
            return;
        }
        if (block >= __builtin_popcountll(leaders))
            return;
        if (f.r.M == 1)
            first = block, rows = 1, expert = __builtin_amdgcn_readlane(e, block);
        else {
            const int of = __builtin_ctzll(__ballot(leader == lane && __builtin_popcountll(leaders & ((1ull << lane) - 1)) == block));
            expert = __builtin_amdgcn_readlane(e, of);
            uint64_t pairs = __ballot(leader == of);
            first = __builtin_popcountll(__ballot(leader < of)), rows = __builtin_popcountll(pairs);
#pragma unroll
            for (int r = 0; r < ROWS - 1; r++) // a lane's row, the last one again behind it
                if (r < min(S::row_of(c), rows - 1))
                    pairs &= pairs - 1;
            row += __builtin_ctzll(pairs) / top * a.x_stride;
        }
    } else {
        const W4Block b = f.r.block[block]; // read before it is known whether it is there
        if (block >= *f.r.count)
            return;
        first = b.first, rows = b.end - first, expert = b.array;
        row += (int64_t)f.r.row[first + min(S::row_of(c), rows - 1)] * a.x_stride;
    }
    const uint8_t *const q = a.q + expert * f.q_bytes, *const scales = a.scales + expert * f.s_bytes;
    S stream;
    stream.clear();
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
        if (wave + d * WAVES < a.blocks)
            stream.load(d, a, q, scales, row, tile0, wave + d * WAVES, lane);
    for (int kb = wave; kb < a.blocks; kb += DEPTH * WAVES)
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            if (kb + d * WAVES < a.blocks) {
                stream.multiply(d);
                if (kb + (d + DEPTH) * WAVES < a.blocks)
                    stream.load(d, a, q, scales, row, tile0, kb + (d + DEPTH) * WAVES, lane);
            }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
        red[wave][nt][lane] = stream.total[nt];
    __syncthreads();
    if (wave == 0) {
        f32x4 gate = red[0][0][lane], up = red[0][1][lane];
#pragma unroll
        for (int o = 1; o < WAVES; o++)
            gate += red[o][0][lane], up += red[o][1][lane];
        const int n = tile0 / 2 * 16 + c;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (n < a.N && 4 * j + i < rows)
                a.y[(int64_t)(first + 4 * j + i) * a.y_stride + n] = rounded<TYPE>(activate(gate[i], a.activation) * up[i]);
    }
}

// The result: a work-group has a tile of outputs, its waves the same number of blocks each - of all blocks of rows and k, one after the other - and every
// wave adds up what it has of each token, in LDS, where they meet.  Where there are fewer tiles than CUs, and much to read, gridDim.y work-groups share them, and
// another launch adds up what they leave.  (The last of them to end could do that, but to have written what others read takes a write-back of the L2: 90 us.)
template <int TYPE, int GPB, bool ZEROS, int ROWS, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void experts_few_down_kernel(const FewArgs f)
{
    constexpr int DEPTH = 2;
    using S = Stream<TYPE, GPB, ZEROS, ROWS, 1, DEPTH>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const RouteArgs &r = f.r;
    const W4Args &a = f.a;
    const int pairs = r.M * r.top;
    float *const sums = (float *)lds;                     // [wave][token][16]
    float *const share = sums + WAVES * r.M * 16;         // [pair]
    int32_t *const token = (int32_t *)(share + pairs);    // [pair]
    int32_t *const block = token + pairs;                 // [block]: expert, first, end
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, j = lane >> 4;
    const int tile = blockIdx.x, items = __builtin_amdgcn_readfirstlane(*r.count) * a.blocks;
    for (int i = tid; i < pairs; i += WAVES * 64) { // what lies behind their ends is not looked at
        share[i] = r.placed_share[i], token[i] = r.row[i];
        if (i < r.most_blocks)
            block[3 * i] = r.block[i].array, block[3 * i + 1] = r.block[i].first, block[3 * i + 2] = r.block[i].end;
    }
    for (int i = tid; i < WAVES * r.M * 16; i += WAVES * 64)
        sums[i] = 0;
    __syncthreads();
    const int split = blockIdx.y, splits = gridDim.y, own = split * WAVES + wave, all = splits * WAVES;
    const int from = (int)((int64_t)items * own / all), to = (int)((int64_t)items * (own + 1) / all);
    S stream;
    stream.clear();
    // the block that is loaded next, and the one that is multiplied next
    int load_at = from / a.blocks, load_kb = from - load_at * a.blocks, at = load_at, kb = load_kb;
    const uint8_t *q = nullptr, *scales = nullptr;
    const uint16_t *row = nullptr;
    auto enter = [&] {
        const int expert = __builtin_amdgcn_readfirstlane(block[3 * load_at]), first = block[3 * load_at + 1], end = block[3 * load_at + 2];
        q = a.q + expert * f.q_bytes, scales = a.scales + expert * f.s_bytes;
        row = a.x + (int64_t)min(first + S::row_of(c), end - 1) * a.x_stride + S::k_of(c, j);
    };
    auto load = [&](int d) {
        stream.load(d, a, q, scales, row, tile, load_kb, lane);
        if (++load_kb == a.blocks) {
            load_kb = 0, load_at++;
            if (load_at * a.blocks < to)
                enter();
        }
    };
    auto leave = [&] { // a block of rows: what they have is added to their tokens'
        const int first = block[3 * at + 1], end = block[3 * at + 2];
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (first + 4 * j + i < end)
                sums[(wave * r.M + token[first + 4 * j + i]) * 16 + c] += share[first + 4 * j + i] * stream.total[0][i];
        stream.clear();
    };
    if (from < to) {
        enter();
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            if (from + d < to)
                load(d);
        for (int i = from; i < to; i += DEPTH)
#pragma unroll
            for (int d = 0; d < DEPTH; d++)
                if (i + d < to) {
                    stream.multiply(d);
                    if (i + d + DEPTH < to)
                        load(d);
                    if (++kb == a.blocks || i + d + 1 == to) {
                        leave();
                        kb = 0, at++;
                    }
                }
    }
    __syncthreads();
    for (int i = tid; i < r.M * 16; i += WAVES * 64) {
        float v = 0;
#pragma unroll
        for (int o = 0; o < WAVES; o++)
            v += sums[o * r.M * 16 + i];
        const int t = i / 16, n = tile * 16 + i % 16;
        if (splits > 1)
            f.part[((int64_t)split * r.M + t) * (gridDim.x * 16) + n] = v;
        else if (n < a.N)
            a.y[(int64_t)t * a.y_stride + n] = rounded<TYPE>(v);
    }
}

template <int TYPE>
__global__ __launch_bounds__(256) void experts_few_join_kernel(const float *part, int splits, int M, int columns, uint16_t *y, int64_t y_stride, int N)
{
    const int per_row = (N + 3) / 4, id = (int)blockIdx.x * 256 + threadIdx.x, t = id / per_row, n = (id - t * per_row) * 4;
    if (t >= M)
        return;
    f32x4 v = {0, 0, 0, 0};
#pragma unroll 4
    for (int s = 0; s < splits; s++)
        v += *(const f32x4 *)(part + ((int64_t)s * M + t) * columns + n);
    put4<TYPE>(y + t * y_stride + n, v, N - n);
}

} // namespace hipq

using namespace hipq;

struct hipq_w4_experts_plan {
    hipq_w4_experts_desc desc;
    int device, tiles[2];      // of an expert: the gated pair, the second product
    uint8_t *memory;
    W4Args args[2];
    W4Groups groups[2];        // where an expert's weights are
};

namespace hipq {

// What lies in a caller's workspace.
struct ExpertsLayout {
    size_t chosen, share, place, row, block, count, hidden, part, xsum, share_by_number, bytes;
    int kernel, splits, block_rows;
    int64_t pairs, blocks; // at most
    int columns;
};
enum { FEW_4, FEW_16, TILE_16, TILE_32, TILE_64, TILE_128_WIDE, SHAPES };
static const struct {
    const char *name;
    int rows, tiles; // of a work-group
} SHAPE[SHAPES] = {{"w4_experts_stream_4", 4, 1}, {"w4_experts_stream_16", 16, 1}, {"w4_experts_16x128", 16, 8}, {"w4_experts_32x128", 32, 8}, {"w4_experts_64x128", 64, 8}, {"w4_experts_128x256", 128, 16}};

// Measured over 1 to 1024 tokens of 8 experts of 4096 x 14336 (two for a token), 64 of 2048 x 1408 (six), 128 of 2048 x 768 (eight), 13 of 1056 x 1120 and 32 of 4096 x 2048,
// us:
//   * up to 64 tokens and 8 rows of an expert the streams: 16 tokens of the first 164 against 167 with tiles of 16 rows, 64 of the second 98 against 106, but 64 of the
//     first, 16 rows each, 280 against 253; with blocks of 4 rows up to 2 each: 4 of the first 77 against 84, but 32 of the second, 3 each, 83 against 78;
//   * tiles of 16, 32, 64 and 128 x 256: 12 rows each 147, 146, 176, 217; 32 each 370, 327, 378, 486; 48 each 282, 239, 233, 253; 96 each 494, 374, 346, 312; but where the
//     widest would have too few work-groups 71, 60, 53, 67 (333 tokens of the fourth, 77 each).
// The rows of an expert are a mean.  One that many tokens choose has several blocks of rows, each of which reads its weights: 64 tokens of two of 64 experts of 2048 x 1408,
// blocks of 4 rows, 64 us with scores at random, 59 where half of them choose one expert, 56 where all do (16 blocks of its rows, but other experts' weights stay unread).
static ExpertsLayout layout_of(const hipq_w4_experts_plan *p, int M)
{
    const hipq_w4_experts_desc &d = p->desc;
    ExpertsLayout l = {};
    l.pairs = (int64_t)M * d.top;
    const int64_t each = l.pairs / d.experts; // an expert's, were all chosen as often
    const int64_t used = l.pairs < d.experts ? l.pairs : d.experts;
    // work-groups of the widest kernel in the first product, half a block of an expert's rows more than there are
    const int64_t wide = (l.pairs / 128 + used / 2) * ((p->tiles[0] + 15) / 16);
    if (M <= FEW_TOKENS && each <= 8)
        l.kernel = each <= 2 ? FEW_4 : FEW_16;
    else
        l.kernel = each <= 16 ? TILE_16 : each <= 40 ? TILE_32 : each <= 64 || wide < 256 ? TILE_64 : TILE_128_WIDE;
    l.block_rows = SHAPE[l.kernel].rows;
    l.blocks = used + l.pairs / l.block_rows;
    l.blocks = l.blocks < l.pairs ? l.blocks : l.pairs;
    const int64_t groups = l.blocks * ((p->tiles[1] + SHAPE[l.kernel].tiles - 1) / SHAPE[l.kernel].tiles); // of the second product
    const int most = p->args[1].blocks / 4;
    l.splits = groups < 256 ? (int)(256 / groups) : 1;
    l.splits = l.splits < most ? l.splits : most;
    l.splits = l.splits < 1 ? 1 : l.splits;
    l.columns = round_up(p->tiles[1], SHAPE[l.kernel].tiles) * 16;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t from = at;
        at += (bytes + 255) / 256 * 256;
        return from;
    };
    l.chosen = take(l.pairs * 4), l.share = take(l.pairs * 4), l.place = take(l.pairs * 4), l.row = take(l.pairs * 4), l.block = take(l.blocks * sizeof(W4Block)), l.count = take(4);
    l.hidden = take((size_t)l.pairs * d.inner * 2);
    if (l.kernel <= FEW_16) {
        l.share_by_number = take(l.pairs * 4);
        // a work-group of 16 waves is what a CU holds; with less than 16 KB for each wave the launch that joins takes longer
        const int64_t kb = used * p->args[1].blocks / 16;
        l.splits = kb / 16 < 256 / p->tiles[1] ? (int)(kb / 16) : 256 / p->tiles[1];
        l.splits = l.splits < 1 ? 1 : l.splits > 8 ? 8 : l.splits;
        if (l.splits > 1)
            l.part = take((size_t)p->tiles[1] * l.splits * M * 16 * 4);
        l.bytes = at;
        return l;
    }
    l.part = take((size_t)l.splits * l.pairs * l.columns * 4);
    if (l.kernel == TILE_128_WIDE) {
        const size_t x = (size_t)round_up(M, 128) * p->args[0].blocks, h = (size_t)((l.pairs + 127) / 128 * 128) * p->args[1].blocks;
        l.xsum = take((x > h ? x : h) * (128 / d.group) * 4);
    }
    l.bytes = at;
    return l;
}

template <int TYPE, int GPB, bool ZEROS, int MT, int NT, int WM, int WN, int WK, int STAGES, bool XSUM>
static int launch_experts(const hipq_w4_experts_plan *p, const ExpertsLayout &l, W4Args a, const W4Groups &g, int tiles, int splits, uint8_t *ws, float *part, hipStream_t st)
{
    constexpr int lds = W4Tile<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM>::LDS;
    static thread_local bool done[64] = {};
    const auto kernel = w4_tile_kernel<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM, W4Groups>;
    if (allow_lds((const void *)kernel, lds, p->device, done))
        return 1;
    if (XSUM) {
        a.m_pad = (a.M + 127) / 128 * 128;
        a.xsum = (const float *)(ws + l.xsum);
        const int64_t groups = ((int64_t)a.m_pad * a.blocks * 16 + 255) / 256;
        const dim3 grid((unsigned)(groups < XSUM_ROW ? groups : XSUM_ROW), (unsigned)((groups + XSUM_ROW - 1) / XSUM_ROW));
        w4_xsum_kernel<TYPE, GPB><<<grid, dim3(256), 0, st>>>(a, (float *)(ws + l.xsum), W4Tile<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM>::FACTOR);
        if (launch_status("w4_xsum_kernel"))
            return 1;
    }
    const int tiles_n = (tiles + NT * WN - 1) / (NT * WN);
    kernel<<<dim3((unsigned)((l.blocks * tiles_n + 7) / 8 * 8), splits), dim3(64 * WM * WN * WK), lds, st>>>(a, g, 0, tiles_n, part);
    return launch_status("w4_tile_kernel");
}

template <int TYPE, int GPB, bool ZEROS>
static int launch_experts(const hipq_w4_experts_plan *p, const ExpertsLayout &l, const W4Args &a, const W4Groups &g, int tiles, int splits, uint8_t *ws, float *part, hipStream_t st)
{
    switch (l.kernel) {
    case TILE_16:
        return launch_experts<TYPE, GPB, ZEROS, 1, 2, 1, 4, 2, 5, false>(p, l, a, g, tiles, splits, ws, part, st);
    case TILE_32:
        return launch_experts<TYPE, GPB, ZEROS, 2, 2, 1, 4, 2, 4, false>(p, l, a, g, tiles, splits, ws, part, st);
    case TILE_64:
        return launch_experts<TYPE, GPB, ZEROS, 4, 2, 1, 4, 2, 3, false>(p, l, a, g, tiles, splits, ws, part, st);
    }
    return launch_experts<TYPE, GPB, ZEROS, 4, 4, 2, 4, 1, GPB == 4 && ZEROS ? 2 : 3, true>(p, l, a, g, tiles, splits, ws, part, st);
}

template <int TYPE, int GPB>
static int launch_experts(const hipq_w4_experts_plan *p, const ExpertsLayout &l, const W4Args &a, const W4Groups &g, int tiles, int splits, uint8_t *ws, float *part, hipStream_t st)
{
    return a.zeros ? launch_experts<TYPE, GPB, true>(p, l, a, g, tiles, splits, ws, part, st) : launch_experts<TYPE, GPB, false>(p, l, a, g, tiles, splits, ws, part, st);
}

template <int TYPE>
static int launch_experts(const hipq_w4_experts_plan *p, const ExpertsLayout &l, const W4Args &a, const W4Groups &g, int tiles, int splits, uint8_t *ws, float *part, hipStream_t st)
{
    return p->desc.group == 128  ? launch_experts<TYPE, 1>(p, l, a, g, tiles, splits, ws, part, st)
           : p->desc.group == 64 ? launch_experts<TYPE, 2>(p, l, a, g, tiles, splits, ws, part, st)
                                 : launch_experts<TYPE, 4>(p, l, a, g, tiles, splits, ws, part, st);
}

template <int TYPE, int GPB, bool ZEROS, int ROWS, int WAVES>
static int launch_few_down(const hipq_w4_experts_plan *p, const FewArgs &f, int splits, hipStream_t st)
{
    constexpr int MOST = (WAVES * FEW_TOKENS * 16 + 5 * FEW_PAIRS) * 4;
    const int lds = (WAVES * f.r.M * 16 + 5 * f.r.M * f.r.top) * 4;
    const auto kernel = experts_few_down_kernel<TYPE, GPB, ZEROS, ROWS, WAVES>;
    static thread_local bool done[64] = {};
    if (lds > 65536 && allow_lds((const void *)kernel, MOST, p->device, done))
        return 1;
    kernel<<<dim3(p->tiles[1], splits), dim3(WAVES * 64), lds, st>>>(f);
    return launch_status("experts_few_down_kernel");
}

// a wave for a token, a lane for a pair, blocks that hold all of an expert's rows, and as many scores as a wave keeps in few registers
static bool chooses_itself(const RouteArgs &r) { return r.M <= 4 && r.M * r.top <= 64 && r.block_rows == 4 && r.experts <= 256; }

// 16 waves of a work-group where a CU has one, 8 where it has two: us, one token through one of 16 experts of 5120 x 8192 with 5120 outputs, 320 work-groups, 26 and 24; through 2 of 8
// of 4096 x 14336, 256, 48 and 52
template <int TYPE, int GPB, bool ZEROS, int ROWS>
static int launch_few(const hipq_w4_experts_plan *p, FewArgs f, const uint16_t *x, int64_t x_stride, uint16_t *hidden, float *part, int splits, uint16_t *y, int64_t y_stride, hipStream_t st)
{
    f.a = p->args[0], f.q_bytes = p->groups[0].q_bytes, f.s_bytes = p->groups[0].s_bytes, f.groups = p->tiles[0] / 2;
    f.a.x = x, f.a.x_stride = x_stride, f.a.y = hidden, f.a.y_stride = p->desc.inner;
    const dim3 grid(f.r.most_blocks * f.groups);
    if (ROWS == 4 && chooses_itself(f.r) && f.r.experts <= 64)
        experts_few_up_kernel<TYPE, GPB, ZEROS, 4, 1><<<dim3(grid.x + 1), dim3(256), 0, st>>>(f);
    else if (ROWS == 4 && chooses_itself(f.r))
        experts_few_up_kernel<TYPE, GPB, ZEROS, 4, 4><<<dim3(grid.x + 1), dim3(256), 0, st>>>(f);
    else
        experts_few_up_kernel<TYPE, GPB, ZEROS, ROWS, 0><<<grid, dim3(256), 0, st>>>(f);
    if (launch_status("experts_few_up_kernel"))
        return 1;
    f.a = p->args[1], f.q_bytes = p->groups[1].q_bytes, f.s_bytes = p->groups[1].s_bytes;
    f.a.x = hidden, f.a.x_stride = p->desc.inner, f.a.y = y, f.a.y_stride = y_stride, f.part = part;
    if (p->tiles[1] <= 256 ? launch_few_down<TYPE, GPB, ZEROS, ROWS, 16>(p, f, splits, st) : launch_few_down<TYPE, GPB, ZEROS, ROWS, 8>(p, f, splits, st))
        return 1;
    if (splits == 1)
        return 0;
    const int64_t threads = (int64_t)f.r.M * ((p->desc.N + 3) / 4);
    experts_few_join_kernel<TYPE><<<dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st>>>(part, splits, f.r.M, p->tiles[1] * 16, y, y_stride, p->desc.N);
    return launch_status("experts_few_join_kernel");
}

template <int TYPE, int GPB, bool ZEROS>
static int launch_few(const hipq_w4_experts_plan *p, const FewArgs &f, const uint16_t *x, int64_t x_stride, uint16_t *hidden, float *part, int splits, uint16_t *y, int64_t y_stride, hipStream_t st)
{
    return f.r.block_rows == 4 ? launch_few<TYPE, GPB, ZEROS, 4>(p, f, x, x_stride, hidden, part, splits, y, y_stride, st) : launch_few<TYPE, GPB, ZEROS, 16>(p, f, x, x_stride, hidden, part, splits, y, y_stride, st);
}

template <int TYPE, int GPB>
static int launch_few(const hipq_w4_experts_plan *p, const FewArgs &f, const uint16_t *x, int64_t x_stride, uint16_t *hidden, float *part, int splits, uint16_t *y, int64_t y_stride, hipStream_t st)
{
    return p->args[0].zeros ? launch_few<TYPE, GPB, true>(p, f, x, x_stride, hidden, part, splits, y, y_stride, st) : launch_few<TYPE, GPB, false>(p, f, x, x_stride, hidden, part, splits, y, y_stride, st);
}

template <int TYPE>
static int launch_few(const hipq_w4_experts_plan *p, const RouteArgs &r, const uint16_t *x, int64_t x_stride, uint16_t *hidden, float *part, int splits, uint16_t *y, int64_t y_stride, hipStream_t st)
{
    FewArgs f = {};
    f.r = r;
    return p->desc.group == 128  ? launch_few<TYPE, 1>(p, f, x, x_stride, hidden, part, splits, y, y_stride, st)
           : p->desc.group == 64 ? launch_few<TYPE, 2>(p, f, x, x_stride, hidden, part, splits, y, y_stride, st)
                                 : launch_few<TYPE, 4>(p, f, x, x_stride, hidden, part, splits, y, y_stride, st);
}

template <int EACH>
static int route(const hipq_w4_experts_plan *p, const RouteArgs &r, hipStream_t st)
{
    if (r.M <= CHOOSE_TOKENS) { // 16 waves choose so many tokens' experts in the time of a launch
        const int lds = 16 * r.experts * 4;
        static thread_local bool done[64] = {};
        if (lds + CHOOSE_TOKENS * MOST_TOP * 8 + 128 > 65536 && allow_lds((const void *)experts_route_kernel<EACH>, 16 * MOST_EXPERTS * 4 + 1024, p->device, done))
            return 1;
        experts_route_kernel<EACH><<<dim3(1), dim3(1024), lds, st>>>(r);
        return launch_status("experts_route_kernel");
    }
    experts_choose_kernel<EACH><<<dim3((unsigned)((r.M + 3) / 4)), dim3(256), 0, st>>>(r);
    if (launch_status("experts_choose_kernel"))
        return 1;
    experts_number_kernel<<<dim3(1), dim3(1024), 0, st>>>(r);
    return launch_status("experts_number_kernel");
}

template <int TYPE>
static int run_experts(const hipq_w4_experts_plan *p, const ExpertsLayout &l, RouteArgs r, const void *x, int64_t x_stride, void *y, int64_t y_stride, uint8_t *ws, hipStream_t st)
{
    if (l.kernel <= FEW_16)
        r.placed_share = (float *)(ws + l.share_by_number), r.most_blocks = (int)l.blocks;
    if (!chooses_itself(r) && (r.experts <= 64 ? route<1>(p, r, st) : r.experts <= 256 ? route<4>(p, r, st) : route<16>(p, r, st)))
        return 1;
    if (l.kernel <= FEW_16)
        return launch_few<TYPE>(p, r, (const uint16_t *)x, x_stride, (uint16_t *)(ws + l.hidden), (float *)(ws + l.part), l.splits, (uint16_t *)y, y_stride, st);
    W4Args a = p->args[0];
    W4Groups g = p->groups[0];
    g.block = r.block, g.count = r.count, g.row = r.row;
    a.x = (const uint16_t *)x, a.x_stride = x_stride, a.y = (uint16_t *)(ws + l.hidden), a.y_stride = p->desc.inner;
    // sums of x are those of tokens, results those of pairs
    a.M = r.M;
    if (launch_experts<TYPE>(p, l, a, g, p->tiles[0], 1, ws, nullptr, st))
        return 1;
    a = p->args[1];
    const W4Block *block = g.block;
    g = p->groups[1];
    g.block = block, g.count = r.count, g.row = nullptr;
    a.x = (const uint16_t *)(ws + l.hidden), a.x_stride = p->desc.inner, a.M = (int)l.pairs;
    if (launch_experts<TYPE>(p, l, a, g, p->tiles[1], l.splits, ws, (float *)(ws + l.part), st))
        return 1;
    const int stretches = (p->desc.N + 1023) / 1024;
    experts_join_kernel<TYPE><<<dim3((unsigned)(r.M * stretches)), dim3(256), 0, st>>>(r, (const float *)(ws + l.part), l.splits, l.pairs, l.columns, (uint16_t *)y, y_stride, p->desc.N,
                                                                                       stretches);
    return launch_status("experts_join_kernel");
}

} // namespace hipq

extern "C" int hipq_w4_experts_create(const hipq_w4_experts_desc *d, const uint8_t *gate_up, const void *gate_up_scales, const uint8_t *gate_up_zeros, const uint8_t *down,
                                      const void *down_scales, const uint8_t *down_zeros, void *stream, hipq_w4_experts_plan **out)
{
    clear_error();
    HIPQ_REQUIRE(d && gate_up && gate_up_scales && down && down_scales && out, "experts: a null pointer");
    HIPQ_REQUIRE(is_real16(d->type), "experts: type %d is neither float16 nor bfloat16", d->type);
    HIPQ_REQUIRE(d->group == 32 || d->group == 64 || d->group == 128, "experts: groups of %d (32, 64 and 128 are there)", d->group);
    HIPQ_REQUIRE(d->activation == HIPQ_ACT_SILU || d->activation == HIPQ_ACT_GELU, "experts: activation %d", d->activation);
    HIPQ_REQUIRE(d->scores == HIPQ_SCORES_SOFTMAX || d->scores == HIPQ_SCORES_SIGMOID, "experts: scores %d", d->scores);
    HIPQ_REQUIRE(d->normalize == 0 || d->normalize == 1, "experts: normalize is %d", d->normalize);
    HIPQ_REQUIRE(d->experts >= 1 && d->experts <= MOST_EXPERTS, "experts: %d experts (up to %d are there)", d->experts, MOST_EXPERTS);
    HIPQ_REQUIRE(d->top >= 1 && d->top <= MOST_TOP && d->top <= d->experts, "experts: %d experts of a token (up to %d, and not more than there are)", d->top, MOST_TOP);
    HIPQ_REQUIRE(d->N >= 1 && d->N <= (1 << 20), "experts: %d outputs", d->N);
    HIPQ_REQUIRE(d->K >= 32 && d->K <= (1 << 20) && d->K % 32 == 0, "experts: %d inputs (a multiple of 32 is needed)", d->K);
    HIPQ_REQUIRE(d->inner >= 32 && d->inner <= (1 << 20) && d->inner % 32 == 0, "experts: %d hidden values (a multiple of 32 is needed)", d->inner);
    HIPQ_REQUIRE(!gate_up_zeros == !down_zeros, "experts: zero points for one of the products alone");
    hipq_w4_experts_plan *p = new (std::nothrow) hipq_w4_experts_plan();
    HIPQ_REQUIRE(p, "experts: out of host memory");
    p->desc = *d;
    const int gpb = 128 / d->group;
    size_t q_bytes[2], s_bytes[2], total = 256;
    for (int i = 0; i < 2; i++) {
        W4Args &a = p->args[i];
        a.N = i ? d->N : d->inner, a.K = i ? d->inner : d->K, a.blocks = (a.K + 127) / 128, a.activation = i ? HIPQ_ACT_NONE : d->activation;
        a.zeros = gate_up_zeros != nullptr;
        p->tiles[i] = (a.N + 15) / 16 * (i ? 1 : 2);
        const size_t pieces = (size_t)round_up(p->tiles[i], 16) * a.blocks;
        q_bytes[i] = pieces * 1024, s_bytes[i] = pieces * 16 * gpb * (a.zeros ? 4 : 2);
        total += d->experts * (q_bytes[i] + s_bytes[i]);
    }
    hipError_t e = hipGetDevice(&p->device);
    if (e == hipSuccess)
        e = hipMalloc(&p->memory, total);
    if (e != hipSuccess) {
        delete p;
        return fail("experts: no memory for %zu bytes of weights: %s", total, hipGetErrorString(e));
    }
    uint8_t *at = p->memory + 256;
    int bad = 0;
    for (int i = 0; i < 2; i++) {
        W4Args &a = p->args[i];
        W4Groups &g = p->groups[i];
        g.q_bytes = q_bytes[i], g.s_bytes = s_bytes[i];
        a.q = at, at += d->experts * q_bytes[i];
        a.scales = at, at += d->experts * s_bytes[i];
        a.nothing = (const uint16_t *)p->memory;
        PackArgs k = {};
        k.rows = a.N, k.K = a.K, k.group = d->group, k.groups = (a.K + d->group - 1) / d->group, k.blocks = a.blocks, k.tiles = round_up(p->tiles[i], 16), k.gated = !i;
        const size_t rows = (size_t)a.N * (i ? 1 : 2);
        k.q = i ? down : gate_up, k.scales = (const uint16_t *)(i ? down_scales : gate_up_scales), k.zeros = i ? down_zeros : gate_up_zeros;
        k.to_q = const_cast<uint8_t *>(a.q), k.to_scales = (uint16_t *)const_cast<uint8_t *>(a.scales), k.to_nothing = (u32x4 *)p->memory;
        k.arrays = d->experts, k.q_step = rows * (a.K / 2), k.s_step = rows * k.groups, k.to_q_step = q_bytes[i], k.to_s_step = s_bytes[i];
        bad = bad || w4_pack(k, d->type, (hipStream_t)stream);
    }
    if (!bad && (e = hipStreamSynchronize((hipStream_t)stream)) != hipSuccess)
        bad = fail("experts: laying the weights out failed: %s", hipGetErrorString(e));
    if (bad) {
        (void)hipFree(p->memory);
        delete p;
        return 1;
    }
    *out = p;
    return 0;
}

extern "C" void hipq_w4_experts_destroy(hipq_w4_experts_plan *p)
{
    if (!p)
        return;
    (void)hipFree(p->memory); // waits for what still reads it
    delete p;
}

// byte offsets of 32 bits, numbers of pairs and work-groups of 31
static int experts_fit(const hipq_w4_experts_plan *p, int M)
{
    HIPQ_REQUIRE(p, "experts: a null plan");
    HIPQ_REQUIRE(M >= 0 && M <= (1 << 20), "experts: %d rows", M);
    HIPQ_REQUIRE((int64_t)M * p->desc.top * p->desc.inner < ((int64_t)1 << 31), "experts: %d rows of %d experts, %d hidden values each", M, p->desc.top, p->desc.inner);
    if (M > 0) {
        const ExpertsLayout l = layout_of(p, M);
        const int tiles = p->tiles[0] > p->tiles[1] ? p->tiles[0] : p->tiles[1];
        HIPQ_REQUIRE(l.blocks * ((tiles + 7) / 8) <= (1 << 23) - 8, "experts: %d rows of %d outputs", M, p->desc.N);
        HIPQ_REQUIRE(l.kernel > FEW_16 || l.blocks * (p->tiles[0] / 2) < (1 << 24) - 1, "experts: %d rows of %d experts, %d hidden values each", M, p->desc.top, p->desc.inner);
        HIPQ_REQUIRE((int64_t)M * ((p->desc.N + 1023) / 1024) < (1 << 24), "experts: %d rows of %d outputs", M, p->desc.N);
    }
    return 0;
}

extern "C" const char *hipq_w4_experts_kernel(const hipq_w4_experts_plan *p, int M)
{
    clear_error();
    return experts_fit(p, M) ? "" : SHAPE[layout_of(p, M > 0 ? M : 1).kernel].name;
}

extern "C" size_t hipq_w4_experts_workspace(const hipq_w4_experts_plan *p, int M)
{
    clear_error();
    return experts_fit(p, M) || M == 0 ? 0 : layout_of(p, M).bytes;
}

extern "C" int hipq_w4_experts_run(const hipq_w4_experts_plan *p, const void *x, int64_t x_stride, const void *logits, int logits_type, int64_t logits_stride, void *y,
                                   int64_t y_stride, int M, void *workspace, size_t workspace_bytes, void *stream)
{
    clear_error();
    if (experts_fit(p, M))
        return 1;
    HIPQ_REQUIRE(logits_type == HIPQ_REAL_F32 || is_real16(logits_type), "experts: logits of type %d", logits_type);
    if (M == 0)
        return 0;
    const hipq_w4_experts_desc &d = p->desc;
    HIPQ_REQUIRE(x && logits && y, "experts: a null pointer");
    HIPQ_REQUIRE((uintptr_t)x % 16 == 0 && x_stride % 8 == 0, "experts: rows of x have to start at multiples of 16 bytes");
    const int logit = logits_type == HIPQ_REAL_F32 ? 4 : 2;
    HIPQ_REQUIRE((uintptr_t)y % 2 == 0 && (uintptr_t)logits % logit == 0, "experts: logits or y are not aligned to their type");
    HIPQ_REQUIRE(M == 1 || (x_stride >= d.K && y_stride >= d.N && logits_stride >= d.experts), "experts: rows overlap (strides %lld, %lld and %lld)", (long long)x_stride,
                 (long long)logits_stride, (long long)y_stride);
    HIPQ_REQUIRE(M == 1 || (x_stride < (1 << 30) && (M - 1) * x_stride + d.K < ((int64_t)1 << 31)), "experts: %d rows of x, %lld elements apart", M, (long long)x_stride);
    const ByteRows written = {(int64_t)(uintptr_t)y, M > 1 ? y_stride * 2 : 0, d.N * 2ll, M};
    HIPQ_REQUIRE(!overlap({(int64_t)(uintptr_t)x, M > 1 ? x_stride * 2 : 0, d.K * 2ll, M}, written), "experts: y lies over x");
    HIPQ_REQUIRE(!overlap({(int64_t)(uintptr_t)logits, M > 1 ? logits_stride * logit : 0, (int64_t)d.experts * logit, M}, written), "experts: y lies over the logits");
    const ExpertsLayout l = layout_of(p, M);
    HIPQ_REQUIRE(workspace && workspace_bytes >= l.bytes && (uintptr_t)workspace % 16 == 0, "experts: a workspace of %zu bytes is needed", l.bytes);
    int device;
    HIPQ_CHECK_HIP(hipGetDevice(&device));
    HIPQ_REQUIRE(device == p->device, "experts: the plan is on device %d, the current one is %d", p->device, device);
    uint8_t *ws = (uint8_t *)workspace;
    RouteArgs r = {};
    r.logits = logits, r.stride = M > 1 ? logits_stride : 0, r.type = logits_type, r.M = M, r.experts = d.experts, r.top = d.top;
    r.sigmoid = d.scores == HIPQ_SCORES_SIGMOID, r.normalize = d.normalize, r.block_rows = l.block_rows;
    r.chosen = (int32_t *)(ws + l.chosen), r.share = (float *)(ws + l.share), r.place = (int32_t *)(ws + l.place), r.row = (int32_t *)(ws + l.row);
    r.block = (W4Block *)(ws + l.block), r.count = (int32_t *)(ws + l.count);
    return d.type == HIPQ_REAL_BF16 ? run_experts<HIPQ_REAL_BF16>(p, l, r, x, M > 1 ? x_stride : 0, y, y_stride, ws, (hipStream_t)stream)
                                    : run_experts<HIPQ_REAL_F16>(p, l, r, x, M > 1 ? x_stride : 0, y, y_stride, ws, (hipStream_t)stream);
}
