// The attention that each token of a paged cache receives (hipq_kv_weigh).  gfx950 only.
//
//   weight[t] (+)= sum over the new tokens' rows r of 2^(s_rt - lse_r),   lse_r = log2 sum_t 2^s_rt,   s = scale log2(e) q_r . k_t
//
// A row's sum is known only when all its scores are, so there are two launches.  The first reads the keys once, as attention does (kv_attend.hip: rows are the columns of
// 16x16x32 products, keys in operand order straight into registers, tiles of 32 tokens in turn for the four waves of a work-group, a sequence split over
// work-groups), and leaves each row's maximum and sum of each part.  The second joins those and adds the rows up, token by token, without atomics: each token
// belongs to one lane.  Where rows are few the first leaves its scores as well, 4 bytes a row and token, less than the keys that the second would have to read again;
// where they are many the second multiplies anew, with a tile's keys in registers and the rows going by.
#include <type_traits>

#include "kv_frag.h"

namespace hipq {

int check_attend(const char *name, const hipq_kv_cache *c, const hipq_kv_attend_desc *d);

struct WeighArgs {
    AttendArgs a; // of the attention whose weights they are; a.splits, a.row_blocks and a.rows are the first launch's
    const float *old;
    float *out;
    float *scores;          // [sequence][head][row][stride], or nullptr
    float *lse;             // [sequence][head][row]: without scores
    int64_t stride;
    int splits, chunk;      // the second launch's work-groups for a sequence and head, and their tokens
};

// Scores of a tile's 8 tokens of a lane and one of its rows, to the base 2; -infinity: not seen.
template <bool QUANT, bool MASKED>
__device__ static __forceinline__ void scaled(const f32x4 (&s)[2], const f32x4 (&ksc)[2], float scale2, uint32_t sees, float (&x)[8])
{
#pragma unroll
    for (int e = 0; e < 8; e++) {
        x[e] = s[e / 4][e % 4] * (QUANT ? ksc[e / 4][e % 4] * scale2 : scale2);
        if (MASKED)
            x[e] = (sees >> e) & 1 ? x[e] : NONE;
    }
}

template <int TYPE, int DIM, bool QUANT>
struct Keys {
    static constexpr int KS = DIM / 32, KW = QUANT ? DIM / 64 : DIM / 32, WIDTH = QUANT ? DIM : 2 * DIM;
    u32x4 x[2][KW];
    f32x4 scale[2];
    __device__ __forceinline__ void load(const AttendArgs &a, const Paging &paging, const Pages &p, int h, int c, int j)
    {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int64_t row = paging.row(p, s, h);
            const gbytes_t k = uniform((const uint8_t *)a.cache.k + row * WIDTH);
#pragma unroll
            for (int i = 0; i < KW; i++)
                x[s][i] = at<u32x4>(k, c * WIDTH + j * 16 + i * 64);
            if (QUANT)
                scale[s] = at<f32x4>(uniform(a.cache.k_scale + row), j * 16);
        }
    }
    __device__ __forceinline__ void operands(u32x4 (&k)[2][KS]) const
    {
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                k[half][ks] = QUANT ? widen<TYPE>(x[half][ks / (QUANT ? 2 : 1)][ks % 2 * 2], x[half][ks / (QUANT ? 2 : 1)][ks % 2 * 2 + 1]) : x[half][ks / (QUANT ? 2 : 1)];
    }
    // of a query, the part that belongs to product ks
    __device__ static __forceinline__ const u32x4 *query(const uint16_t *q, int ks, int j) { return (const u32x4 *)(q + (QUANT ? ks / 2 * 64 + j * 16 + ks % 2 * 8 : ks * 32 + j * 8)); }
};

// Rows' maxima and sums over a part, and with SCORES their scores.  A lane keeps both for its own tokens; they meet at the end.  More than two blocks of 16 rows are
// in LDS, in operand order.
template <int TYPE, int DIM, bool QUANT, int RT, bool SCORES>
__global__ __launch_bounds__(256, 2) void kv_scores_kernel(const WeighArgs w)
{
    using R = Real16<TYPE>;
    using K = Keys<TYPE, DIM, QUANT>;
    constexpr int KS = K::KS;
    constexpr bool Q_LDS = RT > 2;
    const AttendArgs &a = w.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, j = lane >> 4;
    const int eighth = gridDim.x / 8, item = (int)(blockIdx.x % 8) * eighth + (int)(blockIdx.x / 8);
    const int rb = item % a.row_blocks, split = item / a.row_blocks % a.splits, rest = item / a.row_blocks / a.splits;
    const int h = rest % a.cache.heads, b = rest / a.cache.heads;
    if (b >= a.d.sequences)
        return;
    const Sequence seq(a, b);
    const int rows = seq.count * a.group, r0 = rb * 16 * RT;
    if (r0 >= rows)
        return;
    const int share = seq.share(a.splits), t0 = split * share;
    // the last row of the block sees no further than its own token
    const int most = a.d.mask ? seq.len : min(seq.len, seq.old + min(rows - 1, r0 + 16 * RT - 1) / a.group + 1);
    const int t1 = min(t0 + share, most);
    __shared__ float lm[4][RT * 16], ll[4][RT * 16];
    __shared__ u32x4 lq[Q_LDS ? RT * KS * 64 : 1];

    u32x4 q[Q_LDS ? 1 : RT][Q_LDS ? 1 : KS];
    const int live = (min(rows - r0, RT * 16) + 15) / 16; // blocks of rows that are there
    int own[RT]; // the lane's rows (the last one again behind it): new token
    float m[RT], l[RT];
    float *to[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int at = r0 + 16 * rt + c, row = min(at, rows - 1);
        own[rt] = row / a.group;
        const uint16_t *x = (const uint16_t *)a.d.q + (int64_t)(seq.row0 + own[rt]) * a.d.q_token + (int64_t)(h * a.group + row - own[rt] * a.group) * a.d.q_head;
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
            if (!Q_LDS)
                q[Q_LDS ? 0 : rt][Q_LDS ? 0 : ks] = *K::query(x, ks, j);
            else if ((rt * KS + ks) % 4 == wave)
                lq[(rt * KS + ks) * 64 + lane] = *K::query(x, ks, j);
        m[rt] = NONE, l[rt] = 0;
        to[rt] = SCORES && at < rows ? w.scores + (((int64_t)b * a.cache.heads + h) * a.rows + row) * w.stride + j * 4 : nullptr;
    }
    if (Q_LDS)
        __syncthreads();
    const Paging paging(a, a.d.blocks + (int64_t)b * a.d.blocks_stride, seq.len);
    K keys;
    auto tile = [&](int t, const Pages &now, const Pages &next, auto MASKED) __attribute__((always_inline)) {
        constexpr bool masked = decltype(MASKED)::value;
        u32x4 k[2][KS];
        keys.operands(k);
        const f32x4 ksc[2] = {keys.scale[0], keys.scale[1]};
        __builtin_amdgcn_sched_barrier(0);
        keys.load(a, paging, next, h, c, j);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            if (rt > 0 && rt >= live)
                break;
            f32x4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int half = 0; half < 2; half++)
                    s[half] = R::mfma(k[half][ks], Q_LDS ? lq[(rt * KS + ks) * 64 + lane] : q[Q_LDS ? 0 : rt][Q_LDS ? 0 : ks], s[half]);
            float x[8], top = m[rt];
            scaled<QUANT, masked>(s, ksc, a.scale2, masked ? seen_by(a, seq, own[rt], t, j, now) : 0, x);
#pragma unroll
            for (int e = 0; e < 8; e++)
                top = fmaxf(top, x[e]);
            if (__any(top > m[rt] + 8.0f)) { // the reference moves, as in attention
                l[rt] *= top == NONE ? 1.0f : exp2_fast(m[rt] - top);
                m[rt] = top;
            }
            const float ref = m[rt] == NONE ? 0.0f : m[rt];
#pragma unroll
            for (int e = 0; e < 8; e++)
                l[rt] += exp2_fast(x[e] - ref);
            if (SCORES && to[rt])
#pragma unroll
                for (int half = 0; half < 2; half++)
                    *(f32x4 *)(to[rt] + t + 16 * half) = f32x4{x[4 * half], x[4 * half + 1], x[4 * half + 2], x[4 * half + 3]};
        }
    };
    int t = t0 + wave * 32;
    if (t < t1) {
        Pages now = paging.of(t), next = paging.of(t + 128);
        keys.load(a, paging, now, h, c, j);
        const int clear = paging.clear_until(min(min(seq.old, seq.len), t1), t0, lane);
        const int whole = clear - t >= 32 ? (clear - t - 32) / 128 + 1 : 0, last = (t1 - t + 127) / 128;
#pragma unroll 1
        for (int i = 0; i < whole; i++, t += 128) {
            const Pages after = paging.of(t + 256);
            tile(t, now, next, std::false_type{});
            now = next, next = after;
        }
#pragma unroll 1
        for (int i = whole; i < last; i++, t += 128) {
            const Pages after = paging.of(t + 256);
            tile(t, now, next, std::true_type{});
            now = next, next = after;
        }
    }
    // over a row's four lanes, then over the waves
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
#pragma unroll
        for (int o = 16; o < 64; o *= 2) {
            const float om = __shfl_xor(m[rt], o), ol = __shfl_xor(l[rt], o), top = fmaxf(m[rt], om), ref = top == NONE ? 0.0f : top;
            l[rt] = l[rt] * exp2_fast(m[rt] - ref) + ol * exp2_fast(om - ref);
            m[rt] = top;
        }
        if (j == 0)
            lm[wave][rt * 16 + c] = m[rt], ll[wave][rt * 16 + c] = l[rt];
    }
    __syncthreads();
    if (tid < RT * 16 && r0 + tid < rows) {
        float top = NONE, sum = 0;
#pragma unroll
        for (int v = 0; v < 4; v++)
            top = fmaxf(top, lm[v][tid]);
        const float ref = top == NONE ? 0.0f : top;
#pragma unroll
        for (int v = 0; v < 4; v++)
            sum += ll[v][tid] * exp2_fast(lm[v][tid] - ref);
        const int64_t at = (((int64_t)b * a.cache.heads + h) * a.splits + split) * a.rows + r0 + tid;
        a.part_ml[2 * at] = top, a.part_ml[2 * at + 1] = sum;
    }
}

// log2 of a row's sum, by 8 neighbouring lanes of which each takes some of the parts; +infinity for a row that sees nothing, so that its weights are 0
__device__ static __forceinline__ float joined(const AttendArgs &a, int bh, int row, int lane8)
{
    const int64_t at = (int64_t)bh * a.splits * a.rows + row;
    float top = NONE, sum = 0;
    for (int s = lane8; s < a.splits; s += 8) {
        const float m = a.part_ml[2 * (at + (int64_t)s * a.rows)], l = a.part_ml[2 * (at + (int64_t)s * a.rows) + 1], both = fmaxf(top, m), ref = both == NONE ? 0.0f : both;
        sum = sum * exp2_fast(top - ref) + l * exp2_fast(m - ref);
        top = both;
    }
#pragma unroll
    for (int o = 1; o < 8; o *= 2) {
        const float m = __shfl_xor(top, o), l = __shfl_xor(sum, o), both = fmaxf(top, m), ref = both == NONE ? 0.0f : both;
        sum = sum * exp2_fast(top - ref) + l * exp2_fast(m - ref);
        top = both;
    }
    return sum == 0 ? __builtin_inff() : top + log2f(sum);
}

// where a token's weight lies, its four neighbours behind it; -1: in no page
__device__ static __forceinline__ int64_t weight_at(const AttendArgs &a, int b, int h, int t)
{
    const int t16 = t / 16, page16 = a.cache.page / 16, block = a.page_magic ? (int)(((uint64_t)(uint32_t)t16 * a.page_magic) >> 32) >> a.page_shift : t16;
    const int page = a.d.blocks[(int64_t)b * a.d.blocks_stride + block];
    return page < 0 || page >= a.cache.pages ? -1 : ((int64_t)page * a.cache.heads + h) * a.cache.page + t - block * (page16 * 16);
}

// four tokens' sums, into the cache: to those before the new ones what they had is added
__device__ static __forceinline__ void put(const WeighArgs &w, const Sequence &seq, int64_t at, int t, const f32x4 &sum, const f32x4 &old)
{
    if (at < 0 || t >= seq.len)
        return;
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; e++)
        v[e] = t + e < seq.old ? old[e] + sum[e] : sum[e];
    if (t + 4 <= seq.len)
        *(f32x4 *)(w.out + at) = v;
    else
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (t + e < seq.len)
                w.out[at + e] = v[e];
}

// From scores: four tokens a thread, row by row.
__global__ __launch_bounds__(256) void kv_sum_scores_kernel(const WeighArgs w)
{
    const AttendArgs &a = w.a;
    __shared__ float lse[32];
    const int chunk = blockIdx.x % w.splits, bh = blockIdx.x / w.splits, h = bh % a.cache.heads, b = bh / a.cache.heads;
    const Sequence seq(a, b);
    const int rows = seq.count * a.group, t = (chunk * 256 + (int)threadIdx.x) * 4;
    if (chunk * 1024 >= seq.len || rows == 0)
        return;
    const int64_t at = t < seq.len ? weight_at(a, b, h, t) : -1;
    f32x4 old = {0, 0, 0, 0}, sum = {0, 0, 0, 0};
    if (at >= 0 && t < seq.old)
        old = *(const f32x4 *)(w.old + at);
    const int row = threadIdx.x / 8;
    const float own = joined(a, bh, min(row, rows - 1), threadIdx.x % 8);
    if (threadIdx.x % 8 == 0)
        lse[row] = own;
    __syncthreads();
    if (at < 0)
        return;
    const float *from = w.scores + (int64_t)bh * a.rows * w.stride + t;
#pragma unroll 4
    for (int r = 0; r < rows; r++) {
        const f32x4 s = *(const f32x4 *)(from + r * w.stride);
#pragma unroll
        for (int e = 0; e < 4; e++)
            sum[e] += s[e] == NONE ? 0.0f : exp2_fast(s[e] - lse[r]); // what a row does not see it leaves alone, even if it is NaN
    }
    put(w, seq, at, t, sum, old);
}

__global__ __launch_bounds__(256) void kv_lse_kernel(const WeighArgs w)
{
    const AttendArgs &a = w.a;
    const int64_t id = (int64_t)blockIdx.x * 32 + threadIdx.x / 8;
    const int bh = (int)(id / a.rows), row = (int)(id % a.rows);
    if (bh >= a.d.sequences * a.cache.heads)
        return;
    const Sequence seq(a, bh / a.cache.heads);
    const float v = row < seq.count * a.group ? joined(a, bh, row, threadIdx.x % 8) : __builtin_inff();
    if (threadIdx.x % 8 == 0)
        w.lse[id] = v;
}

// From the keys: a wave has 32 tokens', and the rows go by, 16 at a time, from LDS, where BLOCKS such blocks are at once, in operand order, with their sums.
template <int TYPE, int DIM, bool QUANT>
__global__ __launch_bounds__(256, 2) void kv_sum_keys_kernel(const WeighArgs w)
{
    using R = Real16<TYPE>;
    using K = Keys<TYPE, DIM, QUANT>;
    constexpr int KS = K::KS, BLOCKS = DIM == 256 ? 4 : 8;
    const AttendArgs &a = w.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, j = lane >> 4;
    const int eighth = gridDim.x / 8, item = (int)(blockIdx.x % 8) * eighth + (int)(blockIdx.x / 8), chunk = item % w.splits, bh = item / w.splits;
    const int h = bh % a.cache.heads, b = bh / a.cache.heads;
    if (b >= a.d.sequences)
        return;
    const Sequence seq(a, b);
    const int rows = seq.count * a.group, from = chunk * w.chunk, to = min(seq.len, from + w.chunk);
    if (rows == 0 || from >= to)
        return;
    __shared__ u32x4 lq[BLOCKS * KS * 64];
    __shared__ float ls[BLOCKS * 16];
    const Paging paging(a, a.d.blocks + (int64_t)b * a.d.blocks_stride, seq.len);
    auto fetch = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < BLOCKS * KS / 4; i++) {
            const int rb = (i * 4 + wave) / KS, ks = (i * 4 + wave) % KS, row = min(r0 + rb * 16 + c, rows - 1), own = row / a.group;
            const uint16_t *x = (const uint16_t *)a.d.q + (int64_t)(seq.row0 + own) * a.d.q_token + (int64_t)(h * a.group + row - own * a.group) * a.d.q_head;
            if (r0 + rb * 16 < rows)
                lq[(i * 4 + wave) * 64 + lane] = *K::query(x, ks, j);
        }
        if (tid < BLOCKS * 16)
            ls[tid] = r0 + tid < rows ? w.lse[(int64_t)bh * a.rows + r0 + tid] : __builtin_inff();
    };
    K keys;
    Pages now = paging.of(from + wave * 32);
    keys.load(a, paging, now, h, c, j);
    fetch(0);
    __syncthreads();
#pragma unroll 1
    for (int t0 = from; t0 < to; t0 += 128) { // all waves alike, as they share the rows
        const int t = t0 + wave * 32;
        u32x4 k[2][KS];
        keys.operands(k);
        f32x4 ksc[2];
        if (QUANT)
            ksc[0] = keys.scale[0] * a.scale2, ksc[1] = keys.scale[1] * a.scale2;
        const Pages next = paging.of(t + 128);
        __builtin_amdgcn_sched_barrier(0);
        keys.load(a, paging, next, h, c, j);
        __builtin_amdgcn_sched_barrier(0);
        const bool masked = t + 32 > min(seq.old, seq.len) || now.page[0] < 0 || now.page[1] < 0;
        // rows of tokens before the tile's first see none of it
        const int first = a.d.mask || t < seq.old ? 0 : (t - seq.old) * a.group / 16 * 16;
        f32x4 sum[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += BLOCKS * 16) {
            if (rows > BLOCKS * 16 && (r0 > 0 || t0 > from)) {
                __syncthreads();
                fetch(r0);
                __syncthreads();
            }
            const int end = min(BLOCKS, (rows - r0 + 15) / 16);
#pragma unroll 1
            for (int rb = max(first - r0, 0) / 16; rb < end; rb++) {
                f32x4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const u32x4 q = lq[(rb * KS + ks) * 64 + lane];
#pragma unroll
                    for (int half = 0; half < 2; half++)
                        s[half] = R::mfma(k[half][ks], q, s[half]);
                }
                const float lse = ls[rb * 16 + c];
                const uint32_t sees = masked ? seen_by(a, seq, min(r0 + rb * 16 + c, rows - 1) / a.group, t, j, now) : 255u;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float p = exp2_fast(__builtin_fmaf(s[e / 4][e % 4], QUANT ? ksc[e / 4][e % 4] : a.scale2, -lse));
                    sum[e / 4][e % 4] += (sees >> e) & 1 ? p : 0.0f;
                }
            }
        }
#pragma unroll
        for (int o = 1; o < 16; o *= 2)
#pragma unroll
            for (int e = 0; e < 8; e++)
                sum[e / 4][e % 4] += __shfl_xor(sum[e / 4][e % 4], o);
        const int t4 = t + 16 * c + 4 * j;
        if (c < 2 && t4 < seq.len) { // a half each
            const int64_t at = weight_at(a, b, h, t4);
            f32x4 old = {0, 0, 0, 0};
            if (at >= 0 && t4 < seq.old)
                old = *(const f32x4 *)(w.old + at);
            put(w, seq, at, t4, c ? sum[1] : sum[0], old);
        }
        now = next;
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
struct WeighShape {
    int rt, row_blocks, rows, splits, chunks, chunk;
    bool scores;
    int64_t stride;
    size_t part, lse, workspace; // bytes: of the parts; where the rest begins; of all
};

static WeighShape shape_of(const hipq_kv_cache *c, const hipq_kv_attend_desc *d)
{
    WeighShape s = {};
    const int group = d->q_heads / c->heads, width = c->quantized ? c->dim : 2 * c->dim;
    s.rows = d->most_new * group;
    s.rt = s.rows <= 16 ? 1 : s.rows <= 32 ? 2 : s.rows <= 64 ? 4 : 8;
    if (c->dim == 256 && s.rt == 8)
        s.rt = 4; // of LDS without asking
    s.row_blocks = (s.rows + 16 * s.rt - 1) / (16 * s.rt);
    const int64_t longest = d->longest < (int64_t)d->blocks_per_sequence * c->page ? d->longest : (int64_t)d->blocks_per_sequence * c->page;
    const int64_t items = (int64_t)d->sequences * c->heads * s.row_blocks;
    const int64_t want = items ? (1024 + items - 1) / items : 1, most = (longest + 255) / 256;
    s.splits = (int)(want < most ? want : most);
    s.splits = s.splits < 1 ? 1 : s.splits > 256 ? 256 : s.splits;
    s.scores = s.rows <= 32 && s.rows * 8 <= width;
    s.chunk = s.scores ? 1024 : 512;
    s.chunks = (int)((longest + s.chunk - 1) / s.chunk);
    const size_t heads = (size_t)d->sequences * c->heads;
    s.stride = (longest + 31) / 32 * 32;
    s.part = (heads * s.splits * s.rows * 8 + 255) / 256 * 256;
    s.workspace = s.part + (s.scores ? heads * s.rows * s.stride * 4 : heads * s.rows * 4);
    return s;
}

template <int TYPE, int DIM, bool QUANT>
static int launch_weigh(const WeighArgs &w, const WeighShape &s, hipStream_t st)
{
    const int64_t heads = (int64_t)w.a.d.sequences * w.a.cache.heads;
    const dim3 grid((unsigned)((heads * s.row_blocks * s.splits + 7) / 8 * 8));
    if (s.scores && s.rt == 1)
        kv_scores_kernel<TYPE, DIM, QUANT, 1, true><<<grid, dim3(256), 0, st>>>(w);
    else if (s.scores)
        kv_scores_kernel<TYPE, DIM, QUANT, 2, true><<<grid, dim3(256), 0, st>>>(w);
    else if (s.rt == 1)
        kv_scores_kernel<TYPE, DIM, QUANT, 1, false><<<grid, dim3(256), 0, st>>>(w);
    else if (s.rt == 2)
        kv_scores_kernel<TYPE, DIM, QUANT, 2, false><<<grid, dim3(256), 0, st>>>(w);
    else if (s.rt == 4)
        kv_scores_kernel<TYPE, DIM, QUANT, 4, false><<<grid, dim3(256), 0, st>>>(w);
    else if constexpr (DIM < 256)
        kv_scores_kernel<TYPE, DIM, QUANT, 8, false><<<grid, dim3(256), 0, st>>>(w);
    if (launch_status("kv_scores_kernel"))
        return 1;
    if (s.scores) {
        kv_sum_scores_kernel<<<dim3((unsigned)(heads * s.chunks)), dim3(256), 0, st>>>(w);
        return launch_status("kv_sum_scores_kernel");
    }
    kv_lse_kernel<<<dim3((unsigned)((heads * s.rows + 31) / 32)), dim3(256), 0, st>>>(w);
    if (launch_status("kv_lse_kernel"))
        return 1;
    kv_sum_keys_kernel<TYPE, DIM, QUANT><<<dim3((unsigned)((heads * s.chunks + 7) / 8 * 8)), dim3(256), 0, st>>>(w);
    return launch_status("kv_sum_keys_kernel");
}

template <int TYPE, int DIM>
static int launch_weigh(const WeighArgs &w, const WeighShape &s, hipStream_t st)
{
    return w.a.cache.quantized ? launch_weigh<TYPE, DIM, true>(w, s, st) : launch_weigh<TYPE, DIM, false>(w, s, st);
}

template <int TYPE>
static int launch_weigh(const WeighArgs &w, const WeighShape &s, hipStream_t st)
{
    return w.a.cache.dim == 64 ? launch_weigh<TYPE, 64>(w, s, st) : w.a.cache.dim == 128 ? launch_weigh<TYPE, 128>(w, s, st) : launch_weigh<TYPE, 256>(w, s, st);
}

static hipq_kv_attend_desc attend_desc(const hipq_kv_weigh_desc *d)
{
    hipq_kv_attend_desc t = {};
    t.q = d->q, t.q_token = d->q_token, t.q_head = d->q_head, t.starts = d->starts, t.lens = d->lens, t.blocks = d->blocks, t.mask = d->mask;
    t.blocks_stride = d->blocks_stride, t.sequences = d->sequences, t.tokens = d->tokens, t.q_heads = d->q_heads, t.blocks_per_sequence = d->blocks_per_sequence;
    t.most_new = d->most_new, t.longest = d->longest, t.scale = d->scale;
    return t;
}

} // namespace hipq

using namespace hipq;

extern "C" size_t hipq_kv_weigh_workspace(const hipq_kv_cache *cache, const hipq_kv_weigh_desc *desc)
{
    clear_error();
    if (!desc)
        return 0;
    const hipq_kv_attend_desc d = attend_desc(desc);
    return check_attend("weigh", cache, &d) ? 0 : shape_of(cache, &d).workspace;
}

extern "C" int hipq_kv_weigh(const hipq_kv_cache *cache, const hipq_kv_weigh_desc *desc, void *workspace, size_t workspace_bytes, void *stream)
{
    clear_error();
    HIPQ_REQUIRE(desc, "weigh: a null pointer");
    const hipq_kv_attend_desc d = attend_desc(desc);
    if (check_attend("weigh", cache, &d))
        return 1;
    const WeighShape s = shape_of(cache, &d);
    const int64_t heads = (int64_t)d.sequences * cache->heads;
    if (heads * s.rows == 0 || d.tokens == 0 || s.chunks == 0 || cache->pages == 0)
        return 0;
    HIPQ_REQUIRE(d.q && d.starts && d.lens && d.blocks && desc->weights && desc->out, "weigh: a null pointer");
    HIPQ_REQUIRE((uintptr_t)d.q % 16 == 0 && (d.q_token | d.q_head) % 8 == 0, "weigh: heads have to start at multiples of 16 bytes");
    HIPQ_REQUIRE(((uintptr_t)desc->weights | (uintptr_t)desc->out) % 16 == 0, "weigh: weights are not at multiples of 16 bytes");
    HIPQ_REQUIRE(workspace && workspace_bytes >= s.workspace && (uintptr_t)workspace % 16 == 0, "weigh: a workspace of %zu bytes is needed", s.workspace);
    // item numbers are 32 bits, and of 2^32 work-items and more only what is left over would run
    HIPQ_REQUIRE(heads * s.row_blocks * s.splits * 16 * s.rt < ((int64_t)1 << 31) && heads * s.row_blocks * s.splits <= (1 << 24) - 8 && heads * s.chunks <= (1 << 24) - 8
                     && heads * s.rows < ((int64_t)1 << 28),
                 "weigh: %lld work-groups", (long long)(heads * (s.chunks > (int64_t)s.row_blocks * s.splits ? s.chunks : (int64_t)s.row_blocks * s.splits)));
    WeighArgs w = {};
    w.a.cache = *cache, w.a.d = d;
    w.a.scale2 = d.scale * 1.4426950408889634f;
    w.a.group = d.q_heads / cache->heads, w.a.splits = s.splits, w.a.row_blocks = s.row_blocks, w.a.rows = s.rows;
    if (hipq_div_magic((uint32_t)cache->page / 16, &w.a.page_magic, &w.a.page_shift))
        return fail("weigh: pages of %d tokens", cache->page);
    w.old = desc->weights, w.out = desc->out, w.stride = s.stride, w.splits = s.chunks, w.chunk = s.chunk;
    w.a.part_ml = (float *)workspace;
    (s.scores ? w.scores : w.lse) = (float *)((uint8_t *)workspace + s.part);
    return cache->type == HIPQ_REAL_BF16 ? launch_weigh<HIPQ_REAL_BF16>(w, s, (hipStream_t)stream) : launch_weigh<HIPQ_REAL_F16>(w, s, (hipStream_t)stream);
}
