// The attention that each token of a paged cache receives (hipq_kv_weigh).  gfx950 only.
//
//   weight[t] (+)= sum over the new tokens' rows r of 2^(s_rt - lse_r),   lse_r = log2 sum_t 2^s_rt,   s = scale log2(e) q_r . k_t
//
// A row's sum is known only when all its scores are, so there are two launches.  The first reads the keys once, as attention does (kv_attend.hip: rows are the columns of
// 16x16x32 products, keys in operand order straight into registers, tiles of 32 tokens in turn for the four waves of a work-group, a sequence split over
// work-groups), and leaves each row's maximum and sum of each part.  The second joins those and adds the rows up, token by token, without atomics: each token
// belongs to one lane.  Where rows are few the first leaves its scores as well, 4 bytes a row and token, less than the keys that the second would have to read again;
// where they are many the second multiplies anew, with a tile's keys in registers and the rows going by.
//
// us of both launches and what bounds them: one token of 2 sequences of up to 131072 (64 query heads on 8) 105 to 124 + 18, 4.7 TB/s of keys and scores, of the 5.1 of a copy; of 8 of up to 2000
// 10.6 + 5.5, latency: two tiles a wave; 32 tokens of one of up to 30000 in 8 bits 21 + 23, vector instructions (a score's scaling, maximum and power, twice: 2700 a wave with
// 460 of the matrix unit).
#include <type_traits>

#include "kv_frag.h"
#include "overlap.h"

namespace hipq {

int check_attend(const char *name, const hipq_kv_cache *c, const hipq_kv_attend_desc *d);

struct WeighArgs {
    AttendArgs a; // of the attention whose weights they are; a.splits, a.row_blocks and a.rows are the first launch's
    const float *old;
    float *out;
    float *scores;          // [sequence][head][row][stride], or by_page [page][head][row][stride], or nullptr
    float *lse;             // [sequence][head][row]; nullptr: the second launch joins the parts itself
    int64_t stride;
    bool by_page;
    uint32_t group_magic;   // of a.group
    int group_shift;
    int splits, chunk;      // the second launch's work-groups for a sequence and head, and their tokens
};

typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ static __forceinline__ int new_token(const WeighArgs &w, int row) { return w.group_magic ? (int)(((uint64_t)(uint32_t)row * w.group_magic) >> 32) >> w.group_shift : row; }
// a row's query
__device__ static __forceinline__ const uint16_t *query(const WeighArgs &w, const Sequence &seq, int h, int row)
{
    const int own = new_token(w, row);
    return (const uint16_t *)w.a.d.q + (int64_t)(seq.row0 + own) * w.a.d.q_token + (int64_t)(h * w.a.group + row - own * w.a.group) * w.a.d.q_head;
}

// where a row's scores of 16 tokens begin, behind those of the row's number times stride: of the tokens from t on, which lie in a cache row and its place of a page
__device__ static __forceinline__ int64_t scores_at(const WeighArgs &w, int bh, int t, int64_t row, int place)
{
    return w.by_page ? (row - place) * w.a.rows + place : (int64_t)bh * w.a.rows * w.stride + t;
}

constexpr float LOWEST = -0x1.fffffep127f; // a reference where nothing has been seen: finite, so that differences are numbers

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

// Up to 32 rows: their maxima and sums over a part, and with SCORES their scores.  A lane keeps both for its own tokens; they meet at the end.
template <int TYPE, int DIM, bool QUANT, int RT, bool SCORES>
__global__ __launch_bounds__(256, 2) void kv_scores_kernel(const WeighArgs w)
{
    using R = Real16<TYPE>;
    using K = Keys<TYPE, DIM, QUANT>;
    constexpr int KS = K::KS;
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

    u32x4 q[RT][KS];
    float m[RT], l[RT]; // of the lane's rows (the last one again behind it)
    float *to[RT];
    auto row_of = [&](int rt) __attribute__((always_inline)) { return min(r0 + 16 * rt + c, rows - 1); };
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        m[rt] = LOWEST, l[rt] = 0;
        to[rt] = SCORES && r0 + 16 * rt + c < rows ? w.scores + row_of(rt) * w.stride + j * 4 : nullptr;
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
            q[rt][ks] = *K::query(query(w, seq, h, row_of(rt)), ks, j);
    }
    const Paging paging(a, a.d.blocks + (int64_t)b * a.d.blocks_stride, seq.len);
    K keys;
    auto tile = [&](int t, const Pages &now, const Pages &next, auto MASKED) __attribute__((always_inline)) {
        constexpr bool masked = decltype(MASKED)::value;
        u32x4 k[2][KS];
        keys.operands(k);
        f32x4 ksc[2];
        if (QUANT)
            ksc[0] = keys.scale[0] * a.scale2, ksc[1] = keys.scale[1] * a.scale2;
        __builtin_amdgcn_sched_barrier(0);
        keys.load(a, paging, next, h, c, j);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            f32x4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int half = 0; half < 2; half++)
                    s[half] = R::mfma(k[half][ks], q[rt][ks], s[half]);
            // scores to the base 2; of 16-bit keys, where nothing needs them, as they are
            constexpr bool RAW = !QUANT && !SCORES;
            const uint32_t sees = masked ? seen_by(a, seq, new_token(w, row_of(rt)), t, j, now) : 255u;
            float x[8], p[8], left[8]; // left: for the next launch, where NONE is what the row does not see, and nothing else
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[e] = RAW ? s[e / 4][e % 4] : s[e / 4][e % 4] * (QUANT ? ksc[e / 4][e % 4] : a.scale2);
                left[e] = fmaxf(x[e], LOWEST);
                if (masked) {
                    left[e] = (sees >> e) & 1 ? left[e] : NONE;
                    x[e] = (sees >> e) & 1 ? x[e] : NONE;
                }
            }
            // no branch for a reference that stays: blocks of rows would wait for each other's
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            top = fmaxf(RAW ? top * a.scale2 : top, m[rt]);
#pragma unroll
            for (int e = 0; e < 8; e++)
                p[e] = exp2_fast(RAW ? __builtin_fmaf(x[e], a.scale2, -top) : x[e] - top);
            l[rt] = __builtin_fmaf(l[rt], exp2_fast(m[rt] - top), ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])));
            m[rt] = top;
            if (SCORES && to[rt])
#pragma unroll
                for (int half = 0; half < 2; half++)
                    if (!w.by_page || now.page[half] >= 0)
                        *(f32x4 *)(to[rt] + scores_at(w, rest, t + 16 * half, paging.row(now, half, h), now.place[half])) = f32x4{left[4 * half], left[4 * half + 1], left[4 * half + 2], left[4 * half + 3]};
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
            const float om = __shfl_xor(m[rt], o), ol = __shfl_xor(l[rt], o), top = fmaxf(m[rt], om);
            l[rt] = l[rt] * exp2_fast(m[rt] - top) + ol * exp2_fast(om - top);
            m[rt] = top;
        }
        if (j == 0)
            lm[wave][rt * 16 + c] = m[rt], ll[wave][rt * 16 + c] = l[rt];
    }
    __syncthreads();
    if (tid < RT * 16 && r0 + tid < rows) {
        float top = LOWEST, sum = 0;
#pragma unroll
        for (int v = 0; v < 4; v++)
            top = fmaxf(top, lm[v][tid]);
#pragma unroll
        for (int v = 0; v < 4; v++)
            sum += ll[v][tid] * exp2_fast(lm[v][tid] - top);
        ((f32x2 *)a.part_ml)[(((int64_t)b * a.cache.heads + h) * a.rows + r0 + tid) * a.splits + split] = f32x2{top, sum};
    }
}

// More rows: BLOCKS blocks of 16 at once in LDS, in operand order, put there by the load unit; a wave has a tile's keys in registers and the rows go by, two blocks at a
// time, whose maxima and sums wait in LDS meanwhile.  (With those in registers, for which all blocks are unrolled, the code alone took longer to arrive than the work.)
template <int DIM>
constexpr int BLOCKS = DIM == 256 ? 4 : 8;
typedef const uint32_t __attribute__((address_space(1))) *gptr_t;
typedef uint32_t __attribute__((address_space(3))) *lptr_t;

// rows r0 .. of a sequence, the last one again behind it, and waits for this wave's part
template <int TYPE, int DIM, bool QUANT>
__device__ static __forceinline__ void fetch_rows(const WeighArgs &w, const Sequence &seq, int h, int r0, int rows, u32x4 *to, int wave, int c, int j)
{
    using K = Keys<TYPE, DIM, QUANT>;
#pragma unroll 1
    for (int i = wave; i < BLOCKS<DIM> * K::KS; i += 4)
        __builtin_amdgcn_global_load_lds((gptr_t)K::query(query(w, seq, h, min(r0 + i / K::KS * 16 + c, rows - 1)), i % K::KS, j), (lptr_t)(to + i * 64), 16, 0, 0);
}

// two blocks' products with a tile
template <int TYPE, int KS>
__device__ static __forceinline__ void two_blocks(const u32x4 (&k)[2][KS], const u32x4 *q, int lane, f32x4 (&s)[2][2])
{
#pragma unroll
    for (int u = 0; u < 2; u++)
        s[u][0] = s[u][1] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const u32x4 v = q[(u * KS + ks) * 64 + lane];
#pragma unroll
            for (int half = 0; half < 2; half++)
                s[u][half] = Real16<TYPE>::mfma(k[half][ks], v, s[u][half]);
        }
}

template <int TYPE, int DIM, bool QUANT>
__global__ __launch_bounds__(256, 2) void kv_row_sums_kernel(const WeighArgs w)
{
    using K = Keys<TYPE, DIM, QUANT>;
    constexpr int KS = K::KS, ROWS = 16 * BLOCKS<DIM>;
    const AttendArgs &a = w.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, j = lane >> 4;
    const int eighth = gridDim.x / 8, item = (int)(blockIdx.x % 8) * eighth + (int)(blockIdx.x / 8);
    const int rb = item % a.row_blocks, split = item / a.row_blocks % a.splits, bh = item / a.row_blocks / a.splits, h = bh % a.cache.heads, b = bh / a.cache.heads;
    if (b >= a.d.sequences)
        return;
    const Sequence seq(a, b);
    const int rows = seq.count * a.group, r0 = rb * ROWS;
    if (r0 >= rows)
        return;
    const int share = seq.share(a.splits), t0 = split * share;
    const int most = a.d.mask ? seq.len : min(seq.len, seq.old + new_token(w, min(rows, r0 + ROWS) - 1) + 1), t1 = min(t0 + share, most);
    __shared__ u32x4 lq[BLOCKS<DIM> * KS * 64];
    __shared__ f32x2 lml[4][BLOCKS<DIM>][64]; // a wave's own: maxima and sums
    const Paging paging(a, a.d.blocks + (int64_t)b * a.d.blocks_stride, seq.len);
    const int blocks = (min(rows - r0, ROWS) + 15) / 16;
    K keys;
    Pages now = paging.of(t0 + wave * 32);
    fetch_rows<TYPE, DIM, QUANT>(w, seq, h, r0, rows, lq, wave, c, j);
    keys.load(a, paging, now, h, c, j);
#pragma unroll 1
    for (int i = 0; i < BLOCKS<DIM>; i++)
        lml[wave][i][lane] = f32x2{LOWEST, 0};
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll 1
    for (int t = t0 + wave * 32; t < t1; t += 128) {
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
#pragma unroll 1
        for (int i = 0; i < blocks; i += 2) {
            f32x4 s[2][2];
            f32x2 ml[2] = {lml[wave][i][lane], lml[wave][i + 1][lane]};
            two_blocks<TYPE, KS>(k, lq + i * KS * 64, lane, s);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                float x[8], p[8];
#pragma unroll
                for (int e = 0; e < 8; e++)
                    x[e] = QUANT ? s[u][e / 4][e % 4] * ksc[e / 4][e % 4] : s[u][e / 4][e % 4];
                if (masked) {
                    const uint32_t sees = seen_by(a, seq, new_token(w, min(r0 + (i + u) * 16 + c, rows - 1)), t, j, now);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        x[e] = (sees >> e) & 1 ? x[e] : NONE;
                }
                float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
                top = fmaxf(QUANT ? top : top * a.scale2, ml[u][0]);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    p[e] = exp2_fast(QUANT ? x[e] - top : __builtin_fmaf(x[e], a.scale2, -top));
                lml[wave][i + u][lane] = f32x2{top, __builtin_fmaf(ml[u][1], exp2_fast(ml[u][0] - top), ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])))};
            }
        }
        now = next;
    }
    __syncthreads();
    // a row's four lanes of each of the four waves
    if (tid < ROWS && r0 + tid < rows) {
        float top = LOWEST, sum = 0;
#pragma unroll 1
        for (int i = 0; i < 16; i++) {
            const f32x2 ml = lml[i / 4][tid / 16][i % 4 * 16 + tid % 16];
            const float both = fmaxf(top, ml[0]);
            sum = sum * exp2_fast(top - both) + ml[1] * exp2_fast(ml[0] - both);
            top = both;
        }
        ((f32x2 *)a.part_ml)[((int64_t)bh * a.rows + r0 + tid) * a.splits + split] = f32x2{top, sum};
    }
}

// log2 of a row's sum, by LANES neighbouring lanes of which each takes some of the parts; +infinity for a row that sees nothing, so that its weights are 0
template <int LANES>
__device__ static __forceinline__ float joined(const AttendArgs &a, int bh, int row, int lane)
{
    const f32x2 *const part = (const f32x2 *)a.part_ml + ((int64_t)bh * a.rows + row) * a.splits;
    float top = LOWEST, sum = 0;
#pragma unroll 1
    for (int s0 = lane; s0 < a.splits; s0 += 8 * LANES) { // eight on their way at once
        f32x2 ml[8];
        float both = top, more = 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
            ml[i] = part[min(s0 + i * LANES, a.splits - 1)];
#pragma unroll
        for (int i = 0; i < 8; i++)
            both = fmaxf(both, ml[i][0]);
#pragma unroll
        for (int i = 0; i < 8; i++)
            more += s0 + i * LANES < a.splits ? ml[i][1] * exp2_fast(ml[i][0] - both) : 0.0f;
        sum = __builtin_fmaf(sum, exp2_fast(top - both), more);
        top = both;
    }
#pragma unroll
    for (int o = 1; o < LANES; o *= 2) {
        const float m = __shfl_xor(top, o), l = __shfl_xor(sum, o), both = fmaxf(top, m);
        sum = sum * exp2_fast(top - both) + l * exp2_fast(m - both);
        top = both;
    }
    return sum == 0 ? __builtin_inff() : top + log2f(sum);
}

// where a token's weight lies, its four neighbours behind it, and its place in its page; -1: in no page
__device__ static __forceinline__ int64_t weight_at(const AttendArgs &a, int b, int h, int t, int &place)
{
    const int t16 = t / 16, page16 = a.cache.page / 16, block = a.page_magic ? (int)(((uint64_t)(uint32_t)t16 * a.page_magic) >> 32) >> a.page_shift : t16;
    const int page = a.d.blocks[(int64_t)b * a.d.blocks_stride + block];
    place = t - block * (page16 * 16);
    return page < 0 || page >= a.cache.pages ? -1 : ((int64_t)page * a.cache.heads + h) * a.cache.page + place;
}

// the sum over 16 neighbouring lanes, in all of them
__device__ static __forceinline__ float over_rows(float v)
{
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xf, 0xf, true)); // turned round by 8, ...
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x124, 0xf, 0xf, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x122, 0xf, 0xf, true));
    return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x121, 0xf, 0xf, true));
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
    int place = 0;
    const int64_t at = t < seq.len ? weight_at(a, b, h, t, place) : -1;
    f32x4 old = {0, 0, 0, 0}, sum = {0, 0, 0, 0};
    if (at >= 0 && t < seq.old)
        old = *(const f32x4 *)(w.old + at);
    const int row = threadIdx.x / 8;
    const float own = joined<8>(a, bh, min(row, rows - 1), threadIdx.x % 8);
    if (threadIdx.x % 8 == 0)
        lse[row] = own;
    __syncthreads();
    if (at < 0)
        return;
    const float *from = w.scores + scores_at(w, bh, t, at, place);
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
    const float v = row < seq.count * a.group ? joined<8>(a, bh, row, threadIdx.x % 8) : __builtin_inff();
    if (threadIdx.x % 8 == 0)
        w.lse[id] = v;
}

// From the keys: as the first launch of more rows.
template <int TYPE, int DIM, bool QUANT>
__global__ __launch_bounds__(256, 2) void kv_sum_keys_kernel(const WeighArgs w)
{
    using K = Keys<TYPE, DIM, QUANT>;
    constexpr int KS = K::KS, ROWS = 16 * BLOCKS<DIM>;
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
    __shared__ u32x4 lq[BLOCKS<DIM> * KS * 64];
    __shared__ float ls[ROWS];
    const Paging paging(a, a.d.blocks + (int64_t)b * a.d.blocks_stride, seq.len);
    auto fetch = [&](int r0) __attribute__((always_inline)) {
        fetch_rows<TYPE, DIM, QUANT>(w, seq, h, r0, rows, lq, wave, c, j);
        constexpr int LANES = 256 / ROWS;
        const int row = r0 + tid / LANES;
        float lse;
        if (w.lse)
            lse = w.lse[(int64_t)bh * a.rows + min(row, rows - 1)];
        else
            lse = joined<LANES>(a, bh, min(row, rows - 1), tid % LANES);
        ls[tid / LANES] = row < rows ? lse : __builtin_inff();
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    K keys;
    Pages now = paging.of(from + wave * 32);
    keys.load(a, paging, now, h, c, j);
    fetch(0);
#pragma unroll 1
    for (int t0 = from; t0 < to; t0 += 128) { // all waves alike, as they share the rows
        const int t = t0 + wave * 32;
        u32x4 k[2][KS];
        keys.operands(k);
        f32x4 ksc[2];
        if (QUANT)
            ksc[0] = keys.scale[0] * a.scale2, ksc[1] = keys.scale[1] * a.scale2;
        const Pages next = paging.of(t + 128);
        // lanes 0 and 1 of 16 write a half's sums each
        const int t4 = t + 16 * c + 4 * j;
        const bool there = c < 2 && t4 < seq.len && (c ? now.page[1] : now.page[0]) >= 0;
        const int64_t at = (c ? paging.row(now, 1, h) : paging.row(now, 0, h)) + 4 * j;
        f32x4 old = {0, 0, 0, 0};
        if (there && t4 < seq.old)
            old = *(const f32x4 *)(w.old + at);
        __builtin_amdgcn_sched_barrier(0);
        keys.load(a, paging, next, h, c, j);
        __builtin_amdgcn_sched_barrier(0);
        const bool masked = t + 32 > min(seq.old, seq.len) || now.page[0] < 0 || now.page[1] < 0;
        // rows of tokens before the tile's first see none of it
        const int first = a.d.mask || t < seq.old ? 0 : (t - seq.old) * a.group / 32 * 2;
        f32x4 sum[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += ROWS) {
            if (rows > ROWS && (r0 > 0 || t0 > from)) {
                __syncthreads();
                fetch(r0);
            }
            const int end = min(BLOCKS<DIM>, (rows - r0 + 15) / 16);
            // two blocks at once, the second of which may be the last row again with a sum of infinity
#pragma unroll 1
            for (int i = max(first - r0 / 16, 0); i < end; i += 2) {
                f32x4 s[2][2];
                two_blocks<TYPE, KS>(k, lq + i * KS * 64, lane, s);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const float lse = ls[(i + u) * 16 + c];
                    float p[8];
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        p[e] = exp2_fast(__builtin_fmaf(s[u][e / 4][e % 4], QUANT ? ksc[e / 4][e % 4] : a.scale2, -lse));
                    if (masked) {
                        const uint32_t sees = seen_by(a, seq, new_token(w, min(r0 + (i + u) * 16 + c, rows - 1)), t, j, now);
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            p[e] = (sees >> e) & 1 ? p[e] : 0.0f;
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        sum[e / 4][e % 4] += p[e];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
            sum[e / 4][e % 4] = over_rows(sum[e / 4][e % 4]);
        put(w, seq, there ? at : -1, t4, c ? sum[1] : sum[0], old);
        now = next;
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
struct WeighShape {
    int rt, row_blocks, rows, splits, chunks, chunk;
    bool scores, lse, by_page;
    int64_t stride;
    size_t part, workspace; // bytes: of the parts; of all
};

static WeighShape shape_of(const hipq_kv_cache *c, const hipq_kv_attend_desc *d)
{
    WeighShape s = {};
    const int group = d->q_heads / c->heads, width = c->quantized ? c->dim : 2 * c->dim;
    s.rows = d->most_new * group;
    s.rt = s.rows <= 16 ? 1 : s.rows <= 32 ? 2 : c->dim == 256 ? BLOCKS<256> : BLOCKS<128>;
    s.row_blocks = (s.rows + 16 * s.rt - 1) / (16 * s.rt);
    const int64_t longest = d->longest < (int64_t)d->blocks_per_sequence * c->page ? d->longest : (int64_t)d->blocks_per_sequence * c->page;
    const int64_t items = (int64_t)d->sequences * c->heads * s.row_blocks;
    // Two work-groups a CU, with two tiles for a wave at least, four where rows are brought into LDS first: us with 256, 512 and 1024, one token of 2 x up to 131072 157, 142,
    // 142, of one of up to 20000 19, 19, 21, four of 4 x up to 8000 31, 29, 31; 32 of one of up to 30000 in 8 bits 41, with 1024 and two tiles 49
    const int64_t target = 512, least = s.rt <= 2 ? 256 : 512, want = items ? target / items : 1, most = (longest + least - 1) / least;
    s.splits = (int)(want < most ? want : most);
    s.splits = s.splits < 1 ? 1 : s.splits > 256 ? 256 : s.splits;
    s.scores = s.rows <= 32 && s.rows * 8 <= width;
    // once all rows are in LDS at once the second launch joins the parts itself
    s.lse = !s.scores && s.rows > 16 * (c->dim == 256 ? BLOCKS<256> : BLOCKS<128>);
    // from scores, four tokens a thread; from keys, as many tokens of a work-group as fill the chip once with two a CU (us with 512, 768, 1536 of them: 41, 44, 44)
    const int64_t share = (longest * d->sequences * c->heads / 512 + 127) / 128 * 128;
    s.chunk = s.scores ? 1024 : (int)(share < 128 ? 128 : share > 1024 ? 1024 : share);
    s.chunks = (int)((longest + s.chunk - 1) / s.chunk);
    const size_t heads = (size_t)d->sequences * c->heads;
    s.stride = (longest + 31) / 32 * 32;
    // a table may be far wider than the sequences are long: where it has more tokens than the cache, scores lie as the cache's tokens do, in at most half of what the keys take
    s.by_page = s.scores && d->sequences * s.stride > (int64_t)c->pages * c->page;
    if (s.by_page)
        s.stride = c->page;
    s.part = (heads * s.splits * s.rows * 8 + 255) / 256 * 256;
    s.workspace = s.part + (s.scores ? (s.by_page ? (size_t)c->pages * c->heads : heads) * s.rows * s.stride * 4 : s.lse ? heads * s.rows * 4 : 0);
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
    else
        kv_row_sums_kernel<TYPE, DIM, QUANT><<<grid, dim3(256), 0, st>>>(w);
    if (launch_status("kv_scores_kernel"))
        return 1;
    if (s.scores) {
        kv_sum_scores_kernel<<<dim3((unsigned)(heads * s.chunks)), dim3(256), 0, st>>>(w);
        return launch_status("kv_sum_scores_kernel");
    }
    if (w.lse) {
        kv_lse_kernel<<<dim3((unsigned)((heads * s.rows + 31) / 32)), dim3(256), 0, st>>>(w);
        if (launch_status("kv_lse_kernel"))
            return 1;
    }
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

static int check_weigh(const hipq_kv_cache *cache, const hipq_kv_attend_desc &d, WeighShape *shape)
{
    if (check_attend("weigh", cache, &d))
        return 1;
    const WeighShape s = shape_of(cache, &d);
    const int64_t heads = (int64_t)d.sequences * cache->heads;
    // item numbers are 32 bits, and of 2^32 work-items and more only what is left over would run
    HIPQ_REQUIRE(heads * s.row_blocks * s.splits * 16 * s.rt < ((int64_t)1 << 31) && heads * s.row_blocks * s.splits <= (1 << 24) - 8 && heads * s.chunks <= (1 << 24) - 8
                     && heads * s.rows < ((int64_t)1 << 28),
                 "weigh: %lld work-groups", (long long)(heads * (s.chunks > (int64_t)s.row_blocks * s.splits ? s.chunks : (int64_t)s.row_blocks * s.splits)));
    *shape = s;
    return 0;
}

} // namespace hipq

using namespace hipq;

extern "C" size_t hipq_kv_weigh_workspace(const hipq_kv_cache *cache, const hipq_kv_weigh_desc *desc)
{
    clear_error();
    if (!desc)
        return 0;
    WeighShape s;
    return check_weigh(cache, attend_desc(desc), &s) ? 0 : s.workspace;
}

extern "C" int hipq_kv_weigh(const hipq_kv_cache *cache, const hipq_kv_weigh_desc *desc, void *workspace, size_t workspace_bytes, void *stream)
{
    clear_error();
    HIPQ_REQUIRE(desc, "weigh: a null pointer");
    const hipq_kv_attend_desc d = attend_desc(desc);
    WeighShape s;
    if (check_weigh(cache, d, &s))
        return 1;
    if (d.sequences == 0 || s.rows == 0 || d.tokens == 0 || s.chunks == 0 || cache->pages == 0)
        return 0;
    HIPQ_REQUIRE(d.q && d.starts && d.lens && d.blocks && desc->weights && desc->out, "weigh: a null pointer");
    HIPQ_REQUIRE((uintptr_t)d.q % 16 == 0 && (d.q_token | d.q_head) % 8 == 0, "weigh: heads have to start at multiples of 16 bytes");
    HIPQ_REQUIRE(((uintptr_t)desc->weights | (uintptr_t)desc->out) % 16 == 0, "weigh: weights are not at multiples of 16 bytes");
    const int64_t pool = (int64_t)cache->pages * cache->heads * cache->page * 4;
    HIPQ_REQUIRE(desc->out == desc->weights || !overlap({(int64_t)(uintptr_t)desc->weights, 0, pool, 1}, {(int64_t)(uintptr_t)desc->out, 0, pool, 1}), "weigh: out lies over the weights");
    HIPQ_REQUIRE(workspace && workspace_bytes >= s.workspace && (uintptr_t)workspace % 16 == 0, "weigh: a workspace of %zu bytes is needed", s.workspace);
    WeighArgs w = {};
    w.a.cache = *cache, w.a.d = d;
    w.a.scale2 = d.scale * 1.4426950408889634f;
    w.a.group = d.q_heads / cache->heads, w.a.splits = s.splits, w.a.row_blocks = s.row_blocks, w.a.rows = s.rows;
    if (hipq_div_magic((uint32_t)cache->page / 16, &w.a.page_magic, &w.a.page_shift))
        return fail("weigh: pages of %d tokens", cache->page);
    if (hipq_div_magic((uint32_t)w.a.group, &w.group_magic, &w.group_shift))
        return fail("weigh: %d query heads on %d heads of the cache", d.q_heads, cache->heads);
    w.old = desc->weights, w.out = desc->out, w.stride = s.stride, w.by_page = s.by_page, w.splits = s.chunks, w.chunk = s.chunk;
    w.a.part_ml = (float *)workspace;
    if (s.scores)
        w.scores = (float *)((uint8_t *)workspace + s.part);
    if (s.lse)
        w.lse = (float *)((uint8_t *)workspace + s.part);
    return cache->type == HIPQ_REAL_BF16 ? launch_weigh<HIPQ_REAL_BF16>(w, s, (hipStream_t)stream) : launch_weigh<HIPQ_REAL_F16>(w, s, (hipStream_t)stream);
}
