// A paged cache held to a budget (hipq_kv_evict): of every sequence and head the first, the last and the heaviest tokens stay.  gfx950 only.
//
// First a sequence's and head's tokens are chosen: a work-group looks for the weight with which the budget is used up, digit by digit of the weights' bits (counts
// in LDS, which are integers, so that the order does not matter), and writes the kept ones' places in their order; of equal weights the first tokens stay.  The next
// launch moves them.  In place a token moves to the front or not at all, so that work-groups may each have a stretch of the heads' width
// and go through the tokens in order: what a step reads lies behind all that steps before it have written.  Into other pages the tokens are shared out as well.
//
// us, into other pages: 4 sequences of up to 4096, 2048 stay, 8 + 17, the second 4 TB/s of reads and writes; 2 of up to 131072 in 8 bits, 32000 stay, 7 + 9 + 10 + 12 for
// choosing - launches that read all weights and each part's counts - and 75 for 330 MB, 4.4 TB/s.
#include "real16.h"

namespace hipq {

int check_cache(const hipq_kv_cache *c);

struct EvictArgs {
    hipq_kv_cache cache;
    hipq_kv_evict_desc d;
    uint32_t page_magic; // of page / 16
    int page_shift;
    int parts, kinds;    // moving: work-groups that share the tokens, and those that share a token's row
    // choosing by several work-groups, `chunks` for a sequence and head
    int chunks;
    uint32_t *hist, *above, *found; // [digit][sequence and head][chunk][bin], [digit][..][chunk], [digit][..][2]
};

// 0: a NaN, or in no page; otherwise in the order of the weights
__device__ static __forceinline__ uint32_t rank_of(float w)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f); // -0 is 0
    return w != w ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}

// where a token lies, in rows of the cache; -1: in no page
__device__ static __forceinline__ int64_t row_of(const EvictArgs &a, const int32_t *blocks, int h, int t)
{
    const int t16 = t / 16, block = a.page_magic ? (int)(((uint64_t)(uint32_t)t16 * a.page_magic) >> 32) >> a.page_shift : t16, page = blocks[block];
    return page < 0 || page >= a.cache.pages ? -1 : ((int64_t)page * a.cache.heads + h) * a.cache.page + t - block * a.cache.page;
}

__device__ static __forceinline__ int length(const EvictArgs &a, int b)
{
    return max(min(min(a.d.lens[b], a.d.longest), a.d.blocks_per_sequence * a.cache.page), 0);
}

constexpr int CHOOSERS = 1024, BINS = 2048, DIGITS = 3;
__device__ static __forceinline__ int digit_of(int pass) { return pass < 2 ? 11 : 10; }
__device__ static __forceinline__ int shift_of(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }

// What a sequence and head has to keep: of tokens lo..hi - 1 the `want` heaviest, and all others.
struct Middle {
    int len, lo, hi, want;
    __device__ __forceinline__ Middle(const EvictArgs &a, int b) : len(length(a, b)), lo(a.d.first), hi(len - a.d.recent), want(a.d.budget - a.d.first - a.d.recent) {}
};

// Ranks of four tokens from t on (a multiple of four); what is no middle token has 0 as well.
__device__ static __forceinline__ void ranks_of(const EvictArgs &a, const Middle &m, const int32_t *blocks, int h, int t, uint32_t (&rank)[4])
{
    f32x4 w = {0, 0, 0, 0};
    int64_t at = -1;
    if (t < m.hi && t + 4 > m.lo) {
        at = row_of(a, blocks, h, t);
        if (at >= 0)
            w = *(const f32x4 *)(a.d.weights + at);
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        rank[e] = at >= 0 ? rank_of(w[e]) : 0;
}

struct Found {
    uint32_t bin, left;
};
// The bin in which the `left`-th largest is, and how many of that bin's are among them: thread i brings the numbers of bins BINS - 1 - 2 i and BINS - 2 - 2 i.
__device__ static __forceinline__ Found find_bin(uint32_t n0, uint32_t n1, uint32_t left, uint32_t (&totals)[16], uint32_t (&found)[2])
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t run = n0 + n1;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const uint32_t u = (uint32_t)__shfl_up((int)run, o);
        run += lane >= o ? u : 0;
    }
    if (lane == 63)
        totals[wave] = run;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 16; v++)
        run += v < wave ? totals[v] : 0;
    const uint32_t before = run - n0 - n1;
    if (before < left && left <= before + n0)
        found[0] = BINS - 1 - 2 * tid, found[1] = left - before;
    else if (before + n0 < left && left <= run)
        found[0] = BINS - 2 - 2 * tid, found[1] = left - before - n0;
    __syncthreads();
    const Found f = {found[0], found[1]};
    __syncthreads();
    return f;
}

// a number of each thread's, summed over the work-group
__device__ static __forceinline__ uint32_t sum_of(uint32_t n, uint32_t (&totals)[16])
{
#pragma unroll
    for (int o = 1; o < 64; o *= 2)
        n += (uint32_t)__shfl_xor((int)n, o);
    if ((threadIdx.x & 63) == 0)
        totals[threadIdx.x >> 6] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int v = 0; v < 16; v++)
        n += totals[v];
    __syncthreads();
    return n;
}

// Writes the kept of four tokens a thread: the forced ones, those above the border, and of those at it the first `left`.  above, equal: how many there are before these
// 4096, and behind them afterwards.
__device__ static __forceinline__ void write_kept(const Middle &m, int t, const uint32_t (&rank)[4], uint32_t border, uint32_t left, uint32_t &above, uint32_t &equal,
                                                  int32_t *kept, uint32_t (&totals)[16])
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t is[4], mine = 0; // above in the lower half, equal in the upper one
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const bool middle = t + e >= m.lo && t + e < m.hi;
        is[e] = t + e >= m.len ? 0u : !middle ? 1u : m.want == 0 ? 0u : rank[e] > border ? 1u : rank[e] == border ? 1u << 16 : 0u;
        mine += is[e];
    }
    uint32_t run = mine;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const uint32_t u = (uint32_t)__shfl_up((int)run, o);
        run += lane >= o ? u : 0;
    }
    if (lane == 63)
        totals[wave] = run;
    __syncthreads();
    uint32_t all = 0, over = 0;
#pragma unroll
    for (int v = 0; v < 16; v++) {
        over += v < wave ? totals[v] : 0;
        all += totals[v];
    }
    const uint32_t start = over + run - mine;
    uint32_t g = above + (start & 0xffff), q = equal + (start >> 16);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (is[e] == 1 || (is[e] && q < left))
            kept[g + min(q, left)] = t + e;
        g += is[e] & 0xffff, q += is[e] >> 16;
    }
    above += all & 0xffff, equal += all >> 16;
    __syncthreads();
}

__device__ static __forceinline__ void keep_all(const EvictArgs &a, int len, int32_t *kept)
{
    for (int j = threadIdx.x; j < a.d.budget; j += CHOOSERS)
        kept[j] = j < len ? j : -1;
}

// A work-group for a sequence and head of up to 4096 HELD tokens, whose ranks stay in registers.
template <int HELD>
__global__ __launch_bounds__(CHOOSERS) void kv_choose_kernel(const EvictArgs a)
{
    __shared__ uint32_t bins[BINS], totals[16], found[2];
    const int tid = threadIdx.x, h = blockIdx.x % a.cache.heads, b = blockIdx.x / a.cache.heads;
    int32_t *const kept = a.d.kept + (int64_t)blockIdx.x * a.d.budget;
    const Middle m(a, b);
    if (m.len <= a.d.budget)
        return keep_all(a, m.len, kept);
    const int32_t *const blocks = a.d.blocks + (int64_t)b * a.d.blocks_stride;
    uint32_t rank[HELD][4];
#pragma unroll
    for (int i = 0; i < HELD; i++)
        ranks_of(a, m, blocks, h, (i * CHOOSERS + tid) * 4, rank[i]);
    uint32_t border = 0, left = (uint32_t)m.want;
    for (int pass = 0; pass < DIGITS && m.want > 0; pass++) {
        const int digit = digit_of(pass), shift = shift_of(pass);
        for (int i = tid; i < BINS; i += CHOOSERS)
            bins[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < HELD; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int t = (i * CHOOSERS + tid) * 4 + e;
                if (t >= m.lo && t < m.hi && (pass == 0 || rank[i][e] >> (shift + digit) == border))
                    atomicAdd(&bins[(rank[i][e] >> shift) & ((1u << digit) - 1)], 1u);
            }
        __syncthreads();
        const Found f = find_bin(bins[BINS - 1 - 2 * tid], bins[BINS - 2 - 2 * tid], left, totals, found);
        border = border << digit | f.bin, left = f.left;
    }
    uint32_t above = 0, equal = 0;
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if (i * CHOOSERS * 4 < m.len)
            write_kept(m, (i * CHOOSERS + tid) * 4, rank[i], border, left, above, equal, kept, totals);
}

// The same for longer ones, shared by work-groups of 4096 QUADS tokens each: a launch for each digit, which leaves the part's numbers of every bin, and one that writes.
// Every work-group finds the bins from all parts' numbers itself; what was found of earlier digits, and how many of a part's tokens are above them, the launches pass on.
constexpr int QUADS = 2;
template <int PASS>
__global__ __launch_bounds__(CHOOSERS) void kv_rank_kernel(const EvictArgs a)
{
    __shared__ uint32_t bins[BINS], totals[16], found[2];
    const int tid = threadIdx.x, part = blockIdx.x % a.chunks, bh = blockIdx.x / a.chunks, h = bh % a.cache.heads, b = bh / a.cache.heads;
    const int heads = a.d.sequences * a.cache.heads, from = part * (QUADS * CHOOSERS * 4);
    const Middle m(a, b);
    int32_t *const kept = a.d.kept + (int64_t)bh * a.d.budget;
    if (m.len <= a.d.budget) {
        if (PASS == DIGITS && part == 0)
            keep_all(a, m.len, kept);
        return;
    }
    const int parts = (m.len + QUADS * CHOOSERS * 4 - 1) / (QUADS * CHOOSERS * 4); // of this sequence
    if (part >= parts || (m.want == 0 && PASS < DIGITS))
        return;
    const int32_t *const blocks = a.d.blocks + (int64_t)b * a.d.blocks_stride;
    uint32_t rank[QUADS][4];
#pragma unroll
    for (int i = 0; i < QUADS; i++)
        ranks_of(a, m, blocks, h, from + (i * CHOOSERS + tid) * 4, rank[i]);
    uint32_t border = 0, left = (uint32_t)m.want, before = 0, equal_before = 0;
    if (PASS > 0 && m.want > 0) {
        if (PASS > 1)
            border = a.found[2 * ((PASS - 2) * heads + bh)], left = a.found[2 * ((PASS - 2) * heads + bh) + 1];
        const u32x2 *const hist = (const u32x2 *)(a.hist + ((int64_t)((PASS - 1) * heads + bh) * a.chunks) * BINS) + BINS / 2 - 1 - tid;
        u32x2 all = {0, 0}, ours = {0, 0};
#pragma unroll 8
        for (int p = 0; p < parts; p++) {
            const u32x2 n = hist[(int64_t)p * (BINS / 2)];
            all += n;
            if (PASS == DIGITS && p < part)
                ours += n;
        }
        const Found f = find_bin(all[1], all[0], left, totals, found);
        constexpr int digit = PASS - 1 < 2 ? 11 : 10;
        if (PASS == DIGITS) {
            const uint32_t b1 = BINS - 1 - 2 * tid, b0 = b1 - 1;
            before = sum_of((b1 > f.bin ? ours[1] : 0) + (b0 > f.bin ? ours[0] : 0), totals);
            equal_before = sum_of((b1 == f.bin ? ours[1] : 0) + (b0 == f.bin ? ours[0] : 0), totals);
            for (int p = 0; p < part; p++)
                before += a.above[(int64_t)bh * a.chunks + p] + a.above[(int64_t)(heads + bh) * a.chunks + p];
        }
        border = border << digit | f.bin, left = f.left;
        if (PASS < DIGITS) {
            if (part == 0 && tid == 0)
                a.found[2 * ((PASS - 1) * heads + bh)] = border, a.found[2 * ((PASS - 1) * heads + bh) + 1] = left;
            uint32_t n = 0; // above the border in this digit, at it in those before
            constexpr int shift = PASS == 1 ? 21 : 10;
#pragma unroll
            for (int i = 0; i < QUADS; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int t = from + (i * CHOOSERS + tid) * 4 + e;
                    const uint32_t r = rank[i][e] >> shift;
                    n += t >= m.lo && t < m.hi && r > border && (PASS == 1 || r >> 11 == border >> 11) ? 1 : 0;
                }
            n = sum_of(n, totals);
            if (tid == 0)
                a.above[(int64_t)((PASS - 1) * heads + bh) * a.chunks + part] = n;
        }
    }
    if constexpr (PASS < DIGITS) {
        constexpr int digit = PASS < 2 ? 11 : 10, shift = PASS == 0 ? 21 : PASS == 1 ? 10 : 0;
        for (int i = tid; i < BINS; i += CHOOSERS)
            bins[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < QUADS; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int t = from + (i * CHOOSERS + tid) * 4 + e;
                if (t >= m.lo && t < m.hi && (PASS == 0 || rank[i][e] >> ((shift + digit) & 31) == border))
                    atomicAdd(&bins[(rank[i][e] >> shift) & ((1u << digit) - 1)], 1u);
            }
        __syncthreads();
        ((u32x2 *)(a.hist + ((int64_t)(PASS * heads + bh) * a.chunks + part) * BINS))[tid] = ((const u32x2 *)bins)[tid];
    } else {
        uint32_t above = before + min(from, m.lo) + max(from - m.hi, 0);
#pragma unroll
        for (int i = 0; i < QUADS; i++)
            write_kept(m, from + (i * CHOOSERS + tid) * 4, rank[i], border, left, above, equal_before, kept, totals);
    }
}

constexpr int MOVERS = 256, STEPS = 4; // loads of a thread on their way at once

// A work-group moves a stretch of 128 bytes (or the whole row where it is shorter) of the keys or values of its part of the tokens; the last kind of work-groups what there
// is one number of for a token: scales and weights.
template <int STRETCH>
__global__ __launch_bounds__(MOVERS) void kv_move_kernel(const EvictArgs a)
{
    constexpr int LANES = STRETCH / 16, TOKENS = MOVERS / LANES * STEPS;
    const int kind = blockIdx.x % a.kinds, part = blockIdx.x / a.kinds % a.parts, bh = blockIdx.x / a.kinds / a.parts, h = bh % a.cache.heads, b = bh / a.cache.heads;
    const int32_t *const kept = a.d.kept + (int64_t)bh * a.d.budget, *const blocks = a.d.blocks + (int64_t)b * a.d.blocks_stride, *const to = a.d.to + (int64_t)b * a.d.to_stride;
    const int tid = threadIdx.x, width = a.cache.dim * (a.cache.quantized ? 1 : 2), stretches = width / STRETCH;
    if (kind == 0 && h == 0 && part == 0 && tid == 0)
        a.d.left[b] = min(length(a, b), a.d.budget);
    if (kind < 2 * stretches) {
        uint8_t *const pool = (uint8_t *)(kind < stretches ? a.cache.k : a.cache.v) + kind % stretches * STRETCH + tid % LANES * 16;
        for (int j0 = part * TOKENS; j0 < a.d.budget; j0 += a.parts * TOKENS) {
            u32x4 v[STEPS];
            int64_t target[STEPS];
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                const int j = j0 + s * (TOKENS / STEPS) + tid / LANES, t = j < a.d.budget ? kept[j] : -1;
                const int64_t source = t < 0 ? -1 : row_of(a, blocks, h, t);
                target[s] = t < 0 ? -1 : row_of(a, to, h, j);
                if (source < 0 || source == target[s])
                    target[s] = -1;
                if (target[s] >= 0)
                    v[s] = *(const u32x4 *)(pool + source * width);
            }
            // every load of the step has arrived before anything is written: what is written may be what another thread read
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
#pragma unroll
            for (int s = 0; s < STEPS; s++)
                if (target[s] >= 0)
                    *(u32x4 *)(pool + target[s] * width) = v[s];
        }
        return;
    }
    for (int j0 = part * TOKENS; j0 < a.d.budget; j0 += a.parts * TOKENS)
        for (int i0 = 0; i0 < TOKENS; i0 += MOVERS) {
            const int i = i0 + tid, j = j0 + i, t = i < TOKENS && j < a.d.budget ? kept[j] : -1;
            const int64_t source = t < 0 ? -1 : row_of(a, blocks, h, t);
            int64_t target = t < 0 ? -1 : row_of(a, to, h, j);
            if (source < 0 || source == target)
                target = -1;
            float w = 0, ks = 0, vs = 0;
            if (target >= 0) {
                w = a.d.weights[source];
                if (a.cache.quantized)
                    ks = a.cache.k_scale[source], vs = a.cache.v_scale[source];
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (target >= 0) {
                a.d.weights[target] = w;
                if (a.cache.quantized)
                    a.cache.k_scale[target] = ks, a.cache.v_scale[target] = vs;
            }
        }
}

static int choose(const EvictArgs &a, int64_t longest, hipStream_t st)
{
    const unsigned heads = (unsigned)(a.d.sequences * a.cache.heads);
    if (a.chunks == 1) {
        if (longest <= 4 * CHOOSERS || longest <= a.d.budget)
            kv_choose_kernel<1><<<dim3(heads), dim3(CHOOSERS), 0, st>>>(a);
        else
            kv_choose_kernel<4><<<dim3(heads), dim3(CHOOSERS), 0, st>>>(a);
        return launch_status("kv_choose_kernel");
    }
    kv_rank_kernel<0><<<dim3(heads * a.chunks), dim3(CHOOSERS), 0, st>>>(a);
    if (launch_status("kv_rank_kernel"))
        return 1;
    kv_rank_kernel<1><<<dim3(heads * a.chunks), dim3(CHOOSERS), 0, st>>>(a);
    if (launch_status("kv_rank_kernel"))
        return 1;
    kv_rank_kernel<2><<<dim3(heads * a.chunks), dim3(CHOOSERS), 0, st>>>(a);
    if (launch_status("kv_rank_kernel"))
        return 1;
    kv_rank_kernel<3><<<dim3(heads * a.chunks), dim3(CHOOSERS), 0, st>>>(a);
    return launch_status("kv_rank_kernel");
}

static int width_of(const hipq_kv_cache *c) { return c->dim * (c->quantized ? 1 : 2); }
static int kinds_of(const hipq_kv_cache *c) { return 2 * ((width_of(c) + 127) / 128) + 1; }

template <int STRETCH>
static int launch_move(EvictArgs &a, bool in_place, hipStream_t st)
{
    constexpr int TOKENS = MOVERS / (STRETCH / 16) * STEPS;
    const int64_t heads = (int64_t)a.d.sequences * a.cache.heads;
    a.kinds = kinds_of(&a.cache);
    const int64_t most = (a.d.budget + TOKENS - 1) / TOKENS, want = (4096 + heads * a.kinds - 1) / (heads * a.kinds);
    a.parts = in_place ? 1 : (int)(want < most ? want : most);
    kv_move_kernel<STRETCH><<<dim3((unsigned)(heads * a.kinds * a.parts)), dim3(MOVERS), 0, st>>>(a);
    return launch_status("kv_move_kernel");
}

} // namespace hipq

using namespace hipq;

namespace hipq {

struct EvictShape {
    int chunks; // 1: one work-group chooses
    size_t hist, above, workspace;
};

static EvictShape shape_of(const hipq_kv_cache *c, const hipq_kv_evict_desc *d)
{
    const int64_t tokens = (int64_t)d->blocks_per_sequence * c->page, longest = d->longest < tokens ? d->longest : tokens;
    const size_t heads = (size_t)d->sequences * c->heads;
    EvictShape s = {1, 0, 0, 0};
    if (longest > 4 * 4 * CHOOSERS && longest > d->budget) {
        s.chunks = (int)((longest + QUADS * CHOOSERS * 4 - 1) / (QUADS * CHOOSERS * 4));
        s.hist = heads * DIGITS * s.chunks * BINS * 4, s.above = s.hist + (heads * 2 * s.chunks * 4 + 15) / 16 * 16;
        s.workspace = s.above + heads * 2 * 2 * 4;
    }
    return s;
}

static int check_evict(const hipq_kv_cache *cache, const hipq_kv_evict_desc *d)
{
    if (check_cache(cache))
        return 1;
    HIPQ_REQUIRE(d, "evict: a null pointer");
    HIPQ_REQUIRE(d->sequences >= 0 && d->sequences <= (1 << 20), "evict: %d sequences", d->sequences);
    HIPQ_REQUIRE(d->blocks_per_sequence >= 0 && (int64_t)d->blocks_per_sequence * cache->page <= ((int64_t)1 << 30), "evict: %d blocks of a sequence", d->blocks_per_sequence);
    HIPQ_REQUIRE(d->budget >= 1 && d->budget <= (1 << 30), "evict: a budget of %d tokens", d->budget);
    HIPQ_REQUIRE(d->recent >= 0 && d->first >= 0 && (int64_t)d->recent + d->first <= d->budget, "evict: %d first and %d recent tokens in a budget of %d", d->first, d->recent,
                 d->budget);
    HIPQ_REQUIRE(d->longest >= 0, "evict: the longest sequence has %d tokens", d->longest);
    HIPQ_REQUIRE(d->sequences <= 1 || (d->blocks_stride >= d->blocks_per_sequence && d->to_stride >= d->to_per_sequence), "evict: rows of blocks overlap");
    const bool in_place = d->blocks && d->to == d->blocks;
    HIPQ_REQUIRE(!in_place || (d->to_stride == d->blocks_stride && d->to_per_sequence <= d->blocks_per_sequence) || d->sequences <= 1, "evict: in place the blocks are the same");
    const int64_t tokens = (int64_t)d->blocks_per_sequence * cache->page, longest = d->longest < tokens ? d->longest : tokens, most = d->budget < longest ? d->budget : longest;
    HIPQ_REQUIRE(d->to_per_sequence >= 0 && (int64_t)d->to_per_sequence * cache->page >= most, "evict: %d blocks for %lld tokens that stay", d->to_per_sequence, (long long)most);
    // of 2^32 work-items and more only what is left over would run
    const int64_t heads = (int64_t)d->sequences * cache->heads;
    HIPQ_REQUIRE(heads * shape_of(cache, d).chunks < (1 << 22) && heads * kinds_of(cache) < (1 << 24) - 4096, "evict: %d sequences of %d heads", d->sequences, cache->heads);
    return 0;
}

} // namespace hipq

extern "C" size_t hipq_kv_evict_workspace(const hipq_kv_cache *cache, const hipq_kv_evict_desc *d)
{
    clear_error();
    return check_evict(cache, d) ? 0 : shape_of(cache, d).workspace;
}

extern "C" int hipq_kv_evict(const hipq_kv_cache *cache, const hipq_kv_evict_desc *d, void *workspace, size_t workspace_bytes, void *stream)
{
    clear_error();
    if (check_evict(cache, d))
        return 1;
    if (d->sequences == 0)
        return 0;
    const bool in_place = d->blocks && d->to == d->blocks;
    const int64_t tokens = (int64_t)d->blocks_per_sequence * cache->page, longest = d->longest < tokens ? d->longest : tokens, most = d->budget < longest ? d->budget : longest;
    HIPQ_REQUIRE(d->lens && d->kept && d->left && (most == 0 || (d->weights && d->blocks && d->to)), "evict: a null pointer");
    HIPQ_REQUIRE((uintptr_t)d->weights % 16 == 0, "evict: weights are not at multiples of 16 bytes");
    const EvictShape s = shape_of(cache, d);
    HIPQ_REQUIRE(s.workspace == 0 || (workspace && workspace_bytes >= s.workspace && (uintptr_t)workspace % 16 == 0), "evict: a workspace of %zu bytes is needed", s.workspace);
    EvictArgs a = {};
    a.cache = *cache, a.d = *d;
    if (hipq_div_magic((uint32_t)cache->page / 16, &a.page_magic, &a.page_shift))
        return fail("evict: pages of %d tokens", cache->page);
    a.chunks = s.chunks;
    a.hist = (uint32_t *)workspace, a.above = (uint32_t *)((uint8_t *)workspace + s.hist), a.found = (uint32_t *)((uint8_t *)workspace + s.above);
    if (choose(a, longest, (hipStream_t)stream))
        return 1;
    return width_of(cache) == 64 ? launch_move<64>(a, in_place, (hipStream_t)stream) : launch_move<128>(a, in_place, (hipStream_t)stream);
}
