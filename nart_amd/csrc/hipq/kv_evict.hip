// A paged cache held to a budget (hipq_kv_evict): of every sequence and head the first, the last and the heaviest tokens stay.  gfx950 only.
//
// Two launches.  The first finds a sequence's and head's tokens: a work-group looks for the weight with which the budget is used up, digit by digit of the
// weights' bits (counts in LDS, which are integers, so that the order does not matter), and writes the kept ones' places in their order; of equal weights the first
// tokens stay.  The second moves them.  In place a token moves to the front or not at all, so that work-groups may each have a stretch of the heads' width
// and go through the tokens in order: what a step reads lies behind all that steps before it have written.  Into other pages the tokens are shared out as well.
#include "real16.h"

namespace hipq {

int check_cache(const hipq_kv_cache *c);

struct EvictArgs {
    hipq_kv_cache cache;
    hipq_kv_evict_desc d;
    uint32_t page_magic; // of page / 16
    int page_shift;
    int parts, kinds;    // of the second launch: work-groups that share the tokens, and those that share a token's row
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

constexpr int CHOOSERS = 1024, BINS = 2048;

__global__ __launch_bounds__(CHOOSERS) void kv_choose_kernel(const EvictArgs a)
{
    __shared__ uint32_t bins[BINS], totals[16], found[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = blockIdx.x % a.cache.heads, b = blockIdx.x / a.cache.heads, len = length(a, b), budget = a.d.budget;
    int32_t *const kept = a.d.kept + (int64_t)blockIdx.x * budget;
    if (len <= budget) {
        for (int j = tid; j < budget; j += CHOOSERS)
            kept[j] = j < len ? j : -1;
        return;
    }
    const int32_t *const blocks = a.d.blocks + (int64_t)b * a.d.blocks_stride;
    const int lo = a.d.first, hi = len - a.d.recent, want = budget - a.d.first - a.d.recent; // of tokens lo .. hi - 1, which are more than that
    auto four = [&](int t, uint32_t (&rank)[4]) __attribute__((always_inline)) { // of tokens t..t + 3
        const int64_t at = row_of(a, blocks, h, t);
        const f32x4 w = at < 0 ? f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")} : *(const f32x4 *)(a.d.weights + at);
#pragma unroll
        for (int e = 0; e < 4; e++)
            rank[e] = rank_of(w[e]);
    };
    // the rank of the last one that stays, from its highest digit on, and how many of those with that rank stay
    uint32_t border = 0, left = (uint32_t)want;
    int known = 0; // bits
    while (known < 32 && left > 0) {
        const int digit = known < 22 ? 11 : 10, shift = 32 - known - digit;
        for (int i = tid; i < BINS; i += CHOOSERS)
            bins[i] = 0;
        __syncthreads();
        for (int t = (lo & ~3) + tid * 4; t < hi; t += CHOOSERS * 4) {
            uint32_t rank[4];
            four(t, rank);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (t + e >= lo && t + e < hi && (known == 0 || (rank[e] >> (32 - known)) == border))
                    atomicAdd(&bins[(rank[e] >> shift) & ((1u << digit) - 1)], 1u);
        }
        __syncthreads();
        // the bin in which the number wanted is reached, from the highest on: thread i has bins 2 i and 2 i + 1 from above
        const uint32_t n0 = bins[BINS - 1 - 2 * tid], n1 = bins[BINS - 2 - 2 * tid];
        uint32_t run = n0 + n1;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const uint32_t u = (uint32_t)__shfl_up((int)run, o);
            run += lane >= o ? u : 0;
        }
        if (lane == 63)
            totals[wave] = run;
        __syncthreads();
        for (int v = 0; v < wave; v++)
            run += totals[v];
        const uint32_t before = run - n0 - n1;
        if (before < left && left <= before + n0)
            found[0] = BINS - 1 - 2 * tid, found[1] = left - before;
        else if (before + n0 < left && left <= run)
            found[0] = BINS - 2 - 2 * tid, found[1] = left - before - n0;
        __syncthreads();
        border = border << digit | found[0];
        left = found[1];
        known += digit;
        __syncthreads();
    }
    // kept: the forced ones, those above the border, and the first `left` of those at it
    const bool none = want == 0;
    uint32_t above = 0, equal = 0; // so far, of all waves
    for (int t0 = 0; t0 < len; t0 += CHOOSERS * 4) {
        const int t = t0 + tid * 4;
        uint32_t rank[4] = {0, 0, 0, 0}, mine = 0; // above in the lower half, equal in the upper one
        if (t < hi && t + 4 > lo)
            four(t, rank);
        uint32_t is[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool middle = t + e >= lo && t + e < hi;
            is[e] = t + e >= len ? 0u : !middle || (!none && rank[e] > border) ? 1u : !none && rank[e] == border ? 1u << 16 : 0u;
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

template <int STRETCH>
static int launch_move(EvictArgs &a, bool in_place, hipStream_t st)
{
    constexpr int TOKENS = MOVERS / (STRETCH / 16) * STEPS;
    const int64_t heads = (int64_t)a.d.sequences * a.cache.heads;
    a.kinds = 2 * (a.cache.dim * (a.cache.quantized ? 1 : 2) / STRETCH) + 1;
    const int64_t most = (a.d.budget + TOKENS - 1) / TOKENS, want = (4096 + heads * a.kinds - 1) / (heads * a.kinds);
    a.parts = in_place ? 1 : (int)(want < most ? want : most);
    HIPQ_REQUIRE(heads * a.kinds * a.parts < (1 << 24), "evict: %d sequences of %d heads", a.d.sequences, a.cache.heads);
    kv_move_kernel<STRETCH><<<dim3((unsigned)(heads * a.kinds * a.parts)), dim3(MOVERS), 0, st>>>(a);
    return launch_status("kv_move_kernel");
}

} // namespace hipq

using namespace hipq;

extern "C" int hipq_kv_evict(const hipq_kv_cache *cache, const hipq_kv_evict_desc *d, void *stream)
{
    clear_error();
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
    const bool in_place = d->to == d->blocks;
    HIPQ_REQUIRE(!in_place || (d->to_stride == d->blocks_stride && d->to_per_sequence <= d->blocks_per_sequence) || d->sequences <= 1, "evict: in place the blocks are the same");
    const int64_t tokens = (int64_t)d->blocks_per_sequence * cache->page, longest = d->longest < tokens ? d->longest : tokens, most = d->budget < longest ? d->budget : longest;
    HIPQ_REQUIRE(d->to_per_sequence >= 0 && (int64_t)d->to_per_sequence * cache->page >= most, "evict: %d blocks for %lld tokens that stay", d->to_per_sequence, (long long)most);
    if (d->sequences == 0)
        return 0;
    HIPQ_REQUIRE(d->lens && d->kept && d->left && (most == 0 || (d->weights && d->blocks && d->to)), "evict: a null pointer");
    HIPQ_REQUIRE((uintptr_t)d->weights % 16 == 0, "evict: weights are not at multiples of 16 bytes");
    const int64_t heads = (int64_t)d->sequences * cache->heads;
    // of 2^32 work-items and more only what is left over would run
    HIPQ_REQUIRE(heads < (1 << 22), "evict: %d sequences of %d heads", d->sequences, cache->heads);
    EvictArgs a = {};
    a.cache = *cache, a.d = *d;
    if (hipq_div_magic((uint32_t)cache->page / 16, &a.page_magic, &a.page_shift))
        return fail("evict: pages of %d tokens", cache->page);
    kv_choose_kernel<<<dim3((unsigned)heads), dim3(CHOOSERS), 0, (hipStream_t)stream>>>(a);
    if (launch_status("kv_choose_kernel"))
        return 1;
    return cache->dim * (cache->quantized ? 1 : 2) == 64 ? launch_move<64>(a, in_place, (hipStream_t)stream) : launch_move<128>(a, in_place, (hipStream_t)stream);
}
