// A sequence's tokens in a paged cache, as the kernels find and read them that attend over it (kv_attend.hip) or weigh it (kv_weigh.hip).  gfx950 only.
#pragma once

#include "real16.h"

namespace hipq {

int check_cache(const hipq_kv_cache *c);

struct AttendArgs {
    hipq_kv_cache cache;
    hipq_kv_attend_desc d;
    float scale2;            // scale * log2(e)
    int group, splits;       // query heads of a cache head; parts of a sequence
    int row_blocks, rows;    // work-groups and rows (new tokens x group) of a sequence and cache head at most
    uint32_t page_magic;     // of page / 16
    int page_shift;
    float *part_o, *part_ml; // [sequence][head][split][row][dim], [...][row][2]
};

// an address that is the same in all lanes, kept in scalar registers: a lane's part of it is then 32 bits that stay
typedef const uint8_t __attribute__((address_space(1))) *gbytes_t;
__device__ static __forceinline__ gbytes_t uniform(const void *p)
{
    gbytes_t g = (gbytes_t)p;
    asm("" : "+s"(g));
    return g;
}
template <class T>
__device__ static __forceinline__ T at(gbytes_t p, uint32_t offset)
{
    return *(const __attribute__((address_space(1))) T *)(p + offset);
}

constexpr float NONE = -__builtin_inff();

// codes 0..7 of two dwords, as 16-bit floats
template <int TYPE>
__device__ static __forceinline__ u32x4 widen(uint32_t lo, uint32_t hi)
{
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = i < 2 ? lo : hi;
        o[i] = Real16<TYPE>::pack_exact((float)(int8_t)(w >> (16 * (i & 1))), (float)(int8_t)(w >> (16 * (i & 1) + 8)));
    }
    return o;
}

struct Sequence {
    int row0, count, len, old; // first row of q, new tokens, tokens in the cache, those before the new ones
    __device__ __forceinline__ Sequence(const AttendArgs &a, int b)
    {
        const int end = max(min(a.d.starts[b + 1], a.d.tokens), 0); // end - row0 fits whatever is in starts
        row0 = max(a.d.starts[b], 0);
        len = max(min(min(a.d.lens[b], a.d.longest), a.d.blocks_per_sequence * a.cache.page), 0);
        count = max(min(end - row0, a.d.most_new), 0);
        old = len - count;
    }
    // the tokens of a part: an equal share in whole rounds of the four waves
    __device__ __forceinline__ int share(int splits) const { return ((len + splits - 1) / splits + 127) / 128 * 128; }
};

// a tile: two halves of 16 tokens, each in one page
struct Pages {
    int page[2]; // -1: not there
    int place[2];
};
// where the tokens of a sequence lie
struct Paging {
    const int32_t *blocks;
    int halves, page16, page, pages, heads, shift;
    uint32_t magic;
    __device__ __forceinline__ Paging(const AttendArgs &a, const int32_t *blocks_, int len)
        : blocks(blocks_), halves((len + 15) / 16), page16(a.cache.page / 16), page(a.cache.page), pages(a.cache.pages), heads(a.cache.heads), shift(a.page_shift), magic(a.page_magic)
    {
    }
    __device__ __forceinline__ Pages of(int t) const
    {
        Pages p;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int t16 = t / 16 + s;
            const int at = magic ? (int)(((uint64_t)(uint32_t)t16 * magic) >> 32) >> shift : t16;
            // through the scalar cache: behind a barrier the compiler would take a vector load, and wait for all those before it
            const int number = __builtin_amdgcn_readfirstlane(t16 < halves ? ((const int32_t __attribute__((address_space(4))) *)(uintptr_t)blocks)[at] : -1);
            p.page[s] = number >= 0 && number < pages ? number : -1;
            p.place[s] = (t16 - at * page16) * 16;
        }
        return p;
    }
    // of a half's first token in the cache; some page's where there is none
    __device__ __forceinline__ int64_t row(const Pages &p, int s, int h) const { return ((int64_t)max(p.page[s], 0) * heads + h) * page + p.place[s]; }
    // All rows see a whole tile unless it holds a new token, the end, or a page that is not there; from the first such tile on each is looked
    // at token by token.  Which that is, is found beforehand: a loop that ends on what it reads kept two sets of all its registers.
    // The first token from t0 on that is not in a page, at most clear.
    __device__ __forceinline__ int clear_until(int clear, int t0, int lane) const
    {
        for (int at = t0 / page + lane; (int64_t)at * page < clear; at += 64)
            if (blocks[at] < 0 || blocks[at] >= pages)
                clear = min(clear, at * page);
#pragma unroll
        for (int s = 1; s < 64; s *= 2)
            clear = min(clear, __shfl_xor(clear, s));
        return __builtin_amdgcn_readfirstlane(clear);
    }
};

// a bit for each of a lane's 8 tokens of the tile at t: seen by new token `own` of the sequence
__device__ static __forceinline__ uint32_t seen_by(const AttendArgs &a, const Sequence &seq, int own, int t, int j, const Pages &now)
{
    const uint64_t mask = a.d.mask ? a.d.mask[seq.row0 + own] : 0;
    uint32_t sees = 0;
#pragma unroll
    for (int half = 0; half < 2; half++) { // four tokens from `first` on
        const int first = t + half * 16 + j * 4, fresh = first - seq.old;
        const int there = now.page[half] >= 0 ? min(max(seq.len - first, 0), 4) : 0;
        uint32_t bits = (1u << min(max(own + 1 - fresh, 0), 4)) - 1;
        if (a.d.mask)
            bits = fresh >= 0 ? (uint32_t)(mask >> min(fresh, 63)) & (fresh < 64 ? 15u : 0u)
                              : (uint32_t)mask << min(-fresh, 4) | ((1u << min(-fresh, 4)) - 1);
        sees |= (bits & ((1u << there) - 1)) << (4 * half);
    }
    return sees;
}

} // namespace hipq
