// New tokens of a paged cache (hipq_kv_append): norms of queries and keys, the rotation, and the write in one pass.  gfx950 only.
//
// A pass over memory: every head is read once and written once, all arithmetic in float32, rounded once.  DIM / 8 neighbouring lanes have a
// head, 16 bytes each.  A lane reads its partners of the rotation (rot / 2 elements away) itself, from lines that its neighbours
// read in the same instruction, instead of asking them for eight values through LDS.  The cosines and sines of a token are as many bytes
// as four of its heads: lanes take up to 8 heads of one token in turn and keep them, the norm's weights multiplied in, the next head on
// its way.  With a division for each 8-bit code and weights read anew for each head its arithmetic took longer than its bytes: 5000 tokens of
// 40 + 8 + 8 heads of 128, fp16 into int8, 50 us; now 35.5 (133 MB at 3.7 TB/s; 2, 4 or 28 heads a lane: 44.5, 36.7, 40.2).
// 32 tokens of 32 + 8 + 8 heads: 3.3 us.
#include "real16.h"

namespace hipq {

struct AppendArgs {
    hipq_kv_cache cache;
    hipq_kv_append_desc d;
    int blocks, per_chunk; // work-groups that all tokens take for the same heads, and how many heads those are
    uint32_t page_magic;
    int page_shift;
};

// codes of a lane's eight values: v / scale, rounded to nearest even
__device__ static __forceinline__ u32x2 codes_of(const float (&v)[8], float scale)
{
    u32x2 w = {0, 0};
    if (scale > 0x1p-100f && scale < __builtin_inff()) {
        // the quotient from one division a head: v r is 1.5 units in the last place off at most, after one correction by what it leaves
        // less than one, and from there a second one rounds correctly (Markstein), as r is rounded.  Adding 1.5 * 2^23 rounds it, and
        // leaves the code in the low byte.  (A division an element was a third of all instructions.)
        const float r = 1.0f / scale;
        uint32_t c[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float q = v[e] * r;
            q = __builtin_fmaf(__builtin_fmaf(-q, scale, v[e]), r, q);
            q = __builtin_fmaf(__builtin_fmaf(-q, scale, v[e]), r, q);
            c[e] = __builtin_bit_cast(uint32_t, q + 12582912.0f);
        }
#pragma unroll
        for (int e = 0; e < 8; e += 4)
            w[e / 4] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[e + 3], c[e + 2], 0x0c0c0400), __builtin_amdgcn_perm(c[e + 1], c[e], 0x0c0c0400), 0x05040100);
    } else
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // a subnormal scale that was rounded down makes more than 127 of the largest
            const float code = scale > 0 ? fminf(fmaxf(rintf(v[e] / scale), -127.0f), 127.0f) : 0.0f;
            w[e / 4] |= ((uint32_t)(int)code & 255) << (8 * (e % 4));
        }
    return w;
}

// QUANT: into an int8 cache
template <int TYPE, int DIM, bool QUANT>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs a)
{
    using R = Real16<TYPE>;
    constexpr int LANES = DIM / 8;
    const hipq_kv_append_desc &d = a.d;
    const int chunk = blockIdx.x / a.blocks, token = (int)((blockIdx.x - chunk * a.blocks) * 256 + threadIdx.x) / LANES;
    const int i0 = (threadIdx.x % LANES) * 8;
    if (token >= d.tokens)
        return;
    const int heads = a.cache.heads;
    const int slot = d.slots[token], pos = d.positions[token];
    const int from = chunk * a.per_chunk, to = min(d.q_heads + 2 * heads, from + a.per_chunk);

    // partners of the lane's elements, and the sign of the sine: side by side the lane has both; otherwise rot / 2 in front or behind
    const int half = d.rot / 2;
    const bool turned = i0 < d.rot, first = i0 < half;
    const int partner = d.interleaved || !turned ? i0 : first ? i0 + half : i0 - half;
    if (slot < 0 || slot >= a.cache.pages * a.cache.page || (d.rot && (pos < 0 || pos >= d.table_rows)))
        return;
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
        cs[e] = 1, sn[e] = 0;
    if (turned && from < d.q_heads + heads) {
        const float *row = d.table + (int64_t)pos * d.rot + (d.interleaved ? i0 / 2 : first ? i0 : i0 - half);
        if (d.interleaved) {
            const f32x4 c = *(const f32x4 *)row, s = *(const f32x4 *)(row + half);
#pragma unroll
            for (int e = 0; e < 8; e++)
                cs[e] = c[e / 2], sn[e] = e & 1 ? s[e / 2] : -s[e / 2];
        } else {
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const f32x4 c = *(const f32x4 *)(row + 4 * p), s = *(const f32x4 *)(row + half + 4 * p);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    cs[4 * p + e] = c[e], sn[4 * p + e] = first ? -s[e] : s[e];
            }
        }
    }
    const int page = (int)(((uint64_t)(uint32_t)slot * a.page_magic) >> 32) >> a.page_shift;
    const int place = slot - page * a.cache.page;
    auto widen = [](const u32x4 &w, float (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] = e & 1 ? R::high(w[e / 2]) : R::low(w[e / 2]);
    };

#pragma unroll 1
    for (int what = 0; what < 3; what++) { // queries, keys, values: those of this work item
        const int before = what == 0 ? 0 : what == 1 ? d.q_heads : d.q_heads + heads;
        const int begin = max(from - before, 0), end = min(to - before, what == 0 ? d.q_heads : heads);
        if (begin >= end)
            continue;
        const uint16_t *x = what == 0 ? (const uint16_t *)d.q + token * d.q_token
                            : what == 1 ? (const uint16_t *)d.k + token * d.k_token
                                        : (const uint16_t *)d.v + token * d.v_token;
        const int64_t step = what == 0 ? d.q_head : what == 1 ? d.k_head : d.v_head;
        x += begin * step;
        u32x4 own = *(const u32x4 *)(x + i0), other = own;
        const bool apart = what < 2 && d.rot && !d.interleaved;
        if (apart)
            other = *(const u32x4 *)(x + partner);
        // the head's weights go into the cosines and sines
        const uint16_t *norm = (const uint16_t *)(what == 0 ? d.q_norm : what == 1 ? d.k_norm : nullptr);
        float c[8], s[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
            c[e] = cs[e], s[e] = sn[e];
        if (norm) {
            float w[8], wo[8];
            widen(*(const u32x4 *)(norm + i0), w);
            widen(*(const u32x4 *)(norm + partner), wo);
#pragma unroll
            for (int e = 0; e < 8; e++)
                c[e] *= w[e], s[e] *= d.interleaved ? w[e ^ 1] : wo[e];
        }
#pragma unroll 1
        for (int h = begin; h < end; h++) {
            float v[8];
            widen(own, v);
            if (what < 2) {
                float o[8];
                if (apart)
                    widen(other, o);
                else
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        o[e] = v[e ^ 1];
                x += step;
                if (h + 1 < end) { // the next head on its way
                    own = *(const u32x4 *)(x + i0);
                    if (apart)
                        other = *(const u32x4 *)(x + partner);
                }
                if (norm) {
                    float sum = 0;
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        sum = __builtin_fmaf(v[e], v[e], sum);
#pragma unroll
                    for (int l = 1; l < LANES; l *= 2)
                        sum += __shfl_xor(sum, l);
                    const float r = 1.0f / sqrtf(sum * (1.0f / DIM) + d.eps);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        v[e] *= r, o[e] *= r;
                }
#pragma unroll
                for (int e = 0; e < 8; e++)
                    v[e] *= c[e];
                if (turned)
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        v[e] = __builtin_fmaf(o[e], s[e], v[e]);
            } else {
                x += step;
                if (h + 1 < end)
                    own = *(const u32x4 *)(x + i0);
            }
            const int64_t row = ((int64_t)page * heads + h) * a.cache.page + place;
            if (what == 0 || !QUANT) {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    w[e] = R::pack(v[2 * e], v[2 * e + 1]);
                uint16_t *y = what == 0 ? (uint16_t *)d.q_out + token * d.out_token + h * d.out_head : (uint16_t *)(what == 1 ? a.cache.k : a.cache.v) + row * DIM;
                *(u32x4 *)(y + i0) = w;
            } else {
                float most = 0;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    most = fmaxf(most, fabsf(v[e]));
#pragma unroll
                for (int l = 1; l < LANES; l *= 2)
                    most = fmaxf(most, __shfl_xor(most, l));
                const float scale = most / 127.0f;
                *(u32x2 *)((uint8_t *)(what == 1 ? a.cache.k : a.cache.v) + row * DIM + i0) = codes_of(v, scale);
                if (i0 == 0)
                    (what == 1 ? a.cache.k_scale : a.cache.v_scale)[row] = scale;
            }
        }
    }
}

int check_cache(const hipq_kv_cache *c)
{
    HIPQ_REQUIRE(c, "cache: a null pointer");
    HIPQ_REQUIRE(is_real16(c->type), "cache: type %d is neither float16 nor bfloat16", c->type);
    HIPQ_REQUIRE(c->quantized == 0 || c->quantized == 1, "cache: quantized is %d", c->quantized);
    HIPQ_REQUIRE(c->dim == 64 || c->dim == 128 || c->dim == 256, "cache: heads of %d (64, 128 and 256 are there)", c->dim);
    HIPQ_REQUIRE(c->page >= 16 && c->page <= 65536 && c->page % 16 == 0, "cache: pages of %d tokens (a multiple of 16 is needed)", c->page);
    HIPQ_REQUIRE(c->heads >= 1 && c->heads <= 4096, "cache: %d heads", c->heads);
    HIPQ_REQUIRE(c->pages >= 0 && (int64_t)c->pages * c->page < ((int64_t)1 << 31), "cache: %d pages of %d tokens", c->pages, c->page);
    HIPQ_REQUIRE(c->pages == 0 || (c->k && c->v && (!c->quantized || (c->k_scale && c->v_scale))), "cache: a null pointer");
    HIPQ_REQUIRE(((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_scale | (uintptr_t)c->v_scale) % 16 == 0, "cache: not at multiples of 16 bytes");
    return 0;
}

template <int TYPE, int DIM>
static int launch_append(AppendArgs &a, hipStream_t st)
{
    const int all = a.d.q_heads + 2 * a.cache.heads, chunks = (all + a.per_chunk - 1) / a.per_chunk;
    a.blocks = (int)(((int64_t)a.d.tokens * (DIM / 8) + 255) / 256);
    // of 2^32 work-items and more only what is left over would run
    HIPQ_REQUIRE((int64_t)a.blocks * chunks < (1 << 24), "append: %d tokens of %d heads", a.d.tokens, all);
    const dim3 grid((unsigned)(a.blocks * chunks));
    if (a.cache.quantized)
        kv_append_kernel<TYPE, DIM, true><<<grid, dim3(256), 0, st>>>(a);
    else
        kv_append_kernel<TYPE, DIM, false><<<grid, dim3(256), 0, st>>>(a);
    return launch_status("kv_append_kernel");
}

template <int TYPE>
static int launch_append(AppendArgs &a, hipStream_t st)
{
    return a.cache.dim == 64 ? launch_append<TYPE, 64>(a, st) : a.cache.dim == 128 ? launch_append<TYPE, 128>(a, st) : launch_append<TYPE, 256>(a, st);
}

} // namespace hipq

using namespace hipq;

extern "C" int hipq_kv_append(const hipq_kv_cache *cache, const hipq_kv_append_desc *d, void *stream)
{
    clear_error();
    if (check_cache(cache))
        return 1;
    HIPQ_REQUIRE(d, "append: a null pointer");
    HIPQ_REQUIRE(d->tokens >= 0 && d->tokens <= (1 << 24), "append: %d tokens", d->tokens);
    HIPQ_REQUIRE(d->q_heads >= 0 && d->q_heads <= 65536, "append: %d query heads", d->q_heads);
    HIPQ_REQUIRE(d->rot >= 0 && d->rot <= cache->dim && d->rot % 16 == 0, "append: %d rotated elements (a multiple of 16 up to %d is needed)", d->rot, cache->dim);
    HIPQ_REQUIRE(d->interleaved == 0 || d->interleaved == 1, "append: interleaved is %d", d->interleaved);
    HIPQ_REQUIRE(d->table_rows >= 0 && (d->rot == 0 || d->table_rows == 0 || d->table), "append: no table");
    HIPQ_REQUIRE(d->eps >= 0, "append: eps is negative");
    if (d->tokens == 0)
        return 0;
    HIPQ_REQUIRE(d->k && d->v && d->positions && d->slots && (d->q_heads == 0 || (d->q && d->q_out)), "append: a null pointer");
    HIPQ_REQUIRE(((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v | (uintptr_t)d->q_out | (uintptr_t)d->table | (uintptr_t)d->q_norm | (uintptr_t)d->k_norm) % 16 == 0,
                 "append: heads have to start at multiples of 16 bytes");
    HIPQ_REQUIRE((d->q_token | d->q_head | d->k_token | d->k_head | d->v_token | d->v_head | d->out_token | d->out_head) % 8 == 0,
                 "append: heads have to start at multiples of 16 bytes (strides are no multiples of 8)");
    AppendArgs a = {};
    a.cache = *cache, a.d = *d;
    if (cache->pages == 0)
        return 0; // no slot is inside
    if (hipq_div_magic((uint32_t)cache->page, &a.page_magic, &a.page_shift))
        return fail("append: pages of %d tokens", cache->page);
    const int all = d->q_heads + 2 * cache->heads;
    const int64_t work = (int64_t)all * d->tokens;
    a.per_chunk = work >= 65536 ? 8 : work >= 16384 ? 2 : 1;
    return cache->type == HIPQ_REAL_BF16 ? launch_append<HIPQ_REAL_BF16>(a, (hipStream_t)stream) : launch_append<HIPQ_REAL_F16>(a, (hipStream_t)stream);
}
