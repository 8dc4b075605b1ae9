// Attention of new tokens over a paged cache (hipq_kv_attend).  gfx950 only.
//
// The cache is read once and every other thing is small: a query head's scores are never written.  With a reference m that is at least the
// running maximum less 8, each tile of tokens adds p_t = 2^(s_t - m) to the sum l and p_t v_t to the output o, all in float32 (p is
// rounded to 16 bits for the product, half a unit in the last place each, as the values themselves are); when a score passes m + 8, m moves there and l
// and o are scaled, which keeps the result and leaves most tiles without any exchange between lanes.
//
// What carries it:
//   * The rows of a work-group are the new tokens of one sequence times the query heads that share a cache head: up to 16 RT of them read
//     each key and value once.  Rows are the columns of the matrix products: s^T = K q^T, o^T = V^T p^T, both 16x16x32, so that a lane
//     has one row's scores, sums and outputs in its own registers, and the scores come out as the second product's operand is
//     wanted (its 8 tokens of k: 4 of one 16-token half of a tile, 4 of the other).
//   * Keys are read in operand order: lane c of 16 has token c, 16 bytes of it.  Values are read row by row as well, lane c the elements
//     c DIM / 16 ..., and turned in registers: half an instruction for each value takes the halves of two tokens into one register.
//     Nothing goes through LDS and no wave waits for another until the end.
//   * Four waves of a work-group take tiles of 32 tokens in turn, each one tile ahead in registers; the tokens of a sequence are split over
//     work-groups until the chip is full, and a second kernel joins the parts.
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

constexpr float NONE = -__builtin_inff();

// DIM values of one row in 16-bit floats or codes: what a lane reads of a key or value
template <int TYPE>
__device__ static __forceinline__ u32x4 widen(uint32_t lo, uint32_t hi) // eight codes + 128 (exact in either type)
{
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = i < 2 ? lo : hi;
        const float a = (float)((w >> (16 * (i & 1))) & 255), b = (float)((w >> (16 * (i & 1) + 8)) & 255);
        o[i] = Real16<TYPE>::pack(a, b);
    }
    return o;
}

struct Sequence {
    int row0, count, len, old; // first row of q, new tokens, tokens in the cache, those before the new ones
    __device__ __forceinline__ Sequence(const AttendArgs &a, int b)
    {
        const int end = min(a.d.starts[b + 1], a.d.tokens);
        row0 = max(a.d.starts[b], 0);
        len = max(min(min(a.d.lens[b], a.d.longest), a.d.blocks_per_sequence * a.cache.page), 0);
        count = max(min(end - row0, a.d.most_new), 0);
        old = len - count;
    }
    // the tokens of a part: an equal share in whole rounds of the four waves
    __device__ __forceinline__ int share(int splits) const { return ((len + splits - 1) / splits + 127) / 128 * 128; }
};

template <int TYPE, int DIM, bool QUANT, int RT>
__global__ __launch_bounds__(256) void kv_attend_kernel(const AttendArgs a)
{
    using R = Real16<TYPE>;
    constexpr int KS = DIM / 32, VD = DIM / 16;       // products of a score; values of a lane
    constexpr int KW = QUANT ? DIM / 64 : DIM / 32;   // 16-byte loads of a key
    constexpr int VW = QUANT ? VD / 4 : VD / 2;       // dwords of a lane's part of a value
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, j = lane >> 4;
    const int split = blockIdx.x % a.splits, rest = blockIdx.x / a.splits;
    const int rb = rest % a.row_blocks, h = rest / a.row_blocks % a.cache.heads, b = rest / a.row_blocks / a.cache.heads;
    const Sequence seq(a, b);
    const int rows = seq.count * a.group, r0 = rb * 16 * RT;
    if (r0 >= rows)
        return;
    const int share = seq.share(a.splits), t0 = split * share;
    // the last row of the block sees no further than its own token
    const int most = a.d.mask ? seq.len : min(seq.len, seq.old + min(rows - 1, r0 + 16 * RT - 1) / a.group + 1);
    const int t1 = min(t0 + share, most);

    // queries, and what a row sees
    u32x4 q[RT][KS];
    f32x4 init[RT]; // codes are stored as code + 128 in the product: less 128 times the sum of q
    int own[RT];
    uint64_t mask[RT];
    bool there[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int row = r0 + 16 * rt + c;
        there[rt] = row < rows;
        own[rt] = there[rt] ? row / a.group : 0;
        const uint16_t *x = (const uint16_t *)a.d.q + (int64_t)(seq.row0 + own[rt]) * a.d.q_token + (int64_t)(h * a.group + (there[rt] ? row % a.group : 0)) * a.d.q_head;
        mask[rt] = a.d.mask ? a.d.mask[seq.row0 + own[rt]] : 0;
        float sum = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            q[rt][ks] = *(const u32x4 *)(x + (QUANT ? ks / 2 * 64 + j * 16 + ks % 2 * 8 : ks * 32 + j * 8));
            if (QUANT)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    sum += R::low(q[rt][ks][e]) + R::high(q[rt][ks][e]);
        }
        if (QUANT) {
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
        }
        const float s = QUANT ? -128.0f * sum : 0.0f;
        init[rt] = f32x4{s, s, s, s};
    }

    float m[RT], l[RT], lv[RT]; // lv: the sum of what multiplies the codes
    float unit = 0;             // float16 codes: p is multiplied by value scale / unit, unit the largest scale so far or more, to stay in range
    f32x4 o[RT][VD];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        m[rt] = NONE, l[rt] = lv[rt] = 0;
#pragma unroll
        for (int i = 0; i < VD; i++)
            o[rt][i] = f32x4{0, 0, 0, 0};
    }

    // a tile: two halves of 16 tokens, each in one page
    u32x4 kx[2][KW];
    uint32_t vx[2][4][VW];
    f32x4 ksc[2], vsc[2];
    bool half_there[2];
    const int32_t *blocks = a.d.blocks + (int64_t)b * a.d.blocks_stride;
    const int halves = (seq.len + 15) / 16, page16 = a.cache.page / 16;
    auto load = [&](int t) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int t16 = t / 16 + s;
            int at = a.page_magic ? (int)(((uint64_t)(uint32_t)t16 * a.page_magic) >> 32) >> a.page_shift : t16;
            const int in = t16 - at * page16;
            int page = t16 < halves ? blocks[at] : -1;
            half_there[s] = page >= 0 && page < a.cache.pages;
            page = half_there[s] ? page : 0;
            const int64_t row = ((int64_t)page * a.cache.heads + h) * a.cache.page + in * 16;
            const uint8_t *k = (const uint8_t *)a.cache.k + row * (QUANT ? DIM : 2 * DIM), *v = (const uint8_t *)a.cache.v + row * (QUANT ? DIM : 2 * DIM);
#pragma unroll
            for (int i = 0; i < KW; i++)
                kx[s][i] = *(const u32x4 *)(k + c * (QUANT ? DIM : 2 * DIM) + i * 64 + j * 16);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint8_t *from = v + (j * 4 + r) * (QUANT ? DIM : 2 * DIM) + c * (4 * VW);
                if (VW == 1)
                    vx[s][r][0] = *(const uint32_t *)from;
                else if (VW == 2) {
                    const u32x2 w = *(const u32x2 *)from;
                    vx[s][r][0] = w[0], vx[s][r][VW - 1] = w[1];
                } else
#pragma unroll
                    for (int i = 0; i < VW; i += 4) {
                        const u32x4 w = *(const u32x4 *)(from + 4 * i);
#pragma unroll
                        for (int e = 0; e < 4 && i + e < VW; e++)
                            vx[s][r][i + e] = w[e];
                    }
            }
            if (QUANT) {
                ksc[s] = *(const f32x4 *)(a.cache.k_scale + row + j * 4);
                vsc[s] = *(const f32x4 *)(a.cache.v_scale + row + j * 4);
            }
        }
    };

    auto tile = [&](int t) {
        // scores
        f32x4 s[RT][2];
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                u32x4 k;
                if (QUANT)
                    k = widen<TYPE>(kx[half][ks / 2][ks % 2 * 2] ^ 0x80808080u, kx[half][ks / 2][ks % 2 * 2 + 1] ^ 0x80808080u);
                else
                    k = kx[half][ks];
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
                    s[rt][half] = R::mfma(k, q[rt][ks], ks ? s[rt][half] : init[rt]);
            }
        // all rows see the whole tile unless it holds a new token, the end, or a page that is not there
        const bool masked = t + 32 > min(seq.old, seq.len) || !half_there[0] || !half_there[1];
        bool strange = false;
        if (masked) {
            // tokens that are not there may hold anything: their values are taken as 0, so that 0 times them is 0
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const bool in = half_there[half] && t + half * 16 + j * 4 + r < seq.len;
                    if (QUANT)
                        vsc[half][r] = in ? vsc[half][r] : 0.0f;
#pragma unroll
                    for (int i = 0; i < VW; i++) {
                        vx[half][r][i] = in ? vx[half][r][i] : 0;
                        if (!QUANT)
                            strange |= !(fabsf(R::low(vx[half][r][i])) < __builtin_inff()) || !(fabsf(R::high(vx[half][r][i])) < __builtin_inff());
                    }
                }
        }
        if (QUANT && TYPE == HIPQ_REAL_F16) {
            float top = 0;
#pragma unroll
            for (int e = 0; e < 8; e++)
                top = fmaxf(top, vsc[e / 4][e % 4]);
            if (__any(top > unit)) {
#pragma unroll
                for (int s = 1; s < 64; s *= 2)
                    top = fmaxf(top, __shfl_xor(top, s));
                top = fminf(top, 3e38f);
                const float f = unit / top; // 0 at the first, where nothing is there to be scaled
                unit = top;
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    lv[rt] *= f;
#pragma unroll
                    for (int i = 0; i < VD; i++)
                        o[rt][i] *= f;
                }
            }
            const float f = unit > 0 ? 1.0f / unit : 0.0f;
            vsc[0] *= f, vsc[1] *= f;
        }
        u32x4 p[RT];
        u32x4 seen[RT]; // where values are infinite or NaN: ones at the tokens that a row sees
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            float x[8], top = NONE;
            uint32_t sees = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int half = e / 4, r = e % 4, token = t + half * 16 + j * 4 + r;
                x[e] = s[rt][half][r] * a.scale2;
                if (QUANT)
                    x[e] *= ksc[half][r];
                if (masked) {
                    const int fresh = token - seq.old;
                    const bool see = half_there[half] && token < seq.len && there[rt] &&
                                     (fresh < 0 || (a.d.mask ? fresh < 64 && ((mask[rt] >> (fresh & 63)) & 1) : fresh <= own[rt]));
                    sees |= (uint32_t)see << e;
                    x[e] = see ? x[e] : NONE;
                }
                top = fmaxf(top, x[e]);
            }
            if (__any(top > m[rt] + 8.0f)) {
                top = fmaxf(top, m[rt]);
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float f = top == NONE ? 1.0f : exp2_fast(m[rt] - top);
                m[rt] = top;
                l[rt] *= f, lv[rt] *= f;
#pragma unroll
                for (int i = 0; i < VD; i++)
                    o[rt][i] *= f;
            }
            const float ref = m[rt] == NONE ? 0.0f : m[rt];
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y[e] = exp2_fast(x[e] - ref);
                l[rt] += y[e];
                if (QUANT) {
                    y[e] *= vsc[e / 4][e % 4];
                    if (masked)
                        y[e] = (sees >> e) & 1 ? y[e] : 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                p[rt][e] = R::pack(y[2 * e], y[2 * e + 1]);
                if (QUANT)
                    lv[rt] += R::low(p[rt][e]) + R::high(p[rt][e]);
                const uint32_t one = R::pack(1.0f, 0.0f);
                seen[rt][e] = ((sees >> (2 * e)) & 1 ? one : 0) | ((sees >> (2 * e + 1)) & 1 ? one << 16 : 0);
            }
        }
        // output
        const bool any_strange = masked && __any(strange);
#pragma unroll
        for (int i = 0; i < VD; i++) {
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int half = e / 2, r = e % 2 * 2;
                if (QUANT) {
                    const float x0 = (float)(((vx[half][r][i / 4] ^ 0x80808080u) >> (8 * (i % 4))) & 255),
                                x1 = (float)(((vx[half][r + 1][i / 4] ^ 0x80808080u) >> (8 * (i % 4))) & 255);
                    v[e] = R::pack(x0, x1);
                } else
                    v[e] = __builtin_amdgcn_perm(vx[half][r + 1][i / 2], vx[half][r][i / 2], i % 2 ? 0x07060302u : 0x05040100u);
            }
            if (!QUANT && any_strange) {
                // an infinity or NaN among the values near the end reaches the rows that see it, as NaN, and no other
                u32x4 bad = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool lo = !(fabsf(R::low(v[e])) < __builtin_inff()), hi = !(fabsf(R::high(v[e])) < __builtin_inff());
                    const uint32_t one = R::pack(1.0f, 0.0f);
                    bad[e] = (lo ? one : 0) | (hi ? one << 16 : 0);
                    v[e] &= (lo ? 0 : 0xffffu) | (hi ? 0 : 0xffff0000u);
                }
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    const f32x4 n = R::mfma(bad, seen[rt], f32x4{0, 0, 0, 0});
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        o[rt][i][r] = n[r] > 0 ? __builtin_nanf("") : o[rt][i][r];
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
                o[rt][i] = R::mfma(v, p[rt], o[rt][i]);
        }
    };

    for (int t = t0 + wave * 32; t < t1; t += 128) {
        load(t);
        tile(t);
    }

    // the four waves' parts: a row's reference and sums over its lanes, then over the waves, then the outputs in two steps
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    float *lm = (float *)lds, *ll = lm + 4 * RT * 16; // [wave][row]
    f32x4 *lo = (f32x4 *)(ll + 4 * RT * 16);          // [2][RT * VD][64]
    float f[RT], sum[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        l[rt] += __shfl_xor(l[rt], 16);
        l[rt] += __shfl_xor(l[rt], 32);
        if (QUANT) {
            lv[rt] += __shfl_xor(lv[rt], 16);
            lv[rt] += __shfl_xor(lv[rt], 32);
            const float less = -128.0f * lv[rt];
#pragma unroll
            for (int i = 0; i < VD; i++)
                o[rt][i] += less;
            if (TYPE == HIPQ_REAL_F16)
#pragma unroll
                for (int i = 0; i < VD; i++)
                    o[rt][i] *= unit;
        }
        if (j == 0)
            lm[wave * RT * 16 + rt * 16 + c] = m[rt], ll[wave * RT * 16 + rt * 16 + c] = l[rt];
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        float top = NONE;
#pragma unroll
        for (int w = 0; w < 4; w++)
            top = fmaxf(top, lm[w * RT * 16 + rt * 16 + c]);
        const float ref = top == NONE ? 0.0f : top;
        sum[rt] = 0;
#pragma unroll
        for (int w = 0; w < 4; w++)
            sum[rt] += ll[w * RT * 16 + rt * 16 + c] * exp2_fast(lm[w * RT * 16 + rt * 16 + c] - ref);
        f[rt] = exp2_fast(m[rt] - ref);
        m[rt] = top;
#pragma unroll
        for (int i = 0; i < VD; i++)
            o[rt][i] *= f[rt];
    }
#pragma unroll
    for (int step = 2; step >= 1; step /= 2) {
        if (wave >= step && wave < 2 * step)
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int i = 0; i < VD; i++)
                    lo[((wave - step) * RT * VD + rt * VD + i) * 64 + lane] = o[rt][i];
        __syncthreads();
        if (wave < step)
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int i = 0; i < VD; i++)
                    o[rt][i] += lo[(wave * RT * VD + rt * VD + i) * 64 + lane];
        __syncthreads();
    }
    if (wave != 0)
        return;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        if (!there[rt])
            continue;
        const int row = r0 + 16 * rt + c;
        if (a.splits == 1) {
            const float inv = sum[rt] > 0 ? 1.0f / sum[rt] : sum[rt] == 0 ? 0.0f : sum[rt];
            uint16_t *y = (uint16_t *)a.d.o + (int64_t)(seq.row0 + own[rt]) * a.d.o_token + (int64_t)(h * a.group + row % a.group) * a.d.o_head;
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int i = 0; i < VD; i += 4) {
                    const u32x2 w = {R::pack(o[rt][i][r] * inv, o[rt][i + 1][r] * inv), R::pack(o[rt][i + 2][r] * inv, o[rt][i + 3][r] * inv)};
                    *(u32x2 *)(y + (j * 4 + r) * VD + i) = w;
                }
        } else {
            const int64_t at = (((int64_t)b * a.cache.heads + h) * a.splits + split) * a.rows + row;
            if (j == 0)
                a.part_ml[2 * at] = m[rt], a.part_ml[2 * at + 1] = sum[rt];
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int i = 0; i < VD; i += 4)
                    *(f32x4 *)(a.part_o + at * DIM + (j * 4 + r) * VD + i) = f32x4{o[rt][i][r], o[rt][i + 1][r], o[rt][i + 2][r], o[rt][i + 3][r]};
        }
    }
}

// Joins the parts of a row: DIM / 4 neighbouring lanes have a row.
template <int TYPE, int DIM>
__global__ __launch_bounds__(256) void kv_attend_join_kernel(const AttendArgs a)
{
    using R = Real16<TYPE>;
    constexpr int LANES = DIM / 4;
    const int64_t id = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;
    const int i0 = threadIdx.x % LANES * 4, bh = (int)(id / a.rows), row = (int)(id % a.rows);
    if (bh >= a.d.sequences * a.cache.heads)
        return;
    const int b = bh / a.cache.heads, h = bh % a.cache.heads;
    const Sequence seq(a, b);
    if (row >= seq.count * a.group)
        return;
    const int64_t at = (int64_t)bh * a.splits * a.rows + row;
    float top = NONE;
    for (int s = 0; s < a.splits; s++)
        top = fmaxf(top, a.part_ml[2 * (at + (int64_t)s * a.rows)]);
    const float ref = top == NONE ? 0.0f : top;
    float l = 0;
    f32x4 o = {0, 0, 0, 0};
    for (int s = 0; s < a.splits; s++) {
        const int64_t p = at + (int64_t)s * a.rows;
        const float f = exp2_fast(a.part_ml[2 * p] - ref);
        l += f * a.part_ml[2 * p + 1];
        o += f * *(const f32x4 *)(a.part_o + p * DIM + i0);
    }
    const float inv = l > 0 ? 1.0f / l : l == 0 ? 0.0f : l;
    uint16_t *y = (uint16_t *)a.d.o + (int64_t)(seq.row0 + row / a.group) * a.d.o_token + (int64_t)(h * a.group + row % a.group) * a.d.o_head;
    const u32x2 w = {R::pack(o[0] * inv, o[1] * inv), R::pack(o[2] * inv, o[3] * inv)};
    *(u32x2 *)(y + i0) = w;
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
struct AttendShape {
    int rt, row_blocks, rows, splits;
    size_t workspace;
};

static int check_attend(const hipq_kv_cache *c, const hipq_kv_attend_desc *d)
{
    if (check_cache(c))
        return 1;
    HIPQ_REQUIRE(d, "attend: a null pointer");
    HIPQ_REQUIRE(d->sequences >= 0 && d->sequences <= (1 << 20), "attend: %d sequences", d->sequences);
    HIPQ_REQUIRE(d->tokens >= 0 && d->tokens <= (1 << 24), "attend: %d new tokens", d->tokens);
    HIPQ_REQUIRE(d->q_heads >= 1 && d->q_heads <= 65536 && d->q_heads % c->heads == 0, "attend: %d query heads on %d heads of the cache", d->q_heads, c->heads);
    HIPQ_REQUIRE(d->most_new >= 0 && d->most_new <= (1 << 20), "attend: %d new tokens of a sequence", d->most_new);
    HIPQ_REQUIRE(!d->mask || d->most_new <= 64, "attend: a mask has bits for 64 new tokens of a sequence, not %d", d->most_new);
    HIPQ_REQUIRE(d->blocks_per_sequence >= 0 && (int64_t)d->blocks_per_sequence * c->page < ((int64_t)1 << 31), "attend: %d blocks of a sequence", d->blocks_per_sequence);
    HIPQ_REQUIRE(d->blocks_stride >= d->blocks_per_sequence || d->sequences <= 1, "attend: rows of blocks overlap");
    HIPQ_REQUIRE(d->longest >= 0, "attend: the longest sequence has %d tokens", d->longest);
    HIPQ_REQUIRE(d->scale == d->scale && d->scale < 1e30f && d->scale > -1e30f, "attend: scale %g", (double)d->scale);
    const int64_t rows = (int64_t)d->most_new * (d->q_heads / c->heads);
    HIPQ_REQUIRE(rows < (1 << 24), "attend: %lld rows of a sequence", (long long)rows);
    return 0;
}

static AttendShape shape_of(const hipq_kv_cache *c, const hipq_kv_attend_desc *d)
{
    AttendShape s = {};
    const int group = d->q_heads / c->heads;
    s.rows = d->most_new * group;
    s.rt = s.rows <= 16 ? 1 : s.rows <= 32 || c->dim == 256 ? 2 : 4;
    s.row_blocks = (s.rows + 16 * s.rt - 1) / (16 * s.rt);
    const int64_t longest = d->longest < (int64_t)d->blocks_per_sequence * c->page ? d->longest : (int64_t)d->blocks_per_sequence * c->page;
    const int64_t items = (int64_t)d->sequences * c->heads * s.row_blocks;
    const int64_t want = items ? (512 + items - 1) / items : 1, most = (longest + 255) / 256;
    s.splits = (int)(want < most ? want : most);
    s.splits = s.splits < 1 ? 1 : s.splits > 64 ? 64 : s.splits;
    if (s.splits > 1)
        s.workspace = (size_t)d->sequences * c->heads * s.splits * s.rows * (c->dim + 2) * sizeof(float);
    return s;
}

template <int TYPE, int DIM, bool QUANT, int RT>
static int launch_attend(const AttendArgs &a, int64_t items, hipStream_t st)
{
    const size_t lds = (2 * 4 * RT * 16) * 4 + (size_t)2 * RT * (DIM / 16) * 64 * 16;
    static thread_local bool allowed[64] = {};
    int device = 0;
    HIPQ_CHECK_HIP(hipGetDevice(&device));
    if (lds > 65536 && (device >= 64 || !allowed[device])) {
        HIPQ_CHECK_HIP(hipFuncSetAttribute((const void *)kv_attend_kernel<TYPE, DIM, QUANT, RT>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        if (device < 64)
            allowed[device] = true;
    }
    kv_attend_kernel<TYPE, DIM, QUANT, RT><<<dim3((unsigned)(items * a.splits)), dim3(256), lds, st>>>(a);
    return launch_status("kv_attend_kernel");
}

template <int TYPE, int DIM, bool QUANT>
static int launch_attend(const AttendArgs &a, int rt, int64_t items, hipStream_t st)
{
    if (rt == 1)
        return launch_attend<TYPE, DIM, QUANT, 1>(a, items, st);
    if (rt == 2 || DIM == 256)
        return launch_attend<TYPE, DIM, QUANT, 2>(a, items, st);
    return launch_attend<TYPE, DIM, QUANT, DIM == 256 ? 2 : 4>(a, items, st);
}

template <int TYPE, int DIM>
static int launch_attend(const AttendArgs &a, int rt, int64_t items, hipStream_t st)
{
    if (a.cache.quantized ? launch_attend<TYPE, DIM, true>(a, rt, items, st) : launch_attend<TYPE, DIM, false>(a, rt, items, st))
        return 1;
    if (a.splits == 1)
        return 0;
    const int64_t threads = (int64_t)a.d.sequences * a.cache.heads * a.rows * (DIM / 4);
    kv_attend_join_kernel<TYPE, DIM><<<dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st>>>(a);
    return launch_status("kv_attend_join_kernel");
}

template <int TYPE>
static int launch_attend(const AttendArgs &a, int rt, int64_t items, hipStream_t st)
{
    return a.cache.dim == 64 ? launch_attend<TYPE, 64>(a, rt, items, st) : a.cache.dim == 128 ? launch_attend<TYPE, 128>(a, rt, items, st) : launch_attend<TYPE, 256>(a, rt, items, st);
}

} // namespace hipq

using namespace hipq;

extern "C" size_t hipq_kv_attend_workspace(const hipq_kv_cache *cache, const hipq_kv_attend_desc *d)
{
    clear_error();
    return check_attend(cache, d) ? 0 : shape_of(cache, d).workspace;
}

extern "C" int hipq_kv_attend(const hipq_kv_cache *cache, const hipq_kv_attend_desc *d, void *workspace, size_t workspace_bytes, void *stream)
{
    clear_error();
    if (check_attend(cache, d))
        return 1;
    const AttendShape s = shape_of(cache, d);
    const int64_t items = (int64_t)d->sequences * cache->heads * s.row_blocks;
    if (items == 0 || d->tokens == 0)
        return 0;
    HIPQ_REQUIRE(d->q && d->o && d->starts && d->lens && (d->blocks || d->blocks_per_sequence == 0), "attend: a null pointer");
    HIPQ_REQUIRE(((uintptr_t)d->q | (uintptr_t)d->o) % 16 == 0 && (d->q_token | d->q_head | d->o_token | d->o_head) % 8 == 0,
                 "attend: heads have to start at multiples of 16 bytes");
    HIPQ_REQUIRE(s.workspace == 0 || (workspace && workspace_bytes >= s.workspace && (uintptr_t)workspace % 16 == 0), "attend: a workspace of %zu bytes is needed", s.workspace);
    HIPQ_REQUIRE(items * s.splits < ((int64_t)1 << 31), "attend: %lld work-groups", (long long)items * s.splits);
    AttendArgs a = {};
    a.cache = *cache, a.d = *d;
    if (cache->pages == 0)
        a.d.longest = 0; // no block is inside: nothing may be read
    a.scale2 = d->scale * 1.4426950408889634f;
    a.group = d->q_heads / cache->heads, a.splits = s.splits, a.row_blocks = s.row_blocks, a.rows = s.rows;
    if (hipq_div_magic((uint32_t)cache->page / 16, &a.page_magic, &a.page_shift))
        return fail("attend: pages of %d tokens", cache->page);
    if (s.splits > 1) {
        a.part_o = (float *)workspace;
        a.part_ml = a.part_o + (size_t)d->sequences * cache->heads * s.splits * s.rows * cache->dim;
    }
    return cache->type == HIPQ_REAL_BF16 ? launch_attend<HIPQ_REAL_BF16>(a, s.rt, items, (hipStream_t)stream) : launch_attend<HIPQ_REAL_F16>(a, s.rt, items, (hipStream_t)stream);
}
