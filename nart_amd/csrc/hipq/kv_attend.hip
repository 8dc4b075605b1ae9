// Attention of new tokens over a paged cache (hipq_kv_attend).  gfx950 only.
//
// The cache is read once and every other thing is small: a query head's scores are never written.  With a reference m that is at least the
// running maximum less 8, each tile of tokens adds p_t = 2^(s_t - m) to the sum l and p_t v_t to the output o, all in float32; when a score
// passes m + 8, m moves there and l and o are scaled, which keeps the result and leaves most tiles without any exchange between lanes.
// For the product p - over codes p times the token's value scale - is rounded to 16 bits, which is what the matrix unit takes (in two parts it
// would do twice the work): half a unit in the last place each, and for float16's small ones see softmax_step.
//
// What carries it:
//   * The rows of a work-group are the new tokens of one sequence times the query heads that share a cache head: up to 16 RT of them read
//     each key and value once.  Rows are the columns of the matrix products: s^T = K q^T, o^T = V^T p^T, both 16x16x32, so that a lane
//     has one row's scores, sums and outputs in its own registers, and the scores come out as the second product's operand is
//     wanted (its 8 tokens of k: 4 of one 16-token half of a tile, 4 of the other).
//   * Keys are read in operand order: lane c of 16 has token c, 16 bytes of it.  Values are read row by row as well, lane c the elements
//     c DIM / 16 ..., and turned in registers: half an instruction for each value takes the halves of two tokens into one register.
//     Nothing goes through LDS and no wave waits for another until the end.
//   * Four waves of a work-group take tiles of 32 tokens in turn, each a tile ahead in its loads; the tokens of a sequence are split over
//     work-groups until the chip is full, and a second kernel joins the parts.
//   * More than 64 rows of heads of 128 have a kernel of their own (kv_attend_wide_kernel), whose four waves share what they bring from the
//     cache.
// What bounds it, measured (32 query heads on 8 of 128 unless said otherwise): one token of 8 sequences of up to 2000 in 16 bits, 14 us and
// 3.8 for the join: latency, about 3.4 TB/s; one token of 2 x 131072 with 64 heads, 170 to 180 us and 5: 4.6 TB/s, a large copy's rate being
// 5.2; 16 trees of 32 tokens on up to 8000 in 8 bits, 111 us with the join: vector instructions (300 a tile and wave, a tenth of them for widening
// codes; the kernel without shared tiles takes 121, a third of its 360 for that).
#include <type_traits>

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
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

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

// infinities or NaN among an operand's 16-bit values
template <int TYPE>
__device__ static __forceinline__ bool strange(const u32x4 &v)
{
    u16x2 largest = {0, 0};
#pragma unroll
    for (int e = 0; e < 4; e++)
        largest = __builtin_elementwise_max(largest, __builtin_bit_cast(u16x2, v[e] & 0x7fff7fffu));
    constexpr uint16_t inf = TYPE == HIPQ_REAL_BF16 ? 0x7f80 : 0x7c00;
    return largest[0] >= inf || largest[1] >= inf;
}
// Where values are infinite or NaN they reach the rows that see them, as NaN, and no other: ones in their places, multiplied by ones at the
// tokens that a row sees.  What is left of the values is finite.
template <int TYPE, int RT, int VD>
__device__ static __forceinline__ void not_finite(u32x4 &v, const uint32_t (&sees)[RT], f32x4 (&o)[RT][VD], int i)
{
    using R = Real16<TYPE>;
    u32x4 bad = {0, 0, 0, 0};
    const uint32_t one = R::pack(1.0f, 0.0f);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const bool lo = !(fabsf(R::low(v[e])) < __builtin_inff()), hi = !(fabsf(R::high(v[e])) < __builtin_inff());
        bad[e] = (lo ? one : 0) | (hi ? one << 16 : 0);
        v[e] &= (lo ? 0 : 0xffffu) | (hi ? 0 : 0xffff0000u);
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        u32x4 seen;
#pragma unroll
        for (int e = 0; e < 4; e++)
            seen[e] = ((sees[rt] >> (2 * e)) & 1 ? one : 0) | ((sees[rt] >> (2 * e + 1)) & 1 ? one << 16 : 0);
        const f32x4 n = R::mfma(bad, seen, f32x4{0, 0, 0, 0});
#pragma unroll
        for (int r = 0; r < 4; r++)
            o[rt][i][r] = n[r] > 0 ? __builtin_nanf("") : o[rt][i][r];
    }
}

// Float16 has few small numbers: below 2^-14 they lose bits, below 2^-25 they are 0, while weights are at most 2^8 and half of its range lies above.
// Over 16 bits they are therefore 2^7 times as large, in their sum as in the outputs, so that a weight is off by at most half a unit in its last
// place or 2^-32 of the row's largest.  Over codes what is rounded is a weight times its token's value scale, whose size has nothing to
// do with the weight's: it has a reference of its own, `unit`, a power of two that it passes by 2^8 at most, and is
// multiplied by 2^7 / unit; outputs are in units of unit / 2^7.  unit is a row's, from what the row sees, and moves with m as the outputs would.
// (With one unit for a wave, its largest value scale, rows of 8192 tokens with some dominant ones were off by up to 94 times what roundings leave.  us, now against
// then, of float16 over codes: one token of 8 sequences of up to 2000 15.4 and 16.3, 16 trees of 32 tokens on up to 8000 117 and 117.)
template <int TYPE, bool QUANT>
constexpr bool UNITS = QUANT && TYPE == HIPQ_REAL_F16;
constexpr float RAISED = 128.0f, LEAST_UNIT = 0x1p-100f; // what lies below that is 0 in float16, however many tokens there are

// A row's weights p of 8 tokens a lane from its scores s: the reference m moves where a score passes it by more than 8, and with it the sums (l
// of codes, lsum of 16-bit values) and outputs are scaled.
template <int TYPE, bool QUANT, bool MASKED, int VD>
__device__ static __forceinline__ void softmax_step(float scale2, const f32x4 (&s)[2], const f32x4 (&kscale)[2], const f32x4 (&vsc)[2], uint32_t sees, float &m, float &l,
                                                    f32x4 &lsum, float &unit, float &per_unit, f32x4 (&o)[VD], u32x4 &p)
{
    using R = Real16<TYPE>;
    constexpr bool units = UNITS<TYPE, QUANT>;
    float x[8], top = NONE;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        x[e] = QUANT ? s[e / 4][e % 4] * kscale[e / 4][e % 4] : s[e / 4][e % 4];
        if (MASKED)
            x[e] = (sees >> e) & 1 ? x[e] : NONE;
        top = fmaxf(top, x[e]);
    }
    if (!QUANT)
        top *= scale2;
    if (__any(top > m + 8.0f)) {
        top = fmaxf(top, m);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (units)
            top = ceilf(top); // units stay powers of two, and scaling exact
        const float f = top == NONE ? 1.0f : exp2_fast(m - top);
        m = top;
        l *= f;
        lsum *= f;
        if (units) {
            unit *= f;
            per_unit = unit >= LEAST_UNIT ? RAISED / unit : 0.0f;
        } else
#pragma unroll
            for (int i = 0; i < VD; i++)
                o[i] *= f;
    }
    const float ref = (m == NONE ? 0.0f : m) - (!QUANT && TYPE == HIPQ_REAL_F16 ? 7.0f : 0.0f);
    float y[8], most = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        y[e] = exp2_fast(QUANT ? x[e] - ref : __builtin_fmaf(x[e], scale2, -ref));
        if (QUANT) {
            l += y[e];
            y[e] *= vsc[e / 4][e % 4];
            if (MASKED)
                y[e] = (sees >> e) & 1 ? y[e] : 0.0f;
            if (units)
                most = fmaxf(most, fabsf(y[e]));
        }
    }
    if (units) {
        if (__any(most > unit * 256.0f)) {
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            most = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, most) & 0x7f800000u); // the power of two below
            most = fmaxf(fminf(fmaxf(most, LEAST_UNIT), 0x1p126f), unit);
            const float f = unit / most; // 0 at the first, where nothing is there to be scaled
            unit = most, per_unit = RAISED / most;
#pragma unroll
            for (int i = 0; i < VD; i++)
                o[i] *= f;
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
            y[e] *= per_unit;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        p[e] = R::pack(y[2 * e], y[2 * e + 1]);
    if (!QUANT) {
        const uint32_t one = R::pack(1.0f, 1.0f);
        lsum = R::mfma(u32x4{one, one, one, one}, p, lsum);
    }
}

template <int TYPE, int DIM, bool QUANT, int RT>
__global__ __launch_bounds__(256, DIM == 256 || (QUANT && TYPE == HIPQ_REAL_F16 && DIM == 128 && RT == 2) ? 1 : 2) void kv_attend_kernel(const AttendArgs a)
{
    using R = Real16<TYPE>;
    constexpr int KS = DIM / 32, VD = DIM / 16;       // products of a score; values of a lane
    constexpr int KW = QUANT ? DIM / 64 : DIM / 32;   // 16-byte loads of a key
    constexpr int VW = QUANT ? VD / 4 : VD / 2;       // dwords of a lane's part of a value
    constexpr int WIDTH = QUANT ? DIM : 2 * DIM;      // bytes of a row of the cache
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, j = lane >> 4;
    // work-groups go to the 8 XCDs in turn: XCD x takes the x-th contiguous eighth, the row blocks that read the same tokens side by side
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

    // queries
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    // in LDS where they would take the registers of a second work-group, in operand order: [rt][ks][lane], behind what the end needs
    constexpr bool Q_LDS = RT > 1;
    float *const lm = (float *)lds, *const ll = lm + 4 * RT * 16; // [wave][row]
    f32x4 *const lo = (f32x4 *)(ll + 4 * RT * 16);                // [2][RT * VD][64]
    u32x4 *const lq = (u32x4 *)(lo + 2 * RT * VD * 64);
    u32x4 q[Q_LDS ? 1 : RT][Q_LDS ? 1 : KS];
    int own[RT], qh[RT]; // the lane's rows (the last one again behind it): new token and query head
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int row = min(r0 + 16 * rt + c, rows - 1);
        own[rt] = row / a.group, qh[rt] = h * a.group + row - own[rt] * a.group;
        const uint16_t *x = (const uint16_t *)a.d.q + (int64_t)(seq.row0 + own[rt]) * a.d.q_token + (int64_t)qh[rt] * a.d.q_head;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const u32x4 *from = (const u32x4 *)(x + (QUANT ? ks / 2 * 64 + j * 16 + ks % 2 * 8 : ks * 32 + j * 8));
            if (!Q_LDS)
                q[Q_LDS ? 0 : rt][Q_LDS ? 0 : ks] = *from;
            else if ((rt * KS + ks) % 4 == wave)
                lq[(rt * KS + ks) * 64 + lane] = *from;
        }
    }
    if (Q_LDS)
        __syncthreads();

    float m[RT], l[RT];
    f32x4 lsum[RT]; // 16 bits: the sums of p, by a multiply by ones
    float unit[RT], per_unit[RT];
    f32x4 o[RT][VD];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        m[rt] = NONE, l[rt] = 0;
        unit[rt] = per_unit[rt] = 0;
        lsum[rt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < VD; i++)
            o[rt][i] = f32x4{0, 0, 0, 0};
    }

    u32x4 kx[2][KW];
    uint32_t vx[2][4][VW];
    f32x4 ksc[2], vsc[2];
    const int32_t *blocks = a.d.blocks + (int64_t)b * a.d.blocks_stride;
    const Paging paging(a, blocks, seq.len);
    auto load_k = [&](const Pages &p) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int64_t row = paging.row(p, s, h);
            const gbytes_t k = uniform((const uint8_t *)a.cache.k + row * WIDTH);
#pragma unroll
            for (int i = 0; i < KW; i++)
                kx[s][i] = at<u32x4>(k, c * WIDTH + j * 16 + i * 64);
            if (QUANT)
                ksc[s] = at<f32x4>(uniform(a.cache.k_scale + row), j * 16);
        }
    };
    auto load_v = [&](const Pages &p) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int64_t row = paging.row(p, s, h);
            const gbytes_t v = uniform((const uint8_t *)a.cache.v + row * WIDTH);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint32_t from = (j * 4 + r) * WIDTH + c * (4 * VW);
                if (VW == 1)
                    vx[s][r][0] = at<uint32_t>(v, from);
                else if (VW == 2) {
                    const u32x2 w = at<u32x2>(v, from);
                    vx[s][r][0] = w[0], vx[s][r][VW - 1] = w[1];
                } else
#pragma unroll
                    for (int i = 0; i < VW; i += 4) {
                        const u32x4 w = at<u32x4>(v, from + 4 * i);
#pragma unroll
                        for (int e = 0; e < 4 && i + e < VW; e++)
                            vx[s][r][i + e] = w[e];
                    }
            }
            if (QUANT)
                vsc[s] = at<f32x4>(uniform(a.cache.v_scale + row), j * 16);
        }
    };

    // The next tile's keys are asked for when this one's are multiplied, its values when this one's are: each has the other's work to
    // arrive in, and no second set of registers.  (Behind the last tile something is loaded once more, for nothing: a branch around it
    // would make every wait one for all loads.)  MASKED: not all rows see the whole tile.
    auto tile = [&](int t, const Pages &now, const Pages &next, auto MASKED) __attribute__((always_inline)) {
        constexpr bool masked = decltype(MASKED)::value;
        u32x4 k[2][KS];
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                k[half][ks] = QUANT ? widen<TYPE>(kx[half][ks / (QUANT ? 2 : 1)][ks % 2 * 2], kx[half][ks / (QUANT ? 2 : 1)][ks % 2 * 2 + 1]) : kx[half][ks / (QUANT ? 2 : 1)];
        f32x4 kscale[2];
        if (QUANT)
            kscale[0] = ksc[0] * a.scale2, kscale[1] = ksc[1] * a.scale2;
        __builtin_amdgcn_sched_barrier(0); // what is done earlier than it is written does not fit the registers
        load_k(next);
        __builtin_amdgcn_sched_barrier(0);
        if (masked) {
            // tokens that are not there may hold anything: their values are taken as 0, so that 0 times them is 0
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int there = now.page[half] >= 0 ? seq.len - t - half * 16 - j * 4 : 0;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if (QUANT)
                        vsc[half][r] = r < there ? vsc[half][r] : 0.0f;
#pragma unroll
                    for (int i = 0; i < VW; i++)
                        vx[half][r][i] = r < there ? vx[half][r][i] : 0;
                }
            }
        }
        u32x4 p[RT];
        uint32_t sees[RT]; // a bit for each of the lane's 8 tokens: seen by the row
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            f32x4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int half = 0; half < 2; half++)
                    s[half] = R::mfma(k[half][ks], Q_LDS ? lq[(rt * KS + ks) * 64 + lane] : q[Q_LDS ? 0 : rt][Q_LDS ? 0 : ks], s[half]);
            if (masked)
                sees[rt] = seen_by(a, seq, own[rt], t, j, now);
            softmax_step<TYPE, QUANT, masked, VD>(a.scale2, s, kscale, vsc, masked ? sees[rt] : 0, m[rt], l[rt], lsum[rt], unit[rt], per_unit[rt], o[rt], p[rt]);
        }
        __builtin_amdgcn_sched_barrier(0);
        // output
#pragma unroll
        for (int i = 0; i < VD; i++) {
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int half = e / 2, r = e % 2 * 2;
                if (QUANT)
                    v[e] = R::pack_exact((float)(int8_t)(vx[half][r][i / 4] >> (8 * (i % 4))), (float)(int8_t)(vx[half][r + 1][i / 4] >> (8 * (i % 4))));
                else
                    v[e] = __builtin_amdgcn_perm(vx[half][r + 1][i / 2], vx[half][r][i / 2], i % 2 ? 0x07060302u : 0x05040100u);
            }
            if (masked && !QUANT && (a.d.mask || seq.count > 1) && __any(strange<TYPE>(v)))
                not_finite<TYPE>(v, sees, o, i);
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
                o[rt][i] = R::mfma(v, p[rt], o[rt][i]);
        }
        load_v(next);
    };

    int t = t0 + wave * 32;
    if (t < t1) {
        Pages now = paging.of(t), next = paging.of(t + 128);
        load_k(now);
        load_v(now);
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

    // the four waves' parts: a row's reference and sums over its lanes, then over the waves, then the outputs in two steps
    float f[RT], sum[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        if (QUANT) {
            l[rt] += __shfl_xor(l[rt], 16);
            l[rt] += __shfl_xor(l[rt], 32);
            if (UNITS<TYPE, QUANT>)
#pragma unroll
                for (int i = 0; i < VD; i++)
                    o[rt][i] *= unit[rt] * (1 / RAISED);
        } else
            l[rt] = lsum[rt][0];
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
        const int row = r0 + 16 * rt + c;
        if (row >= rows)
            continue;
        if (a.splits == 1) {
            const float inv = sum[rt] > 0 ? 1.0f / sum[rt] : sum[rt] == 0 ? 0.0f : sum[rt];
            uint16_t *y = (uint16_t *)a.d.o + (int64_t)(seq.row0 + own[rt]) * a.d.o_token + (int64_t)qh[rt] * a.d.o_head;
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

// For more than 64 rows: 128 of a work-group, 32 of each of its four waves, all at the same tile of 32 tokens.  Each wave brings a quarter of
// the tile - some 16 x 32 operands of keys, turned ones of values - into LDS in operand order, widened from 8 bits once for all 128 rows,
// a tile ahead of the multiplies that read it; one barrier a tile.  Nothing is joined at the end, as a wave sees all tokens of its rows.
template <int TYPE, int DIM, bool QUANT>
__global__ __launch_bounds__(256, 2) void kv_attend_wide_kernel(const AttendArgs a)
{
    using R = Real16<TYPE>;
    constexpr int RT = 2, ROWS = 64 * RT;
    constexpr int KS = DIM / 32, VD = DIM / 16, KF = KS / 2, VF = VD / 4; // operands of a tile's half, of its values; a wave's share of both
    constexpr int WIDTH = QUANT ? DIM : 2 * DIM;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, j = lane >> 4;
    const int eighth = gridDim.x / 8, item = (int)(blockIdx.x % 8) * eighth + (int)(blockIdx.x / 8);
    const int rb = item % a.row_blocks, split = item / a.row_blocks % a.splits, rest = item / a.row_blocks / a.splits;
    const int h = rest % a.cache.heads, b = rest / a.cache.heads;
    if (b >= a.d.sequences)
        return;
    const Sequence seq(a, b);
    const int rows = seq.count * a.group, r0 = rb * ROWS + wave * 16 * RT;
    if (rb * ROWS >= rows)
        return;
    const int share = seq.share(a.splits), t0 = split * share;
    const int most = a.d.mask ? seq.len : min(seq.len, seq.old + min(rows - 1, rb * ROWS + ROWS - 1) / a.group + 1);
    const int t1 = min(t0 + share, most);

    __shared__ u32x4 lkv[2][2 * KS + VD][64]; // keys: [half][ks], then values
    __shared__ f32x4 lsc[2][QUANT ? 16 : 1];  // scales of keys, then of values
    u32x4 q[RT][KS];
    int own[RT], qh[RT]; // the lane's rows (the last one again behind it): new token and query head
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int row = min(r0 + 16 * rt + c, rows - 1);
        own[rt] = row / a.group, qh[rt] = h * a.group + row - own[rt] * a.group;
        const uint16_t *x = (const uint16_t *)a.d.q + (int64_t)(seq.row0 + own[rt]) * a.d.q_token + (int64_t)qh[rt] * a.d.q_head;
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
            q[rt][ks] = *(const u32x4 *)(x + ks * 32 + j * 8);
    }
    float m[RT], l[RT], unit[RT], per_unit[RT];
    f32x4 lsum[RT], o[RT][VD];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        m[rt] = NONE, l[rt] = 0;
        unit[rt] = per_unit[rt] = 0;
        lsum[rt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < VD; i++)
            o[rt][i] = f32x4{0, 0, 0, 0};
    }

    const int32_t *blocks = a.d.blocks + (int64_t)b * a.d.blocks_stride;
    const Paging paging(a, blocks, seq.len);
    // the wave's part of a tile: operands wave KF .. of keys; of values elements (16 VF) wave + VF c ..
    u32x4 kxs[2][KF];
    uint32_t vxs[2][2][4];
    float sxs[2] = {0, 0};
    auto load = [&](auto SET, const Pages &p) __attribute__((always_inline)) {
        auto &kx = kxs[decltype(SET)::value];
        auto &vx = vxs[decltype(SET)::value];
        auto &sx = sxs[decltype(SET)::value];
        const int64_t row0 = paging.row(p, 0, h), row1 = paging.row(p, 1, h);
        const gbytes_t k = uniform((const uint8_t *)a.cache.k + (wave * KF >= KS ? row1 : row0) * WIDTH);
#pragma unroll
        for (int n = 0; n < KF; n++) {
            const uint32_t from = c * WIDTH + ((wave * KF + n) % KS * 32 + j * 8) * (QUANT ? 1 : 2);
            if (QUANT) {
                const u32x2 w = at<u32x2>(k, from);
                kx[n][0] = w[0], kx[n][1] = w[1];
            } else
                kx[n] = at<u32x4>(k, from);
        }
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const gbytes_t v = uniform((const uint8_t *)a.cache.v + (s ? row1 : row0) * WIDTH);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint32_t from = (j * 4 + r) * WIDTH + (16 * wave + c) * (QUANT ? VF : 2 * VF);
                vx[s][r] = (QUANT ? VF : 2 * VF) == 1 ? at<uint8_t>(v, from) : (QUANT ? VF : 2 * VF) == 2 ? at<uint16_t>(v, from) : at<uint32_t>(v, from);
            }
        }
        if (QUANT) // 32 tokens' scales of keys, then of values: every wave has them, or a wait after the branch would be one for all loads
            sx = *((lane < 32 ? a.cache.k_scale : a.cache.v_scale) + (lane & 16 ? row1 : row0) + (lane & 15));
    };
    auto store = [&](auto SET, int t, const Pages &p) __attribute__((always_inline)) {
        constexpr int to = decltype(SET)::value;
        auto &kx = kxs[to];
        auto &vx = vxs[to];
        auto &sx = sxs[to];
        if (QUANT) {
#pragma unroll
            for (int n = 0; n < KF; n++)
                asm volatile("" : "+v"(kx[n][0]), "+v"(kx[n][1]));
#pragma unroll
            for (int n = 0; n < 8; n++)
                asm volatile("" : "+v"(vx[n / 4][n % 4]));
        }
        if (t + 32 > seq.len || p.page[0] < 0 || p.page[1] < 0) {
            // tokens that are not there may hold anything: their values are taken as 0, so that 0 times them is 0
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const int there = p.page[s] >= 0 ? seq.len - t - s * 16 - j * 4 : 0;
#pragma unroll
                for (int r = 0; r < 4; r++)
                    vx[s][r] = r < there ? vx[s][r] : 0;
            }
            if (QUANT && lane >= 32)
                sx = (lane & 16 ? p.page[1] : p.page[0]) >= 0 && t + (lane & 31) < seq.len ? sx : 0.0f;
        }
#pragma unroll
        for (int n = 0; n < KF; n++)
            lkv[to][wave * KF + n][lane] = QUANT ? widen<TYPE>(kx[n][0], kx[n][1]) : kx[n];
#pragma unroll
        for (int n = 0; n < VF; n++) {
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t v0 = vx[e / 2][e % 2 * 2], v1 = vx[e / 2][e % 2 * 2 + 1];
                v[e] = QUANT ? R::pack_exact((float)(int8_t)(v0 >> (8 * n)), (float)(int8_t)(v1 >> (8 * n)))
                             : __builtin_amdgcn_perm(v1, v0, n ? 0x07060302u : 0x05040100u);
            }
            lkv[to][2 * KS + wave * VF + n][lane] = v;
        }
        if (QUANT && wave == 0)
            ((float *)lsc[to])[lane] = lane < 32 ? sx * a.scale2 : sx;
    };

    auto tile = [&](int t, int from, const Pages &now, auto MASKED) __attribute__((always_inline)) {
        constexpr bool masked = decltype(MASKED)::value;
        f32x4 kscale[2], vsc[2];
        if (QUANT)
#pragma unroll
            for (int s = 0; s < 2; s++)
                kscale[s] = lsc[from][s * 4 + j], vsc[s] = lsc[from][8 + s * 4 + j];
        f32x4 s[RT][2];
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const u32x4 k = lkv[from][half * KS + ks][lane];
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
                    s[rt][half] = R::mfma(k, q[rt][ks], ks ? s[rt][half] : f32x4{0, 0, 0, 0});
            }
        u32x4 p[RT];
        uint32_t sees[RT]; // a bit for each of the lane's 8 tokens: seen by the row
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            if (masked)
                sees[rt] = seen_by(a, seq, own[rt], t, j, now);
            softmax_step<TYPE, QUANT, masked, VD>(a.scale2, s[rt], kscale, vsc, masked ? sees[rt] : 0, m[rt], l[rt], lsum[rt], unit[rt], per_unit[rt], o[rt], p[rt]);
        }
#pragma unroll
        for (int i = 0; i < VD; i++) {
            u32x4 v = lkv[from][2 * KS + i][lane];
            if (masked && !QUANT && (a.d.mask || seq.count > 1) && __any(strange<TYPE>(v)))
                not_finite<TYPE>(v, sees, o, i);
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
                o[rt][i] = R::mfma(v, p[rt], o[rt][i]);
        }
    };
    if (t0 < t1) {
        const std::integral_constant<int, 0> EVEN;
        const std::integral_constant<int, 1> ODD;
        Pages now = paging.of(t0), next = paging.of(t0 + 32), then = paging.of(t0 + 64);
        load(EVEN, now);
        load(ODD, next);
        const int clear = paging.clear_until(min(min(seq.old, seq.len), t1), t0, lane);
        const int whole = clear > t0 ? (clear - t0) / 64 * 2 : 0, last = (t1 - t0 + 31) / 32; // two tiles at a time, each with its set of registers
        store(EVEN, t0, now);
        load(EVEN, then);
        __syncthreads();
        int t = t0;
        auto turn = [&](auto SET, auto OTHER, auto MASKED) __attribute__((always_inline)) {
            const Pages after = paging.of(t + 96);
            tile(t, decltype(SET)::value, now, MASKED);
            __builtin_amdgcn_sched_barrier(0); // what is done earlier than it is written does not fit the registers
            store(OTHER, t + 32, next);
            load(OTHER, after);
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
            now = next, next = then, then = after, t += 32;
        };
#pragma unroll 1
        for (int i = 0; i < whole; i += 2) {
            turn(EVEN, ODD, std::false_type{});
            turn(ODD, EVEN, std::false_type{});
        }
#pragma unroll 1
        for (int i = whole; i < last; i += 2) {
            turn(EVEN, ODD, std::true_type{});
            if (i + 1 < last)
                turn(ODD, EVEN, std::true_type{});
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        if (QUANT) {
            l[rt] += __shfl_xor(l[rt], 16);
            l[rt] += __shfl_xor(l[rt], 32);
        } else
            l[rt] = lsum[rt][0];
        const int row = r0 + 16 * rt + c;
        if (row >= rows)
            continue;
        const float f = (UNITS<TYPE, QUANT> ? unit[rt] * (1 / RAISED) : 1.0f) * (a.splits > 1 ? 1.0f : l[rt] > 0 ? 1.0f / l[rt] : l[rt] == 0 ? 0.0f : l[rt]);
        const int64_t at = (((int64_t)b * a.cache.heads + h) * a.splits + split) * a.rows + row;
        if (a.splits > 1 && j == 0)
            a.part_ml[2 * at] = m[rt], a.part_ml[2 * at + 1] = l[rt];
        uint16_t *y = (uint16_t *)a.d.o + (int64_t)(seq.row0 + own[rt]) * a.d.o_token + (int64_t)qh[rt] * a.d.o_head;
#pragma unroll
        for (int w = 0; w < 4; w++) { // elements 16 VF w + VF (4 j + r) + n
            float v[4 * VF];
#pragma unroll
            for (int e = 0; e < 4 * VF; e++)
                v[e] = o[rt][w * VF + e % VF][e / VF] * f;
            const int i0 = (16 * w + 4 * j) * VF;
#pragma unroll
            for (int e = 0; e < 4 * VF; e += 4)
                if (a.splits > 1)
                    *(f32x4 *)(a.part_o + at * DIM + i0 + e) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
                else
                    *(u32x2 *)(y + i0 + e) = u32x2{R::pack(v[e], v[e + 1]), R::pack(v[e + 2], v[e + 3])};
        }
    }
}

// Joins the parts of a row: DIM / 4 lanes side by side have its elements, SIDE such groups of a work-group its parts in turn.
template <int TYPE, int DIM, int SIDE>
__global__ __launch_bounds__(256) void kv_attend_join_kernel(const AttendArgs a)
{
    using R = Real16<TYPE>;
    constexpr int LANES = DIM / 4, ROWS = 256 / LANES / SIDE;
    __shared__ f32x4 lo[SIDE > 1 ? 256 : 1];
    __shared__ float ll[SIDE > 1 ? 256 / LANES : 1];
    const int tid = threadIdx.x, i0 = tid % LANES * 4, side = tid / LANES % SIDE;
    const int64_t id = (int64_t)blockIdx.x * ROWS + tid / LANES / SIDE;
    const int bh = (int)(id / a.rows), row = (int)(id % a.rows), b = bh / a.cache.heads, h = bh % a.cache.heads;
    const bool in = bh < a.d.sequences * a.cache.heads;
    const Sequence seq(a, in ? b : 0);
    const bool there = in && row < seq.count * a.group;
    const int64_t at = (int64_t)bh * a.splits * a.rows + row;
    float top = NONE, l = 0;
    f32x4 o = {0, 0, 0, 0};
    if (there) {
#pragma unroll 4
        for (int s = 0; s < a.splits; s++)
            top = fmaxf(top, a.part_ml[2 * (at + (int64_t)s * a.rows)]);
        const float ref = top == NONE ? 0.0f : top;
#pragma unroll 4
        for (int s = side; s < a.splits; s += SIDE) {
            const int64_t p = at + (int64_t)s * a.rows;
            const float f = exp2_fast(a.part_ml[2 * p] - ref);
            l += f * a.part_ml[2 * p + 1];
            o += f * *(const f32x4 *)(a.part_o + p * DIM + i0);
        }
    }
    if (SIDE > 1) {
        lo[SIDE > 1 ? tid : 0] = o;
        if (i0 == 0)
            ll[SIDE > 1 ? tid / LANES : 0] = l;
        __syncthreads();
        if (side > 0)
            return;
#pragma unroll
        for (int u = 1; u < SIDE; u++)
            o += lo[SIDE > 1 ? u * LANES + tid : 0], l += ll[SIDE > 1 ? tid / LANES + u : 0];
    }
    if (!there)
        return;
    const float inv = l > 0 ? 1.0f / l : l == 0 ? 0.0f : l;
    uint16_t *y = (uint16_t *)a.d.o + (int64_t)(seq.row0 + row / a.group) * a.d.o_token + (int64_t)(h * a.group + row % a.group) * a.d.o_head;
    const u32x2 w = {R::pack(o[0] * inv, o[1] * inv), R::pack(o[2] * inv, o[3] * inv)};
    *(u32x2 *)(y + i0) = w;
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
struct AttendShape {
    int rt, row_blocks, rows, splits; // rt: 16-row blocks of a wave; 8: the wide kernel's work-group
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
    HIPQ_REQUIRE(d->blocks_per_sequence >= 0 && (int64_t)d->blocks_per_sequence * c->page <= ((int64_t)1 << 30), "attend: %d blocks of a sequence", d->blocks_per_sequence);
    HIPQ_REQUIRE(d->blocks_stride >= d->blocks_per_sequence || d->sequences <= 1, "attend: rows of blocks overlap");
    HIPQ_REQUIRE(d->longest >= 0, "attend: the longest sequence has %d tokens", d->longest);
    HIPQ_REQUIRE(d->scale > 0 && d->scale < 1e30f, "attend: scale %g", (double)d->scale);
    const int64_t rows = (int64_t)d->most_new * (d->q_heads / c->heads);
    HIPQ_REQUIRE(rows < (1 << 24), "attend: %lld rows of a sequence", (long long)rows);
    return 0;
}

static AttendShape shape_of(const hipq_kv_cache *c, const hipq_kv_attend_desc *d)
{
    AttendShape s = {};
    const int group = d->q_heads / c->heads;
    s.rows = d->most_new * group;
    s.rt = s.rows <= 16 || c->dim == 256 ? 1 : 2; // two blocks of 256-wide outputs are all of a wave's registers
    const int64_t longest = d->longest < (int64_t)d->blocks_per_sequence * c->page ? d->longest : (int64_t)d->blocks_per_sequence * c->page;
    // The wide kernel, where it has work for the whole chip, two work-groups a CU with the longest sequences: us against the other
    // kernel's, 16 trees of 32 tokens on up to 8000 in 8 bits 111 against 121, of 17 tokens 105 against 103; in 16 bits 8 x 32 on up to 4096 44
    // against 55, 2 x 64 on up to 16000 65 against 89, 41 chains of 34 on up to 825 43 against 53; with less, 64 on 500 of 4 heads, 22 against
    // 14, and with heads of 64, 24 on up to 4000, 25 against 21.5.  (256 work-groups: 168, 48 and 81 of the first, third and fourth.)
    const int64_t wide = (int64_t)d->sequences * c->heads * ((s.rows + 127) / 128);
    if (c->dim == 128 && s.rows > 64 && wide * ((longest + 255) / 256) >= 256)
        s.rt = 8;
    s.row_blocks = (s.rows + 16 * s.rt - 1) / (16 * s.rt);
    const int64_t items = (int64_t)d->sequences * c->heads * s.row_blocks;
    // A work-group a CU is enough, and two where that leaves some with a longer sequence than others: us with 256, 512 and 1024 work-groups of
    // 8 trees of 16 tokens on 4096: 38, 42, 54; one token on 2 x 131072: 186, 197, 201; of 32 sequences up to 4096 in 8 bits: 62, 52, 55
    const int64_t target = items < 256 ? 256 : 512, want = s.rt == 8 ? 512 / (items > 512 ? 512 : items) : items ? (target + items - 1) / items : 1, most = (longest + 255) / 256;
    s.splits = (int)(want < most ? want : most);
    s.splits = s.splits < 1 ? 1 : s.splits > 64 ? 64 : s.splits;
    if (s.splits > 1)
        s.workspace = (size_t)d->sequences * c->heads * s.splits * s.rows * (c->dim + 2) * sizeof(float);
    return s;
}

template <int TYPE, int DIM, bool QUANT, int RT>
static int launch_attend(const AttendArgs &a, int64_t items, hipStream_t st)
{
    const size_t lds = (2 * 4 * RT * 16) * 4 + (size_t)2 * RT * (DIM / 16) * 64 * 16 + (RT > 1 ? (size_t)RT * (DIM / 32) * 1024 : 0);
    static_assert((2 * 4 * RT * 16) * 4 + 2 * RT * (DIM / 16) * 64 * 16 + RT * (DIM / 32) * 1024 <= 65536, "more LDS than a launch has without asking");
    kv_attend_kernel<TYPE, DIM, QUANT, RT><<<dim3((unsigned)((items * a.splits + 7) / 8 * 8)), dim3(256), lds, st>>>(a);
    return launch_status("kv_attend_kernel");
}

template <int TYPE, int DIM, bool QUANT>
static int launch_attend(const AttendArgs &a, int rt, int64_t items, hipStream_t st)
{
    if (rt == 8) {
        if constexpr (DIM == 128)
            kv_attend_wide_kernel<TYPE, DIM, QUANT><<<dim3((unsigned)((items * a.splits + 7) / 8 * 8)), dim3(256), 0, st>>>(a);
        return launch_status("kv_attend_wide_kernel");
    }
    return rt == 1 ? launch_attend<TYPE, DIM, QUANT, 1>(a, items, st) : launch_attend<TYPE, DIM, QUANT, DIM == 256 ? 1 : 2>(a, items, st);
}

template <int TYPE, int DIM>
static int launch_attend(const AttendArgs &a, int rt, int64_t items, hipStream_t st)
{
    if (a.cache.quantized ? launch_attend<TYPE, DIM, true>(a, rt, items, st) : launch_attend<TYPE, DIM, false>(a, rt, items, st))
        return 1;
    if (a.splits == 1)
        return 0;
    // few rows of many parts: the parts side by side, all groups of a work-group at one row
    const int64_t rows = (int64_t)a.d.sequences * a.cache.heads * a.rows;
    constexpr int GROUPS = 1024 / DIM;
    if (rows <= 4096 && a.splits >= 8)
        kv_attend_join_kernel<TYPE, DIM, GROUPS><<<dim3((unsigned)rows), dim3(256), 0, st>>>(a);
    else
        kv_attend_join_kernel<TYPE, DIM, 1><<<dim3((unsigned)((rows + GROUPS - 1) / GROUPS)), dim3(256), 0, st>>>(a);
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
    // item numbers are 32 bits, and of 2^32 work-items and more only what is left over would run
    HIPQ_REQUIRE(items * s.splits * 16 * s.rt < ((int64_t)1 << 31) && items * s.splits <= (1 << 24) - 8, "attend: %lld work-groups", (long long)items * s.splits);
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
