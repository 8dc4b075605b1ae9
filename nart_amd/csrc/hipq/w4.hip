// Products with 4-bit weights and group scales (hipq_w4_*): y[m][n] = sum_g s[n][g] sum_{k in g} x[m][k] (q[n][k] - z[n][g]).  gfx950 only.
//
// The arithmetic of every kernel here.  A weight's four bits become a 16-bit float without a conversion: with the bits at the right place
// of a half dword, one v_and_or makes two floats 16 + q (16 = 2^4 has q's unit at mantissa bit 3 of a bfloat16, bit 6 of a float16), exactly;
// seven instructions make eight of them.  The 16 and the zero point come off behind the product, where x is already summed: with
// X = sum of x over the group, sum x (q - z) = sum x (16 + q) - (16 + z) X.  Both sums are float32; the terms are at most 31 / 8 as
// large as with centred weights, so the difference keeps 21 bits.  The group's sum is then scaled and added in float32: the
// weights themselves are never rounded.
//
// Layout.  k runs in blocks of 128, rows of weights in tiles of 16.  The 1 KB of a tile and block lies together, a lane's 16 bytes the
// operand of four multiplies: dword t holds k = 32 t + 8 (lane / 16) + 0..7 of row lane % 16, bits of element 2 i at 4 i + SHIFT, of element
// 2 i + 1 at 16 + 4 i + SHIFT, rotated at the word's end.  Scales and zero points of a tile and block lie together row by row.
#include <new>

#include "real16.h"

namespace hipq {

struct W4Args {
    const uint8_t *q;       // [tile][block][lane][16 bytes]
    const uint16_t *scales; // [tile][block][row][groups of a block]
    const uint8_t *zeros;   // the same, or nullptr: 8
    const uint16_t *bias;   // [tile][16], or nullptr
    const uint16_t *x;
    uint16_t *y;
    int64_t x_stride, y_stride;
    const float *xsum; // tile kernel: [block][group of the block][m_pad], minus the sums of x (times 24 where there are no zero points)
    int M, N, K, blocks, m_pad;
    int activation; // with one, tiles 2 i and 2 i + 1 hold rows 16 i .. 16 i + 15 of the gate and of the other projection
};

template <int TYPE>
struct Nibbles;
template <>
struct Nibbles<HIPQ_REAL_BF16> {
    static constexpr int SHIFT = 3;
    static constexpr uint32_t MASK = 0x00780078u, BASE = 0x41804180u, MINUS_ONE = 0xbf80bf80u;
};
template <>
struct Nibbles<HIPQ_REAL_F16> {
    static constexpr int SHIFT = 6;
    static constexpr uint32_t MASK = 0x03c003c0u, BASE = 0x4c004c00u, MINUS_ONE = 0xbc00bc00u;
};

// eight floats 16 + q
template <int TYPE>
__device__ static __forceinline__ u32x4 spread(uint32_t w)
{
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++)
        o[i] = (__builtin_amdgcn_alignbit(w, w, 4 * i) & Nibbles<TYPE>::MASK) | Nibbles<TYPE>::BASE;
    return o;
}

__device__ static __forceinline__ float activate(float v, int activation)
{
    // v / (1 + exp(-v)), and with gelu v / (1 + exp(-2 sqrt(2 / pi) (v + 0.044715 v^3))); exp overflows to infinity and v / inf is 0
    const float t = activation == HIPQ_ACT_SILU ? v : 1.5957691216057308f * (v + 0.044715f * v * v * v);
    return v / (1.0f + exp2_fast(-1.4426950408889634f * t));
}

template <int TYPE>
__device__ static __forceinline__ uint16_t rounded(float v) { return (uint16_t)Real16<TYPE>::pack(v, 0.0f); }

// GPB 16-bit scales, GPB bytes of zero points
template <int GPB>
struct Groups {
    uint32_t s[(GPB + 1) / 2], z;
    __device__ __forceinline__ void load(const W4Args &a, size_t at)
    {
        if (GPB == 1)
            s[0] = a.scales[at];
        else if (GPB == 2)
            s[0] = *(const uint32_t *)(a.scales + at);
        else {
            const u32x2 v = *(const u32x2 *)(a.scales + at);
            s[0] = v[0], s[(GPB + 1) / 2 - 1] = v[1];
        }
        z = 0x08080808u;
        if (a.zeros)
            z = GPB == 1 ? a.zeros[at] : GPB == 2 ? *(const uint16_t *)(a.zeros + at) : *(const uint32_t *)(a.zeros + at);
    }
    template <int TYPE>
    __device__ __forceinline__ float scale(int g) const { return g & 1 ? Real16<TYPE>::high(s[g / 2]) : Real16<TYPE>::low(s[g / 2]); }
    __device__ __forceinline__ float offset(int g) const { return 16.0f + (float)((z >> (8 * g)) & 255); }
};

// ---- few rows: a stream of weights ---------------------------------------------------------------------------------------
// Every weight is used by at most 16 MT rows, so the time is what it takes to read the weights, and what counts is how much of them is
// in flight: a work-group owns NT tiles and 16 MT rows, its waves take the blocks of k in turn, each DEPTH blocks ahead and straight
// into registers (a tile's block is 1 KB, in one load), and their sums meet once, in LDS.  No barrier in the loop.
template <int TYPE, int GPB, int MT, int NT, int WAVES, int DEPTH>
__global__ __launch_bounds__(WAVES * 64) void w4_stream_kernel(const W4Args a)
{
    using R = Real16<TYPE>;
    __shared__ f32x4 red[WAVES][MT * NT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, j = lane >> 4;
    const int tile0 = blockIdx.x * NT, m0 = blockIdx.y * (16 * MT);

    u32x4 w[DEPTH][NT], xa[DEPTH][MT][4];
    Groups<GPB> gs[DEPTH][NT];
    f32x4 total[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
            total[mt][nt] = f32x4{0, 0, 0, 0};
    const uint16_t *xrow[MT];
    bool row[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int m = m0 + 16 * mt + c;
        row[mt] = m < a.M;
        xrow[mt] = a.x + (row[mt] ? m : 0) * a.x_stride + 8 * j;
    }
    auto load = [&](int d, int kb) {
        if (kb < a.blocks) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const size_t at = (size_t)(tile0 + nt) * a.blocks + kb;
                w[d][nt] = *(const u32x4 *)(a.q + at * 1024 + lane * 16);
                gs[d][nt].load(a, (at * 16 + c) * GPB);
            }
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    xa[d][mt][t] = u32x4{0, 0, 0, 0};
                    if (row[mt] && kb * 128 + t * 32 < a.K)
                        xa[d][mt][t] = *(const u32x4 *)(xrow[mt] + kb * 128 + t * 32);
                }
        }
    };
    const u32x4 minus_one = {Nibbles<TYPE>::MINUS_ONE, Nibbles<TYPE>::MINUS_ONE, Nibbles<TYPE>::MINUS_ONE, Nibbles<TYPE>::MINUS_ONE};
    auto compute = [&](int d) {
        u32x4 f[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int t = 0; t < 4; t++)
                f[nt][t] = spread<TYPE>(w[d][nt][t]);
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int g = 0; g < GPB; g++) {
                f32x4 less = {0, 0, 0, 0}; // minus the sums of x, in every column
#pragma unroll
                for (int t = g * 4 / GPB; t < (g + 1) * 4 / GPB; t++)
                    less = R::mfma(xa[d][mt][t], minus_one, less);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    f32x4 sum = less * gs[d][nt].offset(g);
#pragma unroll
                    for (int t = g * 4 / GPB; t < (g + 1) * 4 / GPB; t++)
                        sum = R::mfma(xa[d][mt][t], f[nt][t], sum);
                    const float s = gs[d][nt].template scale<TYPE>(g);
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        total[mt][nt][r] = __builtin_fmaf(s, sum[r], total[mt][nt][r]);
                }
            }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
        load(d, wave + d * WAVES);
    for (int kb = wave; kb < a.blocks; kb += DEPTH * WAVES) {
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
            if (kb + d * WAVES < a.blocks) {
                compute(d);
                load(d, kb + (d + DEPTH) * WAVES);
            }
    }
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
            red[wave][mt * NT + nt][lane] = total[mt][nt];
    __syncthreads();

    auto sum_of = [&](int t, int l) {
        f32x4 v = red[0][t][l];
#pragma unroll
        for (int o = 1; o < WAVES; o++)
            v += red[o][t][l];
        if (a.bias) {
            const float b = Real16<TYPE>::low(a.bias[(tile0 + t % NT) * 16 + (l & 15)]);
            v += b;
        }
        return v;
    };
    const bool gated = a.activation != HIPQ_ACT_NONE;
    const int per = gated ? 2 : 1; // tiles of a result
    for (int i = tid; i < MT * NT * 64 / per; i += WAVES * 64) {
        const int l = i & 63, t = (i >> 6) * per;
        f32x4 v = sum_of(t, l);
        if (NT % 2 == 0 && gated) {
            const f32x4 up = sum_of(t + 1, l);
#pragma unroll
            for (int r = 0; r < 4; r++)
                v[r] = activate(v[r], a.activation) * up[r];
        }
        const int n = (tile0 + t % NT) / per * 16 + (l & 15), m = m0 + t / NT * 16 + (l >> 4) * 4;
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (n < a.N && m + r < a.M)
                a.y[(m + r) * a.y_stride + n] = rounded<TYPE>(v[r]);
    }
}

// ---- many rows: tiles --------------------------------------------------------------------------------------------------------
typedef const uint32_t __attribute__((address_space(1))) *gptr_t;
typedef uint32_t __attribute__((address_space(3))) *lptr_t;

// Minus the sums of x over each group, for the tile kernel: a thread has 8 of x, the group's threads are neighbours.
template <int TYPE, int GPB>
__global__ __launch_bounds__(256) void w4_xsum_kernel(const W4Args a, float *xsum, float factor)
{
    using R = Real16<TYPE>;
    const int per_row = a.blocks * 16;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, m = id / per_row;
    const int k8 = (int)(id - m * per_row);
    float s = 0;
    if (m < a.M && k8 * 8 < a.K) {
        const u32x4 v = *(const u32x4 *)(a.x + m * a.x_stride + k8 * 8);
#pragma unroll
        for (int i = 0; i < 4; i++)
            s += R::low(v[i]) + R::high(v[i]);
    }
#pragma unroll
    for (int o = 1; o < 16 / GPB; o *= 2)
        s += __shfl_xor(s, o);
    if (m < a.m_pad && k8 % (16 / GPB) == 0)
        xsum[(size_t)(k8 / (16 / GPB)) * a.m_pad + m] = factor * s;
}

// A work-group of eight waves computes 128 rows x 16 tiles (256 columns), a wave 64 rows x 4 tiles.  The rows' block of k goes through LDS,
// put there by the load unit one block ahead (16-byte piece p of row m at piece p ^ (m % 16), so that the 16 rows of an operand
// fall on different banks); a wave's weights go straight to its registers, one block ahead as well, in the order that the multiplies take.
template <int TYPE, int GPB, bool ZEROS>
__global__ __launch_bounds__(512, 1) void w4_tile_kernel(const W4Args a, int tiles_m, int tiles_n)
{
    using R = Real16<TYPE>;
    constexpr int STAGE = 128 * 256, XS = GPB * 512;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * (STAGE + XS)];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, j = lane >> 4;
    // work-groups go to the 8 XCDs in turn: XCD x takes the x-th contiguous eighth, column by column, so that its L2 holds the weights
    const int count = tiles_m * tiles_n, part = (count + 7) / 8, item = (int)(blockIdx.x % 8) * part + (int)(blockIdx.x / 8);
    if (item >= count)
        return;
    const int m0 = item % tiles_m * 128, tile0 = item / tiles_m * 16;
    const int wm = wave & 1, wn = wave >> 1;

    auto issue = [&](int kb, int stage) {
        uint8_t *to = lds + stage * (STAGE + XS);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = (wave * 4 + i) * 4 + j, m = min(m0 + r, a.M - 1);
            int k = kb * 128 + (c ^ (r & 15)) * 8;
            k = k < a.K ? k : 0; // behind the last k: read anything, nothing multiplies it
            __builtin_amdgcn_global_load_lds((gptr_t)(a.x + m * a.x_stride + k), (lptr_t)(to + (wave * 4 + i) * 1024), 16, 0, 0);
        }
        if (wave < 2 * GPB)
            __builtin_amdgcn_global_load_lds((gptr_t)(a.xsum + (size_t)(kb * GPB + (wave >> 1)) * a.m_pad + m0 + (wave & 1) * 64 + lane),
                                             (lptr_t)(to + STAGE + (wave >> 1) * 512 + (wave & 1) * 256), 4, 0, 0);
    };
    u32x4 w[2][4];
    Groups<GPB> gs[2][4];
    auto weights = [&](int kb, int d) {
#pragma unroll
        for (int nt = 0; nt < 4; nt++) {
            const size_t at = (size_t)(tile0 + wn * 4 + nt) * a.blocks + kb;
            w[d][nt] = *(const u32x4 *)(a.q + at * 1024 + lane * 16);
            gs[d][nt].load(a, (at * 16 + c) * GPB);
        }
    };
    f32x4 total[4][4];
#pragma unroll
    for (int mt = 0; mt < 4; mt++)
#pragma unroll
        for (int nt = 0; nt < 4; nt++)
            total[mt][nt] = f32x4{0, 0, 0, 0};
    auto compute = [&](int kb, int stage, int d) {
        const uint8_t *from = lds + stage * (STAGE + XS);
        f32x4 sum[4][4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            if (kb * 128 + t * 32 < a.K) {
                constexpr int PER = 4 / GPB;
                const int g = t / PER;
                u32x4 xa[4];
#pragma unroll
                for (int mt = 0; mt < 4; mt++)
                    xa[mt] = *(const u32x4 *)(from + (wm * 64 + mt * 16 + c) * 256 + (((t * 4 + j) ^ c) * 16));
                if (t % PER == 0) {
#pragma unroll
                    for (int mt = 0; mt < 4; mt++) {
                        const f32x4 less = *(const f32x4 *)(from + STAGE + g * 512 + (wm * 64 + mt * 16 + j * 4) * 4);
#pragma unroll
                        for (int nt = 0; nt < 4; nt++)
                            sum[mt][nt] = ZEROS ? less * gs[d][nt].offset(g) : less;
                    }
                }
#pragma unroll
                for (int nt = 0; nt < 4; nt++) {
                    const u32x4 f = spread<TYPE>(w[d][nt][t]);
#pragma unroll
                    for (int mt = 0; mt < 4; mt++)
                        sum[mt][nt] = R::mfma(xa[mt], f, sum[mt][nt]);
                }
            }
            constexpr int PER = 4 / GPB;
            if (t % PER == PER - 1) {
                const int g = t / PER;
                if (kb * 128 + g * PER * 32 < a.K) {
#pragma unroll
                    for (int nt = 0; nt < 4; nt++) {
                        const float s = gs[d][nt].template scale<TYPE>(g);
#pragma unroll
                        for (int mt = 0; mt < 4; mt++)
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                total[mt][nt][r] = __builtin_fmaf(s, sum[mt][nt][r], total[mt][nt][r]);
                    }
                }
            }
        }
    };
    issue(0, 0);
    weights(0, 0);
    for (int kb = 0; kb < a.blocks; kb += 2) {
#pragma unroll
        for (int d = 0; d < 2; d++)
            if (kb + d < a.blocks) {
                // this block has arrived, and every wave is done with the stage that the next one goes to
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                if (kb + d + 1 < a.blocks) {
                    issue(kb + d + 1, 1 - d);
                    weights(kb + d + 1, 1 - d);
                }
                compute(kb + d, d, d);
            }
    }
    const bool gated = a.activation != HIPQ_ACT_NONE;
#pragma unroll
    for (int nt = 0; nt < 4; nt++) {
        const int tile = tile0 + wn * 4 + nt;
        const float b = a.bias ? R::low(a.bias[tile * 16 + c]) : 0.0f;
#pragma unroll
        for (int mt = 0; mt < 4; mt++)
            total[mt][nt] += b;
    }
#pragma unroll
    for (int nt = 0; nt < 4; nt++) {
        if (gated && nt % 2)
            continue;
        const int tile = tile0 + wn * 4 + nt, n = (gated ? tile / 2 : tile) * 16 + c;
#pragma unroll
        for (int mt = 0; mt < 4; mt++) {
            const int m = m0 + wm * 64 + mt * 16 + j * 4;
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (n < a.N && m + r < a.M)
                    a.y[(m + r) * a.y_stride + n] = rounded<TYPE>(gated ? activate(total[mt][nt][r], a.activation) * total[mt][nt | 1][r] : total[mt][nt][r]);
        }
    }
}

// ---- setup ---------------------------------------------------------------------------------------------------------------------
struct PackArgs {
    const uint8_t *q, *zeros;
    const uint16_t *scales, *bias;
    uint8_t *to_q, *to_zeros;
    uint16_t *to_scales, *to_bias;
    int rows, K, group, groups, blocks, tiles, gated; // rows: of one projection
    int shift;
};

// the row of the caller's arrays that row r of a tile holds, -1: none
__device__ static __forceinline__ int64_t source_row(const PackArgs &p, int tile, int r)
{
    const int n = (p.gated ? tile / 2 : tile) * 16 + r;
    return n < p.rows ? (int64_t)n + (p.gated && tile % 2 ? p.rows : 0) : -1;
}

__global__ __launch_bounds__(256) void w4_pack_kernel(const PackArgs p)
{
    const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
    const int gpb = 128 / p.group;
    const int64_t items = (int64_t)p.tiles * p.blocks;
    for (int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); item < items; item += (int64_t)gridDim.x * 4) {
        const int tile = (int)(item / p.blocks), kb = (int)(item % p.blocks);
        const int64_t row = source_row(p, tile, c);
        u32x4 o;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            uint32_t v = 0;
            const int k = kb * 128 + t * 32 + j * 8;
            if (row >= 0 && k < p.K)
                for (int e = 0; e < 8; e++) {
                    const uint32_t b = p.q[row * (p.K / 2) + k / 2 + e / 2];
                    v |= ((e & 1 ? b >> 4 : b) & 15) << (4 * (e / 2) + 16 * (e & 1));
                }
            o[t] = (v << p.shift) | (v >> (32 - p.shift));
        }
        *(u32x4 *)(p.to_q + item * 1024 + lane * 16) = o;
        if (lane < 16)
            for (int g = 0; g < gpb; g++) {
                const int from = kb * gpb + g;
                const bool there = row >= 0 && from < p.groups;
                p.to_scales[(item * 16 + c) * gpb + g] = there ? p.scales[row * p.groups + from] : 0;
                if (p.zeros)
                    p.to_zeros[(item * 16 + c) * gpb + g] = there ? p.zeros[row * p.groups + from] & 15 : 8;
            }
        if (p.bias && kb == 0 && lane < 16)
            p.to_bias[tile * 16 + c] = row >= 0 ? p.bias[row] : 0;
    }
}

static int round_up(int v, int to) { return (v + to - 1) / to * to; }

} // namespace hipq

using namespace hipq;

struct hipq_w4_plan {
    hipq_w4_desc desc;
    int device, blocks, tiles; // tiles: those with rows; memory holds a multiple of 16
    uint8_t *memory;
    W4Args args;
};

extern "C" int hipq_w4_plan_create(const hipq_w4_desc *d, const uint8_t *q, const void *scales, const uint8_t *zeros, const void *bias, void *stream,
                                   hipq_w4_plan **out)
{
    clear_error();
    HIPQ_REQUIRE(d && q && scales && out, "w4: a null pointer");
    HIPQ_REQUIRE(is_real16(d->type), "w4: type %d is neither float16 nor bfloat16", d->type);
    HIPQ_REQUIRE(d->group == 32 || d->group == 64 || d->group == 128, "w4: groups of %d (32, 64 and 128 are there)", d->group);
    HIPQ_REQUIRE(d->activation >= HIPQ_ACT_NONE && d->activation <= HIPQ_ACT_GELU, "w4: activation %d", d->activation);
    HIPQ_REQUIRE(d->N >= 1 && d->N <= (1 << 26), "w4: %d outputs", d->N);
    HIPQ_REQUIRE(d->K >= 32 && d->K <= (1 << 24) && d->K % 32 == 0, "w4: %d inputs (a multiple of 32 is needed)", d->K);
    const int gated = d->activation != HIPQ_ACT_NONE, gpb = 128 / d->group;
    hipq_w4_plan *p = new (std::nothrow) hipq_w4_plan();
    HIPQ_REQUIRE(p, "w4: out of host memory");
    p->desc = *d;
    p->blocks = (d->K + 127) / 128;
    p->tiles = (d->N + 15) / 16 * (gated ? 2 : 1);
    const size_t tiles = round_up(p->tiles, 16), pieces = tiles * p->blocks;
    const size_t q_bytes = pieces * 1024, s_bytes = pieces * 16 * gpb * 2, z_bytes = zeros ? pieces * 16 * gpb : 0, b_bytes = bias ? tiles * 32 : 0;
    hipError_t e = hipGetDevice(&p->device);
    if (e == hipSuccess)
        e = hipMalloc(&p->memory, q_bytes + s_bytes + z_bytes + b_bytes);
    if (e != hipSuccess) {
        delete p;
        return fail("w4: no memory for %zu bytes of weights: %s", q_bytes + s_bytes + z_bytes + b_bytes, hipGetErrorString(e));
    }
    PackArgs k = {};
    k.q = q, k.zeros = zeros, k.scales = (const uint16_t *)scales, k.bias = (const uint16_t *)bias;
    k.to_q = p->memory, k.to_scales = (uint16_t *)(p->memory + q_bytes), k.to_zeros = p->memory + q_bytes + s_bytes;
    k.to_bias = (uint16_t *)(p->memory + q_bytes + s_bytes + z_bytes);
    k.rows = d->N, k.K = d->K, k.group = d->group, k.groups = (d->K + d->group - 1) / d->group, k.blocks = p->blocks, k.tiles = (int)tiles, k.gated = gated;
    k.shift = d->type == HIPQ_REAL_BF16 ? Nibbles<HIPQ_REAL_BF16>::SHIFT : Nibbles<HIPQ_REAL_F16>::SHIFT;
    const size_t groups = (pieces + 3) / 4;
    w4_pack_kernel<<<dim3((unsigned)(groups < 16384 ? groups : 16384)), dim3(256), 0, (hipStream_t)stream>>>(k);
    int bad = launch_status("w4_pack_kernel");
    if (!bad && (e = hipStreamSynchronize((hipStream_t)stream)) != hipSuccess)
        bad = fail("w4: laying the weights out failed: %s", hipGetErrorString(e));
    if (bad) {
        (void)hipFree(p->memory);
        delete p;
        return 1;
    }
    W4Args &a = p->args;
    a.q = k.to_q, a.scales = k.to_scales, a.zeros = zeros ? k.to_zeros : nullptr, a.bias = bias ? k.to_bias : nullptr;
    a.N = d->N, a.K = d->K, a.blocks = p->blocks, a.activation = d->activation;
    *out = p;
    return 0;
}

extern "C" void hipq_w4_plan_destroy(hipq_w4_plan *p)
{
    if (!p)
        return;
    (void)hipFree(p->memory); // waits for what still reads it
    delete p;
}

namespace hipq {

enum { KERNEL_STREAM_1, KERNEL_STREAM_2, KERNEL_STREAM_4, KERNEL_TILE };

static int kernel_of(const hipq_w4_plan *p, int M)
{
    return M <= 16 ? KERNEL_STREAM_1 : M <= 32 ? KERNEL_STREAM_2 : M <= 192 ? KERNEL_STREAM_4 : KERNEL_TILE;
}

template <int TYPE, int GPB, int MT, int NT, int WAVES, int DEPTH>
static int launch_stream(const hipq_w4_plan *p, const W4Args &a, hipStream_t st)
{
    const dim3 grid((p->tiles + NT - 1) / NT, (a.M + 16 * MT - 1) / (16 * MT));
    w4_stream_kernel<TYPE, GPB, MT, NT, WAVES, DEPTH><<<grid, dim3(WAVES * 64), 0, st>>>(a);
    return launch_status("w4_stream_kernel");
}

template <int TYPE, int GPB>
static int launch(const hipq_w4_plan *p, W4Args &a, void *workspace, hipStream_t st)
{
    switch (kernel_of(p, a.M)) {
    case KERNEL_STREAM_1:
        return p->desc.activation ? launch_stream<TYPE, GPB, 1, 2, 8, 4>(p, a, st) : launch_stream<TYPE, GPB, 1, 1, 8, 4>(p, a, st);
    case KERNEL_STREAM_2:
        return launch_stream<TYPE, GPB, 2, 2, 8, 2>(p, a, st);
    case KERNEL_STREAM_4:
        return launch_stream<TYPE, GPB, 4, 2, 4, 1>(p, a, st);
    }
    a.m_pad = round_up(a.M, 128);
    a.xsum = (const float *)workspace;
    const int64_t threads = (int64_t)a.m_pad * a.blocks * 16;
    w4_xsum_kernel<TYPE, GPB><<<dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st>>>(a, (float *)workspace, a.zeros ? -1.0f : -24.0f);
    if (launch_status("w4_xsum_kernel"))
        return 1;
    const int tiles_m = a.m_pad / 128, tiles_n = (p->tiles + 15) / 16;
    const dim3 grid((tiles_m * tiles_n + 7) / 8 * 8);
    if (a.zeros)
        w4_tile_kernel<TYPE, GPB, true><<<grid, dim3(512), 0, st>>>(a, tiles_m, tiles_n);
    else
        w4_tile_kernel<TYPE, GPB, false><<<grid, dim3(512), 0, st>>>(a, tiles_m, tiles_n);
    return launch_status("w4_tile_kernel");
}

template <int TYPE>
static int launch(const hipq_w4_plan *p, W4Args &a, void *workspace, hipStream_t st)
{
    return p->desc.group == 128 ? launch<TYPE, 1>(p, a, workspace, st) : p->desc.group == 64 ? launch<TYPE, 2>(p, a, workspace, st) : launch<TYPE, 4>(p, a, workspace, st);
}

} // namespace hipq

extern "C" const char *hipq_w4_plan_kernel(const hipq_w4_plan *p, int M)
{
    if (!p || M < 0 || M > (1 << 24))
        return "";
    static const char *const names[] = {"w4_stream_16", "w4_stream_32", "w4_stream_64", "w4_tile_128x256"};
    return names[kernel_of(p, M)];
}

extern "C" size_t hipq_w4_workspace(const hipq_w4_plan *p, int M)
{
    if (!p || M <= 0 || M > (1 << 24) || kernel_of(p, M) != KERNEL_TILE)
        return 0;
    return (size_t)round_up(M, 128) * p->blocks * (128 / p->desc.group) * sizeof(float);
}

extern "C" int hipq_w4_run(const hipq_w4_plan *p, const void *x, int64_t x_stride, void *y, int64_t y_stride, int M, void *workspace,
                           size_t workspace_bytes, void *stream)
{
    clear_error();
    HIPQ_REQUIRE(p, "w4: a null plan");
    HIPQ_REQUIRE(M >= 0 && M <= (1 << 24), "w4: %d rows", M);
    if (M == 0)
        return 0;
    HIPQ_REQUIRE(x && y, "w4: a null pointer");
    HIPQ_REQUIRE((uintptr_t)x % 16 == 0 && x_stride % 8 == 0, "w4: rows of x have to start at multiples of 16 bytes");
    HIPQ_REQUIRE((uintptr_t)y % 2 == 0, "w4: y is not aligned to its type");
    HIPQ_REQUIRE(M == 1 || (x_stride >= p->desc.K && y_stride >= p->desc.N), "w4: rows overlap (strides %lld and %lld)", (long long)x_stride, (long long)y_stride);
    const size_t need = hipq_w4_workspace(p, M);
    HIPQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), "w4: a workspace of %zu bytes is needed", need);
    int device;
    HIPQ_CHECK_HIP(hipGetDevice(&device));
    HIPQ_REQUIRE(device == p->device, "w4: the plan is on device %d, the current one is %d", p->device, device);
    W4Args a = p->args;
    a.x = (const uint16_t *)x, a.y = (uint16_t *)y, a.x_stride = x_stride, a.y_stride = y_stride, a.M = M;
    return p->desc.type == HIPQ_REAL_BF16 ? launch<HIPQ_REAL_BF16>(p, a, workspace, (hipStream_t)stream)
                                          : launch<HIPQ_REAL_F16>(p, a, workspace, (hipStream_t)stream);
}
