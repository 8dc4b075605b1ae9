// Products with 4-bit weights and group scales (hipq_w4_*): y[m][n] = sum_g s[n][g] sum_{k in g} x[m][k] (q[n][k] - z[n][g]).  gfx950 only.
//
// The arithmetic of every kernel here.  A weight's four bits become a 16-bit float without a conversion: with the bits at the right place
// of a half dword, one v_and_or makes two floats 32 + q (32 = 2^5 has q's unit at mantissa bit 2 of a bfloat16, bit 5 of a float16), exactly;
// seven instructions make eight of them.  The 32 and the zero point come off behind the product, where x is already summed: with
// X = sum of x over the group, sum x (q - z) = sum x (32 + q) - (32 + z) X.  Where a zero point would then cost more instructions for the sums
// than for the weights, 16 - z is added to the mantissas as an integer (to 48 + q - z, below 64), and 48 X comes off for all columns alike,
// as the matrix product's own initial value.  Both sums are float32: a term is up to 63 |x|, however little of it is left, so beside the
// rounding to 16 bits a group's result is off by a few 2^-24 of 63 sum |x| times its scale (of numbers of either sign, whose running sums are
// smaller, of 63 sqrt(sum x^2)).  Infinities meet their opposites, and are NaN.
// The group's sum is then scaled and added in float32: the weights themselves are never rounded.
//
// Layout.  k runs in blocks of 128, rows of weights in tiles of 16.  The 1 KB of a tile and block lies together (weights_at), a lane's 16 bytes the
// operand of four multiplies: dword t holds k = 32 t + 8 (lane / 16) + 0..7 of row lane % 16, bits of element 2 i at 4 i + SHIFT, of element
// 2 i + 1 at 16 + 4 i + SHIFT, rotated at the word's end.  Scales and zero points of a tile and block lie together row by row.
#include <new>
#include <type_traits>

#include "overlap.h"
#include "real16.h"

namespace hipq {

struct W4Args {
    const uint8_t *q;       // [tile / 8][block][tile % 8][lane][16 bytes]
    const uint8_t *scales;  // [tile / 4][block][tile % 4][row], see Scales
    bool zeros;             // with zero points; otherwise they are 8
    const uint16_t *bias;   // [tile][16], or nullptr
    const uint16_t *x;
    uint16_t *y;
    int64_t x_stride, y_stride;
    const uint16_t *nothing; // 16 bytes of zeros: in the place of x behind the last k
    const float *xsum; // tile kernel: [block][group of the block][m_pad], sums of x times what the kernel adds them with (W4Tile::FACTOR)
    int M, N, K, blocks, m_pad;
    int activation; // with one, tiles 2 i and 2 i + 1 hold rows 16 i .. 16 i + 15 of the gate and of the other projection
};

template <int TYPE>
struct Nibbles;
template <>
struct Nibbles<HIPQ_REAL_BF16> {
    static constexpr int SHIFT = 2;
    static constexpr uint32_t MASK = 0x003c003cu, BASE = 0x42004200u, MINUS_ONE = 0xbf80bf80u, MINUS_40 = 0xc220c220u, MINUS_48 = 0xc240c240u;
};
template <>
struct Nibbles<HIPQ_REAL_F16> {
    static constexpr int SHIFT = 5;
    static constexpr uint32_t MASK = 0x01e001e0u, BASE = 0x50005000u, MINUS_ONE = 0xbc00bc00u, MINUS_40 = 0xd100d100u, MINUS_48 = 0xd200d200u;
};

// eight floats 32 + q.  The two constants sit in registers that the compiler knows nothing about: as literals they would not fit one
// v_and_or, and two instructions would do its work
template <int TYPE>
struct Spread {
    uint32_t mask = Nibbles<TYPE>::MASK, base = Nibbles<TYPE>::BASE;
    __device__ __forceinline__ Spread()
    {
        asm("" : "+s"(mask));
        asm("" : "+v"(base));
    }
    __device__ __forceinline__ u32x4 operator()(uint32_t w) const
    {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; i++)
            o[i] = ((i == 0 ? w : __builtin_amdgcn_alignbit(w, w, 4 * i)) & mask) | base;
        return o;
    }
};

__device__ static __forceinline__ float activate(float v, int activation)
{
    // v / (1 + exp(-v)), and with gelu v / (1 + exp(-2 sqrt(2 / pi) (v + 0.044715 v^3))); exp overflows to infinity and v / inf is 0
    const float t = activation == HIPQ_ACT_SILU ? v : 1.5957691216057308f * (v + 0.044715f * v * v * v);
    return v / (1.0f + exp2_fast(-1.4426950408889634f * t));
}

template <int TYPE>
__device__ static __forceinline__ uint16_t rounded(float v) { return (uint16_t)Real16<TYPE>::pack(v, 0.0f); }

// The scales of a row and block: GPB of them, 16 bits each; with zero points GPB words, the scale below, 16 - z at SHIFT of the half above.
template <int TYPE, int GPB, bool ZEROS>
struct Scales {
    static constexpr int DWORDS = ZEROS ? GPB : (GPB + 1) / 2, BYTES = ZEROS ? 4 * GPB : 2 * GPB;
    typedef uint32_t __attribute__((ext_vector_type(DWORDS))) Words;
    // as they were loaded, until they are used: widened at once, a loop that loads ahead would wait for them there
    std::conditional_t<BYTES == 2, uint16_t, Words> w;
    __device__ __forceinline__ void load(const void *at) { w = *(const decltype(w) *)at; }
    __device__ __forceinline__ float scale(int g) const
    {
        if constexpr (BYTES == 2)
            return Real16<TYPE>::low(w);
        else
            return ZEROS ? Real16<TYPE>::low(w[g]) : g & 1 ? Real16<TYPE>::high(w[g / 2]) : Real16<TYPE>::low(w[g / 2]);
    }
    __device__ __forceinline__ float offset(int g) const
    {
        if constexpr (ZEROS)
            return 80.0f - Real16<TYPE>::high(w[g] | (Nibbles<TYPE>::BASE & 0xffff0000u));
        else
            return 40.0f;
    }
    // what makes two floats 48 + q - z of two 32 + q, by an integer addition
    __device__ __forceinline__ uint32_t less_zero(int g) const
    {
        if constexpr (ZEROS)
            return __builtin_amdgcn_perm(w[g], w[g], 0x03020302u);
        else
            return 0;
    }
};
// where the weights of a tile and block begin, in KB: eight tiles lie together, so that what a work-group reads at once lies side by side
// and not in the same channel of the memory
__device__ __host__ static __forceinline__ size_t weights_at(int tile, int block, int blocks) { return ((size_t)(tile >> 3) * blocks + block) * 8 + (tile & 7); }
// where its scales begin, in rows' worth: four tiles lie together
__device__ __host__ static __forceinline__ size_t scales_at(int tile, int block, int blocks) { return (((size_t)(tile >> 2) * blocks + block) * 4 + (tile & 3)) * 16; }

// ---- few rows: a stream of weights ---------------------------------------------------------------------------------------
// Every weight is used by at most 16 MT rows, so the time is what it takes to read the weights, and what counts is how much of them is
// in flight: a work-group owns NT tiles and 16 MT rows, its waves take the blocks of k in turn, each DEPTH blocks ahead and straight
// into registers (a tile's block is 1 KB, in one load), and their sums meet once, in LDS.  No barrier in the loop.  One row of 4096 x 4096: 4.8 us,
// a launch and one round of loads (all of k is asked for before the first multiply); the tile kernel and its join take 9.3.
template <int TYPE, int GPB, bool ZEROS, int MT, int NT, int WAVES, int DEPTH>
__global__ __launch_bounds__(WAVES * 64) void w4_stream_kernel(const W4Args a)
{
    using R = Real16<TYPE>;
    __shared__ f32x4 red[WAVES][MT * NT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, j = lane >> 4;
    const int tile0 = blockIdx.x * NT, m0 = blockIdx.y * (16 * MT);

    u32x4 w[DEPTH][NT], xa[DEPTH][MT][4];
    Scales<TYPE, GPB, ZEROS> gs[DEPTH][NT];
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
                w[d][nt] = *(const u32x4 *)(a.q + weights_at(tile0 + nt, kb, a.blocks) * 1024 + lane * 16);
                gs[d][nt].load(a.scales + (scales_at(tile0 + nt, kb, a.blocks) + c) * gs[d][nt].BYTES);
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
    const Spread<TYPE> spread;
    const u32x4 minus_one = {Nibbles<TYPE>::MINUS_ONE, Nibbles<TYPE>::MINUS_ONE, Nibbles<TYPE>::MINUS_ONE, Nibbles<TYPE>::MINUS_ONE};
    auto compute = [&](int d) {
        u32x4 f[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int t = 0; t < 4; t++)
                f[nt][t] = spread(w[d][nt][t]);
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
                    const float s = gs[d][nt].scale(g);
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

constexpr int64_t XSUM_ROW = 1 << 23; // work-groups side by side

// Minus the sums of x over each group, for the tile kernel: a thread has 8 of x, the group's threads are neighbours.
template <int TYPE, int GPB>
__global__ __launch_bounds__(256) void w4_xsum_kernel(const W4Args a, float *xsum, float factor)
{
    using R = Real16<TYPE>;
    const int per_row = a.blocks * 16;
    const int64_t id = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x, m = id / per_row;
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

// WM x WN waves compute 16 MT WM rows x NT WN tiles; WK such groups of waves take the blocks of k in turn.  Rows, weights and scales of a
// block go through LDS, put there by the load unit STAGES steps ahead: nothing waits in registers, every wave counts its own loads, and
// a step costs one barrier.  16-byte piece p of row m lies at piece p ^ (m % 16), so that the 16 rows of an operand fall on different
// banks; weights lie in the order that the multiplies take them.  Operands are read 32 of k ahead of their multiplies, over the end of a
// block as well: all waves reading at once and multiplying afterwards left the multiplier idle for a third of the time.
// gridDim.y work-groups share the blocks of k: then float32 sums go to `part`, and w4_join_kernel adds them.
// XSUM: the sums of x come from w4_xsum_kernel, otherwise from a multiply by ones.
// What bounds it: up to some dozen rows the weights (17 rows of 14336 x 4096 gated, groups of 64, 18.9 us: 3.4 TB/s in one round of
// work-groups); above, the vector instructions that unpack weights (7 for 8 of them and 16 MT rows) and scale sums (one for an output and group,
// two with zero points), which take turns with the multiplies, as the waves of a SIMD are in step: 2048 rows of 8192 x 8192 in float16, 265 to 297 us
// on different cards with the sums of x, 0.93 to 1.03 PFLOP/s, 49 % of the time the matrix unit's and 43 % theirs; 100 rows of 5000 x 5504 in groups
// of 32, 23 us.
template <int TYPE, int GPB, bool ZEROS, int MT, int NT, int WM, int WN, int WK, int STAGES, bool XSUM>
struct W4Tile {
    static constexpr int WAVES = WM * WN, BM = 16 * MT * WM, TILES = NT * WN, PER = 4 / GPB; // WAVES: of a group
    static constexpr int S_BYTES = Scales<TYPE, GPB, ZEROS>::BYTES;
    // loads of a block, 64 lanes each: 4 rows; a tile; 64 dwords of scales, of sums.  Those that do not go round the waves are done more than once
    static constexpr int X_LOADS = BM / 4 / WAVES, W_LOADS = TILES / WAVES, S_ALL = TILES * 16 * S_BYTES / 256, S_LOADS = (S_ALL + WAVES - 1) / WAVES;
    static constexpr int XS_ALL = XSUM ? GPB * BM / 64 : 0, XS_LOADS = (XS_ALL + WAVES - 1) / WAVES, LOADS = X_LOADS + W_LOADS + S_LOADS + XS_LOADS;
    static constexpr int W_AT = BM * 256, S_AT = W_AT + TILES * 1024, XS_AT = S_AT + S_ALL * 256, BLOCK = XS_AT + XS_ALL * 256;
    static constexpr int STAGE = WK * BLOCK, RED = (WK - 1) * WAVES * MT * NT * 1024, LDS = STAGES * STAGE > RED ? STAGES * STAGE : RED;
    static_assert(BM % (4 * WAVES) == 0 && TILES % WAVES == 0 && S_ALL >= 1 && (STAGES - 1) * LOADS < 64 && LDS <= 160 * 1024, "shape");
    static_assert(XSUM == (MT * NT >= 16), "only there a stage's sums are read before it is filled again, and only there they are needed");
    // Zero points in the weights (one instruction more for two) instead of in the sums (one more for each group and output), and sums of x as the
    // products' initial values: us, 100 rows of 5000 x 5504 in groups of 32, 25.2 against 27.7; 24 of 14336 x 4096 gated, 26.0 against 27.2; 2048 of
    // 8192 x 8192, 446 against 472, in groups of 64 352 against 376; the initial values alone, without zero points, 128 of 14336 x 4096
    // gated, 61 against 72
    static constexpr bool WHOLE = ZEROS && (XSUM ? MT * GPB >= 8 : GPB == 4 && MT >= 2), OFFSETS = ZEROS && !WHOLE, DIRECT = !OFFSETS && GPB == 4;
    static constexpr float FACTOR = WHOLE ? -48.0f : ZEROS ? -1.0f : -40.0f;
};

template <int TYPE, int GPB, bool ZEROS, int MT, int NT, int WM, int WN, int WK, int STAGES, bool XSUM>
__global__ __launch_bounds__(64 * WM * WN * WK) void w4_tile_kernel(const W4Args a, int tiles_m, int tiles_n, float *part)
{
    using R = Real16<TYPE>;
    using T = W4Tile<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM>;
    constexpr int PER = T::PER, WAVES = T::WAVES;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, all_waves = __builtin_amdgcn_readfirstlane(tid >> 6), wk = all_waves / WAVES, wave = all_waves % WAVES;
    const int c = lane & 15, j = lane >> 4;
    // work-groups go to the 8 XCDs in turn: XCD x takes the x-th contiguous eighth, column by column, so that its L2 holds the weights
    const int count = tiles_m * tiles_n, eighth = (count + 7) / 8, item = (int)(blockIdx.x % 8) * eighth + (int)(blockIdx.x / 8);
    if (item >= count)
        return;
    const int m0 = item % tiles_m * T::BM, tile0 = item / tiles_m * T::TILES;
    const int wm = wave % WM, wn = wave / WM;
    const int share = (a.blocks + (int)gridDim.y - 1) / (int)gridDim.y, kb0 = (int)blockIdx.y * share, mine = min(a.blocks - kb0, share);
    const int steps = mine > 0 ? (mine + WK - 1) / WK : 0;
    // Work-groups begin with different blocks, and go round: in step they would all ask for the same lines of x at once (5 % of 64 rows of
    // 14336 gated).  Those that share rows too many for the L2 stay in step.
    const int first = mine > 0 ? (tiles_m >= 8 ? item % tiles_m : item) % mine : 0;

    // A load's address is one of the work-group's that moves on with the blocks, and an offset of the lane's that stays (each over 31 bits
    // is refused by the host).
    constexpr int QUAD = 64 * T::S_BYTES; // bytes of four tiles' scales
    uint32_t x_off[T::X_LOADS], s_off[T::S_LOADS];
    const uint8_t *const x_base = (const uint8_t *)(a.x + m0 * a.x_stride), *const w_base = a.q + weights_at(tile0, 0, a.blocks) * 1024;
    const uint8_t *const s_base = a.scales + scales_at(tile0, 0, a.blocks) * T::S_BYTES;
#pragma unroll
    for (int i = 0; i < T::X_LOADS; i++) {
        const int r = (wave * T::X_LOADS + i) * 4 + j;
        x_off[i] = (uint32_t)(min(r, a.M - 1 - m0) * (int)a.x_stride + (c ^ (r & 15)) * 8) * 2;
    }
#pragma unroll
    for (int i = 0; i < T::S_LOADS; i++) {
        const int at = (wave * T::S_LOADS + i) % T::S_ALL * 256 + lane * 4;
        s_off[i] = (uint32_t)(at / QUAD * a.blocks * QUAD + at % QUAD);
    }
    auto issue = [&](int step, uint8_t *stage) __attribute__((always_inline)) {
        // behind the last block weights are loaded once more, and nothing for rows: every wait counts the same
        const int own = step * WK + wk, turned = min(own, mine - 1) + first, kb = kb0 + (turned < mine ? turned : turned - mine);
        const int left = own < mine ? a.K - kb * 128 : 0;
        const uint8_t *const xk = x_base + (size_t)kb * 256, *const w = w_base + (size_t)kb * 8192, *const s = s_base + (size_t)kb * QUAD;
        uint8_t *to = stage + wk * T::BLOCK;
#pragma unroll
        for (int i = 0; i < T::X_LOADS; i++) { // zeros behind the last k
            const int piece = wave * T::X_LOADS + i, k = (c ^ ((piece * 4 + j) & 15)) * 8;
            __builtin_amdgcn_global_load_lds((gptr_t)(k < left ? xk + x_off[i] : (const uint8_t *)a.nothing), (lptr_t)(to + piece * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < T::W_LOADS; i++) {
            const int tile = wave * T::W_LOADS + i;
            __builtin_amdgcn_global_load_lds((gptr_t)(w + ((size_t)(tile >> 3) * a.blocks * 8 + (tile & 7)) * 1024 + lane * 16), (lptr_t)(to + T::W_AT + tile * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < T::S_LOADS; i++)
            __builtin_amdgcn_global_load_lds((gptr_t)(s + s_off[i]), (lptr_t)(to + T::S_AT + (wave * T::S_LOADS + i) % T::S_ALL * 256), 4, 0, 0);
        if constexpr (XSUM)
#pragma unroll
            for (int i = 0; i < T::XS_LOADS; i++) {
                const int piece = (wave * T::XS_LOADS + i) % T::XS_ALL, g = piece / (T::BM / 64), r = piece % (T::BM / 64) * 64;
                __builtin_amdgcn_global_load_lds((gptr_t)(a.xsum + (size_t)(kb * GPB + g) * a.m_pad + m0 + r + lane), (lptr_t)(to + T::XS_AT + piece * 256), 4, 0, 0);
            }
    };
    f32x4 total[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
            total[mt][nt] = f32x4{0, 0, 0, 0};
    const Spread<TYPE> spread;
    const uint32_t one = T::WHOLE ? Nibbles<TYPE>::MINUS_48 : ZEROS ? Nibbles<TYPE>::MINUS_ONE : Nibbles<TYPE>::MINUS_40;
    const u32x4 ones = {one, one, one, one};
    // With 64 x 64 results a wave there is no room for that: a group's rows are read at once, and multiplied with one tile after the other
    constexpr bool TIGHT = MT * NT >= 16;
    u32x4 w[TIGHT ? 1 : 2][NT], x[TIGHT ? PER : 2][MT];
    Scales<TYPE, GPB, ZEROS> s[TIGHT ? 1 : 2][NT];
    auto read_weights = [&](int d, const uint8_t *from) __attribute__((always_inline)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            w[d][nt] = *(const u32x4 *)(from + T::W_AT + (wn * NT + nt) * 1024 + lane * 16);
            s[d][nt].load(from + T::S_AT + ((wn * NT + nt) * 16 + c) * T::S_BYTES);
        }
    };
    auto read_rows = [&](int t, const uint8_t *from) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
            x[TIGHT ? t % PER : t & 1][mt] = *(const u32x4 *)(from + ((wm * MT + mt) * 16 + c) * 256 + (((t * 4 + j) ^ c) * 16));
    };
    f32x4 sum[MT][NT], less[MT];
    auto multiply = [&](int t, int d, const uint8_t *from) __attribute__((always_inline)) {
        const int g = t / PER;
        const bool begin = t % PER == 0, end = t % PER == PER - 1;
        if (begin)
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
                less[mt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
            less[mt] = R::mfma(x[t & 1][mt], ones, less[mt]);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            u32x4 f = spread(w[d][nt][t]);
            if (T::WHOLE)
                f += s[d][nt].less_zero(g);
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
                sum[mt][nt] = R::mfma(x[t & 1][mt], f, !begin ? sum[mt][nt] : T::DIRECT ? less[mt] : f32x4{0, 0, 0, 0});
        }
        if (end)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float scale = s[d][nt].scale(g);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float v = T::DIRECT ? sum[mt][nt][r] : T::OFFSETS ? __builtin_fmaf(less[mt][r], s[d][nt].offset(g), sum[mt][nt][r]) : sum[mt][nt][r] + less[mt][r];
                        total[mt][nt][r] = __builtin_fmaf(scale, v, total[mt][nt][r]);
                    }
            }
    };
    auto multiply_group = [&](int g, const uint8_t *from) __attribute__((always_inline)) {
        f32x4 first[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
            first[mt] = *(const f32x4 *)(from + T::XS_AT + (g * T::BM + (wm * MT + mt) * 16 + j * 4) * 4);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            f32x4 v[MT];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
                v[mt] = T::OFFSETS ? first[mt] * s[0][nt].offset(g) : first[mt];
#pragma unroll
            for (int t = 0; t < PER; t++) {
                u32x4 f = spread(w[0][nt][g * PER + t]);
                if (T::WHOLE)
                    f += s[0][nt].less_zero(g);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
                    v[mt] = R::mfma(x[t][mt], f, v[mt]);
            }
            const float scale = s[0][nt].scale(g);
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    total[mt][nt][r] = __builtin_fmaf(scale, v[mt][r], total[mt][nt][r]);
        }
    };
    if (steps > 0) {
        constexpr int AHEAD = TIGHT ? STAGES - 1 : STAGES; // steps loaded ahead of the one that is read
        for (int i = 0; i < AHEAD; i++)
            issue(i, lds + i * T::STAGE);
        const uint8_t *const last = lds + (STAGES - 1) * T::STAGE;
        uint8_t *stage = lds;
        // a wait: this wave's loads of the step have arrived (loads return in the order they were asked for), then every wave's; and every wave
        // has read the stage that is filled next
        if constexpr (TIGHT) {
            uint8_t *to = lds + AHEAD * T::STAGE;
            for (int step = 0; step < steps; step++) {
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * T::LOADS) : "memory");
                issue(step + AHEAD, to);
                const uint8_t *from = stage + wk * T::BLOCK;
                read_weights(0, from);
#pragma unroll
                for (int g = 0; g < GPB; g++) {
                    asm volatile("" ::: "memory"); // two groups' rows at once are more than the registers hold
#pragma unroll
                    for (int t = 0; t < PER; t++)
                        read_rows(g * PER + t, from);
                    multiply_group(g, from);
                }
                stage = stage == last ? lds : stage + T::STAGE;
                to = to == last ? lds : to + T::STAGE;
            }
        } else {
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((STAGES - 1) * T::LOADS) : "memory");
            read_weights(0, stage + wk * T::BLOCK);
            read_rows(0, stage + wk * T::BLOCK);
            auto turn = [&](int step, int d) __attribute__((always_inline)) {
                const uint8_t *from = stage + wk * T::BLOCK;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    if (t < 3)
                        read_rows(t + 1, from);
                    else {
                        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * T::LOADS) : "memory");
                        issue(step + STAGES, stage);
                        stage = stage == last ? lds : stage + T::STAGE;
                        read_weights(1 - d, stage + wk * T::BLOCK);
                        read_rows(0, stage + wk * T::BLOCK);
                    }
                    multiply(t, d, from);
                }
            };
            int step = 0;
            for (; step + 1 < steps; step += 2) {
                turn(step, 0);
                turn(step + 1, 1);
            }
            if (step < steps)
                turn(step, 0);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // of what was loaded for nothing
    }
    if (WK > 1) { // the groups' sums
        __syncthreads();
        f32x4 *red = (f32x4 *)lds;
        if (wk > 0)
#pragma unroll
            for (int i = 0; i < MT * NT; i++)
                red[((all_waves - WAVES) * MT * NT + i) * 64 + lane] = total[i / NT][i % NT];
        __syncthreads();
        if (wk > 0)
            return;
#pragma unroll
        for (int g = 1; g < WK; g++)
#pragma unroll
            for (int i = 0; i < MT * NT; i++)
                total[i / NT][i % NT] += red[(((g - 1) * WAVES + wave) * MT * NT + i) * 64 + lane];
    }
    if (part) {
        const int columns = tiles_n * NT * WN * 16;
        float *to = part + ((size_t)blockIdx.y * a.M * columns);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int m = m0 + (wm * MT + mt) * 16 + j * 4 + r;
                    if (m < a.M)
                        to[(size_t)m * columns + (tile0 + wn * NT + nt) * 16 + c] = total[mt][nt][r];
                }
        return;
    }
    const bool gated = a.activation != HIPQ_ACT_NONE;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const float b = a.bias ? R::low(a.bias[(tile0 + wn * NT + nt) * 16 + c]) : 0.0f;
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
            total[mt][nt] += b;
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        if (gated && nt % 2)
            continue;
        const int tile = tile0 + wn * NT + nt, n = (gated ? tile / 2 : tile) * 16 + c;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const int m = m0 + (wm * MT + mt) * 16 + j * 4;
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (n < a.N && m + r < a.M)
                    a.y[(m + r) * a.y_stride + n] = rounded<TYPE>(gated ? activate(total[mt][nt][r], a.activation) * total[mt][nt | 1][r] : total[mt][nt][r]);
        }
    }
}

// Adds the parts of a row's results, four a thread.
template <int TYPE>
__global__ __launch_bounds__(256) void w4_join_kernel(const W4Args a, const float *part, int splits, int columns)
{
    const int per_row = (a.N + 3) / 4;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int m = (int)(id / per_row), n = (int)(id % per_row) * 4;
    if (m >= a.M)
        return;
    const bool gated = a.activation != HIPQ_ACT_NONE;
    const int column = gated ? n / 16 * 32 + n % 16 : n;
    auto sum_of = [&](int at) {
        f32x4 v = {0, 0, 0, 0};
        for (int s = 0; s < splits; s++)
            v += *(const f32x4 *)(part + ((size_t)s * a.M + m) * columns + at);
        if (a.bias)
#pragma unroll
            for (int e = 0; e < 4; e++)
                v[e] += Real16<TYPE>::low(a.bias[at + e]);
        return v;
    };
    f32x4 v = sum_of(column);
    if (gated) {
        const f32x4 up = sum_of(column + 16);
#pragma unroll
        for (int e = 0; e < 4; e++)
            v[e] = activate(v[e], a.activation) * up[e];
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (n + e < a.N)
            a.y[m * a.y_stride + n + e] = rounded<TYPE>(v[e]);
}

// ---- setup ---------------------------------------------------------------------------------------------------------------------
struct PackArgs {
    const uint8_t *q, *zeros;
    const uint16_t *scales, *bias;
    uint8_t *to_q;
    uint16_t *to_scales, *to_bias;
    u32x4 *to_nothing;
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
    if (blockIdx.x == 0 && threadIdx.x < 16)
        p.to_nothing[threadIdx.x] = u32x4{0, 0, 0, 0};
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
        *(u32x4 *)(p.to_q + weights_at(tile, kb, p.blocks) * 1024 + lane * 16) = o;
        if (lane < 16)
            for (int g = 0; g < gpb; g++) {
                const int from = kb * gpb + g;
                const bool there = row >= 0 && from < p.groups;
                const uint32_t s = there ? p.scales[row * p.groups + from] : 0;
                const size_t at = (scales_at(tile, kb, p.blocks) + c) * gpb + g;
                if (p.zeros) {
                    const uint32_t z = there ? p.zeros[row * p.groups + from] & 15 : 8;
                    ((uint32_t *)p.to_scales)[at] = s | (16 - z) << (16 + p.shift);
                } else
                    p.to_scales[at] = (uint16_t)s;
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
    const size_t nothing = 256, q_bytes = pieces * 1024, s_bytes = pieces * 16 * gpb * (zeros ? 4 : 2), b_bytes = bias ? tiles * 32 : 0;
    hipError_t e = hipGetDevice(&p->device);
    if (e == hipSuccess)
        e = hipMalloc(&p->memory, q_bytes + s_bytes + b_bytes + nothing);
    if (e != hipSuccess) {
        delete p;
        return fail("w4: no memory for %zu bytes of weights: %s", q_bytes + s_bytes + b_bytes + nothing, hipGetErrorString(e));
    }
    PackArgs k = {};
    k.q = q, k.zeros = zeros, k.scales = (const uint16_t *)scales, k.bias = (const uint16_t *)bias;
    k.to_q = p->memory, k.to_nothing = (u32x4 *)(p->memory + q_bytes + s_bytes + b_bytes), k.to_scales = (uint16_t *)(p->memory + q_bytes);
    k.to_bias = (uint16_t *)(p->memory + q_bytes + s_bytes);
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
    a.q = k.to_q, a.scales = (const uint8_t *)k.to_scales, a.zeros = zeros != nullptr, a.bias = bias ? k.to_bias : nullptr;
    a.nothing = (const uint16_t *)k.to_nothing;
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

// How M rows run: the kernel, and the work-groups that share the blocks of k.
struct W4Shape {
    int kernel, splits;
};
enum { STREAM_16, TILE_16, TILE_32, TILE_64, TILE_128, TILE_128_WIDE, SHAPES };
static const struct {
    const char *name;
    int rows, tiles; // of a work-group
    bool xsum;
} SHAPE[SHAPES] = {{"w4_stream_16", 16, 1, false},  {"w4_tile_16x128", 16, 8, false},   {"w4_tile_32x128", 32, 8, false},
                   {"w4_tile_64x128", 64, 8, false}, {"w4_tile_128x128", 128, 8, false}, {"w4_tile_128x256", 128, 16, true}};

// Measured over 1 to 2048 rows of 4096 x 4096, 4096 x 14336, 14336 x 4096 (gated), 5504 x 5000 and 8192 x 8192, us of a replayed graph:
//   * few weights (16 MB; 8 MB for up to 32 rows): the stream kernel needs no second launch to fill the chip - 4096 x 4096, 1 row, 5.6
//     against 9.3, 24 rows 9.9 against 11.0; with more the tile kernel's waves are fed further ahead - 14336 gated, 1 row, 15.8 against 25;
//   * otherwise the least rows of a work-group that hold all rows: rows that are not there cost as much as those that are.  Where a
//     work-group a row block fills half of the chip, one of twice the rows reads the weights once (64 rows, 14336 gated: 29.6
//     against 38; 128: 48 against 55), where it does not more work-groups count (64 rows of 4096 x 4096: 13.1 against 14.6);
//   * the widest from 64 of its work-groups on (256 rows of 8192 x 8192: 51 against 55; of 4096 x 4096, 32 work-groups: 28 against 24).
// The blocks of k are shared by as many work-groups as fill the chip, each with four blocks at least: splitting further costs more in the
// sums than it gives.
static W4Shape shape_of(const hipq_w4_plan *p, int M)
{
    const int64_t weights = (int64_t)p->tiles * p->blocks >> 10; // MB
    const int columns = (p->tiles + 7) / 8;
    W4Shape s = {TILE_128_WIDE, 1};
    if (weights <= 8 ? M <= 32 : M <= 16 && weights <= 16 && columns < 160)
        s.kernel = STREAM_16;
    else if (M <= 32)
        s.kernel = M <= 16 ? TILE_16 : TILE_32;
    else if (M <= 128)
        s.kernel = M <= 64 ? (columns < 128 ? TILE_32 : TILE_64) : (columns < 128 ? TILE_64 : TILE_128);
    else if ((int64_t)((M + 127) / 128) * ((p->tiles + 15) / 16) < 64)
        s.kernel = TILE_128;
    if (s.kernel != STREAM_16) {
        const int64_t groups = (int64_t)((M + SHAPE[s.kernel].rows - 1) / SHAPE[s.kernel].rows) * ((p->tiles + SHAPE[s.kernel].tiles - 1) / SHAPE[s.kernel].tiles);
        const int most = p->blocks / 4;
        s.splits = groups < 256 ? (int)(256 / groups) : 1;
        s.splits = s.splits < most ? s.splits : most;
        s.splits = s.splits < 1 ? 1 : s.splits;
    }
    return s;
}

template <int TYPE, int GPB, bool ZEROS, int MT, int NT, int WAVES, int DEPTH>
static int launch_stream(const hipq_w4_plan *p, const W4Args &a, hipStream_t st)
{
    const dim3 grid((p->tiles + NT - 1) / NT, (a.M + 16 * MT - 1) / (16 * MT));
    w4_stream_kernel<TYPE, GPB, ZEROS, MT, NT, WAVES, DEPTH><<<grid, dim3(WAVES * 64), 0, st>>>(a);
    return launch_status("w4_stream_kernel");
}

// More than 64 KB of LDS have to be asked for, once for each kernel and device.
static int allow_lds(const void *kernel, size_t bytes, int device, bool *done)
{
    if (bytes > 65536 && (device >= 64 || !done[device])) {
        HIPQ_CHECK_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
        if (device < 64)
            done[device] = true;
    }
    return 0;
}

template <int TYPE, int GPB, bool ZEROS, int MT, int NT, int WM, int WN, int WK, int STAGES, bool XSUM>
static int launch_tile(const hipq_w4_plan *p, const W4Args &a, int splits, float *workspace, hipStream_t st)
{
    constexpr int BM = 16 * MT * WM, lds = W4Tile<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM>::LDS;
    static thread_local bool done[64] = {};
    const auto kernel = w4_tile_kernel<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM>;
    if (allow_lds((const void *)kernel, lds, p->device, done))
        return 1;
    const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (p->tiles + NT * WN - 1) / (NT * WN);
    const dim3 grid((tiles_m * tiles_n + 7) / 8 * 8, splits);
    kernel<<<grid, dim3(64 * WM * WN * WK), lds, st>>>(a, tiles_m, tiles_n, splits > 1 ? workspace : nullptr);
    if (launch_status("w4_tile_kernel"))
        return 1;
    if (splits > 1) {
        const int64_t threads = (int64_t)a.M * ((a.N + 3) / 4);
        w4_join_kernel<TYPE><<<dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st>>>(a, workspace, splits, tiles_n * NT * WN * 16);
        return launch_status("w4_join_kernel");
    }
    return 0;
}

template <int TYPE, int GPB, bool ZEROS>
static int launch(const hipq_w4_plan *p, W4Args &a, float *workspace, hipStream_t st)
{
    const W4Shape s = shape_of(p, a.M);
    if (SHAPE[s.kernel].xsum) {
        a.m_pad = round_up(a.M, SHAPE[s.kernel].rows);
        a.xsum = workspace;
        // of 2^32 work-items side by side and more only what is left over would run
        const int64_t groups = ((int64_t)a.m_pad * a.blocks * 16 + 255) / 256;
        const dim3 grid((unsigned)(groups < XSUM_ROW ? groups : XSUM_ROW), (unsigned)((groups + XSUM_ROW - 1) / XSUM_ROW));
        w4_xsum_kernel<TYPE, GPB><<<grid, dim3(256), 0, st>>>(a, workspace, W4Tile<TYPE, GPB, ZEROS, 4, 4, 2, 4, 1, GPB == 4 && ZEROS ? 2 : 3, true>::FACTOR);
        if (launch_status("w4_xsum_kernel"))
            return 1;
        workspace += (size_t)a.m_pad * a.blocks * GPB;
    }
    switch (s.kernel) {
    case STREAM_16:
        return p->desc.activation ? launch_stream<TYPE, GPB, ZEROS, 1, 2, 8, 4>(p, a, st) : launch_stream<TYPE, GPB, ZEROS, 1, 1, 8, 4>(p, a, st);
    case TILE_16:
        return launch_tile<TYPE, GPB, ZEROS, 1, 2, 1, 4, 2, 5, false>(p, a, s.splits, workspace, st);
    case TILE_32:
        return launch_tile<TYPE, GPB, ZEROS, 2, 2, 1, 4, 2, 4, false>(p, a, s.splits, workspace, st);
    case TILE_64:
        return launch_tile<TYPE, GPB, ZEROS, 4, 2, 1, 4, 2, 3, false>(p, a, s.splits, workspace, st);
    case TILE_128:
        return launch_tile<TYPE, GPB, ZEROS, 4, 2, 2, 4, 1, 3, false>(p, a, s.splits, workspace, st);
    }
    return launch_tile<TYPE, GPB, ZEROS, 4, 4, 2, 4, 1, GPB == 4 && ZEROS ? 2 : 3, true>(p, a, s.splits, workspace, st);
}

template <int TYPE, int GPB>
static int launch(const hipq_w4_plan *p, W4Args &a, float *workspace, hipStream_t st)
{
    return a.zeros ? launch<TYPE, GPB, true>(p, a, workspace, st) : launch<TYPE, GPB, false>(p, a, workspace, st);
}

template <int TYPE>
static int launch(const hipq_w4_plan *p, W4Args &a, float *workspace, hipStream_t st)
{
    return p->desc.group == 128 ? launch<TYPE, 1>(p, a, workspace, st) : p->desc.group == 64 ? launch<TYPE, 2>(p, a, workspace, st) : launch<TYPE, 4>(p, a, workspace, st);
}

} // namespace hipq

extern "C" const char *hipq_w4_plan_kernel(const hipq_w4_plan *p, int M)
{
    if (!p || M < 0 || M > (1 << 24))
        return "";
    return SHAPE[shape_of(p, M > 0 ? M : 1).kernel].name;
}

extern "C" size_t hipq_w4_workspace(const hipq_w4_plan *p, int M)
{
    if (!p || M <= 0 || M > (1 << 24))
        return 0;
    const W4Shape s = shape_of(p, M);
    const size_t columns = (size_t)round_up(p->tiles, SHAPE[s.kernel].tiles) * 16;
    return (s.splits > 1 ? s.splits * M * columns * sizeof(float) : 0)
           + (SHAPE[s.kernel].xsum ? (size_t)round_up(M, SHAPE[s.kernel].rows) * p->blocks * (128 / p->desc.group) * sizeof(float) : 0);
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
    HIPQ_REQUIRE(x_stride < (1 << 23), "w4: rows of x are %lld elements apart", (long long)x_stride);
    HIPQ_REQUIRE(M == 1 || (x_stride >= p->desc.K && y_stride >= p->desc.N), "w4: rows overlap (strides %lld and %lld)", (long long)x_stride, (long long)y_stride);
    // the widest work-groups' number: of 2^32 work-items and more only what is left over would run
    HIPQ_REQUIRE((int64_t)((M + 127) / 128) * ((p->tiles + 15) / 16) <= (1 << 23) - 8, "w4: %d rows of %d outputs", M, p->desc.N);
    const ByteRows read = {(int64_t)(uintptr_t)x, M > 1 ? x_stride * 2 : 0, p->desc.K * 2ll, M}, written = {(int64_t)(uintptr_t)y, M > 1 ? y_stride * 2 : 0, p->desc.N * 2ll, M};
    HIPQ_REQUIRE(!overlap(read, written), "w4: y lies over x");
    const size_t need = hipq_w4_workspace(p, M);
    HIPQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), "w4: a workspace of %zu bytes is needed", need);
    int device;
    HIPQ_CHECK_HIP(hipGetDevice(&device));
    HIPQ_REQUIRE(device == p->device, "w4: the plan is on device %d, the current one is %d", p->device, device);
    W4Args a = p->args;
    a.x = (const uint16_t *)x, a.y = (uint16_t *)y, a.x_stride = x_stride, a.y_stride = y_stride, a.M = M;
    return p->desc.type == HIPQ_REAL_BF16 ? launch<HIPQ_REAL_BF16>(p, a, (float *)workspace, (hipStream_t)stream)
                                          : launch<HIPQ_REAL_F16>(p, a, (float *)workspace, (hipStream_t)stream);
}
