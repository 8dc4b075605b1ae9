// The tile kernel of 4-bit weights: rows, weights and scales of a block through LDS, for the products of all rows with the same weights (w4.hip) and of
// groups of rows with weights of their own (experts.hip).  gfx950 only.
#pragma once

#include "w4_frag.h"

namespace hipq {

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

// What the rows of a launch are multiplied with: all with the same weights,
struct W4Whole {
    static constexpr bool GROUPS = false;
};
// or blocks of up to BM rows, each with one of many arrays of weights of the same shape.  Rows are numbered so that those of an array lie together; that number
// is the row of the result, and of x either that as well or what `row` has there.  M is how many rows there are.
struct W4Block {
    int32_t array, first, end, base, number; // its rows are first..end - 1; blocks base..base + number - 1 have the same array
};
struct W4Groups {
    static constexpr bool GROUPS = true;
    const W4Block *block;
    const int32_t *count, *row; // how many blocks; or nullptr
    size_t q_bytes, s_bytes;    // of an array
};

template <int TYPE, int GPB, bool ZEROS, int MT, int NT, int WM, int WN, int WK, int STAGES, bool XSUM, class G>
__global__ __launch_bounds__(64 * WM * WN * WK) void w4_tile_kernel(const W4Args a, const G groups, int tiles_m, int tiles_n, float *part)
{
    using R = Real16<TYPE>;
    using T = W4Tile<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM>;
    constexpr int PER = T::PER, WAVES = T::WAVES;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, all_waves = __builtin_amdgcn_readfirstlane(tid >> 6), wk = all_waves / WAVES, wave = all_waves % WAVES;
    const int c = lane & 15, j = lane >> 4;
    // work-groups go to the 8 XCDs in turn: XCD x takes the x-th contiguous eighth, column by column, so that its L2 holds the weights
    // (of an array's, so that it holds the array's rows as well)
    if constexpr (G::GROUPS)
        tiles_m = __builtin_amdgcn_readfirstlane(*groups.count);
    const int count = tiles_m * tiles_n, eighth = (count + 7) / 8, item = (int)(blockIdx.x % 8) * eighth + (int)(blockIdx.x / 8);
    if (blockIdx.x / 8 >= (unsigned)eighth || item >= count)
        return;
    int m0 = item % tiles_m * T::BM, column = item / tiles_m, end = a.M;
    const uint8_t *q = a.q, *scales = a.scales;
    int phase = tiles_m >= 8 ? item % tiles_m : item;
    if constexpr (G::GROUPS) {
        const W4Block *any = groups.block + item / tiles_n; // of the same array
        const int array = __builtin_amdgcn_readfirstlane(any->array), base = __builtin_amdgcn_readfirstlane(any->base), number = __builtin_amdgcn_readfirstlane(any->number);
        const int local = item - base * tiles_n, block = local % number;
        column = local / number;
        m0 = __builtin_amdgcn_readfirstlane(groups.block[base + block].first), end = __builtin_amdgcn_readfirstlane(groups.block[base + block].end);
        q += array * groups.q_bytes, scales += array * groups.s_bytes;
        // in step: an array's columns side by side share their rows, and which rows a block has may change from call to call (us of 2048 tokens of four of 32 experts of 4096 x 2048,
        // in step 606, from the column on 612, from the item on 618; 1024 tokens of six of 64 of 2048 x 1408 248, 248, 248)
        phase = 0;
    }
    const int tile0 = column * T::TILES;
    // blocks of an array may have few rows: waves without any, which share their SIMDs with others, leave the multiplies to those (in groups of 64 the branch takes more
    // registers than there are)
    const int wm = G::GROUPS ? wave / WN : wave % WM, wn = G::GROUPS ? wave % WN : wave / WM;
    const bool live = !G::GROUPS || GPB == 2 || m0 + wm * (16 * MT) < end;
    const int share = (a.blocks + (int)gridDim.y - 1) / (int)gridDim.y, kb0 = (int)blockIdx.y * share, mine = min(a.blocks - kb0, share);
    const int steps = mine > 0 ? (mine + WK - 1) / WK : 0;
    // Work-groups begin with different blocks, and go round: in step they would all ask for the same lines of x at once (5 % of 64 rows of
    // 14336 gated).  Those that share rows too many for the L2 stay in step.
    const int first = mine > 0 ? phase % mine : 0;
    // the row of x that the result's row m0 + r is of, the last one again behind it
    auto x_row = [&](int r) __attribute__((always_inline)) {
        const int m = min(m0 + r, end - 1);
        if constexpr (G::GROUPS)
            return groups.row ? groups.row[m] : m;
        else
            return m - m0;
    };

    // A load's address is one of the work-group's that moves on with the blocks, and an offset of the lane's that stays (each over 31 bits
    // is refused by the host).
    constexpr int QUAD = 64 * T::S_BYTES; // bytes of four tiles' scales
    uint32_t x_off[T::X_LOADS], s_off[T::S_LOADS], xs_off[T::XS_LOADS > 0 ? T::XS_LOADS : 1];
    const uint8_t *const x_base = (const uint8_t *)(G::GROUPS ? a.x : a.x + m0 * a.x_stride), *const w_base = q + weights_at(tile0, 0, a.blocks) * 1024;
    const uint8_t *const s_base = scales + scales_at(tile0, 0, a.blocks) * T::S_BYTES;
#pragma unroll
    for (int i = 0; i < T::X_LOADS; i++) {
        const int r = (wave * T::X_LOADS + i) * 4 + j;
        x_off[i] = ((uint32_t)x_row(r) * (uint32_t)a.x_stride + (c ^ (r & 15)) * 8) * 2;
    }
    if constexpr (XSUM && G::GROUPS)
#pragma unroll
        for (int i = 0; i < T::XS_LOADS; i++)
            xs_off[i] = x_row((wave * T::XS_LOADS + i) % T::XS_ALL % (T::BM / 64) * 64 + lane);
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
                __builtin_amdgcn_global_load_lds((gptr_t)(a.xsum + (size_t)(kb * GPB + g) * a.m_pad + (G::GROUPS ? xs_off[i] : m0 + r + lane)), (lptr_t)(to + T::XS_AT + piece * 256), 4, 0, 0);
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
                if (live) {
                    read_weights(0, from);
#pragma unroll
                    for (int g = 0; g < GPB; g++) {
                        asm volatile("" ::: "memory"); // two groups' rows at once are more than the registers hold
#pragma unroll
                        for (int t = 0; t < PER; t++)
                            read_rows(g * PER + t, from);
                        multiply_group(g, from);
                    }
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
                    if (m < end)
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
                if (n < a.N && m + r < end)
                    a.y[(m + r) * a.y_stride + n] = rounded<TYPE>(gated ? activate(total[mt][nt][r], a.activation) * total[mt][nt | 1][r] : total[mt][nt][r]);
        }
    }
}

} // namespace hipq
