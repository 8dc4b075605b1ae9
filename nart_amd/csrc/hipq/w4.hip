// Products with 4-bit weights and group scales (hipq_w4_*): y[m][n] = sum_g s[n][g] sum_{k in g} x[m][k] (q[n][k] - z[n][g]).  gfx950 only.
//
// Arithmetic and layout of the weights: w4_frag.h.
#include <new>

#include "overlap.h"
#include "w4_tile.h"

namespace hipq {

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

// ---- many rows: tiles (w4_tile.h) ------------------------------------------------------------------------------------------------
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
// the row of the caller's arrays that row r of a tile holds, -1: none
__device__ static __forceinline__ int64_t source_row(const PackArgs &p, int tile, int r)
{
    const int n = (p.gated ? tile / 2 : tile) * 16 + r;
    return n < p.rows ? (int64_t)n + (p.gated && tile % 2 ? p.rows : 0) : -1;
}

__global__ __launch_bounds__(256) void w4_pack_kernel(const PackArgs all)
{
    PackArgs p = all;
    p.q += blockIdx.y * p.q_step, p.scales += blockIdx.y * p.s_step, p.zeros += p.zeros ? blockIdx.y * p.s_step : 0;
    p.to_q += blockIdx.y * p.to_q_step, p.to_scales += blockIdx.y * p.to_s_step / 2;
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

int w4_pack(PackArgs p, int type, hipStream_t st)
{
    p.shift = type == HIPQ_REAL_BF16 ? Nibbles<HIPQ_REAL_BF16>::SHIFT : Nibbles<HIPQ_REAL_F16>::SHIFT;
    const size_t groups = ((size_t)p.tiles * p.blocks + 3) / 4;
    w4_pack_kernel<<<dim3((unsigned)(groups < 16384 ? groups : 16384), p.arrays > 1 ? p.arrays : 1), dim3(256), 0, st>>>(p);
    return launch_status("w4_pack_kernel");
}

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
    int bad = w4_pack(k, d->type, (hipStream_t)stream);
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

template <int TYPE, int GPB, bool ZEROS, int MT, int NT, int WM, int WN, int WK, int STAGES, bool XSUM>
static int launch_tile(const hipq_w4_plan *p, const W4Args &a, int splits, float *workspace, hipStream_t st)
{
    constexpr int BM = 16 * MT * WM, lds = W4Tile<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM>::LDS;
    static thread_local bool done[64] = {};
    const auto kernel = w4_tile_kernel<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM, W4Whole>;
    if (allow_lds((const void *)kernel, lds, p->device, done))
        return 1;
    const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (p->tiles + NT * WN - 1) / (NT * WN);
    const dim3 grid((tiles_m * tiles_n + 7) / 8 * 8, splits);
    kernel<<<grid, dim3(64 * WM * WN * WK), lds, st>>>(a, W4Whole{}, tiles_m, tiles_n, splits > 1 ? workspace : nullptr);
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
