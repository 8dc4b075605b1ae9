// A layer of experts with 4-bit weights (hipq_w4_experts_*): every token's best experts from its scores, their gated products, the second product of
// each and the weighted sum.  gfx950 only.
//
//   y[t] = sum over the chosen e of share[t][e] * down_e (act(gate_e x[t]) * up_e x[t])
//
// A pair is a token and one of its experts.  Choosing and numbering: a wave finds a token's experts (the largest of its scores, `top` times); one work-group then
// counts the pairs of each expert and numbers them, an expert's side by side in the order of their tokens, so that the same rows meet in the same work-groups
// every time.  Both products are those of w4_tile.h, whose blocks of rows then have an expert each; the hidden rows between them are rounded to 16
// bits, as the matrix unit takes them.  The second product's float32 sums go to memory, and a last kernel adds a token's, each times its share.
#include <cmath>
#include <new>

#include "overlap.h"
#include "w4_tile.h"

namespace hipq {

constexpr int MOST_EXPERTS = 1024, MOST_TOP = 16;

struct RouteArgs {
    const void *logits;
    int64_t stride;
    int type, M, experts, top, sigmoid, normalize, block_rows;
    int32_t *chosen; // [M][top]: the expert, -1: none
    float *share;    // [M][top]
    int32_t *place;  // [M][top]: the pair's number, -1: none
    int32_t *row;    // [pairs]: its token
    W4Block *block;
    int32_t *count;  // of blocks
};

// A token's experts, its scores over the lanes of a wave: lane l has those of experts l, l + 64, ..., EACH of them
template <int EACH>
__device__ static __forceinline__ void choose(const RouteArgs &a, int t, int lane)
{
    uint32_t key[EACH]; // in the order of the scores; 0: never taken
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int e = i * 64 + lane;
        key[i] = 0;
        if (e < a.experts) {
            const int64_t at = t * a.stride + e;
            const float x = a.type == HIPQ_REAL_F32 ? ((const float *)a.logits)[at]
                            : a.type == HIPQ_REAL_F16 ? Real16<HIPQ_REAL_F16>::low(((const uint16_t *)a.logits)[at])
                                                      : Real16<HIPQ_REAL_BF16>::low(((const uint16_t *)a.logits)[at]);
            const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f); // -0 is 0
            key[i] = !(x > -__builtin_inff()) ? 0 : u & 0x80000000u ? ~u : u | 0x80000000u;
        }
    }
    auto largest = [&] {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++)
            most = max(most, key[i]);
#pragma unroll
        for (int o = 1; o < 64; o *= 2)
            most = max(most, (uint32_t)__shfl_xor((int)most, o));
        return most;
    };
    auto score = [](uint32_t k) { return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k); };
    const uint32_t most = largest();
    const float top_score = most ? score(most) : 0.0f;
    // e^(x - m); of infinite scores each counts as much, and nothing else does
    auto weight = [&](float v) { return v == top_score ? 1.0f : exp2_fast((v - top_score) * 1.4426950408889634f); };
    float all = 0;
    if (!a.sigmoid && !a.normalize) {
#pragma unroll
        for (int i = 0; i < EACH; i++)
            if (key[i])
                all += weight(score(key[i]));
#pragma unroll
        for (int o = 1; o < 64; o *= 2)
            all += __shfl_xor(all, o);
    }
    // 1 / (1 + e^-x), and where shares are divided by their sum, e^-r times that with r = min(0, the largest): not 0 however small they are
    const float low = a.normalize ? fminf(top_score, 0.0f) : 0.0f, lift = exp2_fast(low * 1.4426950408889634f);
    int mine = -1; // lane s: the s-th expert
    float share = 0, sum = 0;
    for (int s = 0; s < a.top; s++) {
        const uint32_t best = s == 0 ? most : largest();
        if (best == 0)
            break;
        int e = -1; // the lowest of those that have it
#pragma unroll
        for (int i = EACH - 1; i >= 0; i--) {
            const uint64_t equal = __ballot(key[i] == best);
            e = equal ? i * 64 + __builtin_ctzll(equal) : e;
        }
#pragma unroll
        for (int i = 0; i < EACH; i++)
            if (i * 64 + lane == e)
                key[i] = 0;
        const float v = score(best), w = a.sigmoid ? 1.0f / (lift + exp2_fast((low - v) * 1.4426950408889634f)) : weight(v);
        sum += w;
        if (lane == s)
            mine = e, share = w;
    }
    if (lane < a.top) {
        a.chosen[(int64_t)t * a.top + lane] = mine;
        a.share[(int64_t)t * a.top + lane] = mine < 0 ? 0.0f : share / (a.normalize ? sum : a.sigmoid ? 1.0f : all);
    }
}

template <int EACH>
__global__ __launch_bounds__(256) void experts_choose_kernel(const RouteArgs a)
{
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t < a.M)
        choose<EACH>(a, (int)t, threadIdx.x & 63);
}

// Numbers the pairs, by expert and then by token, and lists the blocks of rows.  Each of 16 waves has a contiguous part of the pairs, and goes through it 64 at a time
// twice: to count each expert's, and to number them from where the waves before it end.  EACH above 0: it chooses as well.
template <int EACH>
__global__ __launch_bounds__(1024) void experts_number_kernel(const RouteArgs a)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    int32_t *const counts = (int32_t *)lds, *const scan = counts + 16 * a.experts; // [wave][expert]; pairs and blocks of [wave]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int i = tid; i < 16 * a.experts; i += 1024)
        counts[i] = 0;
    if constexpr (EACH > 0)
        for (int t = wave; t < a.M; t += 16)
            choose<EACH>(a, t, lane);
    __syncthreads(); // the work-group's own writes to memory are in order behind it
    const int pairs = a.M * a.top, share = (pairs + 1023) / 1024 * 64, from = wave * share, to = min(pairs, from + share);
    auto same = [&](int e) { // the lanes with the same expert
        uint64_t lanes = __ballot(e >= 0);
#pragma unroll
        for (int bit = 0; bit < 10; bit++)
            if (a.experts > 1 << bit) {
                const uint64_t set = __ballot((e >> bit) & 1);
                lanes &= (e >> bit) & 1 ? set : ~set;
            }
        return lanes;
    };
    for (int p = from; p < to; p += 64) {
        const int e = p + lane < to ? a.chosen[p + lane] : -1;
        const uint64_t lanes = same(e);
        if (e >= 0 && lane == __builtin_ctzll(lanes))
            counts[wave * a.experts + e] += __builtin_popcountll(lanes);
    }
    __syncthreads();
    // an expert's pairs and blocks, and those before it
    int pairs_of = 0, blocks_of = 0;
    if (tid < a.experts)
        for (int w = 0; w < 16; w++) {
            const int n = counts[w * a.experts + tid];
            counts[w * a.experts + tid] = pairs_of;
            pairs_of += n;
        }
    blocks_of = (pairs_of + a.block_rows - 1) / a.block_rows;
    int first = pairs_of, base = blocks_of;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int u = __shfl_up(first, o), v = __shfl_up(base, o);
        first += lane >= o ? u : 0, base += lane >= o ? v : 0;
    }
    if (lane == 63)
        scan[wave] = first, scan[16 + wave] = base;
    __syncthreads();
    for (int w = 0; w < wave; w++)
        first += scan[w], base += scan[16 + w];
    if (tid == 1023)
        *a.count = base;
    first -= pairs_of, base -= blocks_of;
    if (tid < a.experts) {
        for (int w = 0; w < 16; w++)
            counts[w * a.experts + tid] += first;
        for (int i = 0; i < blocks_of; i++)
            a.block[base + i] = W4Block{tid, first + i * a.block_rows, min(first + pairs_of, first + (i + 1) * a.block_rows), base, blocks_of};
    }
    __syncthreads();
    for (int p = from; p < to; p += 64) {
        const int e = p + lane < to ? a.chosen[p + lane] : -1;
        const uint64_t lanes = same(e);
        int at = -1;
        if (e >= 0) {
            at = counts[wave * a.experts + e] + __builtin_popcountll(lanes & ((1ull << lane) - 1));
            a.row[at] = (p + lane) / a.top;
        }
        if (p + lane < to)
            a.place[p + lane] = at;
        if (e >= 0 && lane == __builtin_ctzll(lanes)) // in order behind the reads above: a wave's LDS accesses are
            counts[wave * a.experts + e] += __builtin_popcountll(lanes);
    }
}

// y[t] = sum of a token's pairs, four values a thread.
template <int TYPE>
__global__ __launch_bounds__(256) void experts_join_kernel(const RouteArgs a, const float *part, int splits, int64_t pairs, int columns, uint16_t *y, int64_t y_stride, int N)
{
    const int per_row = (N + 3) / 4;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, t = id / per_row;
    const int n = (int)(id - t * per_row) * 4;
    if (t >= a.M)
        return;
    f32x4 v = {0, 0, 0, 0};
    for (int s = 0; s < a.top; s++) {
        const int p = a.place[t * a.top + s];
        if (p < 0)
            break;
        f32x4 u = {0, 0, 0, 0};
        for (int i = 0; i < splits; i++)
            u += *(const f32x4 *)(part + (i * pairs + p) * columns + n);
        v += a.share[t * a.top + s] * u;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (n + e < N)
            y[t * y_stride + n + e] = rounded<TYPE>(v[e]);
}

} // namespace hipq

using namespace hipq;

struct hipq_w4_experts_plan {
    hipq_w4_experts_desc desc;
    int device, tiles[2];      // of an expert: the gated pair, the second product
    uint8_t *memory;
    W4Args args[2];
    W4Groups groups[2];        // where an expert's weights are
};

namespace hipq {

// What lies in a caller's workspace.
struct ExpertsLayout {
    size_t chosen, share, place, row, block, count, hidden, part, xsum, bytes;
    int kernel, splits, block_rows;
    int64_t pairs, blocks; // at most
    int columns;
};
enum { TILE_16, TILE_32, TILE_64, TILE_128_WIDE, SHAPES };
static const struct {
    const char *name;
    int rows, tiles; // of a work-group
} SHAPE[SHAPES] = {{"w4_experts_16x128", 16, 8}, {"w4_experts_32x128", 32, 8}, {"w4_experts_64x128", 64, 8}, {"w4_experts_128x256", 128, 16}};

static ExpertsLayout layout_of(const hipq_w4_experts_plan *p, int M)
{
    const hipq_w4_experts_desc &d = p->desc;
    ExpertsLayout l = {};
    l.pairs = (int64_t)M * d.top;
    const int64_t each = l.pairs / d.experts; // an expert's, were all chosen as often
    l.kernel = each <= 16 ? TILE_16 : each <= 32 ? TILE_32 : each <= 64 ? TILE_64 : TILE_128_WIDE;
    l.block_rows = SHAPE[l.kernel].rows;
    const int64_t used = l.pairs < d.experts ? l.pairs : d.experts;
    l.blocks = used + l.pairs / l.block_rows;
    l.blocks = l.blocks < l.pairs ? l.blocks : l.pairs;
    const int64_t groups = l.blocks * ((p->tiles[1] + SHAPE[l.kernel].tiles - 1) / SHAPE[l.kernel].tiles);
    const int most = p->args[1].blocks / 4;
    l.splits = groups < 256 ? (int)(256 / groups) : 1;
    l.splits = l.splits < most ? l.splits : most;
    l.splits = l.splits < 1 ? 1 : l.splits;
    l.columns = round_up(p->tiles[1], SHAPE[l.kernel].tiles) * 16;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t from = at;
        at += (bytes + 255) / 256 * 256;
        return from;
    };
    l.chosen = take(l.pairs * 4), l.share = take(l.pairs * 4), l.place = take(l.pairs * 4), l.row = take(l.pairs * 4), l.block = take(l.blocks * sizeof(W4Block)), l.count = take(4);
    l.hidden = take((size_t)l.pairs * d.inner * 2);
    l.part = take((size_t)l.splits * l.pairs * l.columns * 4);
    if (l.kernel == TILE_128_WIDE) {
        const size_t x = (size_t)round_up(M, 128) * p->args[0].blocks, h = (size_t)((l.pairs + 127) / 128 * 128) * p->args[1].blocks;
        l.xsum = take((x > h ? x : h) * (128 / d.group) * 4);
    }
    l.bytes = at;
    return l;
}

template <int TYPE, int GPB, bool ZEROS, int MT, int NT, int WM, int WN, int WK, int STAGES, bool XSUM>
static int launch_experts(const hipq_w4_experts_plan *p, const ExpertsLayout &l, W4Args a, const W4Groups &g, int tiles, int splits, uint8_t *ws, float *part, hipStream_t st)
{
    constexpr int lds = W4Tile<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM>::LDS;
    static thread_local bool done[64] = {};
    const auto kernel = w4_tile_kernel<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM, W4Groups>;
    if (allow_lds((const void *)kernel, lds, p->device, done))
        return 1;
    if (XSUM) {
        a.m_pad = (a.M + 127) / 128 * 128;
        a.xsum = (const float *)(ws + l.xsum);
        const int64_t groups = ((int64_t)a.m_pad * a.blocks * 16 + 255) / 256;
        const dim3 grid((unsigned)(groups < XSUM_ROW ? groups : XSUM_ROW), (unsigned)((groups + XSUM_ROW - 1) / XSUM_ROW));
        w4_xsum_kernel<TYPE, GPB><<<grid, dim3(256), 0, st>>>(a, (float *)(ws + l.xsum), W4Tile<TYPE, GPB, ZEROS, MT, NT, WM, WN, WK, STAGES, XSUM>::FACTOR);
        if (launch_status("w4_xsum_kernel"))
            return 1;
    }
    const int tiles_n = (tiles + NT * WN - 1) / (NT * WN);
    kernel<<<dim3((unsigned)((l.blocks * tiles_n + 7) / 8 * 8), splits), dim3(64 * WM * WN * WK), lds, st>>>(a, g, 0, tiles_n, part);
    return launch_status("w4_tile_kernel");
}

template <int TYPE, int GPB, bool ZEROS>
static int launch_experts(const hipq_w4_experts_plan *p, const ExpertsLayout &l, const W4Args &a, const W4Groups &g, int tiles, int splits, uint8_t *ws, float *part, hipStream_t st)
{
    switch (l.kernel) {
    case TILE_16:
        return launch_experts<TYPE, GPB, ZEROS, 1, 2, 1, 4, 2, 5, false>(p, l, a, g, tiles, splits, ws, part, st);
    case TILE_32:
        return launch_experts<TYPE, GPB, ZEROS, 2, 2, 1, 4, 2, 4, false>(p, l, a, g, tiles, splits, ws, part, st);
    case TILE_64:
        return launch_experts<TYPE, GPB, ZEROS, 4, 2, 1, 4, 2, 3, false>(p, l, a, g, tiles, splits, ws, part, st);
    }
    return launch_experts<TYPE, GPB, ZEROS, 4, 4, 2, 4, 1, GPB == 4 && ZEROS ? 2 : 3, true>(p, l, a, g, tiles, splits, ws, part, st);
}

template <int TYPE, int GPB>
static int launch_experts(const hipq_w4_experts_plan *p, const ExpertsLayout &l, const W4Args &a, const W4Groups &g, int tiles, int splits, uint8_t *ws, float *part, hipStream_t st)
{
    return a.zeros ? launch_experts<TYPE, GPB, true>(p, l, a, g, tiles, splits, ws, part, st) : launch_experts<TYPE, GPB, false>(p, l, a, g, tiles, splits, ws, part, st);
}

template <int TYPE>
static int launch_experts(const hipq_w4_experts_plan *p, const ExpertsLayout &l, const W4Args &a, const W4Groups &g, int tiles, int splits, uint8_t *ws, float *part, hipStream_t st)
{
    return p->desc.group == 128  ? launch_experts<TYPE, 1>(p, l, a, g, tiles, splits, ws, part, st)
           : p->desc.group == 64 ? launch_experts<TYPE, 2>(p, l, a, g, tiles, splits, ws, part, st)
                                 : launch_experts<TYPE, 4>(p, l, a, g, tiles, splits, ws, part, st);
}

template <int EACH>
static int route(const hipq_w4_experts_plan *p, const RouteArgs &r, hipStream_t st)
{
    const int lds = (16 * r.experts + 32) * 4, most = (16 * MOST_EXPERTS + 32) * 4;
    const bool both = r.M <= 128; // 16 waves choose 128 tokens' experts in the time of a launch
    static thread_local bool done[2][64] = {};
    const auto kernel = both ? experts_number_kernel<EACH> : experts_number_kernel<0>;
    if (!both) {
        experts_choose_kernel<EACH><<<dim3((unsigned)((r.M + 3) / 4)), dim3(256), 0, st>>>(r);
        if (launch_status("experts_choose_kernel"))
            return 1;
    }
    if (lds > 65536 && allow_lds((const void *)kernel, most, p->device, done[both]))
        return 1;
    kernel<<<dim3(1), dim3(1024), lds, st>>>(r);
    return launch_status("experts_number_kernel");
}

template <int TYPE>
static int run_experts(const hipq_w4_experts_plan *p, const ExpertsLayout &l, RouteArgs r, const void *x, int64_t x_stride, void *y, int64_t y_stride, uint8_t *ws, hipStream_t st)
{
    if (r.experts <= 64 ? route<1>(p, r, st) : r.experts <= 256 ? route<4>(p, r, st) : route<16>(p, r, st))
        return 1;
    W4Args a = p->args[0];
    W4Groups g = p->groups[0];
    g.block = r.block, g.count = r.count, g.row = r.row;
    a.x = (const uint16_t *)x, a.x_stride = x_stride, a.y = (uint16_t *)(ws + l.hidden), a.y_stride = p->desc.inner;
    // sums of x are those of tokens, results those of pairs
    a.M = r.M;
    if (launch_experts<TYPE>(p, l, a, g, p->tiles[0], 1, ws, nullptr, st))
        return 1;
    a = p->args[1];
    const W4Block *block = g.block;
    g = p->groups[1];
    g.block = block, g.count = r.count, g.row = nullptr;
    a.x = (const uint16_t *)(ws + l.hidden), a.x_stride = p->desc.inner, a.M = (int)l.pairs;
    if (launch_experts<TYPE>(p, l, a, g, p->tiles[1], l.splits, ws, (float *)(ws + l.part), st))
        return 1;
    const int64_t threads = (int64_t)r.M * ((p->desc.N + 3) / 4);
    experts_join_kernel<TYPE><<<dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st>>>(r, (const float *)(ws + l.part), l.splits, l.pairs, l.columns, (uint16_t *)y, y_stride,
                                                                                          p->desc.N);
    return launch_status("experts_join_kernel");
}

} // namespace hipq

extern "C" int hipq_w4_experts_create(const hipq_w4_experts_desc *d, const uint8_t *gate_up, const void *gate_up_scales, const uint8_t *gate_up_zeros, const uint8_t *down,
                                      const void *down_scales, const uint8_t *down_zeros, void *stream, hipq_w4_experts_plan **out)
{
    clear_error();
    HIPQ_REQUIRE(d && gate_up && gate_up_scales && down && down_scales && out, "experts: a null pointer");
    HIPQ_REQUIRE(is_real16(d->type), "experts: type %d is neither float16 nor bfloat16", d->type);
    HIPQ_REQUIRE(d->group == 32 || d->group == 64 || d->group == 128, "experts: groups of %d (32, 64 and 128 are there)", d->group);
    HIPQ_REQUIRE(d->activation == HIPQ_ACT_SILU || d->activation == HIPQ_ACT_GELU, "experts: activation %d", d->activation);
    HIPQ_REQUIRE(d->scores == HIPQ_SCORES_SOFTMAX || d->scores == HIPQ_SCORES_SIGMOID, "experts: scores %d", d->scores);
    HIPQ_REQUIRE(d->normalize == 0 || d->normalize == 1, "experts: normalize is %d", d->normalize);
    HIPQ_REQUIRE(d->experts >= 1 && d->experts <= MOST_EXPERTS, "experts: %d experts (up to %d are there)", d->experts, MOST_EXPERTS);
    HIPQ_REQUIRE(d->top >= 1 && d->top <= MOST_TOP && d->top <= d->experts, "experts: %d experts of a token (up to %d, and not more than there are)", d->top, MOST_TOP);
    HIPQ_REQUIRE(d->N >= 1 && d->N <= (1 << 20), "experts: %d outputs", d->N);
    HIPQ_REQUIRE(d->K >= 32 && d->K <= (1 << 20) && d->K % 32 == 0, "experts: %d inputs (a multiple of 32 is needed)", d->K);
    HIPQ_REQUIRE(d->inner >= 32 && d->inner <= (1 << 20) && d->inner % 32 == 0, "experts: %d hidden values (a multiple of 32 is needed)", d->inner);
    HIPQ_REQUIRE(!gate_up_zeros == !down_zeros, "experts: zero points for one of the products alone");
    hipq_w4_experts_plan *p = new (std::nothrow) hipq_w4_experts_plan();
    HIPQ_REQUIRE(p, "experts: out of host memory");
    p->desc = *d;
    const int gpb = 128 / d->group;
    size_t q_bytes[2], s_bytes[2], total = 256;
    for (int i = 0; i < 2; i++) {
        W4Args &a = p->args[i];
        a.N = i ? d->N : d->inner, a.K = i ? d->inner : d->K, a.blocks = (a.K + 127) / 128, a.activation = i ? HIPQ_ACT_NONE : d->activation;
        a.zeros = gate_up_zeros != nullptr;
        p->tiles[i] = (a.N + 15) / 16 * (i ? 1 : 2);
        const size_t pieces = (size_t)round_up(p->tiles[i], 16) * a.blocks;
        q_bytes[i] = pieces * 1024, s_bytes[i] = pieces * 16 * gpb * (a.zeros ? 4 : 2);
        total += d->experts * (q_bytes[i] + s_bytes[i]);
    }
    hipError_t e = hipGetDevice(&p->device);
    if (e == hipSuccess)
        e = hipMalloc(&p->memory, total);
    if (e != hipSuccess) {
        delete p;
        return fail("experts: no memory for %zu bytes of weights: %s", total, hipGetErrorString(e));
    }
    uint8_t *at = p->memory + 256;
    int bad = 0;
    for (int i = 0; i < 2; i++) {
        W4Args &a = p->args[i];
        W4Groups &g = p->groups[i];
        g.q_bytes = q_bytes[i], g.s_bytes = s_bytes[i];
        a.q = at, at += d->experts * q_bytes[i];
        a.scales = at, at += d->experts * s_bytes[i];
        a.nothing = (const uint16_t *)p->memory;
        PackArgs k = {};
        k.rows = a.N, k.K = a.K, k.group = d->group, k.groups = (a.K + d->group - 1) / d->group, k.blocks = a.blocks, k.tiles = round_up(p->tiles[i], 16), k.gated = !i;
        const size_t rows = (size_t)a.N * (i ? 1 : 2);
        for (int x = 0; x < d->experts && !bad; x++) {
            k.q = (i ? down : gate_up) + x * rows * (a.K / 2), k.scales = (const uint16_t *)(i ? down_scales : gate_up_scales) + x * rows * k.groups;
            k.zeros = a.zeros ? (i ? down_zeros : gate_up_zeros) + x * rows * k.groups : nullptr;
            k.to_q = const_cast<uint8_t *>(a.q) + x * q_bytes[i], k.to_scales = (uint16_t *)(a.scales + x * s_bytes[i]), k.to_nothing = (u32x4 *)p->memory;
            bad = w4_pack(k, d->type, (hipStream_t)stream);
        }
    }
    if (!bad && (e = hipStreamSynchronize((hipStream_t)stream)) != hipSuccess)
        bad = fail("experts: laying the weights out failed: %s", hipGetErrorString(e));
    if (bad) {
        (void)hipFree(p->memory);
        delete p;
        return 1;
    }
    *out = p;
    return 0;
}

extern "C" void hipq_w4_experts_destroy(hipq_w4_experts_plan *p)
{
    if (!p)
        return;
    (void)hipFree(p->memory); // waits for what still reads it
    delete p;
}

// byte offsets of 32 bits, numbers of pairs and work-groups of 31
static int experts_fit(const hipq_w4_experts_plan *p, int M)
{
    HIPQ_REQUIRE(p, "experts: a null plan");
    HIPQ_REQUIRE(M >= 0 && M <= (1 << 20), "experts: %d rows", M);
    HIPQ_REQUIRE((int64_t)M * p->desc.top * p->desc.inner < ((int64_t)1 << 31), "experts: %d rows of %d experts, %d hidden values each", M, p->desc.top, p->desc.inner);
    if (M > 0) {
        const ExpertsLayout l = layout_of(p, M);
        const int tiles = p->tiles[0] > p->tiles[1] ? p->tiles[0] : p->tiles[1];
        HIPQ_REQUIRE(l.blocks * ((tiles + 7) / 8) <= (1 << 23) - 8, "experts: %d rows of %d outputs", M, p->desc.N);
        HIPQ_REQUIRE((int64_t)M * ((p->desc.N + 3) / 4) < ((int64_t)1 << 32) - 256, "experts: %d rows of %d outputs", M, p->desc.N);
    }
    return 0;
}

extern "C" const char *hipq_w4_experts_kernel(const hipq_w4_experts_plan *p, int M)
{
    clear_error();
    return experts_fit(p, M) ? "" : SHAPE[layout_of(p, M > 0 ? M : 1).kernel].name;
}

extern "C" size_t hipq_w4_experts_workspace(const hipq_w4_experts_plan *p, int M)
{
    clear_error();
    return experts_fit(p, M) || M == 0 ? 0 : layout_of(p, M).bytes;
}

extern "C" int hipq_w4_experts_run(const hipq_w4_experts_plan *p, const void *x, int64_t x_stride, const void *logits, int logits_type, int64_t logits_stride, void *y,
                                   int64_t y_stride, int M, void *workspace, size_t workspace_bytes, void *stream)
{
    clear_error();
    if (experts_fit(p, M))
        return 1;
    HIPQ_REQUIRE(logits_type == HIPQ_REAL_F32 || is_real16(logits_type), "experts: logits of type %d", logits_type);
    if (M == 0)
        return 0;
    const hipq_w4_experts_desc &d = p->desc;
    HIPQ_REQUIRE(x && logits && y, "experts: a null pointer");
    HIPQ_REQUIRE((uintptr_t)x % 16 == 0 && x_stride % 8 == 0, "experts: rows of x have to start at multiples of 16 bytes");
    const int logit = logits_type == HIPQ_REAL_F32 ? 4 : 2;
    HIPQ_REQUIRE((uintptr_t)y % 2 == 0 && (uintptr_t)logits % logit == 0, "experts: logits or y are not aligned to their type");
    HIPQ_REQUIRE(M == 1 || (x_stride >= d.K && y_stride >= d.N && logits_stride >= d.experts), "experts: rows overlap (strides %lld, %lld and %lld)", (long long)x_stride,
                 (long long)logits_stride, (long long)y_stride);
    HIPQ_REQUIRE(M == 1 || (x_stride < (1 << 30) && (M - 1) * x_stride + d.K < ((int64_t)1 << 31)), "experts: %d rows of x, %lld elements apart", M, (long long)x_stride);
    const ByteRows written = {(int64_t)(uintptr_t)y, M > 1 ? y_stride * 2 : 0, d.N * 2ll, M};
    HIPQ_REQUIRE(!overlap({(int64_t)(uintptr_t)x, M > 1 ? x_stride * 2 : 0, d.K * 2ll, M}, written), "experts: y lies over x");
    HIPQ_REQUIRE(!overlap({(int64_t)(uintptr_t)logits, M > 1 ? logits_stride * logit : 0, (int64_t)d.experts * logit, M}, written), "experts: y lies over the logits");
    const ExpertsLayout l = layout_of(p, M);
    HIPQ_REQUIRE(workspace && workspace_bytes >= l.bytes && (uintptr_t)workspace % 16 == 0, "experts: a workspace of %zu bytes is needed", l.bytes);
    int device;
    HIPQ_CHECK_HIP(hipGetDevice(&device));
    HIPQ_REQUIRE(device == p->device, "experts: the plan is on device %d, the current one is %d", p->device, device);
    uint8_t *ws = (uint8_t *)workspace;
    RouteArgs r = {};
    r.logits = logits, r.stride = M > 1 ? logits_stride : 0, r.type = logits_type, r.M = M, r.experts = d.experts, r.top = d.top;
    r.sigmoid = d.scores == HIPQ_SCORES_SIGMOID, r.normalize = d.normalize, r.block_rows = l.block_rows;
    r.chosen = (int32_t *)(ws + l.chosen), r.share = (float *)(ws + l.share), r.place = (int32_t *)(ws + l.place), r.row = (int32_t *)(ws + l.row);
    r.block = (W4Block *)(ws + l.block), r.count = (int32_t *)(ws + l.count);
    return d.type == HIPQ_REAL_BF16 ? run_experts<HIPQ_REAL_BF16>(p, l, r, x, M > 1 ? x_stride : 0, y, y_stride, ws, (hipStream_t)stream)
                                    : run_experts<HIPQ_REAL_F16>(p, l, r, x, M > 1 ? x_stride : 0, y, y_stride, ws, (hipStream_t)stream);
}
