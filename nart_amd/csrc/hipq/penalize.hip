// Scores before a token is drawn from them (hipq_penalize): penalties for repeated tokens, biases, a grammar's bits.  gfx950 only.
//
// A pass over memory: a score is read once and written once.  What a row's history does to a score depends on how often its token has occurred, so a work-group has a
// slice of the vocabulary with a counter for each of its tokens in LDS, reads the whole history, which is short and in the L2 for all but the first of a row's slices,
// and counts what falls into its slice; integers, so that the order does not matter.  Its own scores are on their way meanwhile.  256 rows of 128000 in float32 with histories of up to
// 4000: 270 MB in 60 us, 4.5 TB/s of the 5.1 of a copy; one row 6 us, a launch and three rounds of loads and barriers.
#include "overlap.h"
#include "real16.h"

namespace hipq {

struct PenalizeArgs {
    hipq_penalize_desc d;
    int slices;
};

constexpr uint32_t OCCURRED = 0x80000000u; // in the prompt; a counter below it

// 16 bytes of a row that begins anywhere
template <int BYTES>
struct Piece;
template <>
struct Piece<2> {
    typedef u32x4 __attribute__((aligned(2))) type;
};
template <>
struct Piece<4> {
    typedef u32x4 __attribute__((aligned(4))) type;
};

// THREADS of a work-group, each with 16 tokens of a slice, 16 bytes of scores at a time
template <int TYPE, int THREADS>
__global__ __launch_bounds__(THREADS, 8) void penalize_kernel(const PenalizeArgs a)
{
    constexpr int EACH = 16, SLICE = EACH * THREADS, WIDE = TYPE == HIPQ_REAL_F32 ? 4 : 8, PIECES = EACH / WIDE, BYTES = TYPE == HIPQ_REAL_F32 ? 4 : 2;
    using piece_t = typename Piece<BYTES>::type;
    extern __shared__ __attribute__((aligned(16))) uint32_t counts[]; // [SLICE], then, with biases, the entry of each token's bias + 1
    const hipq_penalize_desc &d = a.d;
    const int64_t group = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, row = group / a.slices;
    if (row >= d.rows)
        return;
    const int tid = threadIdx.x, first = (int)(group - row * a.slices) * SLICE, vocab = d.vocab;
    const uint8_t *const in = (const uint8_t *)d.logits + row * d.stride * BYTES;
    uint8_t *const out = (uint8_t *)d.out + row * d.out_stride * BYTES;

    // the history is on its way before the scores, as loads are waited for in their order
    constexpr int AHEAD = 4;
    const bool history = d.tokens != nullptr, biases = d.bias != nullptr;
    const int32_t *const tokens = d.tokens + row * d.tokens_stride;
    const int len = !history ? 0 : min(d.lens ? max(d.lens[row], 0) : d.longest, d.longest), prompt = d.prompt_lens ? d.prompt_lens[row] : 0;
    const float repetition = d.repetition ? d.repetition[row] : 1.0f, frequency = d.frequency ? d.frequency[row] : 0.0f, presence = d.presence ? d.presence[row] : 0.0f;
    int32_t occurred[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; k++)
        occurred[k] = tid + k * THREADS < len ? tokens[tid + k * THREADS] : -1;

    u32x4 x[PIECES];
    uint32_t bits[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
        const int v = first + (p * THREADS + tid) * WIDE;
        bits[p] = 0xff;
        x[p] = u32x4{0, 0, 0, 0};
        if (v + WIDE <= vocab)
            x[p] = *(const piece_t *)(in + (int64_t)v * BYTES);
        else
#pragma unroll
            for (int e = 0; e < WIDE; e++)
                if (v + e < vocab) {
                    if (BYTES == 4)
                        x[p][e % 4] = ((const uint32_t *)in)[v + e];
                    else
                        x[p][e / 2 % 4] |= (uint32_t)((const uint16_t *)in)[v + e] << (16 * (e % 2));
                }
        if (d.allowed && v < vocab)
            bits[p] = ((const uint8_t *)(d.allowed + row * d.allowed_stride))[v / 8] >> (v % 8);
    }

    uint32_t *const entry = counts + SLICE;
    if (history || biases) {
        const u32x4 none = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < EACH / 4; i++) {
            if (history)
                ((u32x4 *)counts)[i * THREADS + tid] = none;
            if (biases)
                ((u32x4 *)entry)[i * THREADS + tid] = none;
        }
        __syncthreads();
        auto count = [&](int i, int32_t token) {
            const uint32_t at = (uint32_t)token - (uint32_t)first; // outside of the slice: large
            if (at < (uint32_t)SLICE) {
                if (i < prompt)
                    atomicOr(&counts[at], OCCURRED);
                else
                    atomicAdd(&counts[at], 1u);
            }
        };
        if (history) {
#pragma unroll
            for (int k = 0; k < AHEAD; k++)
                if (tid + k * THREADS < len)
                    count(tid + k * THREADS, occurred[k]);
#pragma unroll 4
            for (int i = tid + AHEAD * THREADS; i < len; i += THREADS)
                count(i, tokens[i]);
        }
        if (biases) {
            const int32_t *const tokens = d.bias_tokens + row * d.bias_stride;
            for (int i = tid; i < d.biases; i += THREADS) {
                const uint32_t at = (uint32_t)tokens[i] - (uint32_t)first;
                if (at < (uint32_t)SLICE)
                    atomicMax(&entry[at], (uint32_t)i + 1);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
        const int at = (p * THREADS + tid) * WIDE, v = first + at;
        float s[WIDE];
#pragma unroll
        for (int e = 0; e < WIDE; e++)
            if constexpr (TYPE == HIPQ_REAL_F32) {
                const uint32_t word = x[p][e]; // the cast of a vector's element itself takes the first
                s[e] = __builtin_bit_cast(float, word);
            } else
                s[e] = e & 1 ? Real16<TYPE>::high(x[p][e / 2]) : Real16<TYPE>::low(x[p][e / 2]);
        if (history) {
            uint32_t n[WIDE], any = 0;
#pragma unroll
            for (int i = 0; i < WIDE; i += 4) {
                const u32x4 w = *(const u32x4 *)(counts + at + i);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    n[i + e] = w[e], any |= w[e];
            }
            if (any)
#pragma unroll
                for (int e = 0; e < WIDE; e++)
                    if (n[e]) {
                        if (d.repetition)
                            s[e] = s[e] > 0 ? s[e] / repetition : s[e] * repetition;
                        if (n[e] & ~OCCURRED)
                            s[e] -= (float)(n[e] & ~OCCURRED) * frequency + presence;
                    }
        }
        if (biases)
#pragma unroll
            for (int e = 0; e < WIDE; e++)
                if (entry[at + e])
                    s[e] += d.bias[row * d.bias_stride + entry[at + e] - 1];
#pragma unroll
        for (int e = 0; e < WIDE; e++)
            s[e] = (bits[p] >> e) & 1 ? s[e] : -__builtin_inff();
#pragma unroll
        for (int e = 0; e < 4; e++)
            if constexpr (TYPE == HIPQ_REAL_F32)
                x[p][e] = __builtin_bit_cast(uint32_t, s[e]);
            else
                x[p][e] = Real16<TYPE>::pack(s[2 * e], s[2 * e + 1]);
        if (v + WIDE <= vocab)
            *(piece_t *)(out + (int64_t)v * BYTES) = x[p];
        else
#pragma unroll
            for (int e = 0; e < WIDE; e++)
                if (v + e < vocab) {
                    if (BYTES == 4)
                        ((uint32_t *)out)[v + e] = x[p][e % 4];
                    else
                        ((uint16_t *)out)[v + e] = (uint16_t)(x[p][e / 2 % 4] >> (16 * (e % 2)));
                }
    }
}

constexpr int64_t PENALIZE_ROW = 1 << 20; // work-groups side by side: of 2^32 work-items and more only what is left over would run

template <int TYPE, int THREADS>
static int launch_penalize(PenalizeArgs &a, hipStream_t st)
{
    static thread_local bool done[64] = {};
    constexpr int SLICE = 16 * THREADS;
    const size_t lds = (size_t)SLICE * 4 * ((a.d.tokens ? 1 : a.d.bias ? 1 : 0) + (a.d.bias ? 1 : 0));
    const auto kernel = penalize_kernel<TYPE, THREADS>;
    if (lds > 65536) {
        int device;
        HIPQ_CHECK_HIP(hipGetDevice(&device));
        if (device >= 64 || !done[device])
            HIPQ_CHECK_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, SLICE * 8));
        if (device < 64)
            done[device] = true;
    }
    a.slices = (a.d.vocab + SLICE - 1) / SLICE;
    const int64_t groups = (int64_t)a.slices * a.d.rows, side = groups < PENALIZE_ROW ? groups : PENALIZE_ROW;
    const int64_t rows = (groups + side - 1) / side;
    HIPQ_REQUIRE(rows < 65536, "penalize: %d rows of %d scores", a.d.rows, a.d.vocab);
    kernel<<<dim3((unsigned)side, (unsigned)rows), dim3(THREADS), lds, st>>>(a);
    return launch_status("penalize_kernel");
}

template <int TYPE>
static int launch_penalize(PenalizeArgs &a, hipStream_t st)
{
    // large slices read a row's history less often, small ones fill the chip: us with 512 and 1024 threads, 8 rows of 128000 9.2 and 10.3, 32 rows 10.2 and 9.6, 256 rows 43 and
    // 42 (with 256 threads 10.5, 11.7 and 52)
    return (int64_t)a.d.rows * ((a.d.vocab + 16383) / 16384) >= 256 ? launch_penalize<TYPE, 1024>(a, st) : launch_penalize<TYPE, 512>(a, st);
}

} // namespace hipq

using namespace hipq;

extern "C" int hipq_penalize(const hipq_penalize_desc *d, void *stream)
{
    clear_error();
    HIPQ_REQUIRE(d, "penalize: a null pointer");
    HIPQ_REQUIRE(d->type == HIPQ_REAL_F32 || is_real16(d->type), "penalize: type %d", d->type);
    HIPQ_REQUIRE(d->rows >= 0 && d->rows <= (1 << 24), "penalize: %d rows", d->rows);
    HIPQ_REQUIRE(d->vocab >= 0 && d->vocab <= (1 << 20), "penalize: %d scores of a row (up to 2^20 are there)", d->vocab);
    HIPQ_REQUIRE(d->longest >= 0 && d->longest < (1 << 30), "penalize: histories of %d tokens", d->longest);
    HIPQ_REQUIRE(d->biases >= 0 && d->biases < (1 << 30), "penalize: %d biases", d->biases);
    if (d->rows == 0 || d->vocab == 0)
        return 0;
    const int bytes = d->type == HIPQ_REAL_F32 ? 4 : 2;
    HIPQ_REQUIRE(d->logits && d->out, "penalize: a null pointer");
    HIPQ_REQUIRE(((uintptr_t)d->logits | (uintptr_t)d->out) % bytes == 0, "penalize: scores are not aligned to their type");
    HIPQ_REQUIRE(d->rows == 1 || (d->stride >= d->vocab && d->out_stride >= d->vocab), "penalize: rows overlap (strides %lld and %lld)", (long long)d->stride, (long long)d->out_stride);
    HIPQ_REQUIRE(d->tokens || d->longest == 0, "penalize: histories of %d tokens, and no tokens", d->longest);
    HIPQ_REQUIRE(d->biases == 0 || (d->bias && d->bias_tokens), "penalize: biases and their tokens belong together");
    HIPQ_REQUIRE(d->rows == 1 || ((!d->tokens || d->tokens_stride >= d->longest) && (!d->bias || d->bias_stride >= d->biases)
                                  && (!d->allowed || d->allowed_stride >= (d->vocab + 31) / 32)),
                 "penalize: rows of tokens, biases or bits overlap");
    const ByteRows read = {(int64_t)(uintptr_t)d->logits, d->rows > 1 ? d->stride * bytes : 0, (int64_t)d->vocab * bytes, d->rows};
    const ByteRows written = {(int64_t)(uintptr_t)d->out, d->rows > 1 ? d->out_stride * bytes : 0, (int64_t)d->vocab * bytes, d->rows};
    HIPQ_REQUIRE((d->out == d->logits && (d->rows == 1 || d->stride == d->out_stride)) || !overlap(read, written), "penalize: out lies over the scores");
    PenalizeArgs a = {};
    a.d = *d;
    if (d->rows == 1)
        a.d.stride = a.d.out_stride = a.d.tokens_stride = a.d.bias_stride = a.d.allowed_stride = 0;
    if (d->longest == 0)
        a.d.tokens = nullptr;
    if (d->biases == 0)
        a.d.bias = nullptr;
    return d->type == HIPQ_REAL_F32   ? launch_penalize<HIPQ_REAL_F32>(a, (hipStream_t)stream)
           : d->type == HIPQ_REAL_F16 ? launch_penalize<HIPQ_REAL_F16>(a, (hipStream_t)stream)
                                      : launch_penalize<HIPQ_REAL_BF16>(a, (hipStream_t)stream);
}
