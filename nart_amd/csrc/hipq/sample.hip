// A token of every row of scores (hipq_sample): temperature, top-k, top-p and min-p from given uniform numbers.  gfx950 only.
//
// Ordered by score (equal ones by index), each filter keeps a prefix, so what is kept is one border: a score, and how many of the scores
// equal to it.  Nothing is sorted.  A filter keeps what has less than `need` in front of it - tokens for top-k, weight for top-p: the
// scores are divided into 2048 intervals below the maximum, the interval is found in which the running sum reaches `need`, what lies in it is
// collected and divided again by the bits of the scores, until an interval is a single score.
// Weights are 64-bit fixed point, 2^-43 of the largest: sums do not depend on their order, so that neither atomics nor the number of
// threads show in a result, and they come from a polynomial in 64 bits (2^-43 of their value off at most): a running sum in 32 bits goes wrong
// where two tokens' borders lie closer than its rounding, at 10^5 tokens once in some hundred rows.
//
// One work-group has a row, and reads it some times: the first from memory, the others from the caches.
#include "real16.h"

// a lambda that is called instead of inlined takes the row's state to memory
#define INLINE __attribute__((always_inline))

namespace hipq {

constexpr int THREADS = 1024, WAVES = THREADS / 64, BINS = 2048, LIST = 4096, FRACTION = 43;
constexpr int MOST_VOCAB = 1 << 20; // sums of weights fit 64 bits

struct SampleArgs {
    const void *logits;
    int64_t stride;
    const float *uniform, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int64_t *tokens;
    int vocab;
};

struct SampleShared {
    uint64_t bins[BINS];
    uint32_t list[LIST];
    double powers[256]; // 2^(i / 256)
    uint64_t wave[WAVES];
    uint64_t sum, before;
    uint32_t bin, listed, low, high;
    float top;
    int index;
};

template <int TYPE>
struct Scores {
    static constexpr int E = TYPE == HIPQ_REAL_F32 ? 4 : 8; // of a 16-byte load
    struct __attribute__((packed, aligned(TYPE == HIPQ_REAL_F32 ? 4 : 2))) Vec {
        u32x4 v;
    };
    __device__ static __forceinline__ float clean(float x) { return x == x ? x : -__builtin_inff(); } // NaN: never taken
    __device__ static __forceinline__ float one(const void *row, int i)
    {
        if (TYPE == HIPQ_REAL_F32)
            return clean(((const float *)row)[i]);
        return clean(Real16<TYPE == HIPQ_REAL_F32 ? HIPQ_REAL_F16 : TYPE>::low(((const uint16_t *)row)[i]));
    }
    // elements i .. i + E - 1, those behind the end as -infinity
    __device__ static __forceinline__ void some(const void *row, int i, int end, float (&x)[E])
    {
        if (i + E <= end) {
            const u32x4 v = ((const Vec *)((const uint8_t *)row + (int64_t)i * (16 / E)))->v;
#pragma unroll
            for (int e = 0; e < E; e++) {
                using R = Real16<TYPE == HIPQ_REAL_F32 ? HIPQ_REAL_F16 : TYPE>;
                x[e] = clean(TYPE == HIPQ_REAL_F32 ? __builtin_bit_cast(float, (uint32_t)v[e % 4]) : e & 1 ? R::high(v[e / 2]) : R::low(v[e / 2]));
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; e++)
                x[e] = i + e < end ? one(row, i + e) : -__builtin_inff();
        }
    }
};

// larger scores have larger keys; -0 and 0 are the same score
__device__ static __forceinline__ uint32_t key_of(float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ static __forceinline__ float score_of(uint32_t key)
{
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

template <int TYPE>
struct Row {
    static constexpr int E = Scores<TYPE>::E;
    const SampleArgs &a;
    SampleShared &s;
    const void *row;
    int tid, lane, wave;
    float top, per_bin; // intervals of a unit of score
    double rate;        // log2(e) / temperature
    // the border: scores above key are kept, and of those equal to it the first `ties` (up to index `last`)
    uint32_t key = 0, ties = 0xffffffffu;
    int last = 0x7fffffff;
    uint64_t least = 0; // smallest weight that min-p keeps

    __device__ Row(const SampleArgs &a_, SampleShared &s_) : a(a_), s(s_)
    {
        tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        row = (const uint8_t *)a.logits + (int64_t)blockIdx.x * a.stride * (TYPE == HIPQ_REAL_F32 ? 4 : 2);
    }

    template <class F>
    __device__ __forceinline__ void each(F f)
    {
        constexpr int U = E / 2, STEP = THREADS * E;
        for (int base = tid * E; base < a.vocab; base += U * STEP) {
            float x[U][E];
#pragma unroll
            for (int u = 0; u < U; u++)
                Scores<TYPE>::some(row, base + u * STEP, a.vocab, x[u]);
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < E; e++)
                    f(x[u][e], base + u * STEP + e);
        }
    }

    // 2^(rate (x - top)) in units of 2^-43: 2^(n / 256) from the table times 2^r, |r| <= 1 / 512, to the fourth term (the fifth is under 2^-48)
    __device__ __forceinline__ uint64_t weight(float x) const
    {
        if (x == top)
            return (uint64_t)1 << FRACTION;
        const double y = ((double)x - (double)top) * rate; // below 0
        if (!(y > -44.5))
            return 0;
        const double big = 6755399441055744.0 / 256; // 1.5 * 2^52 / 256: what is added keeps eight bits behind the point
        const double t = y + big, r = y - (t - big);
        const int n = (int)(uint32_t)__builtin_bit_cast(uint64_t, t);
        double p = __builtin_fma(r, 0.0096181291076284772, 0.055504108664821580);
        p = __builtin_fma(p, r, 0.24022650695910071);
        p = __builtin_fma(p, r, 0.69314718055994531);
        p = __builtin_fma(p, r, 1.0);
        const double one = 4503599627370496.0; // 2^52: the sum's lower bits are the rounded number
        return __builtin_bit_cast(uint64_t, __builtin_ldexp(p * s.powers[n & 255], (n >> 8) + FRACTION) + one) - __builtin_bit_cast(uint64_t, one);
    }
    __device__ __forceinline__ int bin_of(float x) const
    {
        const float v = (top - x) * per_bin;
        return v < BINS - 1 ? (int)v : BINS - 1;
    }
    __device__ __forceinline__ bool kept(float x, int i) const
    {
        const uint32_t k = key_of(x);
        return k > key || (k == key && i <= last);
    }

    __device__ __forceinline__ void clear_bins()
    {
        for (int i = tid; i < BINS; i += THREADS)
            s.bins[i] = 0;
    }

    // sum over the threads in front, and s.sum over all; every thread calls it
    __device__ __forceinline__ uint64_t scan(uint64_t v)
    {
        uint64_t in = v;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const uint64_t up = __shfl_up(in, o);
            in += lane >= o ? up : 0;
        }
        __syncthreads(); // s.wave may still be read
        if (lane == 63)
            s.wave[wave] = in;
        __syncthreads();
        uint64_t front = 0, all = 0;
        for (int w = 0; w < WAVES; w++) {
            const uint64_t t = s.wave[w];
            front += w < wave ? t : 0;
            all += t;
        }
        if (tid == 0)
            s.sum = all;
        return front + in - v;
    }

    // the first bin in which the running sum reaches need: s.bin, and s.before what lies in front of it.  false: the sum stays below
    __device__ __forceinline__ bool find(uint64_t need)
    {
        const uint64_t b0 = s.bins[2 * tid], b1 = s.bins[2 * tid + 1];
        const uint64_t front = scan(b0 + b1);
        __syncthreads();
        const bool reached = s.sum >= need;
        if (front < need && need <= front + b0)
            s.bin = 2 * tid, s.before = front;
        else if (front + b0 < need && need <= front + b0 + b1)
            s.bin = 2 * tid + 1, s.before = front + b0;
        __syncthreads();
        return reached;
    }

    // moves the border to where `need` is reached; the bins hold the first division.  MASS: of weight, otherwise of tokens.  The tokens
    // counted are those above the present border, and `ties` at it.
    template <bool MASS>
    __device__ __forceinline__ void cut(uint64_t need)
    {
        if (!find(need))
            return;
        const int bin = (int)s.bin;
        need -= s.before;
        if (tid == 0)
            s.listed = 0, s.low = 0xffffffffu, s.high = 0;
        __syncthreads();
        const uint32_t old = key, old_ties = ties;
        uint32_t low = 0xffffffffu, high = 0;
        each([&](float x, int i) INLINE {
            if (bin_of(x) == bin && x > -__builtin_inff() && i < a.vocab) {
                const uint32_t k = key_of(x);
                if (k > old || (k == old && old_ties == 0xffffffffu)) {
                    low = min(low, k), high = max(high, k);
                    const uint32_t at = atomicAdd(&s.listed, 1u);
                    if (at < LIST)
                        s.list[at] = k;
                }
            }
        });
        const bool tied = old_ties != 0xffffffffu && bin_of(score_of(old)) == bin; // the border's own ties count as many as are kept
        if (tied)
            low = min(low, old), high = max(high, old);
#pragma unroll
        for (int o = 1; o < 64; o *= 2)
            low = min(low, (uint32_t)__shfl_xor((int)low, o)), high = max(high, (uint32_t)__shfl_xor((int)high, o));
        if (lane == 0)
            atomicMin(&s.low, low), atomicMax(&s.high, high);
        __syncthreads();
        low = s.low, high = s.high;
        const uint32_t listed = s.listed;
        for (int level = 0; level < 4; level++) { // 11 bits of the interval [low, high] at a time: at most three times
            const int bits = high == low ? 0 : 32 - __clz((int)(high - low)), shift = bits > 11 ? bits - 11 : 0;
            clear_bins();
            __syncthreads();
            auto add = [&](uint32_t k) INLINE {
                if (k >= low && k <= high)
                    atomicAdd((unsigned long long *)&s.bins[(high - k) >> shift], (unsigned long long)(MASS ? weight(score_of(k)) : 1));
            };
            if (listed <= LIST) {
                for (uint32_t i = tid; i < listed; i += THREADS)
                    add(s.list[i]);
            } else
                each([&](float x, int i) INLINE {
                    if (bin_of(x) == bin && x > -__builtin_inff() && i < a.vocab) {
                        const uint32_t k = key_of(x);
                        if (k > old || (k == old && old_ties == 0xffffffffu))
                            add(k);
                    }
                });
            if (tied && tid == 0 && old >= low && old <= high)
                atomicAdd((unsigned long long *)&s.bins[(high - old) >> shift], (unsigned long long)(MASS ? weight(score_of(old)) * old_ties : old_ties));
            __syncthreads();
            find(need);
            need -= s.before;
            const uint32_t at = s.bin, to = high - (at << shift);
            if (shift == 0) {
                const uint64_t each_one = MASS ? weight(score_of(to)) : 1, there = s.bins[at] / each_one, wanted = (need + each_one - 1) / each_one;
                key = to;
                // all of them: those of the row, or as many as an earlier border left
                ties = wanted < there ? (uint32_t)wanted : tied && to == old ? old_ties : 0xffffffffu;
                __syncthreads();
                return;
            }
            const uint32_t down = (1u << shift) - 1;
            low = to - low > down ? to - down : low;
            high = to;
            __syncthreads();
        }
    }

    // The first index, in order, at which the running sum of f exceeds `target(sum)`; f: 64-bit whole numbers, their sum above 0.
    template <class F, class T>
    __device__ __forceinline__ int locate(F f, T target)
    {
        const int part = (a.vocab + WAVES * E - 1) / (WAVES * E) * E, from = wave * part, to = min(a.vocab, from + part);
        uint64_t v = 0;
        constexpr int U = E / 2, STEP = 64 * E;
        for (int base = from + lane * E; base < to; base += U * STEP) {
            float x[U][E];
#pragma unroll
            for (int u = 0; u < U; u++)
                Scores<TYPE>::some(row, base + u * STEP, to, x[u]);
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < E; e++)
                    v += f(x[u][e], base + u * STEP + e);
        }
#pragma unroll
        for (int o = 1; o < 64; o *= 2)
            v += __shfl_xor(v, o);
        __syncthreads();
        if (lane == 0)
            s.wave[wave] = v;
        __syncthreads();
        uint64_t all = 0, front = 0;
        for (int i = 0; i < WAVES; i++)
            all += s.wave[i];
        const uint64_t goal = target(all);
        int w = 0;
        for (; w < WAVES - 1 && front + s.wave[w] <= goal; w++)
            front += s.wave[w];
        const int begin = w * part, end = min(a.vocab, begin + part);
        if (tid == 0)
            s.index = -1;
        for (int base = begin; base < end; base += THREADS * E) {
            float x[E];
            const int i = base + tid * E;
            Scores<TYPE>::some(row, i, end, x);
            uint64_t own = 0;
#pragma unroll
            for (int e = 0; e < E; e++)
                own += f(x[e], i + e);
            uint64_t run = front + scan(own);
            if (run <= goal && goal < run + own) {
                int e = 0;
                for (; e < E - 1; e++) {
                    run += f(x[e], i + e);
                    if (run > goal)
                        break;
                }
                s.index = i + e;
            }
            __syncthreads();
            front += s.sum;
            if (s.index >= 0)
                break;
        }
        return s.index;
    }
};

template <int TYPE>
__global__ __launch_bounds__(THREADS) void sample_kernel(const SampleArgs a)
{
    __shared__ SampleShared s;
    Row<TYPE> r(a, s);
    const int tid = threadIdx.x;
    const float none = -__builtin_inff();

    if (tid < 256)
        s.powers[tid] = exp2((double)tid / 256);
    float top = none;
    r.each([&](float x, int) INLINE { top = fmaxf(top, x); });
#pragma unroll
    for (int o = 1; o < 64; o *= 2)
        top = fmaxf(top, __shfl_xor(top, o));
    if (r.lane == 0)
        s.list[r.wave] = __builtin_bit_cast(uint32_t, top);
    __syncthreads();
    for (int w = 0; w < WAVES; w++)
        top = fmaxf(top, __builtin_bit_cast(float, s.list[w]));
    __syncthreads();
    r.top = top;
    const float t = a.temperature ? a.temperature[blockIdx.x] : 1.0f;
    if (top == none) {
        if (tid == 0)
            a.tokens[blockIdx.x] = -1;
        return;
    }
    if (!(t > 0)) {
        if (tid == 0)
            s.index = 0x7fffffff;
        __syncthreads();
        int first = 0x7fffffff;
        r.each([&](float x, int i) INLINE { first = x == top ? min(first, i) : first; });
#pragma unroll
        for (int o = 1; o < 64; o *= 2)
            first = min(first, __shfl_xor(first, o));
        if (r.lane == 0)
            atomicMin(&s.index, first);
        __syncthreads();
        if (tid == 0)
            a.tokens[blockIdx.x] = s.index;
        return;
    }
    r.rate = 1.4426950408889634 / (double)t;
    // 2047 intervals down to where weights are 0, the last one for all below
    r.per_bin = (float)((BINS - 1) * r.rate / 44.5);
    r.per_bin = r.per_bin < 1e30f ? r.per_bin : 1e30f;
    if (a.min_p) {
        const double p = (double)a.min_p[blockIdx.x] * (double)((uint64_t)1 << FRACTION);
        r.least = p > 0 ? p < (double)((uint64_t)1 << FRACTION) ? (uint64_t)ceil(p) : (uint64_t)1 << FRACTION : 0;
    }
    const int k = a.top_k ? a.top_k[blockIdx.x] : 0;
    const float p = a.top_p ? a.top_p[blockIdx.x] : 1.0f;
    const bool by_count = k > 0 && k < a.vocab, by_mass = p < 1;
    if (by_count) {
        r.clear_bins();
        __syncthreads();
        r.each([&](float x, int i) INLINE {
            if (x > none)
                atomicAdd((unsigned long long *)&s.bins[r.bin_of(x)], 1ull);
        });
        __syncthreads();
        // a border among scores without weight changes nothing
        r.template cut<false>((uint64_t)k);
    }
    if (by_mass) {
        r.clear_bins();
        __syncthreads();
        const uint32_t key = r.key, ties = r.ties;
        r.each([&](float x, int i) INLINE {
            const uint32_t own = key_of(x);
            if (x > none && (own > key || (own == key && ties == 0xffffffffu))) {
                const uint64_t w = r.weight(x);
                if (w)
                    atomicAdd((unsigned long long *)&s.bins[r.bin_of(x)], (unsigned long long)w);
            }
        });
        if (tid == 0 && ties != 0xffffffffu)
            atomicAdd((unsigned long long *)&s.bins[r.bin_of(score_of(key))], (unsigned long long)(r.weight(score_of(key)) * ties));
        __syncthreads();
        r.scan(s.bins[2 * tid] + s.bins[2 * tid + 1]);
        __syncthreads();
        const double goal = p > 0 ? ceil((double)p * (double)s.sum) : 1;
        r.template cut<true>(goal > 1 ? (uint64_t)goal : 1);
    }
    if (r.ties != 0xffffffffu) {
        const uint32_t key = r.key;
        const uint64_t before = r.ties - 1;
        r.last = r.locate([&](float x, int) INLINE { return (uint64_t)(key_of(x) == key); }, [&](uint64_t) INLINE { return before; });
        __syncthreads();
    }
    const double u = (double)a.uniform[blockIdx.x];
    const int index = r.locate(
        [&](float x, int i) INLINE -> uint64_t {
            if (!r.kept(x, i))
                return 0;
            const uint64_t w = r.weight(x);
            return w >= r.least ? w : 0;
        },
        [&](uint64_t all) INLINE {
            const double at = u > 0 ? u * (double)all : 0;
            return at < (double)all ? (uint64_t)at : all - 1;
        });
    if (tid == 0)
        a.tokens[blockIdx.x] = index;
}

} // namespace hipq

using namespace hipq;

extern "C" int hipq_sample(const void *logits, int type, int rows, int vocab, int64_t stride, const float *uniform, const float *temperature,
                           const int32_t *top_k, const float *top_p, const float *min_p, int64_t *tokens, void *stream)
{
    clear_error();
    HIPQ_REQUIRE(type == HIPQ_REAL_F32 || is_real16(type), "sample: type %d", type);
    HIPQ_REQUIRE(rows >= 0 && rows <= (1 << 24), "sample: %d rows", rows);
    HIPQ_REQUIRE(vocab >= 1 && vocab <= MOST_VOCAB, "sample: %d scores (1 to %d are possible)", vocab, MOST_VOCAB);
    if (rows == 0)
        return 0;
    HIPQ_REQUIRE(logits && uniform && tokens, "sample: a null pointer");
    HIPQ_REQUIRE((uintptr_t)logits % (type == HIPQ_REAL_F32 ? 4 : 2) == 0, "sample: scores are not aligned to their type");
    HIPQ_REQUIRE(rows == 1 || stride >= vocab, "sample: rows overlap (stride %lld)", (long long)stride);
    SampleArgs a = {};
    a.logits = logits, a.stride = stride, a.uniform = uniform, a.temperature = temperature, a.top_p = top_p, a.min_p = min_p, a.top_k = top_k;
    a.tokens = tokens, a.vocab = vocab;
    const dim3 grid(rows), block(THREADS);
    if (type == HIPQ_REAL_F32)
        sample_kernel<HIPQ_REAL_F32><<<grid, block, 0, (hipStream_t)stream>>>(a);
    else if (type == HIPQ_REAL_F16)
        sample_kernel<HIPQ_REAL_F16><<<grid, block, 0, (hipStream_t)stream>>>(a);
    else
        sample_kernel<HIPQ_REAL_BF16><<<grid, block, 0, (hipStream_t)stream>>>(a);
    return launch_status("sample_kernel");
}
