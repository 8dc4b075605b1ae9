// A token of every row of scores (hipq_sample): temperature, top-k, top-p and min-p from given uniform numbers.  gfx950 only.
//
// Ordered by score (equal ones by index), each filter keeps a prefix, so what is kept is one border: a score, and how many of the scores
// equal to it; the row is never sorted.  A filter keeps what has less than `need` in front of it - tokens for top-k, weight for top-p: the
// scores are divided into 2048 intervals below the maximum, and the interval is found in which the running sum reaches `need`.  Mostly few
// scores are in it (for top-k, with all above): they are put in order in LDS, and decide everything (top-k), or the border (top-p).
// Where they are many they are divided again by the bits of the scores, until an interval is a single score.
// Weights are 64-bit fixed point, 2^-43 of the largest: sums do not depend on their order, so that neither atomics nor the number of
// threads show in a result, and they come from a polynomial in 64 bits (2^-37 of their value off at most): a running sum in 32 bits goes wrong
// where two tokens' borders lie closer than its rounding, at 10^5 tokens once in some hundred rows.
//
// One work-group has a row, and reads it two to four times: the first from memory, the others from the caches.  What bounds it is vector
// instructions (15 to 30 a score and pass) and, for one row, the fetch of code that runs once.  Measured, us: 1 x 32000 bf16, temperature alone
// 14, top-k 100 with top-p 0.9 13.5, top-p alone 27; 24 x 50257 fp16 22, 19, 40; 256 x 128000 fp32 58, 45, 97 (a pass that does nothing but look
// for the maximum takes 18).  All of a row's work in a work-group of its own and no part of a row in another: two parts a row would need the
// sums of both twice in a pass each.
#include "real16.h"

// a lambda that is called instead of inlined takes the row's state to memory
#define INLINE __attribute__((always_inline))

namespace hipq {

constexpr int THREADS = 1024, WAVES = THREADS / 64, BINS = 2048, LIST = 4096, FEW = THREADS, FRACTION = 43;
constexpr int MOST_VOCAB = 1 << 20; // sums of weights fit 64 bits
constexpr int MOST_ROWS = 1 << 21;  // of a launch

// 2^(i / 32) and 2^(i / 1024)
__constant__ const double POWERS[2][32] = {
    {1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
     1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332, 1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
     1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
     1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002},
    {1.0, 1.0006771306930664, 1.0013547198921082, 1.002032767907594, 1.0027112750502025, 1.0033902416308227, 1.004069667960554, 1.0047495543507072,
     1.0054299011128027, 1.006110708558573, 1.0067919769999607, 1.0074737067491204, 1.0081558981184175, 1.0088385514204294, 1.0095216669679448, 1.0102052450739643,
     1.0108892860517005, 1.011573790214578, 1.0122587578762337, 1.0129441893505169, 1.0136300849514894, 1.0143164449934257, 1.0150032697908125, 1.0156905596583505,
     1.016378314910953, 1.0170665358637463, 1.0177552228320703, 1.0184443761314785, 1.019133996077738, 1.0198240829868295, 1.0205146371749483, 1.0212056589585028},
};

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
    union {
        uint32_t list[LIST];
        uint64_t few[FEW];
    };
    double powers[1024]; // 2^(43 + i / 1024)
    uint64_t wave[WAVES], region[WAVES];
    uint64_t before;
    uint32_t bin, listed, low, high;
    float top;
    int index; // of a border
    int found; // locate's alone: a border's index may still be read when locate begins
};

template <int TYPE>
struct Scores {
    static constexpr int SIZE = TYPE == HIPQ_REAL_F32 ? 4 : 2, WORD = 4 / SIZE, LOAD = 4 * WORD; // scores of a word and of a 16-byte load
    static constexpr uint32_t NONE = TYPE == HIPQ_REAL_F32 ? 0xff800000u : TYPE == HIPQ_REAL_F16 ? 0xfc00fc00u : 0xff80ff80u; // -infinity
    template <int N>
    struct __attribute__((packed, aligned(SIZE))) Words {
        uint32_t v __attribute__((ext_vector_type(N)));
    };
    // N words from score i on, those behind the end as -infinity
    template <int N>
    __device__ static __forceinline__ void load(const void *row, int i, int end, uint32_t (&v)[N])
    {
        if (i + N * WORD <= end) {
            const auto w = ((const Words<N> *)((const uint8_t *)row + (int64_t)i * SIZE))->v;
#pragma unroll
            for (int n = 0; n < N; n++)
                v[n] = w[n];
        } else {
#pragma unroll
            for (int n = 0; n < N; n++)
                v[n] = NONE;
            if (i < end) { // all at once: one after the other, eight loads took 3 us
                uint32_t y[N * WORD];
#pragma unroll
                for (int e = 0; e < N * WORD; e++) {
                    const int at = min(i + e, end - 1);
                    y[e] = SIZE == 4 ? ((const uint32_t *)row)[at] : ((const uint16_t *)row)[at];
                }
#pragma unroll
                for (int e = 0; e < N * WORD; e++) {
                    const uint32_t one = i + e < end ? y[e] : SIZE == 4 ? NONE : NONE & 0xffffu;
                    v[e / WORD] = SIZE == 4 ? one : e % WORD ? v[e / WORD] | one << 16 : one;
                }
            }
        }
    }
    __device__ static __forceinline__ void four(const uint32_t *v, float (&x)[4])
    {
        using R = Real16<TYPE == HIPQ_REAL_F32 ? HIPQ_REAL_F16 : TYPE>;
#pragma unroll
        for (int e = 0; e < 4; e++)
            x[e] = SIZE == 4 ? __builtin_bit_cast(float, v[e]) : e & 1 ? R::high(v[e / 2]) : R::low(v[e / 2]);
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

__device__ static __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ static __forceinline__ uint64_t uniform(uint64_t v) { return (uint64_t)uniform((uint32_t)(v >> 32)) << 32 | uniform((uint32_t)v); }
__device__ static __forceinline__ float uniform(float v) { return __builtin_bit_cast(float, uniform(__builtin_bit_cast(uint32_t, v))); }
__device__ static __forceinline__ double uniform(double v) { return __builtin_bit_cast(double, uniform(__builtin_bit_cast(uint64_t, v))); }
__device__ static __forceinline__ uint64_t of_lane(uint64_t v, int lane)
{
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
// v plus that of the lane which HOW names, in the rows of 16 lanes that ROWS has a bit for; 0 where there is none
template <int HOW, int ROWS = 15>
__device__ static __forceinline__ uint64_t plus(uint64_t v)
{
    return v + ((uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), HOW, ROWS, 15, false) << 32 |
                (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, HOW, ROWS, 15, false));
}
// sums up to each lane: of its 16 lanes, and of all 64
__device__ static __forceinline__ uint64_t sums16(uint64_t v)
{
    return plus<0x118>(plus<0x114>(plus<0x112>(plus<0x111>(v)))); // lanes 1, 2, 4, 8 in front
}
__device__ static __forceinline__ uint64_t sums64(uint64_t v)
{
    return plus<0x143, 12>(plus<0x142, 10>(sums16(v))); // the last lane of the row in front, that of the first two rows
}

template <int TYPE>
struct Row {
    using S = Scores<TYPE>;
    static constexpr int E = 4; // scores that a pass works on at a time
    const SampleArgs &a;
    SampleShared &s;
    const void *row;
    int tid, lane, wave;
    float top, per_bin; // intervals of a unit of score
    bool infinite = false;
    double rate, lowest; // log2(e) / temperature; the difference to the top from which on nothing has a weight
    // the border: scores above that of key are kept, and of those equal to it the first `ties` (up to index `last`)
    uint32_t key = 0x007fffffu /* -infinity's */, ties = 0xffffffffu;
    int last = 0x7fffffff;
    uint64_t least = 0; // smallest weight that min-p keeps
    uint64_t sum = 0;   // of the last scan

    __device__ Row(const SampleArgs &a_, SampleShared &s_) : a(a_), s(s_)
    {
        tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        row = (const uint8_t *)a.logits + (int64_t)blockIdx.x * a.stride * (TYPE == HIPQ_REAL_F32 ? 4 : 2);
    }

    // where there are infinities they are all that counts, one like the other
    __device__ __forceinline__ void settle(float (&x)[E]) const
    {
        if (infinite)
#pragma unroll
            for (int e = 0; e < E; e++)
                x[e] = x[e] == __builtin_inff() ? 0.0f : -__builtin_inff();
    }

    // f(four scores, index of the first) of the row's part [from, to), 16 bytes at a time, `lanes` threads side by side, the next 16 bytes
    // on their way.  The loops are short on purpose: what runs once is bound by the fetch of its instructions
    template <class F>
    __device__ __forceinline__ void each(int from, int to, int id, int lanes, F f)
    {
        asm volatile("" : "+v"(id)); // or every pass's addresses are made at the beginning, and kept
        uint32_t v[4], ahead[4];
        S::load(row, from + id * S::LOAD, to, v);
#pragma unroll 1
        for (int base = from; base < to; base += lanes * S::LOAD) {
            const int i = base + id * S::LOAD;
            S::load(row, i + lanes * S::LOAD, to, ahead);
#pragma unroll 1
            for (int part = 0; part < S::LOAD; part += E) {
                float x[E];
                S::four(v, x);
                settle(x);
                f(x, i + part);
                v[0] = v[2], v[1] = v[3]; // of 16-bit scores the second four
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                v[e] = ahead[e];
        }
    }
    template <class F>
    __device__ __forceinline__ void each(F f) { each(0, a.vocab, tid, THREADS, f); }

    // 2^(rate (x - top)) in units of 2^-43: 2^(n / 1024) from the table times 2^r, |r| <= 1 / 2048, to the second power (the third is under
    // 2^-37 of the whole).  No branch, and no instruction to spare: a pass takes 64 / 16 of a wave's clocks for each.  The power of two
    // goes into the table's number by its exponent, and the sum that rounds is the last product's.  The result is RAW more.
    static constexpr uint64_t RAW = 0x4330000000000000ull; // 2^52: a sum's lower bits are the rounded number
    __device__ __forceinline__ uint64_t raw_weight(float x) const
    {
        const double d = fmax((double)x - (double)top, lowest); // NaN and all below the lowest weigh 2^-17 units, which rounds to 0
        const double big = 6755399441055744.0 / 1024;            // 1.5 * 2^52 / 1024: what is added keeps ten bits behind the point
        const double t = __builtin_fma(d, rate, big), r = __builtin_fma(d, rate, big - t);
        const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, t);
        const double p = __builtin_fma(__builtin_fma(r, 0.24022650695910071, 0.69314718055994531), r, 1.0);
        const uint64_t power = __builtin_bit_cast(uint64_t, s.powers[n & 1023]) + ((uint64_t)((n & ~1023u) << 10) << 32);
        return __builtin_bit_cast(uint64_t, __builtin_fma(p, __builtin_bit_cast(double, power), 4503599627370496.0));
    }
    __device__ __forceinline__ uint64_t weight(float x) const { return raw_weight(x) - RAW; }
    __device__ __forceinline__ int bin_of(float x) const
    {
        const float v = (top - x) * per_bin;
        return v < BINS - 1 ? (int)v : BINS - 1;
    }
    __device__ __forceinline__ void clear_bins()
    {
        for (int i = tid; i < BINS; i += THREADS)
            s.bins[i] = 0;
    }

    // sum over the threads in front, and `sum` over all; every thread calls it
    __device__ __forceinline__ uint64_t scan(uint64_t v)
    {
        const uint64_t in = sums64(v);
        __syncthreads(); // s.wave may still be read
        if (lane == 63)
            s.wave[wave] = in;
        __syncthreads();
        const uint64_t waves = sums16(s.wave[lane & 15]);
        sum = of_lane(waves, 15);
        return (uniform((uint32_t)wave) ? of_lane(waves, (int)uniform((uint32_t)wave) - 1) : 0) + in - v;
    }

    // the first bin in which the running sum reaches need: s.bin, and s.before what lies in front of it.  false: the sum stays below
    __device__ __forceinline__ bool find(uint64_t need)
    {
        const uint64_t b0 = s.bins[2 * tid], b1 = s.bins[2 * tid + 1];
        const uint64_t front = scan(b0 + b1);
        const bool reached = sum >= need;
        if (front < need && need <= front + b0)
            s.bin = 2 * tid, s.before = front;
        else if (front + b0 < need && need <= front + b0 + b1)
            s.bin = 2 * tid + 1, s.before = front + b0;
        __syncthreads();
        return reached;
    }

    // moves the border to where `need` is reached; the bins hold the first division.  mass: of weight, otherwise of tokens.  The tokens
    // counted are those above the present border, and `ties` at it.
    __device__ __forceinline__ void cut(bool mass, uint64_t need)
    {
        if (!find(need))
            return;
        const int bin = (int)uniform(s.bin);
        need -= uniform(s.before);
        if (tid == 0)
            s.listed = 0, s.low = 0xffffffffu, s.high = 0;
        __syncthreads();
        const uint32_t old = key, old_ties = ties;
        // the border's own ties count as many as are kept
        const bool tied = old_ties != 0xffffffffu && bin_of(score_of(old)) == bin;
        uint32_t low = tied ? old : 0xffffffffu, high = tied ? old : 0, listed = 0;
#pragma unroll 1
        for (int level = 0; level < 5; level++) { // 0: what lies in the bin is listed; then 11 bits of the interval [low, high] at a time: at most three times
            const int bits = high == low ? 0 : 32 - __clz((int)(high - low)), shift = bits > 11 ? bits - 11 : 0;
            auto add = [&](uint32_t k, uint64_t times) INLINE {
                if (k >= low && k <= high)
                    atomicAdd((unsigned long long *)&s.bins[(high - k) >> shift], (unsigned long long)(mass ? weight(score_of(k)) * times : times));
            };
            if (level > 0) {
                clear_bins();
                __syncthreads();
            }
            if (level == 0 || listed > LIST)
                each([&](const float(&x)[E], int) INLINE {
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const uint32_t k = key_of(x[e]);
                        if (bin_of(x[e]) == bin && x[e] > -__builtin_inff() && (k > old || (k == old && old_ties == 0xffffffffu))) {
                            if (level == 0) {
                                low = min(low, k), high = max(high, k);
                                const uint32_t at = atomicAdd(&s.listed, 1u);
                                if (at < LIST)
                                    s.list[at] = k;
                            } else
                                add(k, 1);
                        }
                    }
                });
            else
                for (uint32_t i = tid; i < listed; i += THREADS)
                    add(s.list[i], 1);
            if (level == 0) {
#pragma unroll
                for (int o = 1; o < 64; o *= 2)
                    low = min(low, (uint32_t)__shfl_xor((int)low, o)), high = max(high, (uint32_t)__shfl_xor((int)high, o));
                if (lane == 0)
                    atomicMin(&s.low, low), atomicMax(&s.high, high);
                __syncthreads();
                low = uniform(s.low), high = uniform(s.high), listed = uniform(s.listed);
                continue;
            }
            if (tied && tid == 0)
                add(old, old_ties);
            __syncthreads();
            find(need);
            need -= uniform(s.before);
            const uint32_t at = uniform(s.bin), to = high - (at << shift);
            if (shift == 0) {
                const uint64_t each_one = mass ? uniform(weight(score_of(to))) : 1, there = uniform(s.bins[at]) / each_one, wanted = (need + each_one - 1) / each_one;
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

    // The row in WAVES parts, one for each wave: where that of wave w begins and ends
    __device__ __forceinline__ int part() const { return (a.vocab + WAVES * S::LOAD - 1) / (WAVES * S::LOAD) * S::LOAD; }
    __device__ __forceinline__ int from() const { return min(a.vocab, wave * part()); }
    __device__ __forceinline__ int to() const { return min(a.vocab, from() + part()); }
    // the parts' sums: v is a thread's
    __device__ __forceinline__ void set_regions(uint64_t v)
    {
        v = sums64(v);
        if (lane == 63)
            s.region[wave] = v;
        __syncthreads();
    }

    // The threads' numbers, the first n of them and all different, from the largest to the smallest (those behind are 0).  Few are each
    // compared with all, by 4 to 16 threads; more by exchanges over distances that halve, in the wave's registers where both ends are in
    // it.  (100 numbers: 1.5 us and 4; a step of the latter takes 140 ns.)
    __device__ __forceinline__ uint64_t sort(uint64_t v, int n)
    {
        if (n <= 256) {
            const int shift = n <= 64 ? 4 : n <= 128 ? 3 : 2, own = tid >> shift, part = tid & ((1 << shift) - 1);
            __syncthreads();
            s.few[tid] = v;
            __syncthreads();
            v = s.few[own];
            int rank = 0;
#pragma unroll 4
            for (int i = part; i < n; i += 1 << shift)
                rank += s.few[i] > v;
            for (int o = 1; o < 1 << shift; o *= 2)
                rank += __shfl_xor(rank, o);
            __syncthreads();
            if (own < n && part == 0)
                s.few[rank] = v;
            __syncthreads();
            return tid < n ? s.few[tid] : 0;
        }
        const bool some = wave * 64 < 2 * n; // waves that can hold some on their way
#pragma unroll 1
        for (int size = 2; size < 2 * n; size *= 2)
#pragma unroll 1
            for (int apart = size / 2; apart > 0; apart /= 2) {
                if (apart >= 64) {
                    __syncthreads();
                    s.few[tid] = v;
                    __syncthreads();
                }
                if (some) {
                    const uint64_t other = apart < 64 ? __shfl_xor(v, apart) : s.few[tid ^ apart];
                    v = (v > other) == (((tid & size) == 0) == ((tid & apart) == 0)) ? v : other;
                }
            }
        return v;
    }

    // The first index, in order, at which the running sum exceeds `target(sum)`; f: the sum of some scores' numbers, and each, if asked for.
    // known: the regions hold their sums.
    template <class F, class T>
    __device__ __forceinline__ int locate(bool known, F f, T target)
    {
        if (!known) {
            uint64_t v = 0;
            each(from(), to(), lane, 64, [&](const float(&x)[E], int i) INLINE { v += f(x, i, nullptr); });
            set_regions(v);
        }
        const int part = this->part();
        const uint64_t regions = sums16(s.region[lane & 15]), goal = target(of_lane(regions, 15));
        const int w = min(WAVES - 1, (int)__popcll(__ballot(lane < WAVES && regions <= goal)));
        uint64_t front = w ? of_lane(regions, w - 1) : 0;
        const int begin = w * part, end = min(a.vocab, begin + part);
        if (tid == 0)
            s.found = -1;
#pragma unroll 1
        for (int base = begin; base < end; base += THREADS * E) {
            float x[E];
            const int i = base + tid * E;
            uint32_t v[E / S::WORD];
            S::load(row, i, end, v);
            S::four(v, x);
            settle(x);
            uint64_t own, each_one[E];
            own = f(x, i, each_one);
            uint64_t run = front + scan(own);
            if (run <= goal && goal < run + own) {
                int at = i;
#pragma unroll
                for (int e = 0; e < E - 1; e++) {
                    run += each_one[e];
                    at += run <= goal;
                }
                s.found = at;
            }
            __syncthreads();
            front += sum;
            if ((int)uniform((uint32_t)s.found) >= 0)
                break;
        }
        return (int)uniform((uint32_t)s.found);
    }
};

template <int TYPE>
__global__ __launch_bounds__(THREADS) void sample_kernel(const SampleArgs a)
{
    __shared__ SampleShared s;
    Row<TYPE> r(a, s);
    constexpr int E = Row<TYPE>::E;
    const int tid = threadIdx.x;
    const float none = -__builtin_inff();

    s.powers[tid] = POWERS[0][tid >> 5] * POWERS[1][tid & 31] * (double)((uint64_t)1 << FRACTION);
    float top = none;
    r.each([&](const float(&x)[E], int) INLINE {
#pragma unroll
        for (int e = 0; e < E; e++)
            top = fmaxf(top, x[e]);
    });
    float own = top; // the largest of this thread's scores
#pragma unroll
    for (int o = 1; o < 64; o *= 2)
        top = fmaxf(top, __shfl_xor(top, o));
    if (r.lane == 0)
        s.list[r.wave] = __builtin_bit_cast(uint32_t, top);
    __syncthreads();
    top = __builtin_bit_cast(float, s.list[r.lane & (WAVES - 1)]);
#pragma unroll
    for (int o = 1; o < WAVES; o *= 2)
        top = fmaxf(top, __shfl_xor(top, o));
    top = uniform(top);
    __syncthreads();
    r.infinite = top == __builtin_inff();
    r.top = r.infinite ? 0.0f : top;
    own = !r.infinite ? own : own == top ? 0.0f : none;
    const float t = a.temperature ? a.temperature[blockIdx.x] : 1.0f;
    if (top == none) {
        if (tid == 0)
            a.tokens[blockIdx.x] = -1;
        return;
    }
    top = r.top;
    if (!(t > 0)) {
        if (tid == 0)
            s.index = 0x7fffffff;
        __syncthreads();
        int first = 0x7fffffff;
        r.each([&](const float(&x)[E], int i) INLINE {
#pragma unroll
            for (int e = 0; e < E; e++)
                first = x[e] == top ? min(first, i + e) : first;
        });
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
    r.rate = uniform(1.4426950408889634 / (double)t);
    r.lowest = fmax(-60.0 / r.rate, -1e300);
    // 2047 intervals down to where weights are 0, the last one for all below
    r.per_bin = (float)((BINS - 1) * r.rate / 44.5);
    r.per_bin = uniform(r.per_bin < 1e30f ? r.per_bin : 1e30f);
    if (a.min_p) {
        const double p = (double)a.min_p[blockIdx.x] * (double)((uint64_t)1 << FRACTION);
        r.least = uniform(p > 0 ? p < (double)((uint64_t)1 << FRACTION) ? (uint64_t)ceil(p) : (uint64_t)1 << FRACTION : (uint64_t)0);
    }
    const int k = a.top_k ? (int)uniform((uint32_t)a.top_k[blockIdx.x]) : 0;
    const float p = a.top_p ? uniform(a.top_p[blockIdx.x]) : 1.0f;
    const bool by_count = k > 0 && k < a.vocab, by_mass = p < 1;
    bool known = false;
    const double u = uniform((double)a.uniform[blockIdx.x]);
    auto goal_of = [&](uint64_t all) INLINE -> uint64_t {
        const double at = u > 0 ? u * (double)all : 0;
        return at < (double)all ? (uint64_t)at : all - 1;
    };
    auto need_of = [&](uint64_t all) INLINE -> uint64_t {
        const double goal = p > 0 ? ceil((double)p * (double)all) : 1;
        return goal > 1 ? (uint64_t)goal : 1;
    };
    constexpr uint64_t RAW = Row<TYPE>::RAW;
#pragma unroll 1
    for (int step = 0; step < 3; step++) { // top-k, then top-p among what it keeps
        // The first k are not below the k-th largest of the threads' largest scores, and hardly more scores are above that: where k
        // is small it is looked for among those alone (0), and in all scores (1) only if that was no use.
        const bool mass = step == 2;
        if (!(mass ? by_mass : by_count && (step == 1 || k <= FEW / 2)))
            continue;
        r.clear_bins();
        __syncthreads();
        const uint32_t key = r.key, ties = r.ties;
        const float border = score_of(key);
        const bool all_ties = ties == 0xffffffffu && border > none;
        if (step == 0) {
            if (own > none)
                atomicAdd((unsigned long long *)&s.bins[r.bin_of(own)], 1ull);
        } else
            r.each([&](const float(&x)[E], int) INLINE {
                bool in[E], any = false;
#pragma unroll
                for (int e = 0; e < E; e++)
                    any |= in[e] = (x[e] > border) | ((x[e] == border) & all_ties); // no branches: a loop of them took twice the instructions
                if (any) {
                    uint64_t w[E];
                    if (mass)
#pragma unroll
                        for (int e = 0; e < E; e++)
                            w[e] = r.weight(x[e]);
#pragma unroll
                    for (int e = 0; e < E; e++)
                        if (in[e])
                            atomicAdd((unsigned long long *)&s.bins[r.bin_of(x[e])], mass ? (unsigned long long)w[e] : 1ull);
                }
            });
        if (tid == 0 && ties != 0xffffffffu)
            atomicAdd((unsigned long long *)&s.bins[r.bin_of(score_of(key))], (unsigned long long)(mass ? r.weight(score_of(key)) * ties : ties));
        __syncthreads();
        uint64_t need = (uint64_t)k; // a border among scores without weight changes nothing
        if (mass) {
            r.scan(s.bins[2 * tid] + s.bins[2 * tid + 1]);
            need = need_of(r.sum);
        }
        // The quick way, where the scores around the border are few: top-k's are all that can be taken, with it everything is decided among
        // them; top-p's border is decided among those of its interval, while the weight of all above is summed in the same pass.
        if (mass ? key == 0x007fffffu : k <= FEW / 2) {
            const bool found = r.find(need);
            const int bin = (int)uniform(s.bin);
            const uint64_t before = uniform(s.before);
            if (!found || bin == BINS - 1)
                continue; // nothing with a weight is cut
            if (tid == 0)
                s.listed = 0, s.low = 0xffffffffu, s.index = -1;
            __syncthreads();
            uint64_t above = 0;
            const float first = mass ? (float)bin : 0.0f, behind = (float)(bin + 1); // the intervals that are listed
            r.each(r.from(), r.to(), r.lane, 64, [&](const float(&x)[E], int i) INLINE {
                // in place of intervals, what their numbers are the whole part of
                float v[E];
                bool here = false, over = false;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    v[e] = (r.top - x[e]) * r.per_bin; // infinite or NaN where a score is never taken
                    here |= (v[e] >= first) & (v[e] < behind);
                    over |= v[e] < first;
                }
                if (here)
#pragma unroll
                    for (int e = 0; e < E; e++)
                        if ((v[e] >= first) & (v[e] < behind)) {
                            const uint32_t at = atomicAdd(&s.listed, 1u);
                            if (at < FEW)
                                s.few[at] = (uint64_t)key_of(x[e]) << 32 | ~(uint32_t)(i + e); // a larger one comes first
                        }
                if (mass && over)
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const uint64_t w = r.weight(x[e]);
                        above += ((v[e] < first) & (w >= r.least)) ? w : 0;
                    }
            });
            r.set_regions(above);
            const int n = (int)uniform(s.listed);
            if (n <= FEW) {
                const uint64_t entry = r.sort(tid < n ? s.few[tid] : 0, n);
                const int index = (int)~(uint32_t)entry;
                uint64_t w = tid < (mass ? n : min(n, k)) ? r.weight(score_of((uint32_t)(entry >> 32))) : 0;
                const uint64_t front = r.scan(w);
                if (mass) {
                    if (tid < n && before + front < need) {
                        if (w >= r.least)
                            atomicAdd((unsigned long long *)&s.region[(uint32_t)index / (uint32_t)r.part()], (unsigned long long)w);
                        if (before + front + w >= need)
                            s.low = (uint32_t)(entry >> 32), s.index = index;
                    }
                    __syncthreads();
                    r.key = uniform(s.low), r.last = (int)uniform((uint32_t)s.index);
                    known = true;
                    continue;
                }
                const uint64_t most = by_mass ? need_of(r.sum) : ~0ull;
                w = front < most && w >= r.least ? w : 0;
                // in the order of their indices
                const uint64_t at = r.sort(tid < min(n, k) ? (uint64_t)(MOST_VOCAB - 1 - index) << (FRACTION + 1) | w : 0, min(n, k));
                w = at & ((2ull << FRACTION) - 1);
                const uint64_t run = r.scan(w);
                const uint64_t goal = goal_of(r.sum);
                if (run <= goal && goal < run + w)
                    a.tokens[blockIdx.x] = MOST_VOCAB - 1 - (int)(at >> (FRACTION + 1));
                return;
            }
        }
        if (step > 0)
            r.cut(mass, need);
    }
    if (r.key == 0x007fffffu)
        r.last = -1; // a score of -infinity is never taken
    const uint64_t least = RAW + r.least;
    const float border = score_of(r.key);
#pragma unroll 1
    for (int last = r.ties == 0xffffffffu; last < 2; last++) { // the last of the ties that are kept, then the token
        const int index = r.locate(
            known,
            [&](const float(&x)[E], int i, uint64_t *each_one) INLINE -> uint64_t {
                const int upto = last == 0 ? 0x7fffffff : r.last;
                uint64_t sum = 0, raw[E];
#pragma unroll
                for (int e = 0; e < E; e++) // side by side, and for a count as well: behind a branch each waits for its own number of the table
                    raw[e] = r.raw_weight(x[e]);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const bool in = ((x[e] > border) & (last != 0)) | ((x[e] == border) & (i + e <= upto));
                    uint64_t w = last == 0 ? RAW + 1 : raw[e];
                    w = (in & (w >= (last == 0 ? RAW : least))) ? w - RAW : 0;
                    sum += w;
                    if (each_one)
                        each_one[e] = w;
                }
                return sum;
            },
            [&](uint64_t all) INLINE -> uint64_t { return last == 0 ? r.ties - 1 : goal_of(all); });
        if (last == 0)
            r.last = index;
        else if (tid == 0)
            a.tokens[blockIdx.x] = index;
        __syncthreads();
    }
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
    // of 2^32 work-items and more only what is left over would run
    for (int done = 0; done < rows; done += MOST_ROWS) {
        const dim3 grid(rows - done < MOST_ROWS ? rows - done : MOST_ROWS), block(THREADS);
        if (type == HIPQ_REAL_F32)
            sample_kernel<HIPQ_REAL_F32><<<grid, block, 0, (hipStream_t)stream>>>(a);
        else if (type == HIPQ_REAL_F16)
            sample_kernel<HIPQ_REAL_F16><<<grid, block, 0, (hipStream_t)stream>>>(a);
        else
            sample_kernel<HIPQ_REAL_BF16><<<grid, block, 0, (hipStream_t)stream>>>(a);
        if (launch_status("sample_kernel"))
            return 1;
        a.logits = (const uint8_t *)a.logits + MOST_ROWS * stride * (type == HIPQ_REAL_F32 ? 4 : 2);
        a.uniform += MOST_ROWS, a.tokens += MOST_ROWS;
        a.temperature += a.temperature ? MOST_ROWS : 0, a.top_k += a.top_k ? MOST_ROWS : 0;
        a.top_p += a.top_p ? MOST_ROWS : 0, a.min_p += a.min_p ? MOST_ROWS : 0;
    }
    return 0;
}
