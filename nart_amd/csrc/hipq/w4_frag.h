// 4-bit weights in the kernels that multiply with them: the arithmetic, the layout, the scales.  gfx950 only.
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
#pragma once

#include <type_traits>

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

// What lays N rows (with an activation 2 N, the gate's first) out in the kernels' order.
struct PackArgs { // `shift` is w4_pack's
    const uint8_t *q, *zeros;
    const uint16_t *scales, *bias;
    uint8_t *to_q;
    uint16_t *to_scales, *to_bias;
    u32x4 *to_nothing;
    int rows, K, group, groups, blocks, tiles, gated; // rows: of one projection
    int shift;
    // several arrays of the same shape in one launch (0: one), and how far apart they lie: q and zeros in bytes, scales in numbers, where they go in bytes
    int arrays;
    size_t q_step, s_step, to_q_step, to_s_step;
};
int w4_pack(PackArgs p, int type, hipStream_t st); // a launch; `tiles` of 16 rows of each array are written, those behind the last row as zeros

static int round_up(int v, int to) { return (v + to - 1) / to * to; }

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

} // namespace hipq
