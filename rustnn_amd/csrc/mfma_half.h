// fp32 products on the fp16 matrix cores, for operands that the loading threads
// split themselves (differential attention, Linear with an activation).
//
// A float times a power of two is hi + lo, hi its nearest fp16 and lo the
// nearest fp16 of the rest: hi + lo is within half a step of 2^-22, so 2^-23, of
// it, as long as lo is no subnormal, which ends 2^-25 at 2^15.  With the power
// chosen so that the largest magnitude of a row or tile comes to
// [2^14, 2^15), every element down to 2^-16 of the largest keeps 2^-23, and
// below that all keep 2^-39 of the largest (2^-12 and 2^-35 for operands whose
// power of two has to last for a whole sum, sticky_up).  a b is then hi hi + hi lo + lo hi:
// products of 22 bits, exact in the matrix core, summed in its fp32
// accumulator; lo lo, left out, is below 2^-22 of the product and of no common
// sign.  Three products an element and four bytes in LDS, where three bf16
// parts (mfma_split.h) take six and six; their range of exponents is not needed
// here, since rows and tiles carry their power of two beside them.
#pragma once

#include "rnn_internal.h"

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __fp16 g4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f2u __attribute__((ext_vector_type(2), aligned(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

struct Half2 {
    h8 hi, lo;
};

// x - (the lower / upper half of h): the rest of a rounding, exact.
__device__ __forceinline__ float rest_lo(uint32_t h, float x) {
    float d;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "v"(x));
    return d;
}
__device__ __forceinline__ float rest_hi(uint32_t h, float x) {
    float d;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "v"(x));
    return d;
}
// Two floats' parts, each pair in a register.
__device__ __forceinline__ void half_pair(float a, float b, uint32_t &hi, uint32_t &lo) {
    const f2 v = {a, b};
    hi = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
    const f2 d = {rest_lo(hi, a), rest_hi(hi, b)};
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(d, h2));
}

// The two parts of 8 floats (times up, a power of two).
__device__ __forceinline__ Half2 half_split(const float (&x)[8]) {
    u32x4 hi, lo;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t a, b;
        half_pair(x[2 * j], x[2 * j + 1], a, b);
        hi[j] = a;
        lo[j] = b;
    }
    return Half2{__builtin_bit_cast(h8, hi), __builtin_bit_cast(h8, lo)};
}
__device__ __forceinline__ Half2 half_split(const float (&x)[8], float up) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = x[e] * up;
    return half_split(y);
}
// The parts of an accumulator's registers 0..7 and 8..15, as they are.
__device__ __forceinline__ void split16(const f32x16 &x, Half2 (&d)[2]) {
#pragma unroll
    for (int s = 0; s < 2; s++) {
        u32x4 hi, lo;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t a, b;
            half_pair(x[8 * s + 2 * j], x[8 * s + 2 * j + 1], a, b);
            hi[j] = a;
            lo[j] = b;
        }
        d[s] = Half2{__builtin_bit_cast(h8, hi), __builtin_bit_cast(h8, lo)};
    }
}

// The power of two that takes a largest magnitude m to [2^14, 2^15) (m of 0,
// an infinity or a NaN: 1), and its reciprocal.  Magnitudes below 2^-112 stay
// smaller.
__device__ __forceinline__ float up_of(float m) {
    const int e = (int)(__float_as_uint(m) >> 23) & 255;
    const int f = (e == 255 || m == 0.0f) ? 127 : min(268 - e, 253);
    return __uint_as_float((uint32_t)f << 23);
}
__device__ __forceinline__ float down_of(float up) {
    return __uint_as_float((254u << 23) - __float_as_uint(up));
}

// The power of two of a sum's operand from tile to tile: it stays until a
// magnitude m times it passes 2^15, and then takes m to [2^10, 2^11), so that it
// hardly moves again and the accumulators with it (which a change rescales).
// FIRST_UP: before any tile.
constexpr float FIRST_UP = 0x1p112f;
__device__ __forceinline__ float sticky_up(float m, float up) {
    return m * up < 0x1p15f ? up : up_of(m) * 0x1p-4f;
}

__device__ __forceinline__ f32x16 mm(h8 a, h8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Where row r of a tile is kept: the rows of a block of 16 as the transpose of a
// 4 x 4.  Rows are an odd number of 16-byte slots long, so that 16 of them at one
// slot are on distinct banks, and four consecutive ones, 4 positions apart, on
// distinct quarters of them, of which a transposing read takes 64 bytes a row (in
// order, conflicts were 58% of the LDS's busy cycles of differential attention's
// forward).
__device__ __forceinline__ constexpr int row_pos(int r) {
    return (r & ~15) | (r & 3) << 2 | (r >> 2 & 3);
}

// A tile of ROWS rows of W channels in LDS, both parts: row r's hi at
// row_pos(r) * STRIDE, its lo PART further on.
template <int ROWS, int W>
struct HalfTile {
    static constexpr int STRIDE = W + 8;  // in halves
    static constexpr int PART = ROWS * STRIDE;
    static constexpr int HALVES = 2 * PART;
    // 8 consecutive channels of a row: an operand with its k along channels
    static __device__ __forceinline__ h8 along(const _Float16 *t, int row, int c) {
        return *(const h8 *)(t + row_pos(row) * STRIDE + c);
    }
    // Rows row0 + {0..3, 8..11} (row0 + 4 for the upper half wave) of channel
    // c0 + lane % 32: an operand with its k along rows, in the order in which
    // a 32 x 32 accumulator's registers 8 s .. 8 s + 7 hold the rows of the
    // block of 16 at row0.  Each 16 lanes read 4 rows of 16 channels, which
    // the LDS hands back transposed.
    static __device__ __forceinline__ h8 across(const _Float16 *t, int row0, int c0) {
        const int l = threadIdx.x & 63;
        const _Float16 *p = t + (row0 + (l >> 5) + (l & 12)) * STRIDE + c0 +
                            16 * ((l >> 4) & 1) + 4 * (l & 3);
        typedef __attribute__((address_space(3))) g4 *lds_g4;
        const h4 a = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_g4)p));
        const h4 b = __builtin_bit_cast(
            h4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_g4)(p + 2 * STRIDE)));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// 8 consecutive channels, `off` floats into a buffer resource, zero from `lim`
// channels on and past the resource's end.  The loads need 4-byte alignment alone,
// and each float past the end is zero by itself.  VEC: lim is a multiple of 4.
template <bool VEC>
__device__ __forceinline__ void load8(__amdgpu_buffer_rsrc_t rs, uint32_t off, int lim,
                                      float (&x)[8]) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
        const uint32_t at = 4 * q < lim ? (off + 4 * q) * 4 : DMA_OOB;
        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; e++)
            x[4 * q + e] = VEC || 4 * q + e < lim ? __uint_as_float(v[e]) : 0.f;
    }
}

// A resource over `rows` rows (at most 64) of `stride` floats from p on, the last
// of them `width` floats long.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const float *p, int rows, long long stride,
                                                            int width) {
    return make_rsrc(p, rows > 0 ? ((uint32_t)(rows - 1) * (uint32_t)stride + width) * 4u : 0u);
}

// Maxima in one instruction each (fmaxf takes a second one to quiet NaNs).
__device__ __forceinline__ float max2(float a, float b) {
    float d;
    asm("v_max_f32 %0, %1, %2" : "=v"(d) : "v"(a), "v"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}
__device__ __forceinline__ float max3abs(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}
template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
    return __uint_as_float(__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CTRL, 0xf, 0xf, false));
}
// Both lanes of each pair (l, l xor 32), or (l, l xor 16): f of the two values.
template <typename F>
__device__ __forceinline__ float pair32(float v, F f) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <typename F>
__device__ __forceinline__ float pair16(float v, F f) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add2(float a, float b) { return a + b; }
// f over the 64 lanes, every lane receiving it, in a fixed tree.
template <typename F>
__device__ __forceinline__ float wave_all(float v, F f) {
    v = f(v, dpp_f<0xB1>(v));
    v = f(v, dpp_f<0x4E>(v));
    v = f(v, dpp_f<0x141>(v));
    v = f(v, dpp_f<0x140>(v));
    return pair32(pair16(v, f), f);
}
__device__ __forceinline__ float wave_max(float v) { return wave_all(v, max2); }
__device__ __forceinline__ float wave_sum(float v) { return wave_all(v, add2); }

__device__ __forceinline__ float absmax8(const float (&x)[8], float m) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) m = max3abs(m, x[e], x[e + 1]);
    return m;
}

// The wave's largest magnitude where it passes what its power of two is good for,
// else 0: the reduction is rarely taken.
__device__ __forceinline__ float wave_over(float m, float good) {
    return __any(m > good) ? wave_max(m) : 0.f;
}
// What sticky_up's power is good for.
__device__ __forceinline__ float good_for(float up) { return 0x1p15f * down_of(up); }

// How NT threads stage a tile of ROWS rows of W channels: RPP rows a pass, 8
// channels a thread, so that a thread keeps its channels from pass to pass
// (W = 96: the last quarter of the threads idle).
template <int ROWS, int W, int NT>
struct StagePlan {
    static constexpr int C8 = W / 8;
    static constexpr int fit = NT / C8;
    static constexpr int most = fit >= 128 ? 128 : fit >= 64 ? 64 : fit >= 32 ? 32 : fit >= 16 ? 16 : fit >= 8 ? 8 : 4;
    static constexpr int RPP = most < ROWS ? most : ROWS;
    static constexpr int PASSES = ROWS / RPP;
    static constexpr bool ALL = RPP * C8 == NT;
    static_assert(RPP * C8 <= NT && PASSES * RPP == ROWS, "whole passes");
};

// The block's number in an order in which each XCD (block id % 8) gets a
// contiguous run: the blocks that share a problem's keys meet in one L2.
__device__ __forceinline__ long long xcd_order(long long id, long long total) {
    const long long per = total >> 3, rem = total & 7, x = id & 7, loc = id >> 3;
    return x < rem ? x * (per + 1) + loc : rem * (per + 1) + (x - rem) * per + loc;
}
