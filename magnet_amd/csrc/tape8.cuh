// The 8-bit tape: activations kept for a backward pass as one code of 8 bits per value and one byte per block of 32 columns.
//
// A block's byte b stands for the step 2^(b - 127), the smallest power of two whose largest code reaches the block's largest magnitude
// (top <= 127 steps signed, <= 255 steps behind a ReLU), so dividing by the step and multiplying by it again are exact in fp32: a value
// comes back with the error of ONE rounding to its code, at most half a step.
//   signed: code = rint(x / step) in [-127, 127], two's complement
//   relu:   code = 0 where x <= 0, else rint(x / step) raised to at least 1 - the mask x > 0 survives exactly, at the price of an error of
//           up to a whole step for positive values under half a step
// b = 0: every value of the block is zero; b in [1, 248]: the step (of the last one, 2^121, codes end at 127: 128 steps are no fp32 number); b = 255: the block holds a value that is not finite and reads as NaN
// in all 32 columns (a run that diverges stays visible); its relu codes are 255 / 0 so that the mask survives there too.
// Columns past the width carry zero.  A code has 8 significant bits at most: bf16 and fp16 hold it exactly.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef float t8_f4 __attribute__((ext_vector_type(4)));
typedef unsigned t8_u2 __attribute__((ext_vector_type(2)));
typedef unsigned t8_u4 __attribute__((ext_vector_type(4)));

enum { T8_SIGNED = 0, T8_RELU = 1 };
enum { T8_F32 = 0, T8_BF16 = 1, T8_F16 = 2 };
#define T8_WIDEST (INT32_MAX - 255)      // columns are counted in 32 bits, up to the end of their block (of 128 in the Linear)

// four neighbouring values of any alignment (the hardware takes 16-byte accesses at 4-byte, 8-byte ones at 2-byte addresses)
template <typename T>
using t8_v4 = T __attribute__((ext_vector_type(4), aligned(sizeof(T))));
// ... as fp32; of fewer than four (a row's end) the ones that are there, the rest zero
template <typename T>
__device__ __forceinline__ t8_f4 t8_load4(const T* __restrict__ p, int n) {
    t8_f4 v = {0.f, 0.f, 0.f, 0.f};
    if (n >= 4) {
        const t8_v4<T> t = *reinterpret_cast<const t8_v4<T>*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)t[i];
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < n) v[i] = (float)p[i];
    }
    return v;
}
// ... and back, each value rounded to T once (to nearest, ties to even)
template <typename T>
__device__ __forceinline__ void t8_store4(T* __restrict__ p, int n, const t8_f4& v) {
    if (n >= 4) {
        t8_v4<T> t;
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = (T)v[i];
        *reinterpret_cast<t8_v4<T>*>(p) = t;
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

// what a value adds to its block's top: the bits of its magnitude (of what a ReLU leaves of it), ordered like the magnitudes; NaN on top
template <int KIND>
__device__ __forceinline__ unsigned t8_top(float x) {
    const unsigned b = __float_as_uint(x), m = b & 0x7FFFFFFFu;
    if (KIND == T8_SIGNED) return m;
    return (m > 0x7F800000u || (int)b > 0) ? m : 0u;
}
template <int KIND>
__device__ __forceinline__ unsigned t8_top4(const t8_f4& v) {
    return max(max(t8_top<KIND>(v[0]), t8_top<KIND>(v[1])), max(t8_top<KIND>(v[2]), t8_top<KIND>(v[3])));
}
// a block's byte from its top: 255 steps = 2^8 * 255/256 (mantissa 0x7F0000), 127 steps = 2^7 * 127/128 (mantissa 0x7E0000)
template <int KIND>
__device__ __forceinline__ unsigned t8_byte(unsigned top) {
    const int e = (int)(top >> 23);
    const unsigned f = top & 0x7FFFFFu;
    int b = KIND == T8_RELU ? e - 7 + (f > 0x7F0000u ? 1 : 0) : e - 6 + (f > 0x7E0000u ? 1 : 0);
    b = min(max(b, 1), 248);
    return top == 0u ? 0u : top >= 0x7F800000u ? 255u : (unsigned)b;
}
// 1 / step of a byte (0 and 255: any finite value will do)
__device__ __forceinline__ float t8_inv_step(unsigned b) { return __uint_as_float((254u - min(max(b, 1u), 248u)) << 23); }
// the step of a byte: 0 for 0, NaN for 255
__device__ __forceinline__ float t8_step(unsigned b) { return b == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(b << 23); }

template <int KIND>
__device__ __forceinline__ unsigned t8_code(float x, float inv, float most, bool bad) {
    if (KIND == T8_RELU) {
        const float q = fminf(fmaxf(rintf(x * inv), 1.f), most);
        if (bad) return x <= 0.f ? 0u : 255u;
        return x > 0.f ? (unsigned)q : 0u;
    }
    const float q = fminf(fmaxf(rintf(x * inv), -127.f), 127.f);
    return bad ? 0u : (unsigned)(int)q & 0xFFu;
}
template <int KIND>
__device__ __forceinline__ unsigned t8_code4(const t8_f4& v, unsigned byte) {
    const float inv = t8_inv_step(byte);
    const float most = byte == 248u ? 127.f : 255.f;
    const bool bad = byte == 255u;
    return t8_code<KIND>(v[0], inv, most, bad) | t8_code<KIND>(v[1], inv, most, bad) << 8 | t8_code<KIND>(v[2], inv, most, bad) << 16 |
           t8_code<KIND>(v[3], inv, most, bad) << 24;
}
// code c of a word of four as a float
template <int KIND>
__device__ __forceinline__ float t8_q(unsigned w, int c) {
    return KIND == T8_RELU ? (float)((w >> (8 * c)) & 0xFFu) : (float)((int)(w << (24 - 8 * c)) >> 24);
}
template <int KIND>
__device__ __forceinline__ t8_f4 t8_decode4(unsigned w, unsigned byte) {
    const float s = t8_step(byte);
    return t8_f4{t8_q<KIND>(w, 0) * s, t8_q<KIND>(w, 1) * s, t8_q<KIND>(w, 2) * s, t8_q<KIND>(w, 3) * s};
}
// the top of a block of 32 columns: eight neighbouring lanes hold four columns each (quad_perm 1 0 3 2, 2 3 0 1, row_half_mirror)
__device__ __forceinline__ unsigned t8_max8(unsigned t) {
    t = max(t, (unsigned)__builtin_amdgcn_update_dpp(0, (int)t, 0xB1, 0xF, 0xF, true));
    t = max(t, (unsigned)__builtin_amdgcn_update_dpp(0, (int)t, 0x4E, 0xF, 0xF, true));
    return max(t, (unsigned)__builtin_amdgcn_update_dpp(0, (int)t, 0x141, 0xF, 0xF, true));
}
