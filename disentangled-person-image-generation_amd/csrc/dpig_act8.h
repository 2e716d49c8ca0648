// 8-bit activation checkpoints on rows of channels: the format, and its device-side encoding and decoding.
//
// A checkpoint of [rows][C] is codes [rows][ld] (ld = C rounded up to 32; columns >= C hold zero codes) and scales [rows][ld / 32].
// The 32 channels of a group share a power of two s = 2^e, stored as the byte e + 127, e the smallest exponent with
// max|x| <= 448 s (E4M3) or 127 s (INT8); code = x / s rounded to nearest even:
//   E4M3   an OCP 8-bit float (1 + 4 + 3 bits)            zero code 0x00
//   INT8   an integer of -127 .. 127, stored plus 128       zero code 0x80
// Choices, and why:
//   * a power of two: code * s is exact in bfloat16 (4 or 7 significant bits), so a product that reads a checkpoint loses nothing
//     beyond the stored rounding; and x / s is exact, so the rounding is one rounding of x;
//   * a value that is not zero never becomes the zero code: below the smallest code it is stored as that code with its sign.  The
//     checkpoint of a ReLU / LeakyReLU output then has the sign pattern of the output and serves as the activation's mask.  It costs
//     at most one smallest code of error there (2^-9 s, 1 s) instead of half of one;
//   * a group that holds a NaN or an infinity gets the scale byte 255 and zero codes: it comes back as NaN throughout, so an overflow
//     of the forward pass is seen where values are read (filter gradients, norms' gradients), and none has to be tested then.  A mask is
//     read from the codes alone: the whole group counts as not positive, its finite neighbours of an infinity included;
//   * e is kept within [-116, 119] (E4M3) / [-116, 121] (INT8): every decoded value is a normal, finite fp32 / bf16 number.  What is larger than
//     the last scale's largest code (1.75 * 2^127) is stored as that code.
#pragma once
#include "dpig_common.h"

namespace dpig {
namespace act8 {

constexpr int GROUP = 32;
constexpr int EXP_MIN = -116;

typedef float f32x2 __attribute__((ext_vector_type(2)));

__host__ __device__ __forceinline__ int padded(int C) { return (C + GROUP - 1) / GROUP * GROUP; }

template <int F> struct Fmt;
template <> struct Fmt<DPIG_ACT8_E4M3> {
    static constexpr float most = 448.f, least = 0x1p-9f;
    static constexpr int bias = 135, exp_max = 119;                 // e = E - bias (+ 1 above `edge`), E the biased exponent of max|x|
    static constexpr unsigned edge = 0x600000u;                      // mantissa of 1.75: 448 = 1.75 * 2^8
};
template <> struct Fmt<DPIG_ACT8_INT8> {
    static constexpr float most = 127.f, least = 1.f;
    static constexpr int bias = 133, exp_max = 121;
    static constexpr unsigned edge = 0x7e0000u;                      // mantissa of 127 / 64
};

// scale byte of a group from the bits of max|x| (255: not finite), and 1 / s
template <int F> __device__ __forceinline__ unsigned scale_byte(unsigned amax_bits, float* inv) {
    int e = (int)(amax_bits >> 23) - Fmt<F>::bias + ((amax_bits & 0x7fffffu) > Fmt<F>::edge ? 1 : 0);
    e = e < EXP_MIN ? EXP_MIN : (e > Fmt<F>::exp_max ? Fmt<F>::exp_max : e);
    const bool bad = amax_bits >= 0x7f800000u;
    *inv = bad ? 0.f : __uint_as_float((unsigned)(127 - e) << 23);
    return bad ? 255u : (unsigned)(e + 127);
}
// x / s with the sign kept, inside the format's range
template <int F> __device__ __forceinline__ float to_grid(float x, float inv) {
    const float m = __builtin_amdgcn_fmed3f(fabsf(x) * inv, Fmt<F>::least, Fmt<F>::most);
    return x == 0.f ? 0.f : copysignf(m, x);
}
// eight codes; inv = 0 marks a group that is not finite (all codes zero)
template <int F> __device__ __forceinline__ uint2 encode8(const float (&x)[8], float inv) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = inv == 0.f ? 0.f : to_grid<F>(x[e], inv);
    unsigned q[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (F == DPIG_ACT8_E4M3) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h], v[4 * h + 1], 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2], v[4 * h + 3], w, true);
            q[h] = (unsigned)w;
        } else {
            // adding 1.5 * 2^23 leaves the integer nearest to v (ties to even) in the low bits of the sum
            unsigned b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(v[4 * h + e] + (12582912.f + 128.f));
            const unsigned lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
            q[h] = lo | hi;
        }
    }
    return make_uint2(q[0], q[1]);
}
__device__ __forceinline__ float scale_value(unsigned byte) { return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23); }

template <int F> __device__ __forceinline__ void decode4(unsigned q, float s, float* v) {
    if constexpr (F == DPIG_ACT8_E4M3) {
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
        v[0] = a[0] * s; v[1] = a[1] * s; v[2] = b[0] * s; v[3] = b[1] * s;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ((float)((q >> (8 * e)) & 255u) - 128.f) * s;      // (no fma with -128 s: 128 * 2^121 overflows)
    }
}
template <int F> __device__ __forceinline__ void decode8(uint2 q, float s, float (&v)[8]) {
    decode4<F>(q.x, s, v);
    decode4<F>(q.y, s, v + 4);
}
// value > 0, for the byte `e` of q (a group that was not finite has zero codes: not positive, as a NaN is not)
template <int F> __device__ __forceinline__ bool positive(unsigned q, int e) {
    const unsigned c = (q >> (8 * e)) & 255u;
    return F == DPIG_ACT8_E4M3 ? (c - 1u < 0x7eu) : c > 128u;
}

}  // namespace act8
}  // namespace dpig
