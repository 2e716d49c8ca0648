// Shared device code of the kernels that norm rows of channels (dpig_rows_fwd.hip, dpig_rows_bwd.hip).
//
// A row of C channels belongs to LPR lanes (8 .. 64 of one wave, or the 256 of a workgroup), NV vectors of 8 channels each: vector j of lane l is
// channels 8 (l + LPR j) .. + 7.  The row stays in registers between its statistics and its result: HBM sees every operand once.
// Rows whose start or length is not a multiple of 16 bytes take the RAG instances: 16-byte accesses at element alignment (which the part's
// memory pipe takes), and element accesses for the one partial vector at a row's end.
#pragma once
#include "dpig_act8.h"

namespace dpig {
namespace rows {

constexpr int NT = 256;
constexpr int C_MAX = 8192;

typedef unsigned short bf16_t;

template <typename T> struct Raw8;
template <> struct Raw8<float> { uint4 a, b; };
template <> struct Raw8<bf16_t> { uint4 a; };

__device__ __forceinline__ unsigned short f2bf(float f) { return __builtin_bit_cast(unsigned short, (__bf16)f); }
__device__ __forceinline__ float round_to(float f, float*) { return f; }
__device__ __forceinline__ float round_to(float f, bf16_t*) { return __uint_as_float((unsigned)f2bf(f) << 16); }

__device__ __forceinline__ void unpack(const Raw8<float>& r, float (&v)[8]) {
    v[0] = __uint_as_float(r.a.x); v[1] = __uint_as_float(r.a.y); v[2] = __uint_as_float(r.a.z); v[3] = __uint_as_float(r.a.w);
    v[4] = __uint_as_float(r.b.x); v[5] = __uint_as_float(r.b.y); v[6] = __uint_as_float(r.b.z); v[7] = __uint_as_float(r.b.w);
}
__device__ __forceinline__ void unpack(const Raw8<bf16_t>& r, float (&v)[8]) {
    v[0] = __uint_as_float(r.a.x << 16); v[1] = __uint_as_float(r.a.x & 0xffff0000u);
    v[2] = __uint_as_float(r.a.y << 16); v[3] = __uint_as_float(r.a.y & 0xffff0000u);
    v[4] = __uint_as_float(r.a.z << 16); v[5] = __uint_as_float(r.a.z & 0xffff0000u);
    v[6] = __uint_as_float(r.a.w << 16); v[7] = __uint_as_float(r.a.w & 0xffff0000u);
}
__device__ __forceinline__ void pack(const float (&v)[8], Raw8<float>& r) {
    r.a = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    r.b = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
}
__device__ __forceinline__ void pack(const float (&v)[8], Raw8<bf16_t>& r) {
    r.a.x = (unsigned)f2bf(v[0]) | ((unsigned)f2bf(v[1]) << 16); r.a.y = (unsigned)f2bf(v[2]) | ((unsigned)f2bf(v[3]) << 16);
    r.a.z = (unsigned)f2bf(v[4]) | ((unsigned)f2bf(v[5]) << 16); r.a.w = (unsigned)f2bf(v[6]) | ((unsigned)f2bf(v[7]) << 16);
}

// n (<= 0: none, >= 8: all) elements at p.  RAG: what lies behind the n is not to be used -- `beyond` says that 8 elements may be read at p
// all the same, which holds for every row but the last where C >= 8 (see `safe_rows`), so that only the last row's partial vector is read
// element by element.
// Rows whose partial vector may be read whole: its 8 elements end before column C + 7 <= ld + C, the end of the next row, if there is one.
__device__ __forceinline__ long safe_rows(long nrows, int C) { return C >= 8 ? nrows - 1 : 0; }
template <bool RAG, typename T> __device__ __forceinline__ Raw8<T> ld8(const T* p, int n, bool beyond) {
    Raw8<T> r = {};
    if (!RAG) {
        if (n > 0) r = *reinterpret_cast<const Raw8<T>*>(p);
    } else if (n >= 8 || (n > 0 && beyond)) {
        __builtin_memcpy(&r, p, sizeof(r));
    } else if (n > 0) {
        T t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = e < n ? p[e] : T(0);
        __builtin_memcpy(&r, t, sizeof(r));
    }
    return r;
}
template <bool RAG, typename T> __device__ __forceinline__ void st8(T* p, const float (&v)[8], int n) {
    Raw8<T> r;
    pack(v, r);
    if (!RAG) {
        if (n > 0) *reinterpret_cast<Raw8<T>*>(p) = r;
    } else if (n >= 8) {
        __builtin_memcpy(p, &r, sizeof(r));
    } else if (n > 0) {                                  // 4 + 2 + 1 elements
        T t[8];
        __builtin_memcpy(t, &r, sizeof(r));
        if (n & 4) __builtin_memcpy(p, t, 4 * sizeof(T));
        if (n & 2) {
            const T u[2] = {n & 4 ? t[4] : t[0], n & 4 ? t[5] : t[1]};
            __builtin_memcpy(p + (n & 4), u, 2 * sizeof(T));
        }
        if (n & 1) p[n & 6] = n & 4 ? (n & 2 ? t[6] : t[4]) : (n & 2 ? t[2] : t[0]);
    }
}
// per-channel fp32 parameters (any 4-byte alignment); `def` where there is no tensor or no channel
__device__ __forceinline__ void ldp(const float* p, int c, int C, float def, float (&v)[8]) {
    if (p != nullptr && c + 8 <= C) {
        __builtin_memcpy(v, p + c, 32);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (p != nullptr && c + e < C) ? p[c + e] : def;
    }
}
__device__ __forceinline__ void ldp(const bf16_t* p, int c, int C, float def, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (c + e < C) ? __uint_as_float((unsigned)p[c + e] << 16) : def;
}

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL> __device__ __forceinline__ unsigned dppu(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
constexpr int QP_XOR1 = 0xb1, QP_XOR2 = 0x4e, ROW_HALF_MIRROR = 0x141, ROW_MIRROR = 0x140;

// sums over the LPR lanes of a row, the same in each of them; always the same order
template <int LPR, int NS> __device__ __forceinline__ void row_sums(float (&s)[NS], float (*red)[4]) {
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        s[k] += dpp<QP_XOR1>(s[k]);
        s[k] += dpp<QP_XOR2>(s[k]);
        s[k] += dpp<ROW_HALF_MIRROR>(s[k]);
        if (LPR >= 16) s[k] += dpp<ROW_MIRROR>(s[k]);
        if (LPR >= 32) s[k] += __shfl_xor(s[k], 16, 64);
        if (LPR >= 64) s[k] += __shfl_xor(s[k], 32, 64);
    }
    if (LPR == NT) {
        __syncthreads();                                 // (red may still be read from the call before)
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < NS; ++k) red[k][threadIdx.x >> 6] = s[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NS; ++k) s[k] = (red[k][0] + red[k][1]) + (red[k][2] + red[k][3]);
    }
}

// s / C and 1 / sqrt(a), each within about half a step: the scale of a whole row hangs on them, and with it the side on which every value of the
// row falls when it is rounded to 8 bits
__device__ __forceinline__ float over_count(float s, float C, float rC) {
    const float q = s * rC, f = fmaf(fmaf(-q, C, s), rC, q);
    return f == f ? f : q;                                    // (a sum that overflowed stays infinite)
}
__device__ __forceinline__ float inv_sqrt(float a) {
    const float r = __builtin_amdgcn_rsqf(a);
    const float h = a * r, l = fmaf(a, r, -h);
    const float e = fmaf(-l, r, fmaf(-h, r, 1.f));           // 1 - a r r
    const float f = fmaf(0.5f * r, e, r);
    return f == f ? f : r;                                    // (1 / sqrt of infinity is zero, of zero infinite)
}

// A row's sum from the sums of its vectors in a lane.  One of 8 lanes x 3 vectors is (S0 + S1) + S2 with S the sums over lanes of one vector each, which is
// the order in which 32 lanes of one vector add up ((S2 + zeros) there); likewise 16 x 3 and 64 x 1, 64 x 3 and 256 x 1, and 32 x 3 and 64 x 2 with the two
// vectors apart.  So a row's statistics do not depend on its layout: the exit's norms are the entry's bit for bit whatever either chooses.
template <int LPR, int NV> constexpr bool vectors_apart() { return NV == 3 || (LPR == 64 && NV == 2); }
template <int LPR, int NV, int NS> __device__ __forceinline__ float row_sum(float (&s)[NS], float (*red)[4]) {
    row_sums<LPR, NS>(s, red);
    float t = s[0];
#pragma unroll
    for (int j = 1; j < NS; ++j) t += s[j];
    return t;
}
// Statistics of a row held in registers, and the row normed in place: mean first, then the sum of squares about it (no cancellation).
// n[j] <= 0: a vector outside the row (zero); what is behind a partial vector's end is ignored and comes out as zero.
template <int LPR, int NV, bool RAG>
__device__ __forceinline__ void whiten(float (&v)[NV][8], const int (&n)[NV], float C, float rC, bool layer, float eps, float (*red)[4], float* mean,
                                       float* rstd) {
    constexpr bool APART = vectors_apart<LPR, NV>();
    constexpr int NS = APART ? NV : 1;
    float s[NS];
    float mu = 0.f;
    if (layer) {
#pragma unroll
        for (int j = 0; j < NS; ++j) s[j] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[APART ? j : 0] += !RAG || e < n[j] ? v[j][e] : 0.f;
        mu = over_count(row_sum<LPR, NV>(s, red), C, rC);
    }
#pragma unroll
    for (int j = 0; j < NS; ++j) s[j] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = RAG ? e < n[j] : n[j] > 0;
            v[j][e] = in ? v[j][e] - mu : 0.f;
            s[APART ? j : 0] = fmaf(v[j][e], v[j][e], s[APART ? j : 0]);
        }
    const float r = inv_sqrt(over_count(row_sum<LPR, NV>(s, red), C, rC) + eps);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] *= r;
    *mean = mu;
    *rstd = r;
}

// The checkpoint is of xh as rounded to fp32: one value in about 10^6 lies so near the edge between two codes that this, and the last bits of the
// statistics, decide which it gets (141 of 127 million values against sums and products in 64 bits; 153 for elementary operations in fp32).
// Products rounded to odd bring it to 102 and cost the 131072 x 256 bf16 norm 37.2 us instead of 30.7.
// One vector of a row into its checkpoint; the four lanes of a quad hold the 32 channels of a group.  `in`: the vector lies within
// the padded row (the same for the whole quad).
template <int F> __device__ __forceinline__ void save8_as(const float (&v)[8], uint8_t* code, uint8_t* scale, bool first) {
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
    m = max(m, dppu<QP_XOR1>(m));
    m = max(m, dppu<QP_XOR2>(m));
    float inv;
    const unsigned byte = act8::scale_byte<F>(m, &inv);
    *reinterpret_cast<uint2*>(code) = act8::encode8<F>(v, inv);
    if (first) *scale = (uint8_t)byte;
}
struct Save {                  // codes == nullptr: nothing is saved
    uint8_t *codes, *scales;
    int fmt, ld;               // ld = padded(C)
};
template <int LPR, int NV>
__device__ __forceinline__ void save8(const Save& q, long r, int lane, const float (&v)[NV][8]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = 8 * (lane + LPR * j);
        if (c < q.ld) {
            uint8_t* code = q.codes + r * q.ld + c;
            uint8_t* scale = q.scales + r * (q.ld >> 5) + (c >> 5);
            if (q.fmt == DPIG_ACT8_E4M3) save8_as<DPIG_ACT8_E4M3>(v[j], code, scale, (lane & 3) == 0);
            else save8_as<DPIG_ACT8_INT8>(v[j], code, scale, (lane & 3) == 0);
        }
    }
}

// Launch shape of a row length: lanes per row and vectors per lane.  One or two vectors a lane up to 4096 channels.
#define DPIG_ROWS_DISPATCH2(C, CALL)                     \
    do {                                                 \
        if ((C) <= 64) { CALL(8, 1); }                   \
        else if ((C) <= 128) { CALL(16, 1); }            \
        else if ((C) <= 256) { CALL(32, 1); }            \
        else if ((C) <= 512) { CALL(64, 1); }            \
        else if ((C) <= 1024) { CALL(64, 2); }           \
        else if ((C) <= 2048) { CALL(256, 1); }          \
        else if ((C) <= 4096) { CALL(256, 2); }          \
        else { CALL(256, 4); }                           \
    } while (0)
inline int lanes_per_row2(int C) { return C <= 64 ? 8 : C <= 128 ? 16 : C <= 256 ? 32 : C <= 1024 ? 64 : 256; }
// Between a power of two and one and a half of it (129 .. 192, 257 .. 384, 513 .. 768, 1025 .. 1536 channels) a quarter to a half of those lanes' vectors are
// idle.  A quarter of the lanes (half of them at 513 .. 768) with three vectors each leave fewer idle and ask for more at a time, once there are rows for four
// sets a CU; what a lane holds of three vectors must be small for that.  Where they are taken, us with one or two / three:
//   entry, bf16 whole rows         32768 x 136 9.8 / 8.7, 131072 x 320 48.1 / 36.7, 65536 x 640 40.7 / 36.2, 32768 x 1280 43.7 / 36.1
//   entry, fp32 with a checkpoint  131072 x 320 90.1 / 81.1, 32768 x 1280 87.8 / 80.5, 16384 x 320 14.1 / 14.1, 32768 x 160 13.4 / 14.2
//   gradients, bf16                from x 262144 x 136 59.2 / 45.8, 32768 x 1280 68.6 / 48.8, 16384 x 320 17.4 / 17.0, 32768 x 160 16.7 / 17.8
//   gradients, from a checkpoint   bf16 262144 x 136 53.0 / 41.6, 32768 x 1280 64.7 / 43.9; fp32 131072 x 320 95.4 / 88.0, 16384 x 320 20.8 / 21.9
//   exits, bf16 whole rows of 513 .. 768 with the next norm or a gate per row: 65536 x 640 98.9 / 79.7 and 135.0 / 127.5, 8192 x 640 21.1 / 19.5 and
//                                  22.9 / 20.7; with both 193 / 221, with neither 30.8 / 34.9 (32768 rows)
// Elsewhere one or two vectors are as fast or faster, three over that: fp32 entry without a checkpoint 0.85 .. 1.08, fp32 gradients from x 0.92 .. 1.25, ragged bf16
// entry 0.84 .. 1.14, the other exits 0.81 .. 1.97 (two operands and five rows of parameters).
inline bool three_vectors(int64_t nrows, int C) {
    const int lanes = C > 1024 ? 64 : C > 512 ? 32 : C > 256 ? 16 : 8;
    return C > 16 * lanes && C <= 24 * lanes && nrows * lanes >= 4L * kNumCU * NT;
}
#define DPIG_ROWS_DISPATCH3(C, CALL)                     \
    do {                                                 \
        if ((C) <= 192) { CALL(8, 3); }                  \
        else if ((C) <= 384) { CALL(16, 3); }            \
        else if ((C) <= 768) { CALL(32, 3); }            \
        else { CALL(64, 3); }                            \
    } while (0)
inline int lanes_per_row3(int C) { return C <= 192 ? 8 : C <= 384 ? 16 : C <= 768 ? 32 : 64; }
inline bool vec_ok(const void* p, int64_t ld, int esize) { return aligned16(p) && (ld * esize) % 16 == 0; }

}  // namespace rows
}  // namespace dpig
