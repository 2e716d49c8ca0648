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

// Statistics of a row held in registers, and the row normed in place: mean first, then the sum of squares about it (no cancellation).
// n[j] <= 0: a vector outside the row (zero); what is behind a partial vector's end is ignored and comes out as zero.
template <int LPR, int NV, bool RAG>
__device__ __forceinline__ void whiten(float (&v)[NV][8], const int (&n)[NV], float C, float rC, bool layer, float eps, float (*red)[4], float* mean,
                                       float* rstd) {
    float s[1];
    float mu = 0.f;
    if (layer) {
        s[0] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[0] += !RAG || e < n[j] ? v[j][e] : 0.f;
        row_sums<LPR, 1>(s, red);
        mu = over_count(s[0], C, rC);
    }
    s[0] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = RAG ? e < n[j] : n[j] > 0;
            v[j][e] = in ? v[j][e] - mu : 0.f;
            s[0] += v[j][e] * v[j][e];
        }
    row_sums<LPR, 1>(s, red);
    const float r = inv_sqrt(over_count(s[0], C, rC) + eps);
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

// Launch shape of a row length: lanes per row and vectors per lane.  One or two vectors a lane up to 4096 channels; where that leaves a lane in
// three or more idle (just above a power of two) and there are rows enough for four sets a CU, a quarter of the lanes with three each: 32768 rows of 640
// channels, the exit's gradient, 24 us instead of 30.  Where the lanes are better filled it does not pay (384 channels: 41.6 against 39.9 us).
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
#define DPIG_ROWS_DISPATCH(C, THREE, CALL)               \
    do {                                                 \
        if (!(THREE)) DPIG_ROWS_DISPATCH2(C, CALL);      \
        else if ((C) <= 160) { CALL(8, 3); }             \
        else if ((C) <= 320) { CALL(16, 3); }            \
        else if ((C) <= 640) { CALL(32, 3); }            \
        else { CALL(64, 3); }                            \
    } while (0)
inline int lanes_per_row2(int C) { return C <= 64 ? 8 : C <= 128 ? 16 : C <= 256 ? 32 : C <= 1024 ? 64 : 256; }
inline bool three_vectors(int64_t nrows, int C) {
    const int lanes = C > 1024 ? 64 : C > 512 ? 32 : C > 256 ? 16 : 8;
    const bool thin = (C > 128 && C <= 160) || (C > 256 && C <= 320) || (C > 512 && C <= 640) || (C > 1024 && C <= 1280);
    return thin && nrows * lanes >= 4L * kNumCU * NT;
}
inline int lanes_per_row(int64_t nrows, int C) {
    return !three_vectors(nrows, C) ? lanes_per_row2(C) : C <= 160 ? 8 : C <= 320 ? 16 : C <= 640 ? 32 : 64;
}
inline bool vec_ok(const void* p, int64_t ld, int esize) { return aligned16(p) && (ld * esize) % 16 == 0; }

}  // namespace rows
}  // namespace dpig
