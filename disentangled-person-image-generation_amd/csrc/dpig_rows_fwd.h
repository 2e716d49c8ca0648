// Norms over the channels of a row, at a residual block's entry and at its exit, forward:
//   entry  y   = scale * xh + offset,            xh = (x - mean) rstd   (kind 'rms': mean = 0)
//   exit   out = x + res_scale * gate * (scale * fh + offset),  fh the normed f; optionally the next block's entry norm of `out` (as stored) too
// and, on request, xh (or fh, or the next norm's xh) as an 8-bit checkpoint from the same registers.
//
// Bound by HBM: every operand is read once and every result written once, one wave (or less, or a workgroup) per row with the row in
// registers; a lane asks for the next row before it works on the present one.  A workgroup takes a contiguous range of rows, so the
// per-channel operands stay in registers and a gate row is loaded when its group begins.
// Measured (averages under the profiler): entry 131072 x 256 bf16 with its e4m3 checkpoint 30 .. 32 us (168 MB, 5.4 TB/s); exit with the next norm
// 131072 x 128 bf16, a gate per 8192 rows, 28.5 us (134 MB, 4.7 TB/s), 131072 x 640 152 us (4.4 TB/s); exit 9001 x 333 fp32 with a gate per row 13.3 us
// (48 MB, 3.6 TB/s: three rows a wave, whose ends share lines; 60001 rows 66 us, 4.8 TB/s); 64 x 512 fp32 3.2 us, the latency of one load, two sums
// and one store.
#pragma once
#include "dpig_rows.h"

namespace dpig {
namespace rows {

struct EntryP {
    const void* x; void* y;
    const float *scale, *offset;
    float *mean, *rstd;
    long ldx, ldy, nrows, chunk;
    int C, layer;
    float eps, rC;
    Save save;
};

template <typename T, int LPR, int NV, bool RAG, bool SAVE>
__global__ __launch_bounds__(NT) void entry_fwd_kernel(const EntryP p) {
    constexpr int RPB = NT / LPR;
    __shared__ float red[1][4];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const long safe = safe_rows(p.nrows, p.C);
    const T* x = static_cast<const T*>(p.x);
    T* y = static_cast<T*>(p.y);
    int n[NV];
    float sc[NV][8], of[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = 8 * (lane + LPR * j);
        n[j] = p.C - c;
        ldp(p.scale, c, p.C, 1.f, sc[j]);
        ldp(p.offset, c, p.C, 0.f, of[j]);
    }
    const long r0 = blockIdx.x * p.chunk, r1 = min(r0 + p.chunk, p.nrows);
    long r = r0 + sub;
    Raw8<T> nx[NV];
    auto fetch = [&](long row) {
#pragma unroll
        for (int j = 0; j < NV; ++j) nx[j] = ld8<RAG>(x + row * p.ldx + 8 * (lane + LPR * j), n[j], row < safe);
    };
    if (r < r1) fetch(r);
    for (; r < r1; r += RPB) {
        float v[NV][8];
#pragma unroll
        for (int j = 0; j < NV; ++j) unpack(nx[j], v[j]);
        if (r + RPB < r1) fetch(r + RPB);
        float mean, rstd;
        whiten<LPR, NV, RAG>(v, n, (float)p.C, p.rC, p.layer != 0, p.eps, red, &mean, &rstd);
        if (lane == 0) {
            if (p.mean != nullptr) p.mean[r] = mean;
            p.rstd[r] = rstd;
        }
        if (SAVE) save8<LPR, NV>(p.save, r, lane, v);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = fmaf(v[j][e], sc[j][e], of[j][e]);
            st8<RAG>(y + r * p.ldy + 8 * (lane + LPR * j), v[j], n[j]);
        }
    }
}

struct ExitP {
    const void *x, *f;
    void *out, *h;                       // h == nullptr: no next norm
    const float *scale, *offset, *res, *scale2, *offset2;
    const void* gate;
    float *mean, *rstd, *mean2, *rstd2;
    long ldx, ldf, ldo, ldh, nrows, chunk, per;      // per = rows of a gate group
    int C, layer, layer2, gate_bf16;
    float eps, eps2, rC;
    Save save, save2;
};

// EACH: every row has a gate of its own, fetched with the row; else a gate row is loaded when its group begins
template <typename T, int LPR, int NV, bool RAG, bool NEXT, bool EACH>
__global__ __launch_bounds__(NT) void exit_fwd_kernel(const ExitP p) {
    constexpr int RPB = NT / LPR;
    __shared__ float red[1][4];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const long safe = safe_rows(p.nrows, p.C);
    const T *x = static_cast<const T*>(p.x), *f = static_cast<const T*>(p.f);
    int n[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) n[j] = p.C - 8 * (lane + LPR * j);
    const long r0 = blockIdx.x * p.chunk, r1 = min(r0 + p.chunk, p.nrows);
    long r = r0 + sub;
    Raw8<T> nx[NV], nf[NV];
    float ng[NV][8];                     // EACH: the next row's gate
    auto load_gate = [&](long g, int j, float (&m)[8]) {
        const int c = 8 * (lane + LPR * j);
        if (p.gate_bf16) ldp(static_cast<const bf16_t*>(p.gate) + g * p.C, c, p.C, 1.f, m);
        else ldp(static_cast<const float*>(p.gate) + g * p.C, c, p.C, 1.f, m);
    };
    auto fetch = [&](long row) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const bool beyond = row < safe;
            nx[j] = ld8<RAG>(x + row * p.ldx + 8 * (lane + LPR * j), n[j], beyond);
            nf[j] = ld8<RAG>(f + row * p.ldf + 8 * (lane + LPR * j), n[j], beyond);
            if (EACH) load_gate(row, j, ng[j]);
        }
    };
    if (r < r1) fetch(r);
    float a[NV][8], b[NV][8], m[NV][8];  // out = x + m (a fh + b): a, b with the residual scale, m the gate
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = 8 * (lane + LPR * j);
        float t[8];
        ldp(p.res, c, p.C, 1.f, t);
        ldp(p.scale, c, p.C, 1.f, a[j]);
        ldp(p.offset, c, p.C, 0.f, b[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) { a[j][e] *= t[e]; b[j][e] *= t[e]; m[j][e] = 1.f; }
    }
    float sc2[NEXT ? NV : 1][8], of2[NEXT ? NV : 1][8];
    if (NEXT) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            ldp(p.scale2, 8 * (lane + LPR * j), p.C, 1.f, sc2[j]);
            ldp(p.offset2, 8 * (lane + LPR * j), p.C, 0.f, of2[j]);
        }
    }
    long g = EACH || p.gate == nullptr ? 0 : r / p.per, until = p.gate == nullptr ? p.nrows : (g + 1) * p.per;     // r's group, and its end
    if (!EACH && p.gate != nullptr && r < r1) {
#pragma unroll
        for (int j = 0; j < NV; ++j) load_gate(g, j, m[j]);
    }
    for (; r < r1; r += RPB) {
        float v[NV][8], xv[NV][8];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            unpack(nf[j], v[j]);
            unpack(nx[j], xv[j]);
            if (EACH) {
#pragma unroll
                for (int e = 0; e < 8; ++e) m[j][e] = ng[j][e];
            }
        }
        if (r + RPB < r1) fetch(r + RPB);
        if (!EACH && r >= until) {
            while (r >= until) { ++g; until += p.per; }
#pragma unroll
            for (int j = 0; j < NV; ++j) load_gate(g, j, m[j]);
        }
        float mean, rstd;
        whiten<LPR, NV, RAG>(v, n, (float)p.C, p.rC, p.layer != 0, p.eps, red, &mean, &rstd);
        if (lane == 0) {
            if (p.mean != nullptr) p.mean[r] = mean;
            p.rstd[r] = rstd;
        }
        if (p.save.codes != nullptr) save8<LPR, NV>(p.save, r, lane, v);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = fmaf(m[j][e], fmaf(v[j][e], a[j][e], b[j][e]), xv[j][e]);
            st8<RAG>(static_cast<T*>(p.out) + r * p.ldo + 8 * (lane + LPR * j), v[j], n[j]);
        }
        if (NEXT) {
            // the next block's norm sees `out` as it is stored, so that its backward pass can start from the stored tensor
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool in = RAG ? e < n[j] : n[j] > 0;
                    v[j][e] = in ? round_to(v[j][e], static_cast<T*>(nullptr)) : 0.f;
                }
            whiten<LPR, NV, RAG>(v, n, (float)p.C, p.rC, p.layer2 != 0, p.eps2, red, &mean, &rstd);
            if (lane == 0) {
                if (p.mean2 != nullptr) p.mean2[r] = mean;
                p.rstd2[r] = rstd;
            }
            if (p.save2.codes != nullptr) save8<LPR, NV>(p.save2, r, lane, v);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j][e] = fmaf(v[j][e], sc2[j][e], of2[j][e]);
                st8<RAG>(static_cast<T*>(p.h) + r * p.ldh + 8 * (lane + LPR * j), v[j], n[j]);
            }
        }
    }
}

// rows per workgroup: a multiple of the rows it takes at a time, at most `per_cu` workgroups per CU
inline long fwd_chunk(int64_t nrows, int lanes, long per_cu) {
    const long rpb = NT / lanes;
    const long want = per_cu * kNumCU;
    long it = (nrows + rpb * want - 1) / (rpb * want);
    return (it < 1 ? 1 : it) * rpb;
}
// The entry's registers let eight workgroups share a CU, the exit's four.  More of them than fit come in rounds: that evens out HBM where there is much
// to move (32768 x 256 fp32 with the next norm, 134 MB: 25.0 us in two rounds, 27.0 in one) but costs each round's start where there is little
// (4096 x 2048 bf16 with the next norm, 67 MB: 16.4 / 14.7; 8192 x 512: 11.0 / 9.6), and a last round that is not full costs as much as a full one
// (9001 x 333 fp32: 1.1 rounds 17.0, one 13.2; 60001 x 333: 1.8 rounds 74, one 71).
constexpr long ENTRY_PER_CU = 8, EXIT_PER_CU = 4, EXIT_ONE_ROUND_BYTES = 96L << 20;
inline long exit_chunk(int64_t nrows, int lanes, long bytes) {
    const long one = fwd_chunk(nrows, lanes, EXIT_PER_CU), two = fwd_chunk(nrows, lanes, 2 * EXIT_PER_CU);
    const long groups = (nrows + two - 1) / two, rounds = (groups + EXIT_PER_CU * kNumCU - 1) / (EXIT_PER_CU * kNumCU);
    return bytes < EXIT_ONE_ROUND_BYTES || one < rounds * two ? one : two;
}

// the kernels on tensors of type T; each type is compiled in a file of its own
template <typename T> int entry_fwd(EntryP p, hipStream_t st);
template <typename T> int exit_fwd(ExitP p, hipStream_t st);

template <typename T> inline int entry_fwd_as(EntryP p, hipStream_t st) {
    const bool rag = p.C % 8 != 0 || !vec_ok(p.x, p.ldx, sizeof(T)) || !vec_ok(p.y, p.ldy, sizeof(T));
    const bool save = p.save.codes != nullptr;
    const bool three = (sizeof(T) == 2 ? !rag : save) && three_vectors(p.nrows, p.C);
    p.chunk = fwd_chunk(p.nrows, three ? lanes_per_row3(p.C) : lanes_per_row2(p.C), ENTRY_PER_CU);
    const dim3 grid((unsigned)((p.nrows + p.chunk - 1) / p.chunk));
#define CALL_RS(L, N, R, S) hipLaunchKernelGGL((entry_fwd_kernel<T, L, N, R, S>), grid, dim3(NT), 0, st, p)
#define CALL(L, N)                                                                                                         \
    do {                                                                                                                  \
        if (rag) { if (save) CALL_RS(L, N, true, true); else CALL_RS(L, N, true, false); }                                 \
        else { if (save) CALL_RS(L, N, false, true); else CALL_RS(L, N, false, false); }                                   \
    } while (0)
#define CALL_WHOLE(L, N) do { if (save) CALL_RS(L, N, false, true); else CALL_RS(L, N, false, false); } while (0)
#define CALL_SAVE(L, N) do { if (rag) CALL_RS(L, N, true, true); else CALL_RS(L, N, false, true); } while (0)
    if (!three) DPIG_ROWS_DISPATCH2(p.C, CALL);
    else if constexpr (sizeof(T) == 2) DPIG_ROWS_DISPATCH3(p.C, CALL_WHOLE);
    else DPIG_ROWS_DISPATCH3(p.C, CALL_SAVE);
#undef CALL
#undef CALL_WHOLE
#undef CALL_SAVE
#undef CALL_RS
    return check_launch("rownorm_fwd");
}
template <typename T> inline int exit_fwd_as(ExitP p, hipStream_t st) {
    const int z = sizeof(T);
    const bool rag = p.C % 8 != 0 || !vec_ok(p.x, p.ldx, z) || !vec_ok(p.f, p.ldf, z) || !vec_ok(p.out, p.ldo, z) ||
                     (p.h != nullptr && !vec_ok(p.h, p.ldh, z));
    const bool next = p.h != nullptr, each = p.gate != nullptr && p.per == 1;
    const bool three = sizeof(T) == 2 && !rag && next != each && p.C > 512 && p.C <= 768 && three_vectors(p.nrows, p.C);
    p.chunk = exit_chunk(p.nrows, three ? lanes_per_row3(p.C) : lanes_per_row2(p.C), (long)p.nrows * p.C * z * (next ? 4 : 3));
    const dim3 grid((unsigned)((p.nrows + p.chunk - 1) / p.chunk));
#define CALL_E(L, N, R, S, E) hipLaunchKernelGGL((exit_fwd_kernel<T, L, N, R, S, E>), grid, dim3(NT), 0, st, p)
#define CALL_RS(L, N, R, S) do { if (each) CALL_E(L, N, R, S, true); else CALL_E(L, N, R, S, false); } while (0)
#define CALL(L, N)                                                                                                         \
    do {                                                                                                                  \
        if (rag) { if (next) CALL_RS(L, N, true, true); else CALL_RS(L, N, true, false); }                                 \
        else { if (next) CALL_RS(L, N, false, true); else CALL_RS(L, N, false, false); }                                   \
    } while (0)
    if (!three) DPIG_ROWS_DISPATCH2(p.C, CALL);
    else if constexpr (sizeof(T) == 2) {
        if (next) CALL_E(32, 3, false, true, false); else CALL_E(32, 3, false, false, true);
    }
#undef CALL
#undef CALL_E
#undef CALL_RS
    return check_launch("gated_residual_fwd");
}

}  // namespace rows
}  // namespace dpig
