// Gradients of the row norms (dpig_rows_fwd.hip).  With xh from the saved input (mean, rstd) or from its 8-bit checkpoint, and per-channel weights
// w = scale (entry) or res_scale * gate * scale (exit):
//   g = dy w,   dx = rstd (g - mean_c g - xh mean_c(g xh)) (+ accum);      kind 'rms' has no mean_c g
// Every parameter gradient follows from two sums per channel and gate group g: A = sum_r dy xh, B = sum_r dy.  With t = scale A + offset B:
//   dgate[g] = res_scale t[g],  dres_scale = sum_g gate t,  dscale = res_scale sum_g gate A,  doffset = res_scale sum_g gate B
// (no gate: one group), so the row pass keeps two accumulators a channel whatever is asked for, and the small products are done once per
// group at the end.  Two ways to cut the rows:
//   pieces   a workgroup takes a contiguous piece of ONE group and leaves (A, B): partial [group][piece][2][C]
//   groups   a row's lanes take WHOLE groups (short ones: down to a row each), write dgate themselves and keep gate-weighted sums:
//            partial [workgroup][2][C]
// The partials are added in a fixed order by one or two small launches: no atomics, the same bits every time.
// Bound by HBM (2 to 4 row tensors in and out).  Measured (averages under the profiler), row pass + sums: 32768 x 384 fp32 with accum 39.0 + 4.5 us (201 MB,
// 5.2 TB/s in the pass); 131072 x 256 bf16 with accum 52.2 + 4.8; 47915 x 250 bf16 from an int8 checkpoint 17.0 .. 17.9 + 4; exit, a gate per eighth of
// the rows: 32768 x 640 bf16 from its e4m3 checkpoint 24.0 + 5.2 (105 MB, 4.4 TB/s), from f 27.1 + 5.2 (126 MB, 4.6 TB/s), 8192 x 2048 bf16 from f
// 22.2 + 6.2; 32768 x 512 bf16 with a gate per row 43.3 + 4.9.
#pragma once
#include "dpig_rows.h"

namespace dpig {
namespace rows {

struct BwdP {
    const void *dy, *x, *accum;          // x: the saved input, or nullptr with a checkpoint
    void* dx;
    const uint8_t *codes, *scales;
    const float *mean, *rstd, *scale, *offset, *res;
    const void* gate;
    void* dgate;                         // groups form only
    float* partial;
    long lddy, ldx, ldacc, lddx, nrows, chunk, per, ngroups;     // chunk: rows of a piece / groups of a workgroup
    int C, layer, fmt, ld8, gate_bf16, pieces;
    bool three;                          // pieces form: three vectors a lane
    float rC;
};

// what a lane asks for of a row: dy, and the saved input or its codes and scales
template <typename T, int LPR, int NV, bool RAG, bool SAVED> struct RowIn {
    Raw8<T> d[NV], x[SAVED ? 1 : NV];
    uint2 q[SAVED ? NV : 1];
    unsigned s[SAVED ? NV : 1];
    float mean, rstd;
    __device__ __forceinline__ void fetch(const BwdP& p, long row, int lane, const int (&n)[NV], long safe) {
        rstd = p.rstd[row];
        if (!SAVED && p.layer) mean = p.mean[row];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = 8 * (lane + LPR * j);
            d[j] = ld8<RAG>(static_cast<const T*>(p.dy) + row * p.lddy + c, n[j], row < safe);
            if constexpr (SAVED) {
                q[j] = make_uint2(0, 0);
                s[j] = 0;
                if (n[j] > 0) {
                    q[j] = *reinterpret_cast<const uint2*>(p.codes + row * p.ld8 + c);
                    s[j] = p.scales[row * (p.ld8 >> 5) + (c >> 5)];
                }
            } else {
                x[j] = ld8<RAG>(static_cast<const T*>(p.x) + row * p.ldx + c, n[j], row < safe);
            }
        }
    }
    __device__ __forceinline__ void values(const BwdP& p, const int (&n)[NV], float (&dv)[NV][8], float (&xh)[NV][8]) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            unpack(d[j], dv[j]);
            if (RAG) {
#pragma unroll
                for (int e = 0; e < 8; ++e) dv[j][e] = e < n[j] ? dv[j][e] : 0.f;
            }
            if constexpr (SAVED) {
                const float sv = act8::scale_value(s[j]);
                if (p.fmt == DPIG_ACT8_E4M3) act8::decode8<DPIG_ACT8_E4M3>(q[j], sv, xh[j]);
                else act8::decode8<DPIG_ACT8_INT8>(q[j], sv, xh[j]);
                if (RAG || n[j] <= 0) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) xh[j][e] = e < n[j] ? xh[j][e] : 0.f;
                }
            } else {
                unpack(x[j], xh[j]);
#pragma unroll
                for (int e = 0; e < 8; ++e) xh[j][e] = (RAG ? e < n[j] : n[j] > 0) ? (xh[j][e] - (p.layer ? mean : 0.f)) * rstd : 0.f;
            }
        }
    }
};

// (A, B) of a workgroup's lanes -> partial [2][C]: the RPB rows' lanes hold sums of the same channels, added over the workgroup in order
template <int LPR, int NV> __device__ __forceinline__ void leave_sums(const BwdP& p, int lane, const int (&n)[NV], const float (&A)[NV][8], const float (&B)[NV][8]) {
    constexpr int RPB = NT / LPR;
    float* out = p.partial + (long)blockIdx.x * 2 * p.C;
    if constexpr (LPR == NT) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = 8 * (lane + LPR * j);
            st8<true>(out + c, A[j], n[j]);
            st8<true>(out + p.C + c, B[j], n[j]);
        }
    } else {
        __shared__ float col[2][NT * 8];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (j > 0) __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) { col[0][threadIdx.x * 8 + e] = A[j][e]; col[1][threadIdx.x * 8 + e] = B[j][e]; }
            __syncthreads();
            for (int i = threadIdx.x; i < LPR * 8; i += NT) {
                const int c = 8 * LPR * j + i;
                if (c < p.C) {
                    float ta = 0.f, tb = 0.f;
#pragma unroll 4
                    for (int q = 0; q < RPB; ++q) { ta += col[0][q * LPR * 8 + i]; tb += col[1][q * LPR * 8 + i]; }
                    out[c] = ta;
                    out[p.C + c] = tb;
                }
            }
        }
    }
}

// Pieces form.  The next row (and its accum) is asked for before the present one is worked on.
template <typename T, int LPR, int NV, bool RAG, bool SAVED>
__global__ __launch_bounds__(NT, NV >= 4 ? 1 : 2) void rows_bwd_kernel(const BwdP p) {
    constexpr int RPB = NT / LPR;
    __shared__ float red[2][4];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const long safe = safe_rows(p.nrows, p.C);
    const long grp = blockIdx.x / p.pieces, pc = blockIdx.x - grp * p.pieces;
    const T* ac = static_cast<const T*>(p.accum);
    int n[NV];
    float w[NV][8], A[NV][8], B[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = 8 * (lane + LPR * j);
        n[j] = p.C - c;
        float t[8];
        ldp(p.scale, c, p.C, 1.f, w[j]);
        ldp(p.res, c, p.C, 1.f, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) { w[j][e] *= t[e]; A[j][e] = 0.f; B[j][e] = 0.f; }
        if (p.gate != nullptr) {
            if (p.gate_bf16) ldp(static_cast<const bf16_t*>(p.gate) + grp * p.C, c, p.C, 0.f, t);
            else ldp(static_cast<const float*>(p.gate) + grp * p.C, c, p.C, 0.f, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[j][e] *= t[e];
        }
    }
    const long lo = grp * p.per + pc * p.chunk, hi = min(lo + p.chunk, (grp + 1) * p.per);
    long r = lo + sub;
    RowIn<T, LPR, NV, RAG, SAVED> in;
    Raw8<T> na[NV];
    auto fetch = [&](long row) {
        in.fetch(p, row, lane, n, safe);
        if (ac != nullptr) {
#pragma unroll
            for (int j = 0; j < NV; ++j) na[j] = ld8<RAG>(ac + row * p.ldacc + 8 * (lane + LPR * j), n[j], row < safe);
        }
    };
    if (r < hi) fetch(r);
    for (; r < hi; r += RPB) {
        float d[NV][8], xh[NV][8], a[NV][8];
        in.values(p, n, d, xh);
        const float rstd = in.rstd;
        if (ac != nullptr) {
#pragma unroll
            for (int j = 0; j < NV; ++j) unpack(na[j], a[j]);
        }
        if (r + RPB < hi) fetch(r + RPB);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                A[j][e] = fmaf(d[j][e], xh[j][e], A[j][e]);
                B[j][e] += d[j][e];
                const float g = d[j][e] * w[j][e];
                s[0] += g;
                s[1] = fmaf(g, xh[j][e], s[1]);
            }
        row_sums<LPR, 2>(s, red);
        const float m1 = p.layer ? s[0] * p.rC : 0.f, m2 = s[1] * p.rC;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                o[e] = rstd * (fmaf(d[j][e], w[j][e], -m1) - xh[j][e] * m2);
                if (ac != nullptr) o[e] += a[j][e];
            }
            st8<RAG>(static_cast<T*>(p.dx) + r * p.lddx + 8 * (lane + LPR * j), o, n[j]);
        }
    }
    if (p.partial != nullptr) leave_sums<LPR, NV>(p, lane, n, A, B);
}

// Groups form: a row's lanes walk through the rows of their groups without a pause, the next row -- and the gate, where it begins a group -- on its
// way.  (Instances for ragged rows only: they read whole ones as well.)
template <typename T, int LPR, int NV, bool SAVED>
__global__ __launch_bounds__(NT, NV >= 4 ? 1 : 2) void rows_bwd_groups_kernel(const BwdP p) {
    constexpr int RPB = NT / LPR;
    constexpr bool RAG = true;
    __shared__ float red[2][4];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const long safe = safe_rows(p.nrows, p.C);
    int n[NV];
    float ws[NV][8], wo[NV][8], A[NV][8], B[NV][8];          // res_scale * scale, res_scale * offset; the gate-weighted sums
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = 8 * (lane + LPR * j);
        n[j] = p.C - c;
        float t[8];
        ldp(p.scale, c, p.C, 1.f, ws[j]);
        ldp(p.offset, c, p.C, 0.f, wo[j]);
        ldp(p.res, c, p.C, 1.f, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) { ws[j][e] *= t[e]; wo[j][e] *= t[e]; A[j][e] = 0.f; B[j][e] = 0.f; }
    }
    float m[NV][8], ng[NV][8], Ag[NV][8], Bg[NV][8];
    auto load_gate = [&](long g) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = 8 * (lane + LPR * j);
            if (p.gate_bf16) ldp(static_cast<const bf16_t*>(p.gate) + g * p.C, c, p.C, 0.f, ng[j]);
            else ldp(static_cast<const float*>(p.gate) + g * p.C, c, p.C, 0.f, ng[j]);
        }
    };
    const long g1 = min((blockIdx.x + 1L) * p.chunk, p.ngroups);
    long g = blockIdx.x * p.chunk + sub, k = 0;              // row k of group g
    RowIn<T, LPR, NV, RAG, SAVED> in;
    if (g < g1) { in.fetch(p, g * p.per, lane, n, safe); load_gate(g); }
    while (g < g1) {
        float d[NV][8], xh[NV][8];
        in.values(p, n, d, xh);
        const float rstd = in.rstd;
        const long r = g * p.per + k;
        if (k == 0) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    m[j][e] = ng[j][e];
                    Ag[j][e] = 0.f;
                    Bg[j][e] = 0.f;
                }
        }
        const bool last = k + 1 == p.per;
        const long gn = last ? g + RPB : g, kn = last ? 0 : k + 1;
        if (gn < g1) {
            in.fetch(p, gn * p.per + kn, lane, n, safe);
            if (last) load_gate(gn);
        }
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                Ag[j][e] = fmaf(d[j][e], xh[j][e], Ag[j][e]);
                Bg[j][e] += d[j][e];
                const float t = d[j][e] * ws[j][e] * m[j][e];
                s[0] += t;
                s[1] = fmaf(t, xh[j][e], s[1]);
            }
        row_sums<LPR, 2>(s, red);
        const float m1 = p.layer ? s[0] * p.rC : 0.f, m2 = s[1] * p.rC;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = 8 * (lane + LPR * j);
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = rstd * (fmaf(d[j][e] * ws[j][e], m[j][e], -m1) - xh[j][e] * m2);
            st8<RAG>(static_cast<T*>(p.dx) + r * p.lddx + c, o, n[j]);
            if (last) {
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    t[e] = fmaf(ws[j][e], Ag[j][e], wo[j][e] * Bg[j][e]);
                    A[j][e] = fmaf(m[j][e], Ag[j][e], A[j][e]);
                    B[j][e] = fmaf(m[j][e], Bg[j][e], B[j][e]);
                }
                if (p.dgate != nullptr) {
                    if (p.gate_bf16) st8<true>(static_cast<bf16_t*>(p.dgate) + g * p.C + c, t, n[j]);
                    else st8<true>(static_cast<float*>(p.dgate) + g * p.C + c, t, n[j]);
                }
            }
        }
        g = gn;
        k = kn;
    }
    if (p.partial != nullptr) leave_sums<LPR, NV>(p, lane, n, A, B);
}

// the row pass on tensors of type T; each type is compiled in a file of its own
template <typename T> void launch_rows(const BwdP& p, bool groups, unsigned blocks, hipStream_t st);

template <typename T> inline void launch_rows_as(const BwdP& p, bool groups, unsigned blocks, hipStream_t st) {
    const int z = sizeof(T);
    const bool rag = p.C % 8 != 0 || !vec_ok(p.dy, p.lddy, z) || !vec_ok(p.dx, p.lddx, z) || (p.x != nullptr && !vec_ok(p.x, p.ldx, z)) ||
                     (p.accum != nullptr && !vec_ok(p.accum, p.ldacc, z));
    const bool saved = p.x == nullptr;
    const dim3 grid(blocks);
#define CALL_RS(L, N, R, S) hipLaunchKernelGGL((rows_bwd_kernel<T, L, N, R, S>), grid, dim3(NT), 0, st, p)
#define CALL(L, N)                                                                                                         \
    do {                                                                                                                  \
        if (rag) { if (saved) CALL_RS(L, N, true, true); else CALL_RS(L, N, true, false); }                                \
        else { if (saved) CALL_RS(L, N, false, true); else CALL_RS(L, N, false, false); }                                  \
    } while (0)
#define CALL_GROUPS(L, N)                                                                                                  \
    do {                                                                                                                  \
        if (saved) hipLaunchKernelGGL((rows_bwd_groups_kernel<T, L, N, true>), grid, dim3(NT), 0, st, p);                 \
        else hipLaunchKernelGGL((rows_bwd_groups_kernel<T, L, N, false>), grid, dim3(NT), 0, st, p);                      \
    } while (0)
#define CALL_SAVED(L, N) do { if (rag) CALL_RS(L, N, true, true); else CALL_RS(L, N, false, true); } while (0)
    if (groups) DPIG_ROWS_DISPATCH2(p.C, CALL_GROUPS);
    else if (!p.three) DPIG_ROWS_DISPATCH2(p.C, CALL);
    else if constexpr (sizeof(T) == 2) DPIG_ROWS_DISPATCH3(p.C, CALL);
    else DPIG_ROWS_DISPATCH3(p.C, CALL_SAVED);
#undef CALL
#undef CALL_SAVED
#undef CALL_GROUPS
#undef CALL_RS
}

}  // namespace rows
}  // namespace dpig
