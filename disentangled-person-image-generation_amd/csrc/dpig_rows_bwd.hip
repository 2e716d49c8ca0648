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
    float rC;
};

template <int LPR, int NV> struct Codes8 { uint2 q[NV]; unsigned s[NV]; };

template <typename T, int LPR, int NV, bool RAG, bool SAVED, bool GROUPS>
__global__ __launch_bounds__(NT) void rows_bwd_kernel(const BwdP p) {
    constexpr int RPB = NT / LPR;
    __shared__ float red[2][4];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const long safe = safe_rows(p.nrows, p.C);
    const T *dy = static_cast<const T*>(p.dy), *x = static_cast<const T*>(p.x), *ac = static_cast<const T*>(p.accum);
    int n[NV];
    float w[NV][8], A[NV][8], B[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        n[j] = p.C - 8 * (lane + LPR * j);
#pragma unroll
        for (int e = 0; e < 8; ++e) { A[j][e] = 0.f; B[j][e] = 0.f; }
    }
    auto load_gate = [&](long g, int j, float (&m)[8]) {
        const int c = 8 * (lane + LPR * j);
        if (p.gate == nullptr) {
#pragma unroll
            for (int e = 0; e < 8; ++e) m[e] = 1.f;
        } else if (p.gate_bf16) ldp(static_cast<const bf16_t*>(p.gate) + g * p.C, c, p.C, 0.f, m);
        else ldp(static_cast<const float*>(p.gate) + g * p.C, c, p.C, 0.f, m);
    };
    auto load_w = [&](long g) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = 8 * (lane + LPR * j);
            float m[8], t[8];
            load_gate(g, j, m);
            ldp(p.scale, c, p.C, 1.f, w[j]);
            ldp(p.res, c, p.C, 1.f, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[j][e] *= m[e] * t[e];
        }
    };
    // rows [r, r1) in steps of `step`; groups form: the rows of group g, then of the group RPB further
    long r, r1, step, g = 0, g1 = 0;
    if (GROUPS) {
        g = blockIdx.x * p.chunk + sub;
        g1 = min((blockIdx.x + 1L) * p.chunk, p.ngroups);
        r = g * p.per; r1 = g < g1 ? r + p.per : r; step = 1;
    } else {
        const long grp = blockIdx.x / p.pieces, pc = blockIdx.x - grp * p.pieces;
        const long lo = grp * p.per + pc * p.chunk, hi = (grp + 1) * p.per;
        r = lo + sub; r1 = min(lo + p.chunk, hi); step = RPB;
        load_w(grp);
    }
    Raw8<T> nd[NV], nx[NV], na[NV];
    Codes8<LPR, NV> nc;
    float nmean = 0.f, nrstd = 0.f;
    auto fetch = [&](long row) {
        nrstd = p.rstd[row];
        if (!SAVED && p.layer) nmean = p.mean[row];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = 8 * (lane + LPR * j);
            nd[j] = ld8<RAG>(dy + row * p.lddy + c, n[j], row < safe);
            if (SAVED) {
                nc.q[j] = make_uint2(0, 0);
                nc.s[j] = 0;
                if (n[j] > 0) {
                    nc.q[j] = *reinterpret_cast<const uint2*>(p.codes + row * p.ld8 + c);
                    nc.s[j] = p.scales[row * (p.ld8 >> 5) + (c >> 5)];
                }
            } else {
                nx[j] = ld8<RAG>(x + row * p.ldx + c, n[j], row < safe);
            }
            if (!GROUPS && ac != nullptr) na[j] = ld8<RAG>(ac + row * p.ldacc + c, n[j], row < safe);
        }
    };
    float Ag[NV][8], Bg[NV][8];          // groups form: the present group's sums
    auto pass = [&]() {
        for (; r < r1; r += step) {
            float d[NV][8], xh[NV][8], a[NV][8];
            const float rstd = nrstd;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                unpack(nd[j], d[j]);
                if (RAG) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[j][e] = e < n[j] ? d[j][e] : 0.f;
                }
                if (SAVED) {
                    const float s = act8::scale_value(nc.s[j]);
                    if (p.fmt == DPIG_ACT8_E4M3) act8::decode8<DPIG_ACT8_E4M3>(nc.q[j], s, xh[j]);
                    else act8::decode8<DPIG_ACT8_INT8>(nc.q[j], s, xh[j]);
                    if (RAG || n[j] <= 0) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) xh[j][e] = e < n[j] ? xh[j][e] : 0.f;
                    }
                } else {
                    unpack(nx[j], xh[j]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) xh[j][e] = (RAG ? e < n[j] : n[j] > 0) ? (xh[j][e] - nmean) * rstd : 0.f;
                }
                if (!GROUPS && ac != nullptr) unpack(na[j], a[j]);
            }
            if (r + step < r1) fetch(r + step);
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (GROUPS) { Ag[j][e] = fmaf(d[j][e], xh[j][e], Ag[j][e]); Bg[j][e] += d[j][e]; }
                    else { A[j][e] = fmaf(d[j][e], xh[j][e], A[j][e]); B[j][e] += d[j][e]; }
                    const float gg = d[j][e] * w[j][e];
                    s[0] += gg;
                    s[1] = fmaf(gg, xh[j][e], s[1]);
                }
            row_sums<LPR, 2>(s, red);
            const float m1 = p.layer ? s[0] * p.rC : 0.f, m2 = s[1] * p.rC;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float o[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    o[e] = rstd * (fmaf(d[j][e], w[j][e], -m1) - xh[j][e] * m2);
                    if (!GROUPS && ac != nullptr) o[e] += a[j][e];
                }
                st8<RAG>(static_cast<T*>(p.dx) + r * p.lddx + 8 * (lane + LPR * j), o, n[j]);
            }
        }
    };
    if (!GROUPS) {
        if (r < r1) fetch(r);
        pass();
    } else {
        for (; g < g1; g += RPB) {
            r = g * p.per;
            r1 = r + p.per;
            fetch(r);
            load_w(g);
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) { Ag[j][e] = 0.f; Bg[j][e] = 0.f; }
            pass();
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = 8 * (lane + LPR * j);
                float m[8];
                load_gate(g, j, m);
                if (p.dgate != nullptr) {
                    float sc[8], of[8], rs[8], t[8];
                    ldp(p.scale, c, p.C, 1.f, sc);
                    ldp(p.offset, c, p.C, 0.f, of);
                    ldp(p.res, c, p.C, 1.f, rs);
#pragma unroll
                    for (int e = 0; e < 8; ++e) t[e] = rs[e] * fmaf(sc[e], Ag[j][e], of[e] * Bg[j][e]);
                    if (p.gate_bf16) st8<true>(static_cast<bf16_t*>(p.dgate) + g * p.C + c, t, n[j]);
                    else st8<true>(static_cast<float*>(p.dgate) + g * p.C + c, t, n[j]);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) { A[j][e] = fmaf(m[e], Ag[j][e], A[j][e]); B[j][e] = fmaf(m[e], Bg[j][e], B[j][e]); }
            }
        }
    }
    if (p.partial == nullptr) return;
    float* out = p.partial + (long)blockIdx.x * 2 * p.C;
    if constexpr (LPR == NT) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = 8 * (lane + LPR * j);
            st8<true>(out + c, A[j], n[j]);
            st8<true>(out + p.C + c, B[j], n[j]);
        }
    } else {
        // the RPB rows' lanes hold sums of the same channels: add them over the workgroup, in order
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

// ---- the partials' sums ---------------------------------------------------------------------------------------------------------------
constexpr int FC = 16, FL = 64, FW = FC * FL / 64;          // channels, summing lanes and waves of a workgroup (1024 threads)
constexpr int FG = 8;                                       // groups that rows_groups_kernel sums at a time
struct FinP {
    const float* partial;                // [n][2][C]
    float* partial2;                     // [gridDim.y][2][C]: gate-weighted sums over the groups of a workgroup (first launch of two)
    const float *scale, *offset, *res;
    const void* gate;
    void* dgate;
    float *dscale, *doffset, *dres;
    long n, ngroups, gpb;                // n: partials per group; gpb: groups of a workgroup
    int C, gate_bf16;
};
// sums over the four lanes of a wave that hold one channel; then thread (k, channel) adds the waves' values, always in the same order
template <int NG> __device__ __forceinline__ void fin_waves(float (&a)[NG], float (&b)[NG], float (*red)[FW][2][FC]) {
#pragma unroll
    for (int k = 0; k < NG; ++k) {
        a[k] += __shfl_xor(a[k], 16, 64);
        b[k] += __shfl_xor(b[k], 16, 64);
        a[k] += __shfl_xor(a[k], 32, 64);
        b[k] += __shfl_xor(b[k], 32, 64);
    }
    __syncthreads();                     // (red may still be read from the call before)
    if ((threadIdx.x & 63) < FC) {
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            red[k][threadIdx.x >> 6][0][threadIdx.x & 15] = a[k];
            red[k][threadIdx.x >> 6][1][threadIdx.x & 15] = b[k];
        }
    }
    __syncthreads();
}
__device__ __forceinline__ void fin_add(const float (*red)[2][FC], int cl, float* a, float* b) {
    *a = *b = 0.f;
#pragma unroll
    for (int w = 0; w < FW; ++w) { *a += red[w][0][cl]; *b += red[w][1][cl]; }
}
__device__ __forceinline__ void fin_outputs(const FinP& p, int c, float a, float b) {
    const float rs = p.res ? p.res[c] : 1.f;
    if (p.dscale) p.dscale[c] = rs * a;
    if (p.doffset) p.doffset[c] = rs * b;
    if (p.dres) p.dres[c] = (p.scale ? p.scale[c] : 1.f) * a + (p.offset ? p.offset[c] : 0.f) * b;
}
// pieces form with a gate: per group the sums over its pieces, dgate, and the gate-weighted sums over the groups of this workgroup.
// FG groups at a time, all their loads in flight together; thread (k, channel) closes group k.
__global__ __launch_bounds__(FC * FL) void rows_groups_kernel(const FinP p) {
    __shared__ float red[FG][FW][2][FC];
    const int cl = threadIdx.x % FC, ln = threadIdx.x / FC, c = blockIdx.x * FC + cl;
    const bool in = c < p.C;
    const float sc = in && p.scale ? p.scale[c] : 1.f, of = in && p.offset ? p.offset[c] : 0.f, rs = in && p.res ? p.res[c] : 1.f;
    const long g0 = blockIdx.y * p.gpb, g1 = min(g0 + p.gpb, p.ngroups);
    float wa = 0.f, wb = 0.f;
    auto close = [&](long g, float a, float b) {
        float m = 1.f;
        if (p.gate) m = p.gate_bf16 ? __uint_as_float((unsigned)static_cast<const bf16_t*>(p.gate)[g * p.C + c] << 16)
                                    : static_cast<const float*>(p.gate)[g * p.C + c];
        if (p.dgate) {
            const float t = rs * (sc * a + of * b);
            if (p.gate_bf16) static_cast<bf16_t*>(p.dgate)[g * p.C + c] = f2bf(t);
            else static_cast<float*>(p.dgate)[g * p.C + c] = t;
        }
        wa += m * a;
        wb += m * b;
    };
    if (p.n == 1) {                      // a lane takes whole groups
        for (long g = g0 + ln; g < g1; g += FL)
            if (in) close(g, p.partial[g * 2 * p.C + c], p.partial[(g * 2 + 1) * p.C + c]);
    } else {
        for (long g = g0; g < g1; g += FG) {
            float a[FG], b[FG];
#pragma unroll
            for (int k = 0; k < FG; ++k) {
                a[k] = b[k] = 0.f;
                if (in && g + k < g1)
                    for (long s = ln; s < p.n; s += FL) {
                        const float* q = p.partial + ((g + k) * p.n + s) * 2 * p.C + c;
                        a[k] += q[0];
                        b[k] += q[p.C];
                    }
            }
            fin_waves<FG>(a, b, red);
            if (in && ln < FG && g + ln < g1) {
                float ta, tb;
                fin_add(red[ln], cl, &ta, &tb);
                close(g + ln, ta, tb);
            }
        }
    }
    float a[1] = {wa}, b[1] = {wb};
    fin_waves<1>(a, b, red);
    if (!in || ln != 0) return;
    fin_add(red[0], cl, &wa, &wb);
    if (gridDim.y == 1) { fin_outputs(p, c, wa, wb); return; }
    p.partial2[(long)blockIdx.y * 2 * p.C + c] = wa;
    p.partial2[((long)blockIdx.y * 2 + 1) * p.C + c] = wb;
}
__global__ __launch_bounds__(FC * FL) void rows_final_kernel(const FinP p) {
    __shared__ float red[1][FW][2][FC];
    const int cl = threadIdx.x % FC, ln = threadIdx.x / FC, c = blockIdx.x * FC + cl;
    float a[1] = {0.f}, b[1] = {0.f};
    if (c < p.C)
#pragma unroll 4
        for (long s = ln; s < p.n; s += FL) { a[0] += p.partial[s * 2 * p.C + c]; b[0] += p.partial[(s * 2 + 1) * p.C + c]; }
    fin_waves<1>(a, b, red);
    if (c >= p.C || ln != 0) return;
    fin_add(red[0], cl, a, b);
    fin_outputs(p, c, a[0], b[0]);
}

// ---- plan ------------------------------------------------------------------------------------------------------------------------------
// Groups shorter than this run in the groups form: a piece of fewer rows would leave more partial sums than it reads.
constexpr long SHORT_GROUP = 16;
struct Plan {
    bool groups;
    long chunk, pieces, blocks, blocks2;          // blocks2 > 1: workgroups (y) of rows_groups_kernel, whose sums a second launch adds
};
// workgroups: one per set of rows taken at a time while that is at most one per CU, then about eight sets each, at most four per CU
static long want_blocks(long sets) {
    if (sets <= kNumCU) return sets;
    const long b = sets / 8;
    return b < kNumCU ? kNumCU : (b > 4 * kNumCU ? 4 * kNumCU : b);
}
static Plan plan(int64_t nrows, int C, bool gated, int64_t groups) {
    Plan q = {};
    const long rpb = NT / lanes_per_row(C), per = nrows / groups;
    auto up = [](long a, long b) { return (a + b - 1) / b; };
    if (gated && groups > 1 && per < SHORT_GROUP) {
        q.groups = true;
        q.chunk = up(up(groups, rpb), want_blocks(up(groups, rpb))) * rpb;
        q.blocks = up(groups, q.chunk);
        q.pieces = 1;
        q.blocks2 = 1;
        return q;
    }
    const long sets = up(per, rpb);
    long pieces = want_blocks(sets * groups) / groups;
    pieces = pieces < 1 ? 1 : (pieces > sets ? sets : pieces);
    q.chunk = up(sets, pieces) * rpb;
    q.pieces = up(per, q.chunk);
    q.blocks = q.pieces * groups;
    q.blocks2 = groups <= 4 * FG ? 1 : (groups / (2 * FG) < 256 ? groups / (2 * FG) : 256);
    return q;
}
static size_t ws_bytes(const Plan& q, int C) {
    return (size_t)(q.blocks + (!q.groups && q.blocks2 > 1 ? q.blocks2 : 0)) * 2 * C * sizeof(float);
}

template <typename T> static void launch_rows(const BwdP& p, const Plan& q, hipStream_t st) {
    const int z = sizeof(T);
    const bool rag = p.C % 8 != 0 || !vec_ok(p.dy, p.lddy, z) || !vec_ok(p.dx, p.lddx, z) || (p.x != nullptr && !vec_ok(p.x, p.ldx, z)) ||
                     (p.accum != nullptr && !vec_ok(p.accum, p.ldacc, z));
    const bool saved = p.x == nullptr;
    const dim3 grid((unsigned)q.blocks);
#define CALL_RSG(L, N, R, S, G) hipLaunchKernelGGL((rows_bwd_kernel<T, L, N, R, S, G>), grid, dim3(NT), 0, st, p)
#define CALL_RS(L, N, R, S) do { if (q.groups) CALL_RSG(L, N, R, S, true); else CALL_RSG(L, N, R, S, false); } while (0)
#define CALL(L, N)                                                                                                         \
    do {                                                                                                                  \
        if (rag) { if (saved) CALL_RS(L, N, true, true); else CALL_RS(L, N, true, false); }                                \
        else { if (saved) CALL_RS(L, N, false, true); else CALL_RS(L, N, false, false); }                                  \
    } while (0)
    DPIG_ROWS_DISPATCH(p.C, CALL);
#undef CALL
#undef CALL_RS
#undef CALL_RSG
}
static void launch_sums(FinP f, const Plan& q, int64_t groups, hipStream_t st) {
    const unsigned gx = (unsigned)((f.C + FC - 1) / FC);
    const float* first = f.partial;
    if (!q.groups && (groups > 1 || f.gate)) {
        f.n = q.pieces;
        f.ngroups = groups;
        f.gpb = (groups + q.blocks2 - 1) / q.blocks2;
        const unsigned gy = (unsigned)((groups + f.gpb - 1) / f.gpb);
        f.partial2 = const_cast<float*>(first) + q.blocks * 2 * f.C;
        hipLaunchKernelGGL(rows_groups_kernel, dim3(gx, gy), dim3(FC * FL), 0, st, f);
        if (gy == 1) return;
        f.partial = f.partial2;
        f.n = gy;
    } else {
        f.n = q.blocks;
    }
    if (f.dscale || f.doffset || f.dres) hipLaunchKernelGGL(rows_final_kernel, dim3(gx), dim3(FC * FL), 0, st, f);
}

static int check_bwd(const char* who, int64_t nrows, int C, int kind, const void* dy, const void* x, const uint8_t* codes, const uint8_t* scales,
                     int fmt, const float* mean, const float* rstd, const void* dx, int64_t lddy, int64_t ldx, int64_t lddx) {
    if (nrows <= 0 || nrows > (1L << 40)) return fail(DPIG_EINVAL, "%s: bad row count", who);
    if (C <= 0 || C > C_MAX) return fail(DPIG_EINVAL, "%s: channels must be 1 .. %d", who, C_MAX);
    if (kind != DPIG_NORM_LAYER && kind != DPIG_NORM_RMS) return fail(DPIG_EINVAL, "%s: unknown kind of norm", who);
    if (!dy || !dx || !rstd) return fail(DPIG_EINVAL, "%s: null pointer", who);
    if ((x != nullptr) == (codes != nullptr)) return fail(DPIG_EINVAL, "%s: exactly one of the saved input and its checkpoint is needed", who);
    if (x && kind == DPIG_NORM_LAYER && !mean) return fail(DPIG_EINVAL, "%s: null pointer", who);
    if (codes && !scales) return fail(DPIG_EINVAL, "%s: a checkpoint needs codes and scales", who);
    if (codes && fmt != DPIG_ACT8_E4M3 && fmt != DPIG_ACT8_INT8) return fail(DPIG_EINVAL, "%s: unknown checkpoint format", who);
    if (codes && !aligned16(codes)) return fail(DPIG_EALIGN, "%s: checkpoint codes must be 16-byte aligned", who);
    if (lddy < C || lddx < C || (x && ldx < C)) return fail(DPIG_EINVAL, "%s: row stride below the channel count", who);
    return DPIG_OK;
}

}  // namespace rows
}  // namespace dpig

using namespace dpig;

extern "C" size_t dpig_rownorm_bwd_workspace_bytes(int64_t nrows, int C) {
    if (nrows <= 0 || C <= 0 || C > rows::C_MAX) return 0;
    return rows::ws_bytes(rows::plan(nrows, C, false, 1), C);
}

extern "C" int dpig_rownorm_bwd(const void* dy, int is_bf16, int64_t lddy, const void* x, int64_t ldx, int fmt, const uint8_t* codes,
                                const uint8_t* scales, int64_t nrows, int C, int kind, const float* scale, const float* mean,
                                const float* rstd, const void* accum, int64_t ldacc, void* dx, int64_t lddx, float* dscale,
                                float* doffset, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = rows::check_bwd("rownorm_bwd", nrows, C, kind, dy, x, codes, scales, fmt, mean, rstd, dx, lddy, ldx, lddx)) return rc;
    if (accum && ldacc < C) return fail(DPIG_EINVAL, "rownorm_bwd: row stride below the channel count");
    const bool params = dscale || doffset;
    const rows::Plan q = rows::plan(nrows, C, false, 1);
    if (params && (!ws || ws_bytes < rows::ws_bytes(q, C))) return fail(DPIG_ENOMEM, "rownorm_bwd: workspace too small");
    hipStream_t st = static_cast<hipStream_t>(stream);
    rows::BwdP p = {};
    p.dy = dy; p.x = x; p.accum = accum; p.dx = dx; p.codes = codes; p.scales = scales; p.mean = mean; p.rstd = rstd; p.scale = scale;
    p.partial = params ? static_cast<float*>(ws) : nullptr;
    p.lddy = lddy; p.ldx = ldx; p.ldacc = ldacc; p.lddx = lddx; p.nrows = nrows; p.chunk = q.chunk; p.per = nrows; p.ngroups = 1;
    p.C = C; p.layer = kind == DPIG_NORM_LAYER; p.fmt = fmt; p.ld8 = act8::padded(C); p.pieces = (int)q.pieces; p.rC = 1.0f / (float)C;
    if (is_bf16) rows::launch_rows<rows::bf16_t>(p, q, st);
    else rows::launch_rows<float>(p, q, st);
    if (params) {
        rows::FinP f = {};
        f.partial = p.partial; f.dscale = dscale; f.doffset = doffset; f.C = C;
        rows::launch_sums(f, q, 1, st);
    }
    return check_launch("rownorm_bwd");
}

extern "C" size_t dpig_gated_residual_bwd_workspace_bytes(int64_t nrows, int C, int64_t groups) {
    if (nrows <= 0 || C <= 0 || C > rows::C_MAX || groups < 0 || (groups > 0 && nrows % groups != 0)) return 0;
    return rows::ws_bytes(rows::plan(nrows, C, groups > 0, groups > 0 ? groups : 1), C);
}

extern "C" int dpig_gated_residual_bwd(const void* dout, int is_bf16, int64_t lddo, const void* f, int64_t ldf, int fmt, const uint8_t* codes,
                                       const uint8_t* scales, int64_t nrows, int C, int kind, const float* scale, const float* offset,
                                       const void* gate, int gate_bf16, int64_t groups, const float* res_scale, const float* mean,
                                       const float* rstd, void* df, int64_t lddf, float* dscale, float* doffset, void* dgate,
                                       float* dres_scale, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = rows::check_bwd("gated_residual_bwd", nrows, C, kind, dout, f, codes, scales, fmt, mean, rstd, df, lddo, ldf, lddf)) return rc;
    if (gate && (groups <= 0 || nrows % groups != 0)) return fail(DPIG_EINVAL, "gated_residual_bwd: rows must be a multiple of the gate's groups");
    if (dgate && !gate) return fail(DPIG_EINVAL, "gated_residual_bwd: a gate gradient without a gate");
    if (!gate) groups = 1;
    const bool sums = dscale || doffset || dres_scale, params = sums || dgate;
    const rows::Plan q = rows::plan(nrows, C, gate != nullptr, groups);
    if (q.blocks > 0x7fffffffL) return fail(DPIG_EINVAL, "gated_residual_bwd: too many gate groups");
    if (params && (!ws || ws_bytes < rows::ws_bytes(q, C))) return fail(DPIG_ENOMEM, "gated_residual_bwd: workspace too small");
    hipStream_t st = static_cast<hipStream_t>(stream);
    rows::BwdP p = {};
    p.dy = dout; p.x = f; p.dx = df; p.codes = codes; p.scales = scales; p.mean = mean; p.rstd = rstd; p.scale = scale; p.offset = offset;
    p.res = res_scale; p.gate = gate; p.dgate = q.groups ? dgate : nullptr;
    p.partial = (q.groups ? sums : params) ? static_cast<float*>(ws) : nullptr;
    p.lddy = lddo; p.ldx = ldf; p.lddx = lddf; p.nrows = nrows; p.chunk = q.chunk; p.per = nrows / groups; p.ngroups = groups;
    p.C = C; p.layer = kind == DPIG_NORM_LAYER; p.fmt = fmt; p.ld8 = act8::padded(C); p.gate_bf16 = gate_bf16; p.pieces = (int)q.pieces;
    p.rC = 1.0f / (float)C;
    if (is_bf16) rows::launch_rows<rows::bf16_t>(p, q, st);
    else rows::launch_rows<float>(p, q, st);
    if (p.partial) {
        rows::FinP z = {};
        z.partial = p.partial; z.scale = scale; z.offset = offset; z.res = res_scale; z.gate = gate; z.gate_bf16 = gate_bf16;
        z.dgate = q.groups ? nullptr : dgate;
        z.dscale = dscale; z.doffset = doffset; z.dres = dres_scale; z.C = C;
        rows::launch_sums(z, q, groups, st);
    }
    return check_launch("gated_residual_bwd");
}
