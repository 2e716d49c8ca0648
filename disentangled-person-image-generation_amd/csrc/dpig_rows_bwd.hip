// The row pass of the norms' gradients on fp32 tensors (dpig_rows_bwd.h), the sums behind it, and the C entries of both types.
#include "dpig_rows_bwd.h"

template <> void dpig::rows::launch_rows<float>(const BwdP& p, bool groups, unsigned blocks, hipStream_t st) {
    launch_rows_as<float>(p, groups, blocks, st);
}

namespace dpig {
namespace rows {

template <> void launch_rows<bf16_t>(const BwdP& p, bool groups, unsigned blocks, hipStream_t st);      // dpig_rows_bwd_bf16.hip

// ---- the partials' sums ---------------------------------------------------------------------------------------------------------------
constexpr int FC = 16, FL = 64, FW = FC * FL / 64;          // channels, summing lanes and waves of a workgroup (1024 threads)
struct FinP {
    const float* partial;                // [n][2][C]
    float* partial2;                     // [gridDim.y][2][C]: gate-weighted sums over the groups of a workgroup (first launch of two)
    const float *scale, *offset, *res;
    const void* gate;
    void* dgate;
    float *dscale, *doffset, *dres;
    long n, ngroups, gpb;                // n: partials per group; gpb: groups of a workgroup
    int C, gate_bf16, wpg;               // wpg: waves that share a group
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
// a channel's parameters, asked for before the sums they are needed after
struct FinChan {
    float sc, of, rs;
    __device__ __forceinline__ FinChan(const FinP& p, int c, bool in)
        : sc(in && p.scale ? p.scale[c] : 1.f), of(in && p.offset ? p.offset[c] : 0.f), rs(in && p.res ? p.res[c] : 1.f) {}
    __device__ __forceinline__ void outputs(const FinP& p, int c, float a, float b) const {
        if (p.dscale) p.dscale[c] = rs * a;
        if (p.doffset) p.doffset[c] = rs * b;
        if (p.dres) p.dres[c] = sc * a + of * b;
    }
};
// Sums of n pairs (A, B) `step` apart, in order, N of them on their way at a time: all loads of a batch are issued before the first is waited for (behind
// the n-th the last one is read again and left out).  Left to itself the compiler waits for each pair: 7.1 us instead of 5.5 for 8 groups of 64.
template <int N> __device__ __forceinline__ void fin_batch(const float* p, int C, long step, int n, float* a, float* b) {
    float va[N], vb[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const float* q = p + min(u, n - 1) * step;
        va[u] = q[0];
        vb[u] = q[C];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < N; ++u) {
        *a = u < n ? *a + va[u] : *a;
        *b = u < n ? *b + vb[u] : *b;
    }
}
__device__ __forceinline__ void fin_sums(const float* p, int C, long step, int n, float* a, float* b) {
    for (; n > 2; n -= 8, p += 8 * step) fin_batch<8>(p, C, step, n, a, b);
    if (n > 0) fin_batch<2>(p, C, step, n, a, b);
}
// pieces form with a gate: per group the sums over its pieces, dgate, and the gate-weighted sums over the groups of this workgroup.  `wpg` waves take a
// group, four lanes a channel each, and sixteen / wpg groups are summed together with all their loads in flight; where every group is one
// piece, a lane takes one.
__global__ __launch_bounds__(FC * FL) void rows_groups_kernel(const FinP p) {
    __shared__ float red[1][FW][2][FC];
    const int cl = threadIdx.x % FC, ln = threadIdx.x / FC, c = blockIdx.x * FC + cl;
    const bool in = c < p.C;
    const FinChan ch(p, c, in);
    const long g0 = blockIdx.y * p.gpb, g1 = min(g0 + p.gpb, p.ngroups);
    float wa = 0.f, wb = 0.f;
    auto gate_of = [&](long g) -> float {
        if (!p.gate || !in) return 1.f;
        return p.gate_bf16 ? __uint_as_float((unsigned)static_cast<const bf16_t*>(p.gate)[g * p.C + c] << 16)
                           : static_cast<const float*>(p.gate)[g * p.C + c];
    };
    auto close = [&](long g, float m, float a, float b) {
        if (p.dgate) {
            const float t = ch.rs * (ch.sc * a + ch.of * b);
            if (p.gate_bf16) static_cast<bf16_t*>(p.dgate)[g * p.C + c] = f2bf(t);
            else static_cast<float*>(p.dgate)[g * p.C + c] = t;
        }
        wa += m * a;
        wb += m * b;
    };
    if (p.n == 1) {
        for (long g = g0 + ln; g < g1; g += FL)
            if (in) close(g, gate_of(g), p.partial[g * 2 * p.C + c], p.partial[(g * 2 + 1) * p.C + c]);
    } else {
        const int wave = threadIdx.x >> 6, slots = FW / p.wpg, part = (wave % p.wpg) * 4 + (ln & 3);
        for (long gb = g0; gb < g1; gb += slots) {
            const bool closer = in && ln < slots && gb + ln < g1;
            const float m = closer ? gate_of(gb + ln) : 1.f;
            const long g = gb + wave / p.wpg;
            float a[1] = {0.f}, b[1] = {0.f};
            if (in && g < g1) {
                const int each = 4 * p.wpg;
                fin_sums(p.partial + (g * p.n + part) * 2 * p.C + c, p.C, 2L * each * p.C, ((int)p.n - part + each - 1) / each, &a[0], &b[0]);
            }
            fin_waves<1>(a, b, red);
            if (closer) {
                float ta = 0.f, tb = 0.f;
                for (int k = 0; k < p.wpg; ++k) { ta += red[0][ln * p.wpg + k][0][cl]; tb += red[0][ln * p.wpg + k][1][cl]; }
                close(gb + ln, m, ta, tb);
            }
        }
    }
    float a[1] = {wa}, b[1] = {wb};
    fin_waves<1>(a, b, red);
    if (!in || ln != 0) return;
    fin_add(red[0], cl, &wa, &wb);
    if (gridDim.y == 1) { ch.outputs(p, c, wa, wb); return; }
    p.partial2[(long)blockIdx.y * 2 * p.C + c] = wa;
    p.partial2[((long)blockIdx.y * 2 + 1) * p.C + c] = wb;
}
__global__ __launch_bounds__(FC * FL) void rows_final_kernel(const FinP p) {
    __shared__ float red[1][FW][2][FC];
    const int cl = threadIdx.x % FC, ln = threadIdx.x / FC, c = blockIdx.x * FC + cl;
    const FinChan ch(p, c, c < p.C);
    float a[1] = {0.f}, b[1] = {0.f};
    if (c < p.C) fin_sums(p.partial + 2L * ln * p.C + c, p.C, 2L * FL * p.C, (int)((p.n - ln + FL - 1) / FL), &a[0], &b[0]);
    fin_waves<1>(a, b, red);
    if (c >= p.C || ln != 0) return;
    fin_add(red[0], cl, a, b);
    ch.outputs(p, c, a[0], b[0]);
}

// ---- plan ------------------------------------------------------------------------------------------------------------------------------
// Groups shorter than this run in the groups form: a piece of fewer rows would leave more partial sums than it reads.
constexpr long SHORT_GROUP = 16;
struct Plan {
    bool groups, three;
    long chunk, pieces, blocks, blocks2;          // blocks2 > 1: workgroups (y) of rows_groups_kernel, whose sums a second launch adds
};
// workgroups: one per set of rows taken at a time while that is at most one per CU, then about eight sets each, at most two per CU: more of them
// leave more partial sums than their loads in flight are worth (131072 x 256 bf16: 55.5 us with two per CU, 58.2 with four, 68.3 with one)
static long want_blocks(long sets) {
    if (sets <= kNumCU) return sets;
    const long b = sets / 8;
    return b < kNumCU ? kNumCU : (b > 2 * kNumCU ? 2 * kNumCU : b);
}
// (three: the tensors' type, or a checkpoint, allows three vectors a lane)
static Plan plan(int64_t nrows, int C, bool gated, int64_t groups, bool three) {
    Plan q = {};
    const long per = nrows / groups;
    q.three = three && three_vectors(nrows, C);
    long rpb = NT / (q.three ? lanes_per_row3(C) : lanes_per_row2(C));
    auto up = [](long a, long b) { return (a + b - 1) / b; };
    if (gated && groups > 1 && per < SHORT_GROUP) {
        q.groups = true;
        rpb = NT / lanes_per_row2(C);
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
    // (where a group is one piece, a lane takes a group: sixteen times as many of them keep a workgroup of the sums busy)
    q.blocks2 = groups <= 2 * FW ? 1 : q.pieces == 1 ? up(groups, FL) : groups / FW;
    if (q.blocks2 > 256) q.blocks2 = 256;
    return q;
}
static size_t ws_bytes(const Plan& q, int C) {
    return (size_t)(q.blocks + (!q.groups && q.blocks2 > 1 ? q.blocks2 : 0)) * 2 * C * sizeof(float);
}
// what is enough for either layout: the queries know neither the tensors' type nor whether they come from a checkpoint
static size_t ws_bytes(int64_t nrows, int C, bool gated, int64_t groups) {
    const size_t a = ws_bytes(plan(nrows, C, gated, groups, false), C), b = ws_bytes(plan(nrows, C, gated, groups, true), C);
    return a > b ? a : b;
}

static void launch_sums(FinP f, const Plan& q, int64_t groups, hipStream_t st) {
    const unsigned gx = (unsigned)((f.C + FC - 1) / FC);
    const float* first = f.partial;
    if (!q.groups && (groups > 1 || f.gate)) {
        f.n = q.pieces;
        f.ngroups = groups;
        f.gpb = (groups + q.blocks2 - 1) / q.blocks2;
        const unsigned gy = (unsigned)((groups + f.gpb - 1) / f.gpb);
        f.wpg = f.gpb <= 1 ? 16 : f.gpb <= 2 ? 8 : f.gpb <= 4 ? 4 : f.gpb <= 8 ? 2 : 1;
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
    return rows::ws_bytes(nrows, C, false, 1);
}

extern "C" int dpig_rownorm_bwd(const void* dy, int is_bf16, int64_t lddy, const void* x, int64_t ldx, int fmt, const uint8_t* codes,
                                const uint8_t* scales, int64_t nrows, int C, int kind, const float* scale, const float* mean,
                                const float* rstd, const void* accum, int64_t ldacc, void* dx, int64_t lddx, float* dscale,
                                float* doffset, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = rows::check_bwd("rownorm_bwd", nrows, C, kind, dy, x, codes, scales, fmt, mean, rstd, dx, lddy, ldx, lddx)) return rc;
    if (accum && ldacc < C) return fail(DPIG_EINVAL, "rownorm_bwd: row stride below the channel count");
    const bool params = dscale || doffset;
    const rows::Plan q = rows::plan(nrows, C, false, 1, is_bf16 || codes);
    if (params && (!ws || ws_bytes < rows::ws_bytes(q, C))) return fail(DPIG_ENOMEM, "rownorm_bwd: workspace too small");
    hipStream_t st = static_cast<hipStream_t>(stream);
    rows::BwdP p = {};
    p.dy = dy; p.x = x; p.accum = accum; p.dx = dx; p.codes = codes; p.scales = scales; p.mean = mean; p.rstd = rstd; p.scale = scale;
    p.partial = params ? static_cast<float*>(ws) : nullptr;
    p.lddy = lddy; p.ldx = ldx; p.ldacc = ldacc; p.lddx = lddx; p.nrows = nrows; p.chunk = q.chunk; p.per = nrows; p.ngroups = 1;
    p.C = C; p.layer = kind == DPIG_NORM_LAYER; p.fmt = fmt; p.ld8 = act8::padded(C); p.pieces = (int)q.pieces; p.three = q.three; p.rC = 1.0f / (float)C;
    if (is_bf16) rows::launch_rows<rows::bf16_t>(p, q.groups, (unsigned)q.blocks, st);
    else rows::launch_rows<float>(p, q.groups, (unsigned)q.blocks, st);
    if (params) {
        rows::FinP f = {};
        f.partial = p.partial; f.dscale = dscale; f.doffset = doffset; f.C = C;
        rows::launch_sums(f, q, 1, st);
    }
    return check_launch("rownorm_bwd");
}

extern "C" size_t dpig_gated_residual_bwd_workspace_bytes(int64_t nrows, int C, int64_t groups) {
    if (nrows <= 0 || C <= 0 || C > rows::C_MAX || groups < 0 || (groups > 0 && nrows % groups != 0)) return 0;
    return rows::ws_bytes(nrows, C, groups > 0, groups > 0 ? groups : 1);
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
    const rows::Plan q = rows::plan(nrows, C, gate != nullptr, groups, is_bf16 || codes);
    if (q.blocks > 0x7fffffffL) return fail(DPIG_EINVAL, "gated_residual_bwd: too many gate groups");
    if (params && (!ws || ws_bytes < rows::ws_bytes(q, C))) return fail(DPIG_ENOMEM, "gated_residual_bwd: workspace too small");
    hipStream_t st = static_cast<hipStream_t>(stream);
    rows::BwdP p = {};
    p.dy = dout; p.x = f; p.dx = df; p.codes = codes; p.scales = scales; p.mean = mean; p.rstd = rstd; p.scale = scale; p.offset = offset;
    p.res = res_scale; p.gate = gate; p.dgate = q.groups ? dgate : nullptr;
    p.partial = (q.groups ? sums : params) ? static_cast<float*>(ws) : nullptr;
    p.lddy = lddo; p.ldx = ldf; p.lddx = lddf; p.nrows = nrows; p.chunk = q.chunk; p.per = nrows / groups; p.ngroups = groups;
    p.C = C; p.layer = kind == DPIG_NORM_LAYER; p.fmt = fmt; p.ld8 = act8::padded(C); p.gate_bf16 = gate_bf16; p.pieces = (int)q.pieces;
    p.three = q.three;
    p.rC = 1.0f / (float)C;
    if (is_bf16) rows::launch_rows<rows::bf16_t>(p, q.groups, (unsigned)q.blocks, st);
    else rows::launch_rows<float>(p, q.groups, (unsigned)q.blocks, st);
    if (p.partial) {
        rows::FinP z = {};
        z.partial = p.partial; z.scale = scale; z.offset = offset; z.res = res_scale; z.gate = gate; z.gate_bf16 = gate_bf16;
        z.dgate = q.groups ? nullptr : dgate;
        z.dscale = dscale; z.doffset = doffset; z.dres = dres_scale; z.C = C;
        rows::launch_sums(z, q, groups, st);
    }
    return check_launch("gated_residual_bwd");
}
