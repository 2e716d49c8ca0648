// Filter gradient of a fully connected layer (or 1x1 conv on its rows) whose saved input is an 8-bit checkpoint:
//   dw[c][k] = beta dw + sum_r (scale[c] q[r][c] + offset[c]) dy[r][k],   db[k] = beta_b db + sum_r dy[r][k],
// q the values the checkpoint stands for.  The affine part is pulled out of the sum, dw = scale[c] (q^T dy) + offset[c] (x) sum_r dy: the checkpoint of a
// norm's xh serves both the norm's gradient and this product, and the scale / offset cost one multiply-add per element of dw.
//
// Products on the bf16 matrix pipe, accumulation in fp32.  q is exact in bf16 (dpig_act8.h).  A bf16 dy is used as it is; an fp32 dy is cut
// into three bf16 terms (8 + 8 + 8 significand bits) whose products are exact in fp32, so the result is that of fp32 products -- at three of the bf16
// pipe's MFMAs, 16 / 3 times the fp32 pipe's rate.
//
// GEMM rows = c (128 per workgroup), columns = k (128), reduction = rows r (TR per tile).  Both operands lie reduction-major in HBM while an
// MFMA lane wants 8 consecutive r of one column: tiles are staged [r][128 columns] as bf16 (codes are decoded, fp32 gradients cut, on their
// way into LDS) and read with the transposing LDS read.  The rows are split over workgroups until the chip is full; partial sums are
// joined by a second launch in a fixed order.
#include "dpig_rows.h"

namespace dpig {
namespace wg8 {

using namespace rows;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int TM = 128, TN = 128, ROWB = 256;      // bytes of a staged row of 128 bf16 columns

struct P {
    const uint8_t *codes, *scales;
    const void* dy;
    float *dw, *db, *partial, *bias_partial;       // partial == nullptr: one split, written in place
    long lddy, nrows;
    int C, K, ld8, mtiles, ntiles, nsplit;
    long tiles_per_split;
    float beta, beta_b;
    bool want_db;
};

// granule g (8 columns) of staged row r lies at slot g ^ ((r & 3) << 2): the lanes a transposing read serves together cover all banks once
__device__ __forceinline__ int slot(int r, int g) { return r * ROWB + ((g ^ ((r & 3) << 2)) << 4); }

__device__ __forceinline__ uint4 to_bf16(const float (&v)[8]) {
    Raw8<bf16_t> r;
    pack(v, r);
    return r.a;
}

template <typename T, int F, bool RAG, int TR>
__global__ __launch_bounds__(256, 2) void wgrad8_kernel(const P p) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int TERMS = F32 ? 3 : 1;
    constexpr int TILE = TR * ROWB, STAGE = (1 + TERMS) * TILE;
    constexpr int NV = TR / 32;                    // staged rows per thread
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wrow = (wave >> 1) * 64, wcol = (wave & 1) * 64, l31 = lane & 31, half = lane >> 5;
    const int ntl = p.mtiles * p.ntiles;
    const int item = xcd_remap((int)blockIdx.x, ntl * p.nsplit);       // tile fastest: an XCD's L2 holds whole row ranges
    const int split = item / ntl, tile = item - split * ntl;
    const int mt = tile / p.ntiles, nt = tile - mt * p.ntiles;
    const int c0 = mt * TM, k0 = nt * TN;
    const long row0 = split * p.tiles_per_split * TR;
    const long row1 = min(row0 + p.tiles_per_split * TR, p.nrows);
    const bool do_bias = p.want_db && mt == 0;

    // staging roles: thread -> row tid / 8 (+ 32 i) of the tile, columns 16 (tid % 8) .. + 15 of both operands
    const int sr = tid >> 3, sc = (tid & 7) * 16;
    const bool xin = c0 + sc < p.ld8;
    const int nk = p.K - (k0 + sc);
    uint4 xq[NV];
    unsigned xs[NV];
    Raw8<T> yv[NV][2];
    float bias[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) bias[e] = 0.f;
    auto fetch = [&](long base) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const long r = base + sr + 32 * i;
            const bool in = r < row1;
            xq[i] = make_uint4(0, 0, 0, 0);
            xs[i] = 0;
            if (in && xin) {
                xq[i] = *reinterpret_cast<const uint4*>(p.codes + r * p.ld8 + c0 + sc);
                xs[i] = p.scales[r * (p.ld8 >> 5) + ((c0 + sc) >> 5)];
            }
            const T* y = static_cast<const T*>(p.dy) + r * p.lddy + k0 + sc;
#pragma unroll
            for (int h = 0; h < 2; ++h) yv[i][h] = ld8<RAG>(y + 8 * h, in ? nk - 8 * h : 0);
        }
    };
    auto stage = [&](int st) {
        char* xt = smem + st * STAGE;
        char* yt = xt + TILE;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int r = sr + 32 * i;
            const float s = act8::scale_value(xs[i]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
                act8::decode8<F>(h ? make_uint2(xq[i].z, xq[i].w) : make_uint2(xq[i].x, xq[i].y), s, v);
                *reinterpret_cast<uint4*>(xt + slot(r, (tid & 7) * 2 + h)) = to_bf16(v);
                const int o = slot(r, (tid & 7) * 2 + h);
                unpack(yv[i][h], v);
                if (do_bias) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) bias[8 * h + e] += v[e];
                }
#pragma unroll
                for (int t = 0; t < TERMS; ++t) {
                    if constexpr (!F32) {
                        *reinterpret_cast<uint4*>(yt + o) = yv[i][h].a;
                    } else {
                        const uint4 q = to_bf16(v);
                        *reinterpret_cast<uint4*>(yt + t * TILE + o) = q;
                        float w[8];
                        unpack(Raw8<bf16_t>{q}, w);
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] -= w[e];      // exact: the rest of a rounding
                    }
                }
            }
        }
    };

    f32x16 acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
    // transposing reads: 16 lanes serve a [4 rows][16 columns] block; lane q supplies row q / 4, columns 4 (q % 4) .. + 3, and receives the
    // 4 rows of column q.  Two of them make the 8 consecutive r of a 32x32x16 fragment.
    const int q = lane & 15, cg = (lane >> 4) & 1, pq = q >> 2;
    auto frag = [&](const char* t, int col, int ks) -> bf16x8 {
        const int cc = col + cg * 16 + (q & 3) * 4;
        const int r = ks * 16 + half * 8 + pq;
        const char* a = t + r * ROWB + (((cc >> 3) ^ (pq << 2)) << 4) + (cc & 7) * 2;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + 4 * ROWB));
        const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        return __builtin_bit_cast(bf16x8, v);
    };
    auto compute = [&](int st) {
        const char* xt = smem + st * STAGE;
#pragma unroll
        for (int ks = 0; ks < TR / 16; ++ks) {
            bf16x8 fa[2];
#pragma unroll
            for (int a = 0; a < 2; ++a) fa[a] = frag(xt, wrow + 32 * a, ks);
#pragma unroll
            for (int t = TERMS - 1; t >= 0; --t) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const bf16x8 fb = frag(xt + (1 + t) * TILE, wcol + 32 * b, ks);
#pragma unroll
                    for (int a = 0; a < 2; ++a) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[a], fb, acc[a][b], 0, 0, 0);
                }
            }
        }
    };
    fetch(row0);
    stage(0);
    __syncthreads();
    int st = 0;
    for (long base = row0; base < row1; base += TR) {
        const bool more = base + TR < row1;
        if (more) fetch(base + TR);
        compute(st);
        if (more) stage(st ^ 1);
        __syncthreads();
        st ^= 1;
    }

    // ---- result: accumulator register r of lane (half, l31) is row (r & 3) + 8 (r >> 2) + 4 half, column l31 of its 32x32 block ----------
    float* out = p.partial ? p.partial + (long)split * p.C * p.K : p.dw;
    const float beta = p.partial ? 0.f : p.beta;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int c = c0 + wrow + 32 * a + (r & 3) + 8 * (r >> 2) + 4 * half, k = k0 + wcol + 32 * b + l31;
                if (c < p.C && k < p.K) {
                    float* o = out + (long)c * p.K + k;
                    *o = beta != 0.f ? beta * *o + acc[a][b][r] : acc[a][b][r];
                }
            }
    if (do_bias) {                                    // workgroup-uniform; the staging buffers are free
        float(*bs)[TN] = reinterpret_cast<float(*)[TN]>(smem);       // [32 rows][128 columns]
#pragma unroll
        for (int e = 0; e < 16; ++e) bs[sr][sc + e] = bias[e];
        __syncthreads();
        if (tid < TN && k0 + tid < p.K) {
            float s = 0.f;
#pragma unroll 8
            for (int r = 0; r < 32; ++r) s += bs[r][tid];
            if (p.bias_partial) p.bias_partial[(long)split * p.K + k0 + tid] = s;
            else p.db[k0 + tid] = p.beta_b != 0.f ? p.beta_b * p.db[k0 + tid] + s : s;
        }
    }
}

struct JoinP {
    const float *partial, *bias_partial, *scale, *offset;
    float *dw, *db;
    int C, K, nsplit;
    float beta, beta_b;
};
// dw[c][k] = beta dw + scale[c] sum_s partial[s][c][k] + offset[c] sum_s bias[s][k]; the row after the last is db.  Splits are added in order.
__global__ __launch_bounds__(256) void wgrad8_join_kernel(const JoinP p) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    const int c = (int)(i / p.K), k = (int)(i - (long)c * p.K);
    if (c > p.C) return;
    float sb = 0.f;
    if (c == p.C || p.offset) {
#pragma unroll 8
        for (int s = 0; s < p.nsplit; ++s) sb += p.bias_partial[(long)s * p.K + k];
    }
    if (c == p.C) {
        if (p.db) p.db[k] = p.beta_b != 0.f ? p.beta_b * p.db[k] + sb : sb;
        return;
    }
    float sum = 0.f;
    const float* src = p.partial + (long)c * p.K + k;
    const long step = (long)p.C * p.K;
#pragma unroll 8
    for (int s = 0; s < p.nsplit; ++s) sum += src[s * step];
    if (p.scale) sum *= p.scale[c];
    if (p.offset) sum = fmaf(p.offset[c], sb, sum);
    float* o = p.dw + (long)c * p.K + k;
    *o = p.beta != 0.f ? p.beta * *o + sum : sum;
}

struct Plan { int mtiles, ntiles, nsplit, tr; long tiles_per_split; };
static Plan plan(int64_t nrows, int C, int K, bool f32) {
    Plan q;
    q.tr = f32 ? 32 : 64;
    q.mtiles = (C + TM - 1) / TM;
    q.ntiles = (K + TN - 1) / TN;
    const long tiles = (long)q.mtiles * q.ntiles, rt = (nrows + q.tr - 1) / q.tr;
    long want = (2L * kNumCU + tiles / 2) / tiles;
    if (want > (rt + 3) / 4) want = (rt + 3) / 4;      // at least four tiles of rows a split
    if (want < 1) want = 1;
    q.tiles_per_split = (rt + want - 1) / want;
    q.nsplit = (int)((rt + q.tiles_per_split - 1) / q.tiles_per_split);
    return q;
}
static bool joined(const Plan& q, bool affine) { return q.nsplit > 1 || affine; }
static size_t ws_bytes(const Plan& q, int C, int K, bool affine) {
    return joined(q, affine) ? (size_t)q.nsplit * K * (C + 1L) * sizeof(float) : 0;
}

}  // namespace wg8
}  // namespace dpig

using namespace dpig;

extern "C" size_t dpig_linear_wgrad8_workspace_bytes(int64_t nrows, int C, int K, int dy_bf16, int affine) {
    if (nrows <= 0 || C <= 0 || K <= 0) return 0;
    return wg8::ws_bytes(wg8::plan(nrows, C, K, !dy_bf16), C, K, affine != 0);
}

extern "C" int dpig_linear_wgrad8(const uint8_t* codes, const uint8_t* scales, int fmt, int64_t nrows, int C, const void* dy, int dy_bf16,
                                  int64_t lddy, int K, const float* scale, const float* offset, float* dw, float beta, float* db,
                                  float beta_b, void* ws, size_t ws_bytes, void* stream) {
    if (!codes || !scales || !dy || !dw) return fail(DPIG_EINVAL, "linear_wgrad8: null pointer");
    if (nrows <= 0 || C <= 0 || K <= 0 || nrows > (1L << 40) || C > (1 << 20) || K > (1 << 20)) return fail(DPIG_EINVAL, "linear_wgrad8: bad shape");
    if (fmt != DPIG_ACT8_E4M3 && fmt != DPIG_ACT8_INT8) return fail(DPIG_EINVAL, "linear_wgrad8: unknown checkpoint format");
    if (!aligned16(codes)) return fail(DPIG_EALIGN, "linear_wgrad8: checkpoint codes must be 16-byte aligned");
    if (lddy < K) return fail(DPIG_EINVAL, "linear_wgrad8: row stride below the column count");
    const wg8::Plan q = wg8::plan(nrows, C, K, !dy_bf16);
    const bool affine = scale || offset, join = wg8::joined(q, affine);
    if ((long)q.mtiles * q.ntiles * q.nsplit > 0x7fffffffL) return fail(DPIG_EINVAL, "linear_wgrad8: too many tiles");
    if (join && (!ws || ws_bytes < wg8::ws_bytes(q, C, K, affine))) return fail(DPIG_ENOMEM, "linear_wgrad8: workspace too small");
    hipStream_t st = static_cast<hipStream_t>(stream);
    wg8::P p = {};
    p.codes = codes; p.scales = scales; p.dy = dy; p.dw = dw; p.db = db; p.lddy = lddy; p.nrows = nrows; p.C = C; p.K = K;
    p.ld8 = act8::padded(C); p.mtiles = q.mtiles; p.ntiles = q.ntiles; p.nsplit = q.nsplit; p.tiles_per_split = q.tiles_per_split;
    p.beta = beta; p.beta_b = beta_b; p.want_db = db || offset;
    if (join) {
        p.partial = static_cast<float*>(ws);
        p.bias_partial = p.partial + (long)q.nsplit * C * K;
    }
    const dim3 grid((unsigned)(q.mtiles * q.ntiles * q.nsplit));
    const bool rag = K % 8 != 0 || !rows::vec_ok(dy, lddy, dy_bf16 ? 2 : 4);
#define GO(T, F, R, TR) hipLaunchKernelGGL((wg8::wgrad8_kernel<T, F, R, TR>), grid, dim3(256), 0, st, p)
#define BY_RAG(T, F, TR) do { if (rag) GO(T, F, true, TR); else GO(T, F, false, TR); } while (0)
#define BY_FMT(T, TR) do { if (fmt == DPIG_ACT8_E4M3) BY_RAG(T, DPIG_ACT8_E4M3, TR); else BY_RAG(T, DPIG_ACT8_INT8, TR); } while (0)
    if (dy_bf16) BY_FMT(rows::bf16_t, 64);
    else BY_FMT(float, 32);
#undef BY_FMT
#undef BY_RAG
#undef GO
    if (join) {
        const wg8::JoinP j = {p.partial, p.bias_partial, scale, offset, dw, db, C, K, q.nsplit, beta, beta_b};
        const long n = (long)K * (C + (db ? 1 : 0));
        hipLaunchKernelGGL(wg8::wgrad8_join_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, j);
    }
    return check_launch("linear_wgrad8");
}
