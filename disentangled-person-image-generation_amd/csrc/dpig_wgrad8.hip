// Filter gradient of a fully connected layer (or 1x1 conv on its rows) whose saved input is an 8-bit checkpoint:
//   dw[c][k] = beta dw + sum_r (scale[c] q[r][c] + offset[c]) dy[r][k],   db[k] = beta_b db + sum_r dy[r][k],
// q the values the checkpoint stands for.  The affine part is pulled out of the sum, dw = scale[c] (q^T dy) + offset[c] (x) sum_r dy: the checkpoint of a
// norm's xh serves both the norm's gradient and this product, and the scale / offset cost one multiply-add per element of dw.
//
// Products on the bf16 matrix pipe, accumulation in fp32.  q is exact in bf16 (dpig_act8.h).  A bf16 dy is used as it is; an fp32 dy is cut
// into three bf16 terms (8 + 8 + 8 significand bits, each the rest's leading ones) whose products are exact in fp32, so the result is that of fp32
// products -- at three of the bf16 pipe's MFMAs, 16 / 3 times the fp32 pipe's rate.  (An infinite dy leaves a rest that is not a number: NaN.)
//
// GEMM rows = c (128 or 256 per workgroup), columns = k (128 or 256), reduction = rows r (TR per tile).  Both operands lie reduction-major in HBM while
// an MFMA lane wants 8 consecutive r of one column: tiles are staged [r][columns] as bf16 (codes are decoded, fp32 gradients cut, on their
// way into LDS) and read with the transposing LDS read.  The rows are split over workgroups until the chip is full; partial sums are
// joined by a second launch in a fixed order.
//
// Measured (averages under the profiler), product + join: bf16 dy 131072 x 512 x 512 80 .. 94 + 7.8 us, as the chip holds its clock over a run of them
// (68.7 GFLOP: 730 .. 860 TFLOP/s in the product; a library product of two bf16 operands of that shape takes 361 us), 131072 x 768 x 768 168 + 12.2 (920
// TFLOP/s), 32768 x 512 x 512 30.8 + 4.5, 2048 x 512 x 512 11.4 + 4.0, 64 x 512 x 512 5.7 and no join; fp32 dy 131072 x 128 x 128 22.4 + 5.8, 32768 x 512 x 512
// 48.9 + 6.8 (351 TFLOP/s of fp32 products), 20011 x 250 x 390 25.2 .. 27.5 + 5.8, 64 x 512 x 512 6.2.
// Of the large product the matrix instructions and barriers alone take 54 us, without the loads it is 69, without decoding and staging 63: the
// matrix pipe, the LDS port and the loads' waits overlap, but not fully.  Asking L2 for tiles ahead of the loads, or for three and six tiles ahead
// instead of two, changed nothing.  (The steps of the loop as one expression, one exit behind each: 79.4 us; with a branch of its own each, 82.3.)
#include "dpig_rows.h"
#include <type_traits>
#include <utility>

namespace dpig {
namespace wg8 {

using namespace rows;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

struct P {
    const uint8_t *codes, *scales;
    const void* dy;
    float *dw, *db, *partial, *bias_partial;       // partial == nullptr: one split, written in place
    long lddy;
    int nrows, C, K, ld8, mtiles, ntiles, nsplit, rows_per_split;
    float beta, beta_b;
    bool want_db;
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// eight codes -> bf16, exact.  E4M3 has one instruction for two values and their scale; `q` must be the NaN code throughout where the group was not finite
template <int F> __device__ __forceinline__ uint4 decode_bf16(unsigned q0, unsigned q1, float s) {
    uint4 r;
    if constexpr (F == DPIG_ACT8_E4M3) {
        r.x = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q0, s, false));
        r.y = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q0, s, true));
        r.z = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q1, s, false));
        r.w = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q1, s, true));
    } else {
        float v[8];
        q0 ^= 0x80808080u;                              // to two's complement
        q1 ^= 0x80808080u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = (float)(signed char)(q0 >> (8 * e)) * s;
            v[4 + e] = (float)(signed char)(q1 >> (8 * e)) * s;
        }
        Raw8<bf16_t> t;
        pack(v, t);
        r = t.a;
    }
    return r;
}
// The order of a multiplying phase: behind each of its NM matrix instructions (32 cycles of the matrix pipe) some vector instructions and a share of its
// NW LDS writes and NL loads
template <int I, int NM, int NW, int NL> __device__ __forceinline__ void weave() {
    if constexpr (I < NM) {
        constexpr int w = NW * (I + 1) / NM - NW * I / NM, l = NL * (I + 1) / NM - NL * I / NM;
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if constexpr (NW > 0) __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
        if constexpr (w > 0) __builtin_amdgcn_sched_group_barrier(0x200, w, 0);
        if constexpr (l > 0) __builtin_amdgcn_sched_group_barrier(0x020, l, 0);
        weave<I + 1, NM, NW, NL>();
    }
}

// step(0) && step(1) && ...
template <typename S, int... I> __device__ __forceinline__ bool every(S& step, std::integer_sequence<int, I...>) {
    return (step(std::integral_constant<int, I>()) && ...);
}

// Eight waves, WM x 8 / WM, each with MA x NB blocks of 32 x 32; TR rows per tile.
//
// A SIMD holds two waves, one of each half of the workgroup, and the halves run half a tile apart: while one multiplies (its fragments in registers, the
// matrix pipe to itself), the other reads the fragments of its next tile.  Two barriers a tile keep them apart.  In half-steps h the first half reads tile
// t at h = 2 t and multiplies at 2 t + 1, the second at 2 t + 1 and 2 t + 2.  Where a wave decodes its share of a later tile into LDS:
//   LATE  between the matrix instructions of its multiplying phase (their 32 cycles leave room).  Tile t + 2 is written at 2 t + 1 and 2 t + 2 and read
//         from 2 t + 4 on; its stage held tile t - 1, last read at 2 t - 1: three stages.  (65536 x 512 x 512: 46 us, 49 the other way.)
//   else  behind its reads.  Tile t + 1 is written at 2 t and 2 t + 1 and read from 2 t + 2 on; its stage held tile t - 1: two stages.  The
//         256 x 256 tile's accumulators leave no registers for more (262144 x 512 x 512: 157 us; 177 with the decoding late, which spills).
template <typename T, int F, bool RAG, int MA, int NB, int WM, int TR>
__global__ __launch_bounds__(512, 2) void wgrad8_kernel(const P p) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int TERMS = F32 ? 3 : 1, WN = 8 / WM, TM = 32 * MA * WM, TN = 32 * NB * WN;
    constexpr int XROW = 2 * TM, YROW = 2 * TN;                         // bytes of a staged row of bf16 columns
    constexpr int XTILE = TR * XROW, YTILE = TR * YROW, STAGE = XTILE + TERMS * YTILE;
    constexpr int NV = TR / 32, NX = TM / 128, G = TM / 32;             // staging: rows per lane, its pieces of q a row, scales of a row
    constexpr int YC = 16 / (int)sizeof(T), YW = TN / 16 / YC;          // columns of dy a load, loads a row
    constexpr int KS = TR / 16;
    constexpr bool LATE = MA == 2;                                      // (see above)
    constexpr int STAGES = LATE ? 3 : 2;
    __shared__ __attribute__((aligned(16))) char smem[STAGES * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wrow = (wave / WN) * 32 * MA, wcol = (wave % WN) * 32 * NB, l31 = lane & 31, half = lane >> 5;
    const int ntl = p.mtiles * p.ntiles;
    const int item = xcd_remap((int)blockIdx.x, ntl * p.nsplit);       // tile fastest: an XCD's L2 holds whole row ranges
    const int split = item / ntl, tile = item - split * ntl;
    const int mt = tile / p.ntiles, nt = tile - mt * p.ntiles;
    const int c0 = mt * TM, k0 = nt * TN;
    const int row0 = split * p.rows_per_split, row1 = min(row0 + p.rows_per_split, p.nrows);
    const long safe = safe_rows(p.nrows, p.K);

    // A wave stages 4 NV rows, 16 lanes a row: 8 columns of every 128 of q and YC of every 16 YC of dy each.  Every load of a wave covers lines of its
    // own: a line asked for again while it is still on its way stalls the CU's cache until it arrives.  That goes for the scales too, a few
    // bytes a row: a lane loads one of them, and the lanes that need it fetch it from there.
    const int sr = lane >> 4, sg = lane & 15, wr = wave * 4 * NV;
    const int lds8 = p.ld8 >> 5;
    struct Regs { u32x2 xq[NV][NX]; int sb; u32x4 yv[NV][YW]; };
    float bias[YW][YC];
#pragma unroll
    for (int w = 0; w < YW; ++w)
#pragma unroll
        for (int e = 0; e < YC; ++e) bias[w][e] = 0.f;
    auto widen = [](const u32x4& q, float (&v)[YC]) {
        if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(q[e]);
        } else {
            unpack(__builtin_bit_cast(Raw8<bf16_t>, q), v);
        }
    };
    // The split's operands through buffer descriptors: a row behind the split, or a lane whose columns lie behind the matrix (offset OOB), reads zero
    // without a branch.  (The plan keeps a split's bytes below 2^30: offsets and OOB never meet.)  dy whose rows are not 4-byte aligned (RAG) is
    // read by address.
    constexpr unsigned OOB = 0x80000000u;
    const int have_rows = row1 - row0, yld = (int)(p.lddy * sizeof(T));
    const auto rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.codes + (long)row0 * p.ld8), 0, have_rows * p.ld8, 0x00020000);
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.scales + (long)row0 * lds8), 0, have_rows * lds8, 0x00020000);
    const auto ry = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(p.dy) + (long)row0 * yld), 0,
                                                      (have_rows - 1) * yld + p.K * (int)sizeof(T), 0x00020000);
    unsigned xoff[NV][NX], soff, yoff[NV][YW];               // of the next tile to ask for
    int yrow = row0 + wr + sr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int r = wr + 4 * i + sr;
#pragma unroll
        for (int m = 0; m < NX; ++m) {
            const int c = c0 + 128 * m + 8 * sg;
            xoff[i][m] = c < p.ld8 ? (unsigned)(r * p.ld8 + c) : OOB;
        }
#pragma unroll
        for (int w = 0; w < YW; ++w) {
            const int k = k0 + (16 * w + sg) * YC;
            yoff[i][w] = k < p.K ? (unsigned)(r * yld) + (unsigned)(k * sizeof(T)) : OOB;
        }
    }
    soff = lane < 4 * NV * G && (c0 >> 5) + lane % G < lds8 ? (unsigned)((wr + lane / G) * lds8 + (c0 >> 5) + lane % G) : OOB;
    auto fetch = [&](Regs& g) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int m = 0; m < NX; ++m) {
                g.xq[i][m] = __builtin_amdgcn_raw_buffer_load_b64(rx, xoff[i][m], 0, 0);
                xoff[i][m] += TR * p.ld8;
            }
#pragma unroll
            for (int w = 0; w < YW; ++w) {
                if constexpr (RAG) {
                    const int r = yrow + 4 * i, k = k0 + (16 * w + sg) * YC;
                    g.yv[i][w] = __builtin_bit_cast(u32x4, ld8<true>(static_cast<const T*>(p.dy) + r * p.lddy + k, r < row1 ? p.K - k : 0, r < safe));
                } else {
                    g.yv[i][w] = __builtin_amdgcn_raw_buffer_load_b128(ry, yoff[i][w], 0, 0);
                    yoff[i][w] += TR * yld;
                }
            }
        }
        g.sb = __builtin_amdgcn_raw_buffer_load_b8(rs, soff, 0, 0);
        soff += TR * lds8;
        if (RAG) yrow += TR;
    };
    // the scales of this lane's pieces of its row i, a byte each
    auto scales = [&](const Regs& g, int (&byte)[NV]) {
        int v = g.sb;
        if (NX == 2) v |= (int)dppu<0x104>((unsigned)g.sb) << 8;          // (row_shl 4: the lane four on holds the scale four groups on)
#pragma unroll
        for (int i = 0; i < NV; ++i) byte[i] = __builtin_amdgcn_ds_bpermute(4 * ((4 * i + sr) * G + (sg >> 2)), v);
    };
    auto stage = [&](const Regs& g, const int (&byte)[NV], char* xt) {
        char* yt = xt + XTILE;
        const int swz = (sr & 3) << 2;                       // (row & 3 == sr)
        // granule g (8 columns) of staged row r lies at slot g ^ ((r & 3) << 2): the lanes that a transposing read serves together cover all banks
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int r = wr + 4 * i + sr;
#pragma unroll
            for (int w = 0; w < YW; ++w) {
                if constexpr (!F32) {
                    *reinterpret_cast<u32x4*>(yt + r * YROW + (((16 * w + sg) ^ swz) << 4)) = g.yv[i][w];
                } else {
                    // the upper halves of fp32 values are their first eight significand bits in bf16; what is left has the next sixteen
                    float v[4];
                    widen(g.yv[i][w], v);
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        const u32x2 h = {__builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x07060302u),
                                         __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x07060302u)};
                        *reinterpret_cast<u32x2*>(yt + t * YTILE + r * YROW + (((8 * w + (sg >> 1)) ^ swz) << 4) + 8 * (sg & 1)) = h;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] -= __uint_as_float(__float_as_uint(v[e]) & 0xffff0000u);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < NX; ++m) {
                const unsigned e = ((unsigned)byte[i] >> (8 * m)) & 255u;
                const float s = F == DPIG_ACT8_E4M3 ? __uint_as_float(e << 23) : act8::scale_value(e);
                u32x2 q = g.xq[i][m];
                if (F == DPIG_ACT8_E4M3) {
                    q[0] = e == 255u ? 0x7f7f7f7fu : q[0];
                    q[1] = e == 255u ? 0x7f7f7f7fu : q[1];
                }
                *reinterpret_cast<uint4*>(xt + r * XROW + (((16 * m + sg) ^ swz) << 4)) = decode_bf16<F>(q[0], q[1], s);
            }
        }
    };

    f32x16 acc[MA][NB];
#pragma unroll
    for (int a = 0; a < MA; ++a)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
    // transposing reads: 16 lanes serve a [4 rows][16 columns] block; lane q supplies row q / 4, columns 4 (q % 4) .. + 3, and receives the
    // 4 rows of column q.  Two of them make the 8 consecutive r of a 32x32x16 fragment.
    const int q = lane & 15, cg = (lane >> 4) & 1, pq = q >> 2;
    int offa[MA], offb[NB];
#pragma unroll
    for (int b = 0; b < MA; ++b) {
        const int ca = wrow + 32 * b + cg * 16 + (q & 3) * 4;
        offa[b] = (half * 8 + pq) * XROW + (((ca >> 3) ^ (pq << 2)) << 4) + (ca & 7) * 2;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int cb = wcol + 32 * b + cg * 16 + (q & 3) * 4;
        offb[b] = XTILE + (half * 8 + pq) * YROW + (((cb >> 3) ^ (pq << 2)) << 4) + (cb & 7) * 2;
    }
    auto frag = [&](const char* a, int row4) -> bf16x8 {
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + row4));
        const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        return __builtin_bit_cast(bf16x8, v);
    };
    bf16x8 fa[KS][MA], fb[KS][TERMS][NB];                  // a tile's fragments
    auto read = [&](const char* at) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
            for (int a = 0; a < MA; ++a) fa[ks][a] = frag(at + offa[a] + ks * 16 * XROW, 4 * XROW);
#pragma unroll
            for (int t = 0; t < TERMS; ++t)
#pragma unroll
                for (int b = 0; b < NB; ++b) fb[ks][t][b] = frag(at + offb[b] + t * YTILE + ks * 16 * YROW, 4 * YROW);
        }
    };
    auto multiply = [&]() {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int t = TERMS - 1; t >= 0; --t)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int a = 0; a < MA; ++a)
                        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[ks][a], fb[ks][t][b], acc[a][b], 0, 0, 0);
    };
    // The column sums of dy are shared out over the workgroups of a column of tiles, which all read it: every mtiles-th tile each.
    int turn = p.want_db ? (p.nsplit == 1 ? (mt == 0 ? 0 : -1) : mt) : -1;           // tiles until this workgroup's next turn (< 0: never)
    auto bias_turn = [&](const Regs& g) {
        if (turn == 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int w = 0; w < YW; ++w) {
                    float v[YC];
                    widen(g.yv[i][w], v);
#pragma unroll
                    for (int e = 0; e < YC; ++e) bias[w][e] += v[e];
                }
            turn = p.nsplit == 1 ? 1 : p.mtiles;
        }
        if (turn > 0) --turn;
    };
    auto barrier = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    Regs g[2];
    const int ntr = (have_rows + TR - 1) / TR;
    int byte[NV];
    fetch(g[0]);
    fetch(g[1]);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {                // tiles 0 (and 1) into LDS, the two after them on their way
        bias_turn(g[i]);
        scales(g[i], byte);
        stage(g[i], byte, smem + i * STAGE);
        fetch(g[i]);
    }
    barrier();
    if (wave >= 4) barrier();                             // the second half: half a tile behind
    int t = 0;
    auto step = [&](auto I) {
        constexpr int i = decltype(I)::value;             // t % 6
        constexpr int NM = KS * TERMS * MA * NB, NW = LATE ? NV * (NX + YW * TERMS) : 0, NL = NV * (NX + YW) + 1;
        constexpr int later = (i + STAGES - 1) % STAGES;  // the stage of tile t + STAGES - 1
        Regs& s = g[(i + STAGES - 1) & 1];                // that tile
        scales(s, byte);
        read(smem + i % STAGES * STAGE);
        if (!LATE) stage(s, byte, smem + later * STAGE);
        bias_turn(s);
        barrier();
        __builtin_amdgcn_s_setprio(1);
        if (LATE) stage(s, byte, smem + later * STAGE);
        fetch(s);                                         // two tiles further on
        multiply();
        weave<0, NM, NW, NL>();
        __builtin_amdgcn_s_setprio(0);
        barrier();
        return ++t < ntr;
    };
    while (every(step, std::make_integer_sequence<int, LATE ? 6 : 2>())) {}
    if (wave < 4) barrier();

    // ---- result: accumulator register r of lane (half, l31) is row (r & 3) + 8 (r >> 2) + 4 half, column l31 of its 32x32 block ----------
    // (a descriptor of this wave's rows bounds them; a column behind the matrix gets an offset behind the descriptor)
    const int have = min(32 * MA, p.C - (c0 + wrow));
    float* out = (p.partial ? p.partial + (long)split * p.C * p.K : p.dw) + (have > 0 ? (long)(c0 + wrow) * p.K : 0);
    const auto ro = __builtin_amdgcn_make_buffer_rsrc(out, 0, have > 0 ? (int)(have * p.K * 4u) : 0, 0x00020000);
    const bool add = !p.partial && p.beta != 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int k = k0 + wcol + 32 * b + l31;
        const unsigned o = k < p.K ? (unsigned)(4 * half * p.K + k) * 4u : OOB;
#pragma unroll
        for (int a = 0; a < MA; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int so = (32 * a + (r & 3) + 8 * (r >> 2)) * p.K * 4;
                float v = acc[a][b][r];
                if (add) v += p.beta * __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ro, o, so, 0));
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), ro, o, so, 0);
            }
    }
    if (p.want_db && (p.nsplit > 1 || mt == 0)) {     // workgroup-uniform; the staging buffers are free
        float(*sums)[TN] = reinterpret_cast<float(*)[TN]>(smem);     // [32 rows][TN columns]
#pragma unroll
        for (int w = 0; w < YW; ++w)
#pragma unroll
            for (int e = 0; e < YC; ++e) sums[wave * 4 + sr][(16 * w + sg) * YC + e] = bias[w][e];
        __syncthreads();
        if (tid < TN && k0 + tid < p.K) {
            float s = 0.f;
#pragma unroll 8
            for (int r = 0; r < 32; ++r) s += sums[r][tid];
            if (p.bias_partial) p.bias_partial[((long)split * (p.nsplit > 1 ? p.mtiles : 1) + mt) * p.K + k0 + tid] = s;
            else p.db[k0 + tid] = p.beta_b != 0.f ? p.beta_b * p.db[k0 + tid] + s : s;
        }
    }
}

struct JoinP {
    const float *partial, *bias_partial, *scale, *offset;
    float *dw, *db;
    int C, K, nsplit, nbias;
    float beta, beta_b;
};
// dw[c][k] = beta dw + scale[c] sum_s partial[s][c][k] + offset[c] sum_s bias[s][k], and db.  A workgroup has 16 x V columns; its 16 rows of threads take
// 16 rows of dw (few splits, many rows) or, with SPLITS, a share of the splits of one row each.  Every sum in a fixed order.
template <int V, bool SPLITS> __global__ __launch_bounds__(256) void wgrad8_join_kernel(const JoinP p) {
    typedef float vec __attribute__((ext_vector_type(V), aligned(4)));
    __shared__ vec red[16][16];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int k = (blockIdx.x * 16 + tx) * V;
    const bool in = k < p.K;
    vec sb = 0.f;
    auto across = [&](vec mine) -> vec {                 // sum over the 16 rows of threads
        __syncthreads();
        red[ty][tx] = mine;
        __syncthreads();
        vec t = 0.f;
#pragma unroll
        for (int y = 0; y < 16; ++y) t += red[y][tx];
        return t;
    };
    const bool write_db = p.db && blockIdx.y == 0;
    if (p.offset || write_db) {                          // (uniform in the workgroup)
        if (in) {
#pragma unroll 4
            for (int s = ty; s < p.nbias; s += 16) sb += *reinterpret_cast<const vec*>(p.bias_partial + (long)s * p.K + k);
        }
        sb = across(sb);
        if (write_db && in && ty == 0) {
            vec* o = reinterpret_cast<vec*>(p.db + k);
            *o = p.beta_b != 0.f ? p.beta_b * *o + sb : sb;
        }
    }
    const int c = SPLITS ? blockIdx.y : blockIdx.y * 16 + ty;
    vec sum = 0.f;
    if (in && c < p.C) {
        const float* src = p.partial + (long)c * p.K + k;
        const long step = (long)p.C * p.K;
#pragma unroll 8
        for (int s = SPLITS ? ty : 0; s < p.nsplit; s += SPLITS ? 16 : 1) sum += *reinterpret_cast<const vec*>(src + s * step);
    }
    if (SPLITS) sum = across(sum);
    if (!in || c >= p.C || (SPLITS && ty != 0)) return;
    if (p.scale) sum *= p.scale[c];
    if (p.offset) sum += p.offset[c] * sb;
    vec* o = reinterpret_cast<vec*>(p.dw + (long)c * p.K + k);
    *o = p.beta != 0.f ? p.beta * *o + sum : sum;
}

// Tile shapes: columns of q by columns of dy, rows
struct Shape { int tm, tn, tr; };
constexpr Shape SMALL = {128, 128, 64}, WIDE = {256, 128, 64}, LARGE = {256, 256, 32}, SMALL32 = {128, 128, 32}, WIDE32 = {256, 128, 32};
struct Plan { Shape shape; int mtiles, ntiles, nsplit, rows_per_split; };
static Plan plan(int64_t nrows, int C, int K, bool f32, long row_bytes) {
    Plan q;
    auto up = [](long a, long b) { return (a + b - 1) / b; };
    // Larger tiles read and decode less per product but leave fewer, larger pieces of work and more partial sums.  us with the smaller / larger tile:
    // 256 x 128 pays from about 10^10 products on (bf16 rows x 512 x 512, 24576 rows 29.0 / 30.7, 32768 36.5 / 36.2, 49152 47.3 / 44.5; x 256 x 512, 65536 rows
    // 39.5 / 40.3, 98304 52.4 / 50.8; a third of that for fp32 dy: rows x 512 x 512, 12288 rows 31.2 / 31.6, 16384 rows 37.5 / 36.9), 256 x 256 from 2^36
    // (512 x 512, 131072 rows 95.0 / 98.5, 196608 133 / 131, 262144 171 / 170; 768 x 768, 98304 rows 138 / 142, 131072 186 / 180), unless it is padding
    // that grows.
    const double products = (double)nrows * C * K * (f32 ? 3 : 1);
    auto area = [&](Shape t) { return up(C, t.tm) * t.tm * up(K, t.tn) * t.tn; };
    q.shape = f32 ? SMALL32 : SMALL;
    const Shape wide = f32 ? WIDE32 : WIDE;
    if (products > 0x1.4p33 && area(wide) <= area(q.shape) * 5 / 4) q.shape = wide;
    if (!f32 && products >= 0x1p36 && area(LARGE) <= area(q.shape) * 9 / 8) q.shape = LARGE;
    q.mtiles = (int)up(C, q.shape.tm);
    q.ntiles = (int)up(K, q.shape.tn);
    const long tiles = (long)q.mtiles * q.ntiles, rt = up(nrows, q.shape.tr);
    long want = (kNumCU + tiles / 2) / tiles;              // one workgroup per CU
    if (want > (rt + 3) / 4) want = (rt + 3) / 4;      // at least four tiles of rows a split
    if (want < 1) want = 1;
    const long most = (1L << 30) / row_bytes / q.shape.tr;      // (descriptors of a split's operands stay below 2^30 bytes)
    if (up(rt, want) > most) want = up(rt, most);
    q.rows_per_split = (int)(up(rt, want) * q.shape.tr);
    q.nsplit = (int)up(nrows, q.rows_per_split);
    return q;
}
static long row_bytes(int C, int64_t lddy, int dy_bf16) {
    const long y = lddy * (dy_bf16 ? 2 : 4), x = act8::padded(C);
    return x > y ? x : y;
}
static bool joined(const Plan& q, bool affine) { return q.nsplit > 1 || affine; }
static int bias_slots(const Plan& q) { return q.nsplit > 1 ? q.nsplit * q.mtiles : 1; }
static size_t ws_bytes(const Plan& q, int C, int K, bool affine) {
    return joined(q, affine) ? ((size_t)q.nsplit * C + bias_slots(q)) * K * sizeof(float) : 0;
}

}  // namespace wg8
}  // namespace dpig

using namespace dpig;

extern "C" size_t dpig_linear_wgrad8_workspace_bytes(int64_t nrows, int C, int64_t lddy, int K, int dy_bf16, int affine) {
    if (nrows <= 0 || C <= 0 || K <= 0 || lddy < K || lddy > (1 << 22)) return 0;
    return wg8::ws_bytes(wg8::plan(nrows, C, K, !dy_bf16, wg8::row_bytes(C, lddy, dy_bf16)), C, K, affine != 0);
}

extern "C" int dpig_linear_wgrad8(const uint8_t* codes, const uint8_t* scales, int fmt, int64_t nrows, int C, const void* dy, int dy_bf16,
                                  int64_t lddy, int K, const float* scale, const float* offset, float* dw, float beta, float* db,
                                  float beta_b, void* ws, size_t ws_bytes, void* stream) {
    if (!codes || !scales || !dy || !dw) return fail(DPIG_EINVAL, "linear_wgrad8: null pointer");
    if (nrows <= 0 || C <= 0 || K <= 0 || nrows > (1L << 30) || C > 32768 || K > 32768) return fail(DPIG_EINVAL, "linear_wgrad8: bad shape");
    if (fmt != DPIG_ACT8_E4M3 && fmt != DPIG_ACT8_INT8) return fail(DPIG_EINVAL, "linear_wgrad8: unknown checkpoint format");
    if (!aligned16(codes)) return fail(DPIG_EALIGN, "linear_wgrad8: checkpoint codes must be 16-byte aligned");
    if (lddy < K) return fail(DPIG_EINVAL, "linear_wgrad8: row stride below the column count");
    if (lddy > (1 << 22)) return fail(DPIG_EINVAL, "linear_wgrad8: row stride above %d", 1 << 22);
    const wg8::Plan q = wg8::plan(nrows, C, K, !dy_bf16, wg8::row_bytes(C, lddy, dy_bf16));
    const bool affine = scale || offset, join = wg8::joined(q, affine);
    if ((long)q.mtiles * q.ntiles * q.nsplit > 0x7fffffffL) return fail(DPIG_EINVAL, "linear_wgrad8: too many tiles");
    if (join && (!ws || ws_bytes < wg8::ws_bytes(q, C, K, affine))) return fail(DPIG_ENOMEM, "linear_wgrad8: workspace too small");
    hipStream_t st = static_cast<hipStream_t>(stream);
    wg8::P p = {};
    p.codes = codes; p.scales = scales; p.dy = dy; p.dw = dw; p.db = db; p.lddy = lddy; p.nrows = (int)nrows; p.C = C; p.K = K;
    p.ld8 = act8::padded(C); p.mtiles = q.mtiles; p.ntiles = q.ntiles; p.nsplit = q.nsplit; p.rows_per_split = q.rows_per_split;
    p.beta = beta; p.beta_b = beta_b; p.want_db = db || offset;
    if (join) {
        p.partial = static_cast<float*>(ws);
        p.bias_partial = p.partial + (long)q.nsplit * C * K;
    }
    const dim3 grid((unsigned)(q.mtiles * q.ntiles * q.nsplit));
    const bool rag = dy_bf16 && (K % 2 != 0 || lddy % 2 != 0 || (reinterpret_cast<uintptr_t>(dy) & 3) != 0);
#define GO(T, F, R, MA, NB, WM, TR) hipLaunchKernelGGL((wg8::wgrad8_kernel<T, F, R, MA, NB, WM, TR>), grid, dim3(512), 0, st, p)
#define BF16(F, R)                                                                                                         \
    do {                                                                                                                  \
        if (q.shape.tn == 256) GO(rows::bf16_t, F, R, 4, 2, 2, 32);                                                       \
        else if (q.shape.tm == 256) GO(rows::bf16_t, F, R, 2, 2, 4, 64);                                                  \
        else GO(rows::bf16_t, F, R, 2, 1, 2, 64);                                                                         \
    } while (0)
#define FP32(F) do { if (q.shape.tm == 256) GO(float, F, false, 2, 2, 4, 32); else GO(float, F, false, 2, 1, 2, 32); } while (0)
    const bool e4m3 = fmt == DPIG_ACT8_E4M3;
    if (!dy_bf16) { if (e4m3) FP32(DPIG_ACT8_E4M3); else FP32(DPIG_ACT8_INT8); }
    else if (rag) { if (e4m3) BF16(DPIG_ACT8_E4M3, true); else BF16(DPIG_ACT8_INT8, true); }
    else { if (e4m3) BF16(DPIG_ACT8_E4M3, false); else BF16(DPIG_ACT8_INT8, false); }
#undef FP32
#undef BF16
#undef GO
    if (join) {
        const wg8::JoinP j = {p.partial, p.bias_partial, scale, offset, dw, db, C, K, q.nsplit, wg8::bias_slots(q), beta, beta_b};
        const int v = K % 4 == 0 ? 4 : K % 2 == 0 ? 2 : 1;
        const bool by_split = q.nsplit >= 64;
        const dim3 jg((unsigned)((K / v + 15) / 16), (unsigned)(by_split ? C : (C + 15) / 16));
        if (v == 4 && by_split) hipLaunchKernelGGL((wg8::wgrad8_join_kernel<4, true>), jg, dim3(256), 0, st, j);
        else if (v == 4) hipLaunchKernelGGL((wg8::wgrad8_join_kernel<4, false>), jg, dim3(256), 0, st, j);
        else if (v == 2 && by_split) hipLaunchKernelGGL((wg8::wgrad8_join_kernel<2, true>), jg, dim3(256), 0, st, j);
        else if (v == 2) hipLaunchKernelGGL((wg8::wgrad8_join_kernel<2, false>), jg, dim3(256), 0, st, j);
        else if (by_split) hipLaunchKernelGGL((wg8::wgrad8_join_kernel<1, true>), jg, dim3(256), 0, st, j);
        else hipLaunchKernelGGL((wg8::wgrad8_join_kernel<1, false>), jg, dim3(256), 0, st, j);
    }
    return check_launch("linear_wgrad8");
}
