// 8-bit activation checkpoints (the format: dpig_act8.h): store, load, and an activation's gradient with the mask read from the codes.
// Elementwise and bound by HBM: 8 channels a lane, the 32 channels of a group in a quad of lanes, rows beside each other in a wave.
// Measured: 524288 x 128 bf16 store 42 us + load 32 us (203 MB each way: 4.8 and 6.4 TB/s, the codes still in the cache when loaded); mask of
// 131072 x 256 fp32 51.5 us (302 MB, 5.9 TB/s).
#include "dpig_rows.h"

namespace dpig {
namespace act8k {

using namespace rows;

struct P {
    const void* x; void* y;
    uint8_t *codes, *scales;
    long ldx, ldy, nrows;
    long drow;                              // a step of the whole grid: drow rows and dvec vectors
    int C, ld8, nvec, dvec, act;            // nvec: vectors of a row that are visited
    float alpha;
};
// the vectors of all rows, one after the other, dealt to the threads of the grid; one division a thread, steps after that
#define ACT8_FOR(r, v)                                                                                                     \
    const unsigned long i0 = (unsigned long)blockIdx.x * NT + threadIdx.x;                                                  \
    long r = (long)(i0 / (unsigned)p.nvec);                                                                               \
    int v = (int)(i0 - (unsigned long)r * (unsigned)p.nvec);                                                               \
    for (; r < p.nrows; r += p.drow, v += p.dvec, r += v >= p.nvec ? 1 : 0, v -= v >= p.nvec ? p.nvec : 0)

template <typename T, bool RAG, int F>
__global__ __launch_bounds__(NT) void store_kernel(const P p) {
    ACT8_FOR(r, v) {
        float x[8];
        unpack(ld8<RAG>(static_cast<const T*>(p.x) + r * p.ldx + 8 * v, p.C - 8 * v, false), x);
        save8_as<F>(x, p.codes + r * p.ld8 + 8 * v, p.scales + r * (p.ld8 >> 5) + (v >> 2), (v & 3) == 0);
    }
}
template <typename T, bool RAG, int F>
__global__ __launch_bounds__(NT) void load_kernel(const P p) {
    ACT8_FOR(r, v) {
        const uint2 q = *reinterpret_cast<const uint2*>(p.codes + r * p.ld8 + 8 * v);
        const float s = act8::scale_value(p.scales[r * (p.ld8 >> 5) + (v >> 2)]);
        float x[8];
        act8::decode8<F>(q, s, x);
        st8<RAG>(static_cast<T*>(p.y) + r * p.ldy + 8 * v, x, p.C - 8 * v);
    }
}
template <typename T, bool RAG, int F>
__global__ __launch_bounds__(NT) void mask_kernel(const P p) {
    const long safe = safe_rows(p.nrows, p.C);
    const float off = p.act == DPIG_ACT_RELU ? 0.f : p.alpha;
    ACT8_FOR(r, v) {
        const uint2 q = *reinterpret_cast<const uint2*>(p.codes + r * p.ld8 + 8 * v);
        float d[8];
        unpack(ld8<RAG>(static_cast<const T*>(p.x) + r * p.ldx + 8 * v, p.C - 8 * v, r < safe), d);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] *= act8::positive<F>(e < 4 ? q.x : q.y, e & 3) ? 1.f : off;
        st8<RAG>(static_cast<T*>(p.y) + r * p.ldy + 8 * v, d, p.C - 8 * v);
    }
}

static int check(const char* who, int64_t nrows, int C, int fmt, const uint8_t* codes, const uint8_t* scales) {
    if (nrows <= 0 || C <= 0 || nrows > (1L << 40) || C > (1 << 24)) return fail(DPIG_EINVAL, "%s: bad shape", who);
    if (fmt != DPIG_ACT8_E4M3 && fmt != DPIG_ACT8_INT8) return fail(DPIG_EINVAL, "%s: unknown checkpoint format", who);
    if (!codes || (!scales)) return fail(DPIG_EINVAL, "%s: null pointer", who);
    if (!aligned16(codes)) return fail(DPIG_EALIGN, "%s: checkpoint codes must be 16-byte aligned", who);
    return DPIG_OK;
}
static unsigned geometry(P* p, int nvec) {      // -> workgroups: sixteen per CU at most
    const unsigned long blocks = ((unsigned long)p->nrows * (unsigned)nvec + NT - 1) / NT;
    const unsigned grid = (unsigned)(blocks < 16ul * kNumCU ? blocks : 16ul * kNumCU);
    p->nvec = nvec;
    p->drow = (long)(grid * (unsigned long)NT / (unsigned)nvec);
    p->dvec = (int)(grid * (unsigned long)NT % (unsigned)nvec);
    return grid;
}
#define ACT8_LAUNCH(KERNEL, RAG)                                                                                                   \
    do {                                                                                                                          \
        if (is_bf16) ACT8_FMT(KERNEL, bf16_t, RAG); else ACT8_FMT(KERNEL, float, RAG);                                            \
    } while (0)
#define ACT8_FMT(KERNEL, T, RAG)                                                                                                   \
    do {                                                                                                                          \
        if (RAG) { if (fmt == DPIG_ACT8_E4M3) ACT8_GO((KERNEL<T, true, DPIG_ACT8_E4M3>)); else ACT8_GO((KERNEL<T, true, DPIG_ACT8_INT8>)); }        \
        else { if (fmt == DPIG_ACT8_E4M3) ACT8_GO((KERNEL<T, false, DPIG_ACT8_E4M3>)); else ACT8_GO((KERNEL<T, false, DPIG_ACT8_INT8>)); }          \
    } while (0)
#define ACT8_GO(K) hipLaunchKernelGGL(K, dim3(grid), dim3(NT), 0, static_cast<hipStream_t>(stream), p)

}  // namespace act8k
}  // namespace dpig

using namespace dpig;
using namespace dpig::act8k;

extern "C" int dpig_act8_store(const void* x, int is_bf16, int64_t ldx, int64_t nrows, int C, int fmt, uint8_t* codes, uint8_t* scales,
                               void* stream) {
    if (int rc = check("act8_store", nrows, C, fmt, codes, scales)) return rc;
    if (!x) return fail(DPIG_EINVAL, "act8_store: null pointer");
    if (ldx < C) return fail(DPIG_EINVAL, "act8_store: row stride below the channel count");
    P p = {};
    p.x = x; p.codes = codes; p.scales = scales; p.ldx = ldx; p.nrows = nrows; p.C = C; p.ld8 = act8::padded(C);
    const unsigned grid = geometry(&p, p.ld8 / 8);
    const bool rag = C % 8 != 0 || !vec_ok(x, ldx, is_bf16 ? 2 : 4);
    ACT8_LAUNCH(store_kernel, rag);
    return check_launch("act8_store");
}

extern "C" int dpig_act8_load(const uint8_t* codes, const uint8_t* scales, int64_t nrows, int C, int fmt, void* y, int is_bf16, int64_t ldy,
                              void* stream) {
    if (int rc = check("act8_load", nrows, C, fmt, codes, scales)) return rc;
    if (!y) return fail(DPIG_EINVAL, "act8_load: null pointer");
    if (ldy < C) return fail(DPIG_EINVAL, "act8_load: row stride below the channel count");
    P p = {};
    p.y = y; p.codes = const_cast<uint8_t*>(codes); p.scales = const_cast<uint8_t*>(scales); p.ldy = ldy; p.nrows = nrows; p.C = C;
    p.ld8 = act8::padded(C);
    const unsigned grid = geometry(&p, (C + 7) / 8);
    const bool rag = C % 8 != 0 || !vec_ok(y, ldy, is_bf16 ? 2 : 4);
    ACT8_LAUNCH(load_kernel, rag);
    return check_launch("act8_load");
}

extern "C" int dpig_act8_act_bwd(const void* dy, int is_bf16, int64_t lddy, const uint8_t* codes, int64_t nrows, int C, int fmt, int act,
                                 float alpha, void* dz, int64_t lddz, void* stream) {
    if (int rc = check("act8_act_bwd", nrows, C, fmt, codes, codes)) return rc;
    if (!dy || !dz) return fail(DPIG_EINVAL, "act8_act_bwd: null pointer");
    if (act != DPIG_ACT_RELU && act != DPIG_ACT_LRELU) return fail(DPIG_EINVAL, "act8_act_bwd: the activation must be ReLU or LeakyReLU");
    if (lddy < C || lddz < C) return fail(DPIG_EINVAL, "act8_act_bwd: row stride below the channel count");
    P p = {};
    p.x = dy; p.y = dz; p.codes = const_cast<uint8_t*>(codes); p.ldx = lddy; p.ldy = lddz; p.nrows = nrows; p.C = C; p.ld8 = act8::padded(C);
    p.act = act; p.alpha = alpha;
    const unsigned grid = geometry(&p, (C + 7) / 8);
    const bool rag = C % 8 != 0 || !vec_ok(dy, lddy, is_bf16 ? 2 : 4) || !vec_ok(dz, lddz, is_bf16 ? 2 : 4);
    ACT8_LAUNCH(mask_kernel, rag);
    return check_launch("act8_act_bwd");
}
