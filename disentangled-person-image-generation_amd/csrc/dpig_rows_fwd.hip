// The norms' forward kernels on fp32 tensors (dpig_rows_fwd.h), and the C entries of both types.
#include "dpig_rows_fwd.h"

template <> int dpig::rows::entry_fwd<float>(EntryP p, hipStream_t st) { return entry_fwd_as<float>(p, st); }
template <> int dpig::rows::exit_fwd<float>(ExitP p, hipStream_t st) { return exit_fwd_as<float>(p, st); }

namespace dpig {
namespace rows {

template <> int entry_fwd<bf16_t>(EntryP p, hipStream_t st);      // dpig_rows_fwd_bf16.hip
template <> int exit_fwd<bf16_t>(ExitP p, hipStream_t st);

static int check_rows(const char* who, int64_t nrows, int C, int kind) {
    if (nrows <= 0 || nrows > (1L << 40)) return fail(DPIG_EINVAL, "%s: bad row count", who);
    if (C <= 0 || C > C_MAX) return fail(DPIG_EINVAL, "%s: channels must be 1 .. %d", who, C_MAX);
    if (kind != DPIG_NORM_LAYER && kind != DPIG_NORM_RMS) return fail(DPIG_EINVAL, "%s: unknown kind of norm", who);
    return DPIG_OK;
}
static int check_save(const char* who, int fmt, const uint8_t* codes, const uint8_t* scales) {
    if (!codes && !scales) return DPIG_OK;
    if (!codes || !scales) return fail(DPIG_EINVAL, "%s: a checkpoint needs codes and scales", who);
    if (fmt != DPIG_ACT8_E4M3 && fmt != DPIG_ACT8_INT8) return fail(DPIG_EINVAL, "%s: unknown checkpoint format", who);
    if (!aligned16(codes)) return fail(DPIG_EALIGN, "%s: checkpoint codes must be 16-byte aligned", who);
    return DPIG_OK;
}

}  // namespace rows
}  // namespace dpig

using namespace dpig;

extern "C" int dpig_rownorm_fwd(const void* x, int is_bf16, int64_t ldx, int64_t nrows, int C, int kind, const float* scale, const float* offset,
                                float eps, void* y, int64_t ldy, float* mean, float* rstd, int fmt, uint8_t* codes, uint8_t* scales,
                                void* stream) {
    if (int rc = rows::check_rows("rownorm_fwd", nrows, C, kind)) return rc;
    if (int rc = rows::check_save("rownorm_fwd", fmt, codes, scales)) return rc;
    if (!x || !y || !rstd || (kind == DPIG_NORM_LAYER && !mean)) return fail(DPIG_EINVAL, "rownorm_fwd: null pointer");
    if (ldx < C || ldy < C) return fail(DPIG_EINVAL, "rownorm_fwd: row stride below the channel count");
    rows::EntryP p = {x, y, scale, offset, kind == DPIG_NORM_LAYER ? mean : nullptr, rstd, (long)ldx, (long)ldy, (long)nrows, 0, C,
                      kind == DPIG_NORM_LAYER, eps, 1.0f / (float)C, {codes, scales, fmt, act8::padded(C)}};
    hipStream_t st = static_cast<hipStream_t>(stream);
    return is_bf16 ? rows::entry_fwd<rows::bf16_t>(p, st) : rows::entry_fwd<float>(p, st);
}

extern "C" int dpig_gated_residual_fwd(const void* x, int64_t ldx, const void* f, int64_t ldf, int is_bf16, int64_t nrows, int C, int kind,
                                       const float* scale, const float* offset, float eps, const void* gate, int gate_bf16, int64_t groups,
                                       const float* res_scale, void* out, int64_t ldo, float* mean, float* rstd, int fmt, uint8_t* codes,
                                       uint8_t* scales, int kind2, const float* scale2, const float* offset2, float eps2, void* h,
                                       int64_t ldh, float* mean2, float* rstd2, int fmt2, uint8_t* codes2, uint8_t* scales2,
                                       void* stream) {
    if (int rc = rows::check_rows("gated_residual_fwd", nrows, C, kind)) return rc;
    if (int rc = rows::check_save("gated_residual_fwd", fmt, codes, scales)) return rc;
    if (!x || !f || !out || !rstd || (kind == DPIG_NORM_LAYER && !mean)) return fail(DPIG_EINVAL, "gated_residual_fwd: null pointer");
    if (ldx < C || ldf < C || ldo < C || (h && ldh < C)) return fail(DPIG_EINVAL, "gated_residual_fwd: row stride below the channel count");
    if (gate && (groups <= 0 || nrows % groups != 0)) return fail(DPIG_EINVAL, "gated_residual_fwd: rows must be a multiple of the gate's groups");
    if (h) {
        if (int rc = rows::check_rows("gated_residual_fwd (next norm)", nrows, C, kind2)) return rc;
        if (int rc = rows::check_save("gated_residual_fwd (next norm)", fmt2, codes2, scales2)) return rc;
        if (!rstd2 || (kind2 == DPIG_NORM_LAYER && !mean2)) return fail(DPIG_EINVAL, "gated_residual_fwd: null pointer (next norm)");
    }
    const int ld8 = act8::padded(C);
    rows::ExitP p = {x, f, out, h, scale, offset, res_scale, scale2, offset2, gate, kind == DPIG_NORM_LAYER ? mean : nullptr, rstd,
                     kind2 == DPIG_NORM_LAYER ? mean2 : nullptr, rstd2, (long)ldx, (long)ldf, (long)ldo, (long)ldh, (long)nrows, 0, gate ? (long)(nrows / groups) : (long)nrows, C, kind == DPIG_NORM_LAYER,
                     kind2 == DPIG_NORM_LAYER, gate_bf16, eps, eps2, 1.0f / (float)C, {codes, scales, fmt, ld8},
                     {h ? codes2 : nullptr, scales2, fmt2, ld8}};
    hipStream_t st = static_cast<hipStream_t>(stream);
    return is_bf16 ? rows::exit_fwd<rows::bf16_t>(p, st) : rows::exit_fwd<float>(p, st);
}
