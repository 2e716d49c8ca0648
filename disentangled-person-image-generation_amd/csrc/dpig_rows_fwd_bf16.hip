// The norms' forward kernels on bf16 tensors (dpig_rows_fwd.h).
#include "dpig_rows_fwd.h"

template <> int dpig::rows::entry_fwd<dpig::rows::bf16_t>(EntryP p, hipStream_t st) { return entry_fwd_as<bf16_t>(p, st); }
template <> int dpig::rows::exit_fwd<dpig::rows::bf16_t>(ExitP p, hipStream_t st) { return exit_fwd_as<bf16_t>(p, st); }
