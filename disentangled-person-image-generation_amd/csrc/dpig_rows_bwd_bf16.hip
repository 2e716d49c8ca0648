// The row pass of the norms' gradients on bf16 tensors (dpig_rows_bwd.h).
#include "dpig_rows_bwd.h"

template <> void dpig::rows::launch_rows<dpig::rows::bf16_t>(const BwdP& p, bool groups, unsigned blocks, hipStream_t st) {
    launch_rows_as<bf16_t>(p, groups, blocks, st);
}
