// nn_gated_q8.hip -- the gated block's kernels on 8-bit rows and weights.
#include "nn_gated.h"

namespace g1nn {

template int run_gated<i8, float, false>(const GatedArgs&, bool, hipStream_t);
template int run_gated<i8, bf16, false>(const GatedArgs&, bool, hipStream_t);

}  // namespace g1nn
