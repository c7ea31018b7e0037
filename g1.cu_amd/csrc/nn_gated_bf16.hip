// nn_gated_bf16.hip -- the gated block's kernels in bf16.
#include "nn_gated.h"

namespace g1nn {

template int run_gated<bf16, bf16, false>(const GatedArgs&, bool, hipStream_t);
template int gated_backward<bf16>(GatedArgs, const Split&, hipStream_t);

}  // namespace g1nn
