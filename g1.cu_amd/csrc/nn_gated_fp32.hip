// nn_gated_fp32.hip -- the gated block's kernels in fp32.
#include "nn_gated.h"

namespace g1nn {

template int run_gated<float, float, false>(const GatedArgs&, bool, hipStream_t);
template int gated_backward<float>(GatedArgs, const Split&, hipStream_t);

}  // namespace g1nn
