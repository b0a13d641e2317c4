// One type of x of the layer norm kernels per translation unit (the build sets
// ST_NORM_TYPE to ST_SCORE_F32, ST_SCORE_F16 and ST_SCORE_BF16), so that the
// instantiations compile in parallel.
#include "layer_norm_kernel.hpp"

#ifndef ST_NORM_TYPE
#error "ST_NORM_TYPE must be defined"
#endif
