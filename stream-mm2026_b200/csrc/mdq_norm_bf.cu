// Residual norm with x in __nv_bfloat16 and h in float (mdq_norm.cuh).
#include "mdq_norm.cuh"

MDQ_NORM_INSTANTIATE(__nv_bfloat16, float, bf)
