// Residual norm with x in __nv_bfloat16 and h in __nv_bfloat16 (mdq_norm.cuh).
#include "mdq_norm.cuh"

MDQ_NORM_INSTANTIATE(__nv_bfloat16, __nv_bfloat16, bb)
