// Residual norm with x in float and h in __nv_bfloat16 (mdq_norm.cuh).
#include "mdq_norm.cuh"

MDQ_NORM_INSTANTIATE(float, __nv_bfloat16, fb)
