// Residual norm with x in float and h in float (mdq_norm.cuh).
#include "mdq_norm.cuh"

MDQ_NORM_INSTANTIATE(float, float, ff)
