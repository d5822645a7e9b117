// Layer norm with the residual stream's addition: launches of layer_norm.hip
// and layer_norm_bwd.hip, shared with the C-ABI entry points.
#pragma once

#include <hip/hip_runtime.h>

// dtype codes 0 bf16, 1 fp16, 2 fp32; dtype_r is meaningful where residual is given.
hipError_t hattn_layer_norm_fwd_launch(const void* x, const void* residual, const void* weight,
                                       const void* bias, void* y, void* s, float* mean,
                                       float* rstd, long rows, int n, float eps, int dtype_x,
                                       int dtype_r, int dtype_w, hipStream_t stream);
hipError_t hattn_layer_norm_bwd_launch(const void* s, const void* weight, const float* mean,
                                       const float* rstd, const void* dy, const void* ds, void* dx,
                                       void* dres, void* dweight, void* dbias, float* ws, long rows,
                                       int n, int dtype_x, int dtype_s, int dtype_w,
                                       hipStream_t stream);
size_t hattn_layer_norm_bwd_ws_bytes(long rows, int n);
constexpr int kLayerNormMaxN = 16384;
