// Element types of the operators' tensors: ONNX TensorProto codes, loads widened to 32 bits and
// stores rounded once to the tensor's type (to nearest, ties to even).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/wocr.h"

namespace wocr {
namespace k {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

inline int elem_size(int type) { return type == WOCR_F32 ? 4 : 2; }

}  // namespace k
}  // namespace wocr
