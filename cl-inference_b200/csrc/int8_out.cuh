// int8_out.cuh -- the last step of the 8-bit products: the exact integer sum to
// f32, times the channel's scale, times the token's, plus the residual, rounded
// once to the output type.  Every kernel takes the same steps in the same
// order, so which one ran cannot be told from the result.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace clq {

template <typename OT> __device__ __forceinline__ OT int8_round(float v);
template <> __device__ __forceinline__ float int8_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 int8_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half int8_round<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float int8_scaled(int acc, float ws, float xs) {
    return __fmul_rn(__fmul_rn(__int2float_rn(acc), ws), xs);
}

}  // namespace clq
