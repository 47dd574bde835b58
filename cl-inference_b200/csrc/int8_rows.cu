// int8_rows.cu -- rows of activations (or weights) as 8-bit codes with one f32
// scale a row, the operand form of the integer product (int8_linear.cu), and
// the work a decoder layer does between two products fused into the rounding:
//   rows     v = x
//   norm     h = x + residual, v = h * norm_w, s = 1 / sqrt(mean(h^2) + eps)
//            (the RMSNorm of local/blocks.lisp:115-116 after the residual
//            addition of :387-392); residual_out = h
//   SwiGLU   v = silu(gate) * up (:151-154)
// and then, for peak = max |v| of the row,
//   step  = max(FLT_MIN, peak / 127)     the Q8 codec of local/kv-cache.lisp:37-60
//   code  = clamp(round-half-even(v * (1 / step)), -127, 127)
//   scale = step * s                     (1 for an all-zero row)
// The norm's factor s is common to the row, so the codes need only v and its
// peak, and s enters the scale: one reduction (sum of squares and peak
// together) serves both.  A row that holds a non-finite h or v, or whose sum of
// squares leaves f32, gets codes 0 and the scale NaN, so that every product
// formed with it is NaN.
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/clq.h"
#include "clq_internal.h"

namespace clq {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// silu(g) * u in f32 with the IEEE exponential and quotient: the value is
// rounded to a code, so an error in it moves values across code borders.
__device__ __forceinline__ float silu_times(float g, float u) { return __fmul_rn(__fdiv_rn(g, 1.f + expf(-g)), u); }

constexpr int kRowThreads = 256;

// The row's (sum of squares, peak) over the CTA, the same in every thread.
__device__ __forceinline__ float2 row_reduce(float ss, float peak) {
    __shared__ float2 red[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (int)(blockDim.x >> 5);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, o));
    }
    if (lane == 0) red[warp] = make_float2(ss, peak);
    __syncthreads();
    float2 a = red[0];
    for (int w = 1; w < nw; w++) {
        a.x += red[w].x;
        a.y = fmaxf(a.y, red[w].y);
    }
    return a;
}

// One CTA per row, two passes over it (the second hits L1 / L2).
template <typename XT, typename RT>
__global__ void __launch_bounds__(kRowThreads) quantize_rows_kernel(const QuantRows Q) {
    const int64_t row = blockIdx.x;
    const XT* x = static_cast<const XT*>(Q.x) + row * Q.ldx;
    const XT* gate = Q.gate ? static_cast<const XT*>(Q.gate) + row * Q.ldg : nullptr;
    const RT* res = Q.res ? static_cast<const RT*>(Q.res) + row * Q.ldr : nullptr;
    RT* res_out = Q.res_out ? static_cast<RT*>(Q.res_out) + row * Q.ldro : nullptr;
    int8_t* codes = Q.codes + row * Q.ldc;
    auto value = [&](int64_t i, float& h) {
        h = to_f32(x[i]);
        if (gate) return silu_times(to_f32(gate[i]), h);
        if (res) h = __fadd_rn(h, to_f32(res[i]));
        return Q.norm_w ? __fmul_rn(h, Q.norm_w[i]) : h;
    };
    float ss = 0.f, peak = 0.f;
    for (int64_t i = threadIdx.x; i < Q.k; i += blockDim.x) {
        float h;
        const float v = value(i, h);
        ss = fmaf(h, h, ss);
        peak = v == v ? fmaxf(peak, fabsf(v)) : INFINITY;  // fmaxf drops a NaN
    }
    const float2 r = row_reduce(ss, peak);
    float s = 1.f;
    bool fine = r.y < INFINITY;
    if (Q.norm_w) {
        s = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(r.x, (float)Q.k) + Q.eps));
        fine = fine && r.x < INFINITY;
    }
    const float step = fmaxf(FLT_MIN, __fdiv_rn(r.y, 127.f)), inv = fine ? __fdiv_rn(1.f, step) : 0.f;
    if (threadIdx.x == 0) Q.scales[row] = !fine ? NAN : r.y > 0.f ? __fmul_rn(step, s) : 1.f;
    for (int64_t i = threadIdx.x; i < Q.k; i += blockDim.x) {
        float h;
        const float v = value(i, h);
        if (res_out) res_out[i] = from_f32<RT>(h);
        codes[i] = fine ? (int8_t)fminf(fmaxf(rintf(v * inv), -127.f), 127.f) : (int8_t)0;
    }
}

template <typename OT>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(const int8_t* __restrict__ codes, int64_t ldc,
                                                              const float* __restrict__ scales, int64_t k,
                                                              OT* __restrict__ out, int64_t ldo) {
    const int64_t row = blockIdx.y;
    const float s = scales[row];
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < k; i += (int64_t)gridDim.x * blockDim.x)
        out[row * ldo + i] = from_f32<OT>((float)codes[row * ldc + i] * s);
}

template <typename XT, typename RT>
cudaError_t launch_quant(const QuantRows& q, cudaStream_t s) {
    quantize_rows_kernel<XT, RT><<<(unsigned)q.m, kRowThreads, 0, s>>>(q);
    return cudaGetLastError();
}

template <typename XT>
cudaError_t launch_quant_x(const QuantRows& q, cudaStream_t s) {
    if (!q.res || q.rtype == q.xtype) return launch_quant<XT, XT>(q, s);
    return launch_quant<XT, float>(q, s);
}

template <typename OT>
cudaError_t launch_dequant(const int8_t* codes, int64_t ldc, const float* scales, int64_t m, int64_t k, void* out,
                           int64_t ldo, cudaStream_t s) {
    for (int64_t r0 = 0; r0 < m; r0 += 65535) {
        const int64_t rows = m - r0 < 65535 ? m - r0 : 65535;
        dequantize_rows_kernel<OT><<<dim3((unsigned)((k + 1023) / 1024), (unsigned)rows), 256, 0, s>>>(
            codes + r0 * ldc, ldc, scales + r0, k, static_cast<OT*>(out) + r0 * ldo, ldo);
    }
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize_rows(const QuantRows& q, cudaStream_t s) {
    switch (q.xtype) {
    case CLQ_X_F32: return launch_quant_x<float>(q, s);
    case CLQ_X_BF16: return launch_quant_x<__nv_bfloat16>(q, s);
    case CLQ_X_F16: return launch_quant_x<__half>(q, s);
    default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_dequantize_rows(const int8_t* codes, int64_t ldc, const float* scales, int64_t m, int64_t k, void* out,
                                   int otype, int64_t ldo, cudaStream_t s) {
    switch (otype) {
    case CLQ_X_F32: return launch_dequant<float>(codes, ldc, scales, m, k, out, ldo, s);
    case CLQ_X_BF16: return launch_dequant<__nv_bfloat16>(codes, ldc, scales, m, k, out, ldo, s);
    case CLQ_X_F16: return launch_dequant<__half>(codes, ldc, scales, m, k, out, ldo, s);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace clq
