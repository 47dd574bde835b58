// int8_linear.cu -- the product of 8-bit rows (int8_rows.cu):
//   out[t, j] = round(float(sum_c x[t, c] * w[j, c]) * (w scale j) * (x scale t) + residual[t, j])
// with the sum in 32-bit integers, so it is exact and the same however it is
// split.  This file holds the C entry points of the 8-bit operators, the
// choice of a kernel, and the kernel for operands off the 16-byte grid.
#include <cstdint>

#include <cuda_runtime.h>

#include "../../include/clq.h"
#include "clq_internal.h"
#include "int8_mma.cuh"
#include "int8_out.cuh"
#include "launch.cuh"
#include "pipeline.cuh"

namespace clq {
namespace {

// The product for rows of any address and stride, which TMA cannot read.  A CTA
// forms kLT tokens x kLT weight rows from 128-byte columns of both operands: 16
// codes a load, shifted out of the two 16-byte words around them into shared memory
// after the column before has been multiplied (their words are in flight meanwhile),
// rows 144 bytes apart so that the eight of an ldmatrix take different banks.  Each
// of eight warps forms 32 tokens x 16 rows with m16n8k32 integer MMAs.  Bound by L1 (83%
// busy), which passes every word twice: 2048 x 4096 x 4096 290 us, with four bytes of
// products to an instruction 1210, with 64-byte columns, four of them in flight, 365.
constexpr int kLT = 64, kLK = 128, kLPitch = kLK + 16;
__device__ __forceinline__ void load_fragments(uint32_t (&r)[4], const uint8_t* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p)));
}
template <typename OT>
__global__ void __launch_bounds__(256, 2) int8_loose_kernel(const Int8Product P) {
    __shared__ __align__(16) uint8_t sh[2][2][kLT][kLPitch];  // [column parity][tokens, rows]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = tid >> 3, chunk = tid & 7;  // staged: rows row and row + 32 of both, 16 codes each
    const int wt = (warp >> 2) * 32, wn = (warp & 3) * 16;
    const int64_t n0 = (int64_t)blockIdx.x * kLT, columns = (P.k + kLK - 1) / kLK;
    pipe::grid_dependency_wait();
    pipe::allow_dependents();
    for (int64_t t0 = (int64_t)blockIdx.y * kLT; t0 < P.m; t0 += (int64_t)gridDim.y * kLT) {
        const int8_t* src[4];
#pragma unroll
        for (int i = 0; i < 2; i++) {  // rows past the last repeat it and are not written
            src[i] = P.x + min(t0 + row + 32 * i, P.m - 1) * P.ldx;
            src[2 + i] = P.w + min(n0 + row + 32 * i, P.n - 1) * P.ldw;
        }
        Codes16 next[4];
        const auto fetch = [&](int64_t c) {
#pragma unroll
            for (int i = 0; i < 4; i++) next[i].load(src[i], c * kLK + 16 * chunk, P.k);
        };
        const auto stage = [&](int64_t c) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<uint4*>(&sh[c & 1][i >> 1][row + 32 * (i & 1)][16 * chunk]) = next[i].codes();
        };
        int acc[2][2][4] = {};
        if (columns > 0) {
            fetch(0);
            stage(0);
        }
        __syncthreads();
        for (int64_t c = 0; c < columns; c++) {
            if (c + 1 < columns) fetch(c + 1);
            const auto& tokens = sh[c & 1][0];
            const auto& rows = sh[c & 1][1];
#pragma unroll
            for (int kk = 0; kk < kLK; kk += 32) {
                uint32_t a[2][4], b[4];
#pragma unroll
                for (int i = 0; i < 2; i++) load_fragments(a[i], &tokens[wt + 16 * i + (lane & 15)][kk + 16 * (lane >> 4)]);
                load_fragments(b, &rows[wn + (lane & 7) + 8 * (lane >> 4)][kk + 16 * (lane >> 3 & 1)]);
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        mma_s8(acc[i][j], a[i][0], a[i][1], a[i][2], a[i][3], b[2 * j], b[2 * j + 1]);
            }
            if (c + 1 < columns) stage(c + 1);  // the other buffer: read before the last barrier
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int64_t t = t0 + wt + 16 * i + (lane >> 2) + 8 * (e >> 1), n = n0 + wn + 8 * j + 2 * (lane & 3) + (e & 1);
                    if (t >= P.m || n >= P.n) continue;
                    float v = int8_scaled(acc[i][j][e], P.ws[n], P.xs[t]);
                    if (P.res) v = __fadd_rn(v, P.res[t * P.ldr + n]);
                    static_cast<OT*>(P.out)[t * P.ldo + n] = int8_round<OT>(v);
                }
    }
}

cudaError_t launch_int8_loose(const Int8Product& p, cudaStream_t s) {
    const int64_t bx = (p.n + kLT - 1) / kLT, by = (p.m + kLT - 1) / kLT;
    if (bx > INT32_MAX) return cudaErrorInvalidConfiguration;
    const dim3 grid((unsigned)bx, (unsigned)(by < 65535 ? by : 65535));
    switch (p.otype) {
    case CLQ_X_F32: return pipe::launch_pdl(int8_loose_kernel<float>, grid, 256, 0, s, p);
    case CLQ_X_BF16: return pipe::launch_pdl(int8_loose_kernel<__nv_bfloat16>, grid, 256, 0, s, p);
    case CLQ_X_F16: return pipe::launch_pdl(int8_loose_kernel<__half>, grid, 256, 0, s, p);
    default: return cudaErrorInvalidValue;
    }
}

int i8_fail(int code, const char* what) { return set_error(code, "%s", what); }

bool known_type(int t) { return t == CLQ_X_F32 || t == CLQ_X_BF16 || t == CLQ_X_F16; }

// Whether P may hold elements of TYPE: kernels load whole ones.
bool off_type(const void* p, int type) { return (uintptr_t)p % (type == CLQ_X_F32 ? 4 : 2) != 0; }

int check_codes(const char* what, int64_t m, int64_t k, int64_t ld) {
    if (m < 0 || k < 0) return set_error(CLQ_ERR_SHAPE, "%s: negative shape (%lld %lld)", what, (long long)m, (long long)k);
    if (ld < k && m > 1)
        return set_error(CLQ_ERR_SHAPE, "%s: row stride %lld below the row length %lld", what, (long long)ld, (long long)k);
    return CLQ_OK;
}

int run_quantize(const QuantRows& q, void* stream) {
    int dev = 0, rc;
    if (q.m == 0) return CLQ_OK;
    if (q.k > 0 && (!q.x || !q.codes)) return i8_fail(CLQ_ERR_ARGUMENT, "null rows or codes");
    if (!q.scales) return i8_fail(CLQ_ERR_ARGUMENT, "null scales");
    if (off_type(q.x, q.xtype) || off_type(q.gate, q.xtype) || off_type(q.res, q.rtype) || off_type(q.res_out, q.rtype) ||
        off_type(q.norm_w, CLQ_X_F32) || off_type(q.scales, CLQ_X_F32))
        return i8_fail(CLQ_ERR_ARGUMENT, "an address off its element type's alignment");
    if ((rc = sm100_device(&dev))) return rc;
    const cudaError_t e = launch_quantize_rows(q, (cudaStream_t)stream);
    return e == cudaSuccess ? CLQ_OK : set_error(CLQ_ERR_CUDA, "row quantization: %s", cudaGetErrorString(e));
}

}  // namespace

bool int8_aligned(const Int8Product& p) {
    const int64_t strides = (p.m > 1 ? p.ldx : 0) | (p.n > 1 ? p.ldw : 0);  // a single row's is never used
    return !(((uintptr_t)p.x | (uintptr_t)p.w | (uint64_t)strides) & 15);
}

cudaError_t launch_linear_int8(const Int8Product& p, cudaStream_t s) {
    cudaError_t e = launch_int8_gemv(p, s);
    if (e == cudaErrorNotSupported) e = launch_int8_gemm(p, s);
    return e == cudaErrorNotSupported ? launch_int8_loose(p, s) : e;
}

}  // namespace clq

// ---------------------------------------------------------------------------

using clq::i8_fail;

extern "C" {

int clq_quantize_rows_device(const void* x, int xtype, int64_t m, int64_t k, int64_t ldx, int8_t* codes, int64_t ldc,
                             float* scales, void* stream) {
    return clq_norm_quantize_device(x, xtype, m, k, ldx, nullptr, 0.f, nullptr, xtype, 0, nullptr, 0, codes, ldc, scales,
                                    stream);
}

int clq_norm_quantize_device(const void* x, int xtype, int64_t m, int64_t k, int64_t ldx, const float* norm_weight,
                             float norm_epsilon, const void* residual, int rtype, int64_t ldr, void* residual_out,
                             int64_t ldro, int8_t* codes, int64_t ldc, float* scales, void* stream) {
    int rc;
    if (!clq::known_type(xtype)) return clq::set_error(CLQ_ERR_ARGUMENT, "unknown row type %d", xtype);
    if (residual && rtype != xtype && rtype != CLQ_X_F32)
        return clq::set_error(CLQ_ERR_ARGUMENT, "residual type %d beside rows of type %d (the same, or f32)", rtype, xtype);
    if (residual_out && !residual) return i8_fail(CLQ_ERR_ARGUMENT, "a residual output without a residual");
    if ((rc = clq::check_codes("codes", m, k, ldc))) return rc;
    if (ldx < 0 || (residual && ldr < 0)) return i8_fail(CLQ_ERR_SHAPE, "negative row stride");
    if (residual_out && m > 1 && ldro < k)
        return clq::set_error(CLQ_ERR_SHAPE, "residual output stride %lld below the row length %lld", (long long)ldro,
                              (long long)k);
    if (norm_weight && !(norm_epsilon >= 0.f)) return i8_fail(CLQ_ERR_ARGUMENT, "the norm's epsilon must not be negative");
    if (residual_out && residual_out == residual && m > 1 && ldro != ldr)
        return i8_fail(CLQ_ERR_SHAPE, "the residual and its output are one matrix with two row strides");
    if (residual_out && residual_out == x && (rtype != xtype || (m > 1 && ldro != ldx)))
        return i8_fail(CLQ_ERR_SHAPE, "the rows and the residual's output are one matrix with two layouts");
    clq::QuantRows q = {};
    q.x = x;
    q.xtype = xtype;
    q.m = m;
    q.k = k;
    q.ldx = ldx;
    q.norm_w = norm_weight;
    q.eps = norm_epsilon;
    q.res = residual;
    q.rtype = rtype;
    q.ldr = ldr;
    q.res_out = residual_out;
    q.ldro = ldro;
    q.codes = codes;
    q.ldc = ldc;
    q.scales = scales;
    return clq::run_quantize(q, stream);
}

int clq_swiglu_quantize_device(const void* gate, int64_t ldg, const void* up, int64_t ldu, int xtype, int64_t m, int64_t k,
                               int8_t* codes, int64_t ldc, float* scales, void* stream) {
    int rc;
    if (!clq::known_type(xtype)) return clq::set_error(CLQ_ERR_ARGUMENT, "unknown row type %d", xtype);
    if ((rc = clq::check_codes("codes", m, k, ldc))) return rc;
    if (ldg < 0 || ldu < 0) return i8_fail(CLQ_ERR_SHAPE, "negative row stride");
    if (!gate && m > 0 && k > 0) return i8_fail(CLQ_ERR_ARGUMENT, "null gate");
    clq::QuantRows q = {};
    q.x = up;
    q.xtype = xtype;
    q.m = m;
    q.k = k;
    q.ldx = ldu;
    q.gate = gate;
    q.ldg = ldg;
    q.rtype = xtype;
    q.codes = codes;
    q.ldc = ldc;
    q.scales = scales;
    return clq::run_quantize(q, stream);
}

int clq_dequantize_rows_device(const int8_t* codes, int64_t ldc, const float* scales, int64_t m, int64_t k, void* out,
                               int otype, int64_t ldo, void* stream) {
    int rc, dev = 0;
    if (!clq::known_type(otype)) return clq::set_error(CLQ_ERR_ARGUMENT, "unknown output type %d", otype);
    if ((rc = clq::check_codes("codes", m, k, ldc))) return rc;
    if ((rc = clq::check_codes("values", m, k, ldo))) return rc;
    if (m == 0 || k == 0) return CLQ_OK;
    if (!codes || !scales || !out) return i8_fail(CLQ_ERR_ARGUMENT, "null codes, scales or output");
    if (clq::off_type(scales, CLQ_X_F32) || clq::off_type(out, otype))
        return i8_fail(CLQ_ERR_ARGUMENT, "an address off its element type's alignment");
    if ((rc = clq::sm100_device(&dev))) return rc;
    const cudaError_t e = clq::launch_dequantize_rows(codes, ldc, scales, m, k, out, otype, ldo, (cudaStream_t)stream);
    return e == cudaSuccess ? CLQ_OK : clq::set_error(CLQ_ERR_CUDA, "row dequantization: %s", cudaGetErrorString(e));
}

int clq_linear_int8_device(const int8_t* x, int64_t ldx, const float* x_scales, int64_t m, const int8_t* w, int64_t ldw,
                           const float* w_scales, int64_t n, int64_t k, const float* residual, int64_t ldr, void* out,
                           int otype, int64_t ldo, void* stream) {
    int rc, dev = 0;
    if (!clq::known_type(otype)) return clq::set_error(CLQ_ERR_ARGUMENT, "unknown output type %d", otype);
    if ((rc = clq::check_codes("activation codes", m, k, ldx))) return rc;
    if ((rc = clq::check_codes("weight codes", n, k, ldw))) return rc;
    if (k > CLQ_INT8_MAX_K)
        return clq::set_error(CLQ_ERR_UNSUPPORTED, "rows of %lld codes (32-bit sums hold %d)", (long long)k, CLQ_INT8_MAX_K);
    if (m > 1 && (ldo < n || (residual && ldr < n)))
        return clq::set_error(CLQ_ERR_SHAPE, "output or residual stride below %lld columns", (long long)n);
    if (residual && residual == out && (otype != CLQ_X_F32 || (m > 1 && ldr != ldo)))
        return i8_fail(CLQ_ERR_SHAPE, "the residual and the output are one matrix with two layouts");
    if (m == 0 || n == 0) return CLQ_OK;
    if (!out || !x_scales || !w_scales || (k > 0 && (!x || !w))) return i8_fail(CLQ_ERR_ARGUMENT, "null operand or output");
    if (clq::off_type(x_scales, CLQ_X_F32) || clq::off_type(w_scales, CLQ_X_F32) || clq::off_type(residual, CLQ_X_F32) ||
        clq::off_type(out, otype))
        return i8_fail(CLQ_ERR_ARGUMENT, "an address off its element type's alignment");
    if ((rc = clq::sm100_device(&dev))) return rc;
    clq::Int8Product p = {};
    p.x = x;
    p.ldx = ldx;
    p.xs = x_scales;
    p.m = m;
    p.w = w;
    p.ldw = ldw;
    p.ws = w_scales;
    p.n = n;
    p.k = k;
    p.res = residual;
    p.ldr = ldr;
    p.out = out;
    p.otype = otype;
    p.ldo = ldo;
    const cudaError_t e = clq::launch_linear_int8(p, (cudaStream_t)stream);
    return e == cudaSuccess ? CLQ_OK : clq::set_error(CLQ_ERR_CUDA, "8-bit linear: %s", cudaGetErrorString(e));
}

}  // extern "C"
