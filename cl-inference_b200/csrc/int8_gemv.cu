// int8_gemv.cu -- the 8-bit product for up to 16 tokens: every weight byte is
// read once, straight into the registers of an m16n8k32 integer MMA, so the
// kernel is bound by the weight's bytes (and, below a few MB, by latency).
//
// A CTA takes 8 R weight rows; its warps take the 64-byte columns of K in turn
// and add their integer sums in shared memory at the end.  In one 64-byte
// column lane (g, q) = (lane / 4, lane % 4) loads the 16 bytes at 16 q of weight
// row g (eight rows, whole 32-byte sectors) and of token rows g and g + 8.  Words 0
// and 1 of the load are the B (and A) fragments of one MMA, words 2 and 3 those
// of a second: the two operands permute K alike, which a sum does not see.
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

// 16 bytes of the weight stream, read once: past L1, the whole 256-byte L2
// line asked for.  Volatile, so that the loads of a batch stay ahead of its
// MMAs: left to the compiler's order the kernel took 8.3 us for one token at
// 4096 x 4096, and 4.9 with this one (4.4 now).
__device__ __forceinline__ uint4 load_stream(const int8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
// 16 bytes of a token row, zeros where it has none.
__device__ __forceinline__ uint4 load_token(const int8_t* p, bool in) {
    uint4 v;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t"
        "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
        "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
        : "l"(p), "r"((uint32_t)in));
    return v;
}

// Bytes [k0, k0 + 16) of a row of K codes, zeros past its end.
__device__ __forceinline__ uint4 load_tail(const int8_t* row, int64_t k0, int64_t k) {
    if (k0 + 16 <= k) return *reinterpret_cast<const uint4*>(row + k0);
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; k0 + i < k; i++) w[i >> 2] |= (uint32_t)(uint8_t)row[k0 + i] << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// HI: tokens 8..15 are present.  R: groups of eight weight rows to a CTA.  W:
// warps.  U: 64-byte columns a warp has in flight.  LOOSE: rows of any address
// and stride, at twice the loads and their shifts (one token, 4096 x 4096: 8.9 us beside
// 4.4; 14336 x 4096: 28.9 and 11.5).
template <typename OT, int R, bool HI, int W, int U, bool LOOSE>
__global__ void __launch_bounds__(W * 32, 16 / W) int8_gemv_kernel(const Int8Product P) {
    __shared__ int part[W][R][HI ? 4 : 2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int64_t n0 = (int64_t)blockIdx.x * 8 * R;
    // While the previous kernel ends, the columns that the warps load first come
    // into L2, where anything that kernel still writes to them stays visible (a
    // layer of 4096 / 14336 at one token 36.7 -> 35.6 us, of 2048 / 8192 17.4 -> 16.1;
    // whole rows ahead push out the stream's own lines: 41.0).
    if (!LOOSE && threadIdx.x < 8 * R && n0 + threadIdx.x < P.n) {
        const uint32_t bytes = (uint32_t)(P.k < W * U * 64 ? P.k & ~(int64_t)15 : W * U * 64);
        if (bytes) pipe::prefetch_l2(P.w + (n0 + threadIdx.x) * P.ldw, bytes);
    }
    pipe::grid_dependency_wait();
    pipe::allow_dependents();

    const int8_t* wr[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int64_t n = n0 + 8 * r + g;
        wr[r] = P.w + (n < P.n ? n : P.n - 1) * P.ldw;  // rows past the last repeat it and are not written
    }
    const bool lo_in = g < P.m, hi_in = HI && g + 8 < P.m;
    const int8_t* xlo = P.x + (lo_in ? g : 0) * P.ldx;
    const int8_t* xhi = P.x + (hi_in ? g + 8 : 0) * P.ldx;
    int acc[R][4] = {};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    auto column = [&](const uint4 (&w)[R], const uint4& a, const uint4& b) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            mma_s8(acc[r], a.x, b.x, a.y, b.y, w[r].x, w[r].y);
            mma_s8(acc[r], a.z, b.z, a.w, b.w, w[r].z, w[r].w);
        }
    };
    if constexpr (LOOSE) {
        const auto some = [&](int64_t c) {  // one column, wherever it lies
            const int64_t k0 = c * 64 + 16 * q;
            uint4 w[R];
            Codes16 t;
#pragma unroll
            for (int r = 0; r < R; r++) {
                t.load(wr[r], k0, P.k);
                w[r] = t.codes();
            }
            Codes16 lo, hi;
            lo.load(xlo, k0, lo_in ? P.k : 0);
            hi.load(xhi, k0, hi_in ? P.k : 0);
            column(w, lo.codes(), hi.codes());
        };
        // the first column and the last ones have no codes on one side
        const int64_t whole = (P.k - 16) / 64;
        int64_t c = warp;
        if (c == 0 && P.k > 0) {
            some(0);
            c = W;
        }
        for (; c + (U - 1) * W < whole; c += U * W) {
            Codes16 w[U][R], a[U], b[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int64_t k0 = (c + u * W) * 64 + 16 * q;
#pragma unroll
                for (int r = 0; r < R; r++) w[u][r].load_inside(wr[r] + k0);
                a[u].zero();
                b[u].zero();
                if (lo_in) a[u].load_inside(xlo + k0);
                if (hi_in) b[u].load_inside(xhi + k0);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                uint4 v[R];
#pragma unroll
                for (int r = 0; r < R; r++) v[r] = w[u][r].codes();
                column(v, a[u].codes(), b[u].codes());
            }
        }
        for (; c * 64 < P.k; c += W) some(c);
    } else {
        const int64_t whole = P.k / 64;
        int64_t c = warp;
        for (; c + (U - 1) * W < whole; c += U * W) {
            uint4 w[U][R], a[U], b[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int64_t k0 = (c + u * W) * 64 + 16 * q;
#pragma unroll
                for (int r = 0; r < R; r++) w[u][r] = load_stream(wr[r] + k0);
                a[u] = load_token(xlo + k0, lo_in);
                b[u] = HI ? load_token(xhi + k0, hi_in) : zero;
            }
#pragma unroll
            for (int u = 0; u < U; u++) column(w[u], a[u], b[u]);
        }
        for (; c * 64 < P.k; c += W) {  // the last columns, one at a time
            const int64_t k0 = c * 64 + 16 * q;
            uint4 w[R];
#pragma unroll
            for (int r = 0; r < R; r++) w[r] = load_tail(wr[r], k0, P.k);
            column(w, lo_in ? load_tail(xlo, k0, P.k) : zero, hi_in ? load_tail(xhi, k0, P.k) : zero);
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int i = 0; i < (HI ? 4 : 2); i++) part[warp][r][i][lane] = acc[r][i];
    __syncthreads();
    // output (t, 8 r + j): lane 4 (t % 8) + j / 2, register j % 2 + 2 (t / 8)
    OT* out = static_cast<OT*>(P.out);
    for (int e = threadIdx.x; e < (int)P.m * 8 * R; e += W * 32) {
        const int t = e / (8 * R), jn = e % (8 * R), r = jn >> 3, j = jn & 7;
        const int64_t n = n0 + jn;
        if (n >= P.n) continue;
        const int l = 4 * (t & 7) + (j >> 1), i = (j & 1) + (HI ? 2 * (t >> 3) : 0);
        int sum = 0;
#pragma unroll
        for (int w = 0; w < W; w++) sum += part[w][r][i][l];
        float v = int8_scaled(sum, P.ws[n], P.xs[t]);
        if (P.res) v = __fadd_rn(v, P.res[t * P.ldr + n]);
        out[t * P.ldo + n] = int8_round<OT>(v);
    }
}

template <typename OT, int R, int W, int U, bool LOOSE>
cudaError_t launch_gv(const Int8Product& p, cudaStream_t s) {
    const int64_t blocks = (p.n + 8 * R - 1) / (8 * R);
    if (blocks > INT32_MAX) return cudaErrorNotSupported;
    const dim3 grid((unsigned)blocks);
    return p.m > 8 ? pipe::launch_pdl(int8_gemv_kernel<OT, R, true, W, U, LOOSE>, grid, W * 32, 0, s, p)
                   : pipe::launch_pdl(int8_gemv_kernel<OT, R, false, W, U, LOOSE>, grid, W * 32, 0, s, p);
}

// Few rows: eight to a CTA, K over eight warps, so that every SM has a CTA (1024
// x 4096 at one token: 2.3 us; 16 rows to a CTA 3.2).  More: 16 to a CTA, which halves
// what the tokens' rows cost (4096 x 14336: 11.1 us, eight rows 16.6), and from
// four CTAs an SM on four warps, whose longer runs of K keep the loads flowing
// (14336 x 4096: 11.5 us at one token and 14.2 at sixteen, eight warps 12.9 and 14.5).
// Off the grid fewer columns are in flight: each takes twice the registers.
template <typename OT>
cudaError_t launch_gv_type(const Int8Product& p, cudaStream_t s) {
    const int64_t ctas16 = (p.n + 15) / 16, sms = sm_count();
    if (!int8_aligned(p))
        return ctas16 < sms ? launch_gv<OT, 1, 8, 4, true>(p, s) : launch_gv<OT, 2, 8, 2, true>(p, s);
    if (ctas16 < sms) return launch_gv<OT, 1, 8, 8, false>(p, s);
    return ctas16 < 4 * sms ? launch_gv<OT, 2, 8, 4, false>(p, s) : launch_gv<OT, 2, 4, 4, false>(p, s);
}

}  // namespace

cudaError_t launch_int8_gemv(const Int8Product& p, cudaStream_t s) {
    if (p.m > 16) return cudaErrorNotSupported;
    // the second half of the tokens' loads costs a fifth of the rate, the tile kernel 2 us more to
    // start: sixteen tokens at 28672 x 8192 46.9 us here and 41.5 there, at 14336 x 4096 14.2
    // and 13.1, at 4096 x 4096 5.5 and 7.2
    if (int8_aligned(p) && p.m > 8 && p.n * p.k > 40 * 1000 * 1000) return cudaErrorNotSupported;
    switch (p.otype) {
    case CLQ_X_F32: return launch_gv_type<float>(p, s);
    case CLQ_X_BF16: return launch_gv_type<__nv_bfloat16>(p, s);
    case CLQ_X_F16: return launch_gv_type<__half>(p, s);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace clq
