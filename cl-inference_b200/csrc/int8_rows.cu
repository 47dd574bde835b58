// int8_rows.cu -- rows of activations (or weights) as 8-bit codes with one f32
// scale a row, the operand form of the integer product (int8_linear.cu), and
// the work a decoder layer does between two products fused into the rounding:
//   rows     v = x
//   norm     h = x + residual, v = h * norm_w, s = 1 / sqrt(mean(h^2) + eps)
//            (the RMSNorm of local/blocks.lisp:115-116 after the residual
//            addition of :387-392); residual_out = h
//   SwiGLU   v = silu(gate) * up (:151-154)
// and then, for peak = max |v| of the row,
//   step  = max(FLT_MIN, peak / 127)     as the Q8 codec of local/kv-cache.lisp:37-60
//   code  = clamp(round-half-even(v * (1 / step)), -127, 127), where that codec divides
//   scale = step * s                     (1 for an all-zero row)
// The norm's factor s is common to the row, so the codes need only v and its
// peak, and s enters the scale: one reduction (sum of squares and peak
// together) serves both, and a row is read once, its values held in registers
// between the reduction and the rounding.  Bound by memory for many rows and by
// one round trip and the reduction for few.  A row that holds a non-finite h or v, or whose sum of
// squares leaves f32 at either end, gets codes 0 and the scale NaN, so that every
// product formed with it is NaN.
#include <atomic>
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/clq.h"
#include "clq_internal.h"
#include "int8_out.cuh"
#include "launch.cuh"
#include "pipeline.cuh"

namespace clq {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// silu(g) * u = g / (1 + 2^(-g log2 e)) * u for gates from kFarGate, where the power and
// the reciprocal stay normal numbers (below, anything).  The exponent's product is kept
// in two parts (t and what its rounding left), so that the relative error stays that of
// ex2.approx (2^-22); with rcp.approx (2^-23) and four f32 roundings v is within 10
// roundings of 2^-24.  The library's exponential and an IEEE quotient have 7, and take
// the kernel, which instructions bound, from 37 us to 58 (2048 rows of 14336 bf16, where
// 4 codes of 29 million then differ).  A gate that is NaN or infinite gives NaN or an
// infinity.
constexpr float kFarGate = -87.f;
__device__ __forceinline__ float silu_near(float g, float u) {
    constexpr float kLog2e = 1.44269504f, kLog2eLow = 1.92596303e-8f, kLn2 = 0.693147181f;
    const float n = -fminf(g, 200.f);
    const float t = __fmul_rn(n, kLog2e);
    const float low = fmaf(n, kLog2eLow, fmaf(n, kLog2e, -t));
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    const float d = 1.f + fmaf(e, low * kLn2, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return __fmul_rn(__fmul_rn(g, r), u);
}
// And below, where 1 + e^-g is e^-g to f32 and may leave it: g e^g u, the power as two
// factors around u, so that a gate's tail times a large u is kept: within 11 roundings
// (two of the exponential's 2^-22 and three products) and, past -174, where e^(g/2) is
// subnormal, 2^-137 for any u.  -infinity gives NaN.
__device__ __forceinline__ float silu_far(float g, float u) {
    const float h = expf(0.5f * g);
    return __fmul_rn(__fmul_rn(__fmul_rn(g, h), u), h);
}
// V values of it over the u, the far gates behind one branch: a step seldom holds any
// (2048 x 14336 bf16 36.4 us at that step, without far gates 35.8; 38.0 with selects in
// every element, 37.6 with one branch after a thread's whole share).
template <int V>
__device__ __forceinline__ void silu_times(const float (&g)[V], float (&u)[V]) {
    bool far = false;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        far = far || g[j] < kFarGate;
        v[j] = silu_near(g[j], u[j]);
    }
    if (far) {
#pragma unroll
        for (int j = 0; j < V; j++)
            if (g[j] < kFarGate) v[j] = silu_far(g[j], u[j]);
    }
#pragma unroll
    for (int j = 0; j < V; j++) u[j] = v[j];
}

// max(a, |v|), NaN once either is.
__device__ __forceinline__ float peak_of(float a, float v) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(fabsf(v)));
    return m;
}

enum { kPlain, kNorm, kSwiglu };

// V values of v in place of X's, the peak and, for a norm, the sum of squares of h.
template <int MODE, int V>
__device__ __forceinline__ void values_of(float (&x)[V], const float (&other)[V], const float (&w)[V], float& ss, float& peak) {
    if constexpr (MODE == kSwiglu) silu_times(other, x);
#pragma unroll
    for (int j = 0; j < V; j++) {
        if constexpr (MODE != kSwiglu) x[j] = __fadd_rn(x[j], other[j]);
        if constexpr (MODE == kNorm) {
            ss = fmaf(x[j], x[j], ss);
            x[j] = __fmul_rn(x[j], w[j]);
        }
        peak = peak_of(peak, x[j]);
    }
}

struct RowScale {
    float inv, scale;  // v * inv rounds to the code; inv is 0 for a row of codes 0
};
template <int MODE>
__device__ __forceinline__ RowScale row_scale(const QuantRows& Q, float ss, float peak) {
    bool fine = peak < INFINITY;  // not NaN either
    float s = 1.f;
    if constexpr (MODE == kNorm) {
        // Squares under 2^-126 lose bits, 2^-150 of the mean at most and as much in its
        // rounding: no more than 2^-24 of a sum with eps that reaches 2^-125.
        const float mean = __fadd_rn(__fdiv_rn(ss, (float)Q.k), Q.eps);
        s = __fdiv_rn(1.f, __fsqrt_rn(mean));
        fine = fine && ss < INFINITY && (mean >= 2.f * FLT_MIN || peak == 0.f);
    }
    const float step = fmaxf(FLT_MIN, __fdiv_rn(peak, 127.f));
    RowScale r;
    r.inv = fine ? __fdiv_rn(1.f, step) : 0.f;
    r.scale = !fine ? NAN : peak > 0.f ? __fmul_rn(step, s) : 1.f;
    return r;
}
// The code in the low byte: v * inv, itself rounded to f32 (at most 127 (1 + 2^-22) in
// size), lands in the low bits of a float of 2^23, rounded half to even by the
// addition.  The two steps stay apart: one fma takes values on the border of two
// codes to another one than the rule above (58 of 2048 x 14336 normal bf16 values), at 1 to 3% of
// the time (those rows 18.4 us, so 19.0; 1024 x 8192 f32 9.2 and 9.4).
__device__ __forceinline__ uint32_t code_bits(float v, float inv) {
    return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.f));
}

// ---- rows held in registers -------------------------------------------------

// VALUES consecutive elements of T as they lie in memory: one, or VALUES * sizeof(T) a
// multiple of 16 bytes with the address on 16.  Kept so until a batch of loads is
// under way: a conversion beside each of them waits for it (2048 rows of 4097
// bf16, an element at a time: 42 us).
template <typename T, int VALUES>
struct Packed {
    static constexpr int E = 16 / (int)sizeof(T);
    uint4 w[VALUES / E] = {};
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < VALUES / E; i++) w[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void unpack(float (&f)[VALUES]) const {
#pragma unroll
        for (int i = 0; i < VALUES / E; i++) {
            const T* e = reinterpret_cast<const T*>(&w[i]);
#pragma unroll
            for (int j = 0; j < E; j++) f[i * E + j] = to_f32(e[j]);
        }
    }
};
template <typename T>
struct Packed<T, 1> {
    T v = T(0.f);
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ void unpack(float (&f)[1]) const { f[0] = to_f32(v); }
};
template <typename T, int VALUES>
__device__ __forceinline__ void load_values(const T* p, float (&f)[VALUES]) {
    Packed<T, VALUES> a;
    a.load(p);
    a.unpack(f);
}
template <typename T, int VALUES>
__device__ __forceinline__ void store_values(T* p, const float (&f)[VALUES]) {
    if constexpr (VALUES == 1) {
        *p = int8_round<T>(f[0]);
    } else {
        constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < VALUES / E; i++) {
            uint4 w;
            T* e = reinterpret_cast<T*>(&w);
#pragma unroll
            for (int j = 0; j < E; j++) e[j] = int8_round<T>(f[i * E + j]);
            reinterpret_cast<uint4*>(p)[i] = w;
        }
    }
}

// The row's (sum of squares, peak) over a warp, the same in each lane.
__device__ __forceinline__ float2 row_reduce_warp(float ss, float peak) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    // NaN's bits are the largest
    return make_float2(ss, __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(peak))));
}
// And over a CTA of WARPS warps; RED: that many entries of shared memory, not
// in use by an earlier call that some thread may still be in.
__device__ __forceinline__ float2 row_reduce_cta(float ss, float peak, float2* red, int warps) {
    const int lane = threadIdx.x & 31;
    const float2 mine = row_reduce_warp(ss, peak);
    if (lane == 0) red[threadIdx.x >> 5] = mine;
    __syncthreads();
    const float2 a = lane < warps ? red[lane] : make_float2(0.f, 0.f);
    return row_reduce_warp(a.x, a.y);
}

// The codes of V values at P (on 4 or 8 bytes for V = 4 or 8); zeros for inv 0,
// whose values may be anything.
template <int V>
__device__ __forceinline__ void store_codes(int8_t* p, const float (&v)[V], float inv) {
    if constexpr (V == 1) {
        *p = inv > 0.f ? (int8_t)code_bits(v[0], inv) : (int8_t)0;
    } else {
        uint32_t w[V / 4] = {};
        if (inv > 0.f) {  // the same for the whole row
#pragma unroll
            for (int q = 0; q < V / 4; q++) {
                uint32_t b[4];
#pragma unroll
                for (int j = 0; j < 4; j++) b[j] = code_bits(v[4 * q + j], inv);
                w[q] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            }
        }
        if constexpr (V == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
        else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    }
}

constexpr int kSmallRow = 128;  // threads of a CTA that takes a row per warp

// CTAs an SM holds: 16 values a thread leave room for 1024 to 1280 threads, 32
// for 1024 of f32 rows and 512 of 16-bit ones, 64 for 512.  Element by element, 1024
// (more spill: 2048 x 4095 f32 norm 24.6 us, 21.4 so) and three CTAs of 384.
template <typename XT, int V, int G, int C>
constexpr int min_ctas() {
    constexpr int values = C * V, threads = G == 32 ? kSmallRow : G;
    constexpr bool f32 = sizeof(XT) == 4;
    constexpr int at_once = V == 1                   ? threads == 384 ? 1152 : 1024
                            : values > (f32 ? 32 : 16) ? 512
                            : values <= 16 && f32      ? 1280
                                                       : 1024;
    return threads < at_once ? at_once / threads : 1;
}

// The elements of a step: 16 bytes of x, or one where rows may have any base,
// stride and length (neighbouring lanes then take neighbouring elements, which
// keeps single-element accesses whole and free of bank conflicts).
template <typename XT, bool LOOSE>
constexpr int step_of = LOOSE ? 1 : 16 / (int)sizeof(XT);

// G threads a row, C steps of V elements a thread, step c of thread i at element
// (c G + i) V.
template <typename XT, typename RT, int MODE, bool LOOSE, int G, int C>
__global__ void __launch_bounds__(G == 32 ? kSmallRow : G, min_ctas<XT, step_of<XT, LOOSE>, G, C>())
    quantize_rows_kernel(const QuantRows Q) {
    constexpr int V = step_of<XT, LOOSE>;
    __shared__ float2 red[G == 32 ? 1 : G / 32];
    pipe::grid_dependency_wait();
    pipe::allow_dependents();
    const int64_t row = G == 32 ? blockIdx.x * (int64_t)(kSmallRow / 32) + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
    if (row >= Q.m) return;  // whole warps, and only where no barrier follows
    const int tid = G == 32 ? threadIdx.x & 31 : threadIdx.x;
    const XT* x = static_cast<const XT*>(Q.x) + row * Q.ldx;
    // gate (of type RT too) or residual
    const RT* other = MODE == kSwiglu ? static_cast<const RT*>(Q.gate) + row * Q.ldg
                      : Q.res         ? static_cast<const RT*>(Q.res) + row * Q.ldr
                                      : nullptr;
    float v[C][V];
    float ss = 0.f, peak = 0.f;
    const int k = (int)Q.k;
    RT* res_out = Q.res_out ? static_cast<RT*>(Q.res_out) + row * Q.ldro : nullptr;
    // steps whose loads are in flight before any is used (two where 64 values fill the registers)
    constexpr int B = C < 4 || V == 1 ? C : V * C > 32 && V == 8 ? 2 : 4;
#pragma unroll
    for (int c0 = 0; c0 < C; c0 += B) {
        Packed<XT, V> xp[B];
        Packed<RT, V> op[B];  // residual or gate
#pragma unroll
        for (int b = 0; b < B; b++) {
            const int i = ((c0 + b) * G + tid) * V;
            if (i < k) {
                xp[b].load(x + i);
                if constexpr (MODE == kSwiglu) op[b].load(other + i);
            }
        }
        if (MODE != kSwiglu && other) {
#pragma unroll
            for (int b = 0; b < B; b++) {
                const int i = ((c0 + b) * G + tid) * V;
                if (i < k) op[b].load(other + i);
            }
        }
#pragma unroll
        for (int b = 0; b < B; b++) {
            const int i = ((c0 + b) * G + tid) * V;
            float o[V];
            xp[b].unpack(v[c0 + b]);
            op[b].unpack(o);
            if (MODE != kSwiglu && !other) {
#pragma unroll
                for (int j = 0; j < V; j++) o[j] = -0.f;  // x + -0 is x, its sign kept
            }
            if (MODE != kSwiglu && res_out && i < k) {
                float h[V];
#pragma unroll
                for (int j = 0; j < V; j++) h[j] = __fadd_rn(v[c0 + b][j], o[j]);
                store_values<RT, V>(res_out + i, h);
            }
            float w[V];
#pragma unroll
            for (int j = 0; j < V; j++) w[j] = 0.f;
            if constexpr (MODE == kNorm) {
                if (i < k) load_values<float, V>(Q.norm_w + i, w);
            }
            values_of<MODE>(v[c0 + b], o, w, ss, peak);
        }
    }
    const float2 sums = G == 32 ? row_reduce_warp(ss, peak) : row_reduce_cta(ss, peak, red, G / 32);
    const RowScale r = row_scale<MODE>(Q, sums.x, sums.y);
    if (tid == 0) Q.scales[row] = r.scale;
    int8_t* codes = Q.codes + row * Q.ldc;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int i = (c * G + tid) * V;
        if (i >= k) continue;
        store_codes<V>(codes + i, v[c], r.inv);
    }
}

// ---- many rows, streamed through shared memory ------------------------------

// In a peak's place, from a thread whose wait for its row gave up: every thread of the CTA
// then finds it in the reduced peak (the bits are above those of any peak, NaN included).
constexpr uint32_t kGaveUp = 0xffffffffu;
constexpr int kStreamStages = 4;
constexpr int kStreamHeader = 1024;  // barriers and two rows' reductions
// Threads of a CTA at most: rows off the grid, whose reads are longer, gain by more
// of them (SwiGLU of 700 x 20001 bf16 26.1 us, with 512 31.3), the others lose (2048 x
// 14336 37.5, with 1024 49).
constexpr int stream_threads(bool loose) { return loose ? 1024 : 512; }
constexpr int stream_values(bool loose) { return loose ? 32 : 64; }  // of a thread at most

// W[0, N) = the N words that start BYTES (under 16) into W[0, N + 4).
template <int N, bool ODD_HALVES>
__device__ __forceinline__ void shift_words(uint32_t (&w)[N + 4], uint32_t bytes) {
    if (bytes & 8) {
#pragma unroll
        for (int j = 0; j < N + 2; j++) w[j] = w[j + 2];
    }
    if (bytes & 4) {
#pragma unroll
        for (int j = 0; j < N + 1; j++) w[j] = w[j + 1];
    }
    if constexpr (ODD_HALVES) {
#pragma unroll
        for (int j = 0; j < N; j++) w[j] = __funnelshift_r(w[j], w[j + 1], (bytes & 2) * 8);
    }
}

// A row in global memory and its copy in shared memory, which keeps the row's
// distance from the 16-byte grid (OFF bytes): the bulk copy takes the whole
// 16-byte words, and the ends, under 16 bytes each, go element by element.
// Reads take the words around a step of V elements and shift them.
template <typename T, int V, bool LOOSE>
struct StagedRow {
    const T* g;
    uint8_t* s;           // 16-byte aligned; element 0 lies OFF bytes in
    uint32_t off;
    uint32_t head, body;  // elements before the words, and in them

    __device__ __forceinline__ StagedRow(const void* base, int64_t row, int64_t ld, int k, uint8_t* buf) : s(buf) {
        g = static_cast<const T*>(base) + row * ld;
        off = LOOSE ? (uint32_t)reinterpret_cast<uintptr_t>(g) & 15u : 0u;
        head = LOOSE ? min((uint32_t)k, ((16u - off) & 15u) / (uint32_t)sizeof(T)) : 0u;
        body = LOOSE ? ((uint32_t)k - head) / (16u / sizeof(T)) * (16u / sizeof(T)) : (uint32_t)k;
    }
    __device__ __forceinline__ uint32_t bytes() const { return body * (uint32_t)sizeof(T); }
    __device__ __forceinline__ void copy(uint64_t* bar) const {
        if (body) pipe::bulk_copy(s + off + head * sizeof(T), g + head, bytes(), bar);
    }
    // The element of the ends that LANE (0 .. 15) brings, or K for none.
    __device__ __forceinline__ uint32_t end_element(uint32_t lane, uint32_t k) const {
        return lane < 8 ? (lane < head ? lane : k) : min(k, head + body + lane - 8);
    }
    __device__ __forceinline__ T* place(uint32_t i) const { return reinterpret_cast<T*>(s + off) + i; }
    __device__ __forceinline__ void load(int i, int k, float (&f)[V]) const {
        if constexpr (!LOOSE) {
            load_values<T, V>(reinterpret_cast<const T*>(s) + i, f);
        } else {
            constexpr int N = V * (int)sizeof(T) / 4;
            uint32_t w[N + 4];
            const uint4* q = reinterpret_cast<const uint4*>(s + (size_t)i * sizeof(T));
#pragma unroll
            for (int n = 0; n <= N / 4; n++) {
                const uint4 u = q[n];
                w[4 * n] = u.x;
                w[4 * n + 1] = u.y;
                w[4 * n + 2] = u.z;
                w[4 * n + 3] = u.w;
            }
            shift_words<N, sizeof(T) == 2>(w, off);
            const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
            for (int j = 0; j < V; j++) f[j] = i + j < k ? to_f32(e[j]) : 0.f;
        }
    }
};
// Bytes of a buffer for K elements (a multiple of a step) of SIZE bytes, with
// the word that a shifted read looks ahead.
__host__ __device__ constexpr uint32_t staged_bytes(int64_t k, int size) {
    return (uint32_t)((k * size + 15) / 16 * 16 + 16);
}

// Elements I .. I + V - 1 of the row of K at P, which may lie anywhere, by a whole
// warp whose lanes hold neighbouring steps: each lane stores the 16-byte words
// that start within its step, the last of them completed from the next lane;
// what no word covers goes element by element.
template <typename T, int V>
__device__ __forceinline__ void store_shifted(T* p, int i, int k, const float (&f)[V]) {
    constexpr int N = V * (int)sizeof(T) / 4, E = 16 / (int)sizeof(T);
    const int lane = threadIdx.x & 31;
    __align__(16) T mine[V];
#pragma unroll
    for (int j = 0; j < V; j++) mine[j] = int8_round<T>(f[j]);
    uint32_t w[N + 4];
#pragma unroll
    for (int j = 0; j < N; j++) w[j] = reinterpret_cast<const uint32_t*>(mine)[j];
#pragma unroll
    for (int j = 0; j < 4; j++) w[N + j] = __shfl_down_sync(0xffffffffu, w[j], 1);
    const uint32_t skip = (16u - ((uint32_t)reinterpret_cast<uintptr_t>(p) & 15u)) & 15u;  // bytes before the first word
    const int first = (int)(skip / sizeof(T));
    const bool words = skip == 0 ? i + V <= k : lane < 31 && i + V + E <= k;
    const bool led = skip == 0 || (lane > 0 && i + E <= k);  // the lane before writes this one's first elements
    if (words) {
        shift_words<N, sizeof(T) == 2>(w, skip);
        uint4* q = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p + i) + skip);
#pragma unroll
        for (int n = 0; n < N / 4; n++) q[n] = make_uint4(w[4 * n], w[4 * n + 1], w[4 * n + 2], w[4 * n + 3]);
    }
    if (!words || !led) {
#pragma unroll
        for (int j = 0; j < V; j++)
            if (i + j < k && (j < first ? !led : !words)) p[i + j] = mine[j];
    }
}

// CTA b takes rows b, b + gridDim.x, ..: row r's operands are copied into one of
// STAGES buffers by the bulk-copy engine while earlier rows are computed, so the
// memory never waits for the arithmetic (with a CTA per row the two took turns:
// SwiGLU of 2048 x 14336 bf16 44 us, so 37.5, against 22.4 of traffic).  A buffer is
// free once the row's reduction has passed its barrier: every thread then holds
// its values in registers.  LOOSE: rows of any base, stride and length, put back
// on the grid from shared memory.  WTS_HELD: the norm weight is kept there too.
template <typename XT, typename RT, int MODE, bool LOOSE, int C>
__global__ void __launch_bounds__(stream_threads(LOOSE), !LOOSE && C * 16 / (int)sizeof(XT) <= 32 ? 2 : 1)
    quantize_stream_kernel(const QuantRows Q, int stages, bool wts_held, int* err) {
    constexpr int kStreamThreads = stream_threads(LOOSE);
    constexpr int V = 16 / (int)sizeof(XT);
    extern __shared__ __align__(128) uint8_t sh[];
    uint64_t* full = reinterpret_cast<uint64_t*>(sh);
    float2* red = reinterpret_cast<float2*>(sh + 64);  // [2][kStreamThreads / 32]
    const int k = (int)Q.k, kv = (k + V - 1) / V * V, G = (int)blockDim.x, tid = (int)threadIdx.x;
    const bool two = MODE == kSwiglu || Q.res;
    const uint32_t xb = staged_bytes(kv, sizeof(XT)), stage = xb + (two ? staged_bytes(kv, sizeof(RT)) : 0u);
    float* wts = reinterpret_cast<float*>(sh + kStreamHeader);
    uint8_t* buf = sh + kStreamHeader + (MODE == kNorm && wts_held ? staged_bytes(kv, 4) : 0u);
    const void* other = MODE == kSwiglu ? Q.gate : Q.res;
    const int64_t other_ld = MODE == kSwiglu ? Q.ldg : Q.ldr;
    const auto x_row = [&](int64_t row, int s) {
        return StagedRow<XT, V, LOOSE>(Q.x, row, Q.ldx, k, buf + (size_t)s * stage);
    };
    const auto o_row = [&](int64_t row, int s) {
        return StagedRow<RT, V, LOOSE>(other, row, other_ld, k, buf + (size_t)s * stage + xb);
    };
    // Warp 0 brings the ends of a row that is off the grid: lanes 0-15 x's, 16-31 the
    // other operand's, fetched ahead of the time at which the buffer is free.
    XT x_end{};
    RT o_end{};
    const auto fetch_ends = [&](int64_t row) {
        if (!LOOSE || tid >= 32 || row >= Q.m) return;
        if (tid < 16) {
            const auto r = x_row(row, 0);
            const uint32_t e = r.end_element(tid, k);
            if (e < (uint32_t)k) x_end = r.g[e];
        } else if (two) {
            const auto r = o_row(row, 0);
            const uint32_t e = r.end_element(tid - 16, k);
            if (e < (uint32_t)k) o_end = r.g[e];
        }
    };
    const uint32_t wts_bytes = MODE == kNorm && wts_held ? (uint32_t)k / 4 * 16 : 0u;
    const auto issue = [&](int64_t row, int s, bool first) {  // by warp 0
        if (row >= Q.m) return;
        const auto x = x_row(row, s);
        const auto o = o_row(two ? row : 0, s);
        if (LOOSE && tid < 16) {
            const uint32_t e = x.end_element(tid, k);
            if (e < (uint32_t)k) *x.place(e) = x_end;
        } else if (LOOSE && two) {
            const uint32_t e = o.end_element(tid - 16, k);
            if (e < (uint32_t)k) *o.place(e) = o_end;
        }
        // a later row's bulk copy may write where an end lies now
        if (LOOSE) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (tid == 0) {
            pipe::mbar_arrive_tx(&full[s], x.bytes() + (two ? o.bytes() : 0u) + (first ? wts_bytes : 0u));
            x.copy(&full[s]);
            if (two) o.copy(&full[s]);
            if (first && wts_bytes) pipe::bulk_copy(wts, Q.norm_w, wts_bytes, &full[s]);
        }
    };
    if (tid == 0) {
        for (int s = 0; s < stages; s++) pipe::mbar_init(&full[s], 1);
        pipe::mbar_init_fence();
    }
    pipe::grid_dependency_wait();
    pipe::allow_dependents();
    if (wts_bytes && tid < k % 4) wts[k - 1 - tid] = Q.norm_w[k - 1 - tid];
    if (tid < 32) {
        for (int s = 0; s < stages; s++) {
            fetch_ends(blockIdx.x + (int64_t)s * gridDim.x);
            issue(blockIdx.x + (int64_t)s * gridDim.x, s, s == 0);
        }
    }
    __syncthreads();
    int s = 0, turn = 0;
    uint32_t parity = 0;
    for (int64_t row = blockIdx.x; row < Q.m; row += gridDim.x, turn ^= 1) {
        const int64_t next = row + (int64_t)stages * gridDim.x;
        fetch_ends(next);
        // without it, the values formed below are of whatever the buffer holds, and not used
        bool here = pipe::mbar_wait(&full[s], parity, err);
        if (LOOSE && MODE != kSwiglu) here = __all_sync(0xffffffffu, here);  // store_shifted takes whole warps
        const auto x = x_row(row, s);
        const auto o = o_row(two ? row : 0, s);
        RT* res_out = Q.res_out ? static_cast<RT*>(Q.res_out) + row * Q.ldro : nullptr;
        float v[C][V];
        float ss = 0.f, peak = 0.f;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int i = (c * G + tid) * V;
            float ov[V], w[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                v[c][j] = w[j] = 0.f;
                ov[j] = MODE == kSwiglu ? 0.f : -0.f;
            }
            if (i < k) {
                x.load(i, k, v[c]);
                if (two) o.load(i, k, ov);
                if constexpr (MODE == kNorm) {
                    if (wts_held) {
                        load_values<float, V>(wts + i, w);
                    } else if (reinterpret_cast<uintptr_t>(Q.norm_w) % 16 == 0 && i + V <= k) {
                        load_values<float, V>(Q.norm_w + i, w);
                    } else {
#pragma unroll
                        for (int j = 0; j < V; j++) w[j] = i + j < k ? Q.norm_w[i + j] : 0.f;
                    }
                    if (LOOSE && i + V > k) {  // past the end the held copy has whatever was there
#pragma unroll
                        for (int j = 0; j < V; j++) w[j] = i + j < k ? w[j] : 0.f;
                    }
                }
            }
            if (MODE != kSwiglu && res_out && here) {
                float h[V];
#pragma unroll
                for (int j = 0; j < V; j++) h[j] = __fadd_rn(v[c][j], ov[j]);
                if constexpr (LOOSE) store_shifted<RT, V>(res_out, i, k, h);
                else if (i < k) store_values<RT, V>(res_out + i, h);
            }
            values_of<MODE>(v[c], ov, w, ss, peak);
        }
        if (!here) peak = __uint_as_float(kGaveUp);
        const float2 sums = row_reduce_cta(ss, peak, red + turn * (kStreamThreads / 32), G / 32);
        if (__float_as_uint(sums.y) == kGaveUp) {
            // nothing more is copied, read or written; what is in flight lands before the CTA exits
            for (int i = 0; tid == 0 && i < stages && row + (int64_t)i * gridDim.x < Q.m; i++) {
                const bool wrapped = s + i >= stages;
                pipe::mbar_drain(&full[wrapped ? s + i - stages : s + i], parity ^ (wrapped ? 1u : 0u));
            }
            return;
        }
        if (tid < 32) issue(next, s, false);
        if (LOOSE && stages == 1) __syncthreads();  // the ends just written are read in the next turn
        if (++s == stages) {
            s = 0;
            parity ^= 1;
        }
        const RowScale r = row_scale<MODE>(Q, sums.x, sums.y);
        if (tid == 0) Q.scales[row] = r.scale;
        int8_t* codes = Q.codes + row * Q.ldc;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int i = (c * G + tid) * V;
            if (i >= k) continue;
            if (!LOOSE || (i + V <= k && reinterpret_cast<uintptr_t>(codes) % V == 0)) {
                store_codes<V>(codes + i, v[c], r.inv);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (i + j < k) codes[i + j] = r.inv > 0.f ? (int8_t)code_bits(v[c][j], r.inv) : (int8_t)0;
            }
        }
    }
}

// ---- rows longer than the registers of a CTA hold --------------------------

// Two passes over the row (the second mostly from L2); the residual's sum is
// written in the second, when its row has been read for the last time by then.
constexpr int kLongThreads = 1024;
template <typename XT, typename RT, int MODE>
__global__ void __launch_bounds__(kLongThreads) quantize_long_rows_kernel(const QuantRows Q) {
    __shared__ float2 red[kLongThreads / 32];
    pipe::grid_dependency_wait();
    pipe::allow_dependents();
    const int64_t row = blockIdx.x;
    const XT* x = static_cast<const XT*>(Q.x) + row * Q.ldx;
    const XT* gate = MODE == kSwiglu ? static_cast<const XT*>(Q.gate) + row * Q.ldg : nullptr;
    const RT* res = Q.res ? static_cast<const RT*>(Q.res) + row * Q.ldr : nullptr;
    RT* res_out = Q.res_out ? static_cast<RT*>(Q.res_out) + row * Q.ldro : nullptr;
    const auto other = [&](int64_t i) { return MODE == kSwiglu ? to_f32(gate[i]) : res ? to_f32(res[i]) : -0.f; };
    float ss = 0.f, peak = 0.f;
    const auto value = [&](float a, float o, int64_t i) {
        float v[1] = {a};
        const float others[1] = {o}, w[1] = {MODE == kNorm ? Q.norm_w[i] : 0.f};
        values_of<MODE>(v, others, w, ss, peak);
        return v[0];
    };
    for (int64_t i = threadIdx.x; i < Q.k; i += kLongThreads) value(to_f32(x[i]), other(i), i);
    const float2 sums = row_reduce_cta(ss, peak, red, kLongThreads / 32);
    const RowScale r = row_scale<MODE>(Q, sums.x, sums.y);
    if (threadIdx.x == 0) Q.scales[row] = r.scale;
    int8_t* codes = Q.codes + row * Q.ldc;
    for (int64_t i = threadIdx.x; i < Q.k; i += kLongThreads) {
        const float a = to_f32(x[i]), o = other(i);
        if (MODE != kSwiglu && res_out) res_out[i] = int8_round<RT>(__fadd_rn(a, o));
        const float v = value(a, o, i);
        codes[i] = r.inv > 0.f ? (int8_t)code_bits(v, r.inv) : (int8_t)0;
    }
}

// ---- codes back to values ---------------------------------------------------

// R rows of one chunk of 16 codes a thread, rows on the 16-byte grid.
template <typename OT, int R>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(const int8_t* __restrict__ codes, int64_t ldc,
                                                              const float* __restrict__ scales, int64_t m, int64_t k,
                                                              OT* __restrict__ out, int64_t ldo) {
    constexpr int V = 16;
    pipe::grid_dependency_wait();
    pipe::allow_dependents();
    const int64_t i = (blockIdx.y * (int64_t)blockDim.x + threadIdx.x) * V, r0 = (int64_t)blockIdx.x * R;
    if (i >= k) return;
    __align__(16) int8_t c[R][V];
    float s[R];
    const bool whole = i + V <= k;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const bool in = r0 + r < m;
        const int8_t* p = codes + (in ? r0 + r : r0) * ldc + i;
        s[r] = in ? scales[r0 + r] : 0.f;
        if (whole) {
            *reinterpret_cast<uint4*>(c[r]) = *reinterpret_cast<const uint4*>(p);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) c[r][j] = i + j < k ? p[j] : (int8_t)0;
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        if (r0 + r >= m) return;
        OT* o = out + (r0 + r) * ldo + i;
        float f[V];
#pragma unroll
        for (int j = 0; j < V; j++) f[j] = __fmul_rn((float)c[r][j], s[r]);
        if (whole) {
            store_values<OT, V>(o, f);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (i + j < k) o[j] = int8_round<OT>(f[j]);
        }
    }
}

// Rows of any base, stride and length: a thread writes one 16-byte word of the
// output (E values), whose codes lie anywhere; a last thread writes the row's ends.
template <typename OT>
__global__ void __launch_bounds__(256) dequantize_loose_kernel(const int8_t* __restrict__ codes, int64_t ldc,
                                                               const float* __restrict__ scales, int64_t k,
                                                               OT* __restrict__ out, int64_t ldo) {
    constexpr int E = 16 / (int)sizeof(OT);
    pipe::grid_dependency_wait();
    pipe::allow_dependents();
    const int64_t row = blockIdx.x;
    const int8_t* c = codes + row * ldc;
    OT* o = out + row * ldo;
    const float s = scales[row];
    const int64_t to_grid = (int64_t)((16 - (reinterpret_cast<uintptr_t>(o) & 15)) & 15) / (int)sizeof(OT);
    const int64_t head = to_grid < k ? to_grid : k, words = (k - head) / E;
    const int64_t q = blockIdx.y * (int64_t)blockDim.x + threadIdx.x;
    if (q < words) {
        const int64_t i = head + q * E;
        const uintptr_t at = reinterpret_cast<uintptr_t>(c + i);
        const uint32_t off = (uint32_t)at & 3u;
        uint32_t w[E / 4 + 1];
        float f[E];
        if (i >= 4 && i + E + 4 <= k) {  // whole 4-byte words of this row, shifted
            const uint32_t* p = reinterpret_cast<const uint32_t*>(at - off);
#pragma unroll
            for (int j = 0; j <= E / 4; j++) w[j] = p[j];
#pragma unroll
            for (int j = 0; j < E / 4; j++) w[j] = __funnelshift_r(w[j], w[j + 1], off * 8);
#pragma unroll
            for (int j = 0; j < E; j++) f[j] = __fmul_rn((float)(int8_t)(w[j / 4] >> (8 * (j % 4))), s);
        } else {
#pragma unroll
            for (int j = 0; j < E; j++) f[j] = __fmul_rn((float)c[i + j], s);
        }
        store_values<OT, E>(o + i, f);
    } else if (q == words) {
        for (int64_t i = 0; i < head; i++) o[i] = int8_round<OT>(__fmul_rn((float)c[i], s));
        for (int64_t i = head + words * E; i < k; i++) o[i] = int8_round<OT>(__fmul_rn((float)c[i], s));
    }
}

// ---- host -------------------------------------------------------------------

template <typename XT, typename RT, int MODE, bool LOOSE, int G, int C>
cudaError_t launch_held(const QuantRows& q, cudaStream_t s) {
    constexpr int kPerCta = G == 32 ? kSmallRow / 32 : 1;
    const int64_t blocks = (q.m + kPerCta - 1) / kPerCta;
    if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
    return pipe::launch_pdl(quantize_rows_kernel<XT, RT, MODE, LOOSE, G, C>, dim3((unsigned)blocks), G == 32 ? kSmallRow : G, 0, s,
                            q);
}

template <typename XT, typename RT, int MODE>
cudaError_t launch_long(const QuantRows& q, cudaStream_t s) {
    if (q.m > INT32_MAX) return cudaErrorInvalidConfiguration;
    return pipe::launch_pdl(quantize_long_rows_kernel<XT, RT, MODE>, dim3((unsigned)q.m), kLongThreads, 0, s, q);
}

template <typename XT, typename RT, int MODE, bool LOOSE, int C>
cudaError_t launch_stream(const QuantRows& q, int threads, int stages, bool wts_held, int ctas, size_t smem, cudaStream_t s) {
    static std::atomic<uint64_t> allowed{0};
    int* err = device_status_word();
    if (!err) return cudaErrorUnknown;
    const cudaError_t e = pipe::allow_smem(quantize_stream_kernel<XT, RT, MODE, LOOSE, C>, pipe::kSmemPerSm, allowed);
    if (e != cudaSuccess) return e;
    const int64_t at_once = (int64_t)ctas * sm_count();
    return pipe::launch_pdl(quantize_stream_kernel<XT, RT, MODE, LOOSE, C>, dim3((unsigned)(q.m < at_once ? q.m : at_once)),
                            threads, smem, s, q, stages, wts_held, err);
}

// The streaming kernel with as many CTAs to an SM (up to eight) as leave each of
// them two buffers and, together, 1024 threads; one buffer, and the norm weight read
// from global memory, where rows are too long for that.  cudaErrorNotSupported for
// rows that no buffer holds, or more values than stream_values of each thread.
template <typename XT, typename RT, int MODE, bool LOOSE>
cudaError_t try_stream(const QuantRows& q, cudaStream_t s) {
    constexpr int V = 16 / (int)sizeof(XT), kStreamThreads = stream_threads(LOOSE);
    if (q.k > stream_values(LOOSE) * kStreamThreads) return cudaErrorNotSupported;
    const int64_t kv = (q.k + V - 1) / V * V;
    const bool two = MODE == kSwiglu || q.res;
    const size_t stage = staged_bytes(kv, sizeof(XT)) + (two ? staged_bytes(kv, sizeof(RT)) : 0u);
    size_t wts = MODE == kNorm ? staged_bytes(kv, 4) : 0u;
    const int values = q.k <= 16 * kStreamThreads ? 16 : q.k <= 32 * kStreamThreads ? 32 : 64;  // a thread
    const int threads = (int)(((kv + values - 1) / values + 31) / 32 * 32);
    const auto room = [](int ctas) { return pipe::kSmemPerSm / (size_t)ctas - 1024 - kStreamHeader; };
    const int at_once = values <= 32 ? 1024 : 512;  // threads of an SM that the registers leave room for
    int ctas = at_once / threads < 8 ? at_once / threads : 8;
    if ((uintptr_t)q.norm_w % 16) wts = 0;  // the norm weight is held where a bulk copy can bring it
    while (ctas > 1 && room(ctas) < wts + 2 * stage) ctas--;
    const bool held = wts && room(ctas) >= wts + 2 * stage;
    const size_t left = room(ctas) - (held ? wts : 0);
    if (left < stage) return cudaErrorNotSupported;
    const int stages = (int)(left / stage < kStreamStages ? left / stage : kStreamStages);
    const size_t smem = kStreamHeader + (held ? wts : 0) + stages * stage;
    switch (values) {
    case 16: return launch_stream<XT, RT, MODE, LOOSE, 16 / V>(q, threads, stages, held, ctas, smem, s);
    case 32: return launch_stream<XT, RT, MODE, LOOSE, 32 / V>(q, threads, stages, held, ctas, smem, s);
    default:
        if constexpr (!LOOSE) return launch_stream<XT, RT, MODE, LOOSE, 64 / V>(q, threads, stages, held, ctas, smem, s);
        return cudaErrorNotSupported;
    }
}

// One row per CTA (or warp).  Few of them (at most one an SM) wait for one round
// trip, so they are spread over as many threads as they have chunks, up to 1024; more
// take 16 values a thread (2048 x 4096 with an f32 residual: f32 19.0 us, 32 values 19.5),
// short ones a warp, and long ones what fits, 64 values at most.
template <typename XT, typename RT, int MODE>
cudaError_t launch_rows(const QuantRows& q, cudaStream_t s) {
    constexpr int V = 16 / (int)sizeof(XT), C = 16 / V;
    const int64_t chunks = q.k / V;
    if (q.m <= sm_count() && chunks > 128 && chunks <= 1024) {
        return chunks <= 512 ? launch_held<XT, RT, MODE, false, 512, 1>(q, s) : launch_held<XT, RT, MODE, false, 1024, 1>(q, s);
    }
    if (chunks <= 32 * C) return launch_held<XT, RT, MODE, false, 32, C>(q, s);
    if (chunks <= 128 * C) return launch_held<XT, RT, MODE, false, 128, C>(q, s);
    if (chunks <= 256 * C) return launch_held<XT, RT, MODE, false, 256, C>(q, s);
    if (chunks <= 512 * C) return launch_held<XT, RT, MODE, false, 512, C>(q, s);
    if (chunks <= 512 * 4) return launch_held<XT, RT, MODE, false, 512, 4>(q, s);
    if (chunks <= 512 * 8) return launch_held<XT, RT, MODE, false, 512, 8>(q, s);
    if constexpr (V == 4) {
        if (chunks <= 512 * 16) return launch_held<XT, RT, MODE, false, 512, 16>(q, s);
    }
    return launch_long<XT, RT, MODE>(q, s);
}

// Rows off the 16-byte grid, element by element: a warp a row up to 512 elements, then a
// CTA; few rows (at most one an SM), up to 16384 elements, over as many threads as help (one of
// 4097 f32 with norm and residual 2.8 us, streamed 4.0).  cudaErrorNotSupported for those
// that streaming serves better, whose words shared memory puts back together.  Of
// many rows these are the ones of more than 8192 elements (2048 x 14337 SwiGLU
// bf16 51 us, so 73); of more than 4096, 16-bit rows alone, where an element is a small
// part of a request (2048 x 7001 bf16 19.4 us, so 23.6; f32 23.7 and 22.2, with norm
// and residual 67 and 38); and 16-bit SwiGLU of more than 6144 (7001: 27.7 us, so
// 29.8; 6143: 24.7 and 22.3).
template <typename XT, typename RT, int MODE>
cudaError_t launch_loose(const QuantRows& q, cudaStream_t s) {
    if (q.k <= 512) return launch_held<XT, RT, MODE, true, 32, 16>(q, s);
    if (q.m <= sm_count()) {
        if (q.k <= 1024) return launch_held<XT, RT, MODE, true, 256, 4>(q, s);
        if (q.k <= 4096) return launch_held<XT, RT, MODE, true, 1024, 4>(q, s);
        if (q.k <= 8192) return launch_held<XT, RT, MODE, true, 512, 16>(q, s);
        if (q.k <= 16384) return launch_held<XT, RT, MODE, true, 1024, 16>(q, s);
        return cudaErrorNotSupported;
    }
    if (q.k <= 2048) return launch_held<XT, RT, MODE, true, 128, 16>(q, s);
    if (q.k <= 4096) return launch_held<XT, RT, MODE, true, 256, 16>(q, s);
    if (q.k > 8192 || (sizeof(XT) == 2 && (MODE == kSwiglu ? q.k > 6144 : !q.res))) return cudaErrorNotSupported;
    return q.k <= 6144 ? launch_held<XT, RT, MODE, true, 384, 16>(q, s) : launch_held<XT, RT, MODE, true, 512, 16>(q, s);
}

// Streams long rows off the 16-byte grid (launch_loose); and, of at least four rows
// an SM, those whose arithmetic counts beside the traffic: 16-bit rows
// (2048 x 14336 alone 19 us, a CTA per row 32, with an f32 residual and norm 59.7 and 61.6,
// SwiGLU 37.5 and 44) and SwiGLU of long f32 ones (2048 x 12288 38.6 us and 41.1, 28672 96 and
// 107; but 14336, of which an SM holds two rows at a time, 45.5 and 44.6, and 16384 63 and
// 48).  f32 rows otherwise keep a CTA per row (the norm with its residual 60 us, streamed 78).
template <typename XT, typename RT, int MODE>
cudaError_t launch_mode(const QuantRows& q, cudaStream_t s) {
    const uint64_t strides = (uint64_t)q.ldx * sizeof(XT) | (uint64_t)q.ldg * sizeof(XT) | (uint64_t)q.ldr * sizeof(RT) |
                             (uint64_t)q.ldro * sizeof(RT) | (uint64_t)q.ldc * 2;
    const uint64_t bits = (uint64_t)(uintptr_t)q.x | (uint64_t)(uintptr_t)q.gate | (uint64_t)(uintptr_t)q.norm_w |
                          (uint64_t)(uintptr_t)q.res | (uint64_t)(uintptr_t)q.res_out | (uint64_t)(uintptr_t)q.codes * 2 |
                          (uint64_t)q.k * sizeof(XT) | (q.m > 1 ? strides : 0);  // a single row's is never used
    if (bits & 15) {
        cudaError_t e = launch_loose<XT, RT, MODE>(q, s);
        if (e == cudaErrorNotSupported) e = try_stream<XT, RT, MODE, true>(q, s);
        return e != cudaErrorNotSupported ? e : launch_long<XT, RT, MODE>(q, s);
    }
    const bool dense = sizeof(XT) == 2 || (MODE == kSwiglu && q.k > 8192);
    if (dense && q.m >= 4 * sm_count() && q.k >= 1024) {
        const cudaError_t e = try_stream<XT, RT, MODE, false>(q, s);
        if (e != cudaErrorNotSupported) return e;
    }
    return launch_rows<XT, RT, MODE>(q, s);
}

template <typename XT>
cudaError_t launch_quant(const QuantRows& q, cudaStream_t s) {
    if (q.gate) return launch_mode<XT, XT, kSwiglu>(q, s);
    if (q.res && q.rtype != q.xtype)
        return q.norm_w ? launch_mode<XT, float, kNorm>(q, s) : launch_mode<XT, float, kPlain>(q, s);
    return q.norm_w ? launch_mode<XT, XT, kNorm>(q, s) : launch_mode<XT, XT, kPlain>(q, s);
}

template <typename OT, int R>
cudaError_t launch_deq(const int8_t* codes, int64_t ldc, const float* scales, int64_t m, int64_t k, OT* out, int64_t ldo,
                       cudaStream_t s) {
    const int64_t threads = (k + 15) / 16, bx = (m + R - 1) / R;
    const int T = threads > 128 ? 256 : threads > 32 ? 128 : 32;
    const int64_t by = (threads + T - 1) / T;
    if (bx > INT32_MAX || by > 65535) return cudaErrorInvalidConfiguration;
    return pipe::launch_pdl(dequantize_rows_kernel<OT, R>, dim3((unsigned)bx, (unsigned)by), T, 0, s, codes, ldc, scales, m, k,
                            out, ldo);
}

// One row of a chunk a thread (2048 x 4096 to bf16: 6.2 us, four rows 6.7); four of short rows.
template <typename OT>
cudaError_t launch_dequant(const int8_t* codes, int64_t ldc, const float* scales, int64_t m, int64_t k, void* to,
                           int64_t ldo, cudaStream_t s) {
    OT* out = static_cast<OT*>(to);
    const uint64_t strides = m > 1 ? (uint64_t)ldc | (uint64_t)ldo * sizeof(OT) : 0;  // a single row's is never used
    const uint64_t bits = (uint64_t)(uintptr_t)codes | (uint64_t)(uintptr_t)out | strides;
    if (bits & 15) {
        const int64_t threads = k * (int64_t)sizeof(OT) / 16 + 1;
        const int T = threads > 128 ? 256 : threads > 32 ? 128 : 32;
        const int64_t by = (threads + T - 1) / T;
        if (m > INT32_MAX || by > 65535) return cudaErrorInvalidConfiguration;
        return pipe::launch_pdl(dequantize_loose_kernel<OT>, dim3((unsigned)m, (unsigned)by), T, 0, s, codes, ldc, scales, k, out,
                                ldo);
    }
    return k > 1024 ? launch_deq<OT, 1>(codes, ldc, scales, m, k, out, ldo, s)
                    : launch_deq<OT, 4>(codes, ldc, scales, m, k, out, ldo, s);
}

}  // namespace

cudaError_t launch_quantize_rows(const QuantRows& q, cudaStream_t s) {
    switch (q.xtype) {
    case CLQ_X_F32: return launch_quant<float>(q, s);
    case CLQ_X_BF16: return launch_quant<__nv_bfloat16>(q, s);
    case CLQ_X_F16: return launch_quant<__half>(q, s);
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
