// int8_gemm.cu -- the 8-bit product on the 5th-generation tensor cores:
// tcgen05.mma kind::i8 (signed 8-bit operands, 32-bit integer accumulators in
// tensor memory), both operands copied by TMA under the 128-byte swizzle.
//
// The weight's rows are the MMA's M (the accumulator's lanes) and the tokens its
// N (the columns): a warp of the epilogue then holds 32 neighbouring outputs of
// one token in its lanes, so it stores whole sectors of the row-major output
// straight from registers, whatever the output's stride, and few tokens make a
// narrow MMA instead of an empty one.
//
// Two kernels:
//   tile  one CTA per 128 weight rows x TN tokens and part of K; the parts of
//         one tile are the CTAs of a cluster, which exchange their integer
//         sums through distributed shared memory (no scratch, no second launch);
//   pair  two SMs per 256 weight rows x 256 tokens (cta_group::2), persistent,
//         with two accumulators, so that the epilogue of one tile runs under the
//         products of the next.
// Every mbarrier wait is bounded; on expiry the CTA records CLQ_ERR_TIMEOUT in
// the library's device status word, stops issuing, drains what it issued and
// frees its tensor memory.
#include <algorithm>
#include <atomic>
#include <cstdint>

#include <cuda.h>

#include "../../include/clq.h"
#include "clq_internal.h"
#include "int8_out.cuh"
#include "launch.cuh"
#include "pipeline.cuh"
#include "tma_host.h"

namespace clq {
namespace {

using namespace pipe;

constexpr int kRows = 128;                   // weight rows per CTA
constexpr int kKB = 128;                     // codes of K per stage: one swizzle span
constexpr uint32_t kABytes = kRows * kKB;
constexpr int kThreads = 192;                // warps 0-3 epilogue, 4 copies, 5 MMAs

struct GemmI8 {
    CUtensorMap wmap, xmap;
    CUtensorMap xmap_part;  // pair kernel: boxes of a part's tokens
    Int8Product p;
    int64_t kbt;            // 128-wide columns of K
    int64_t row_tiles, token_tiles;
    int64_t whole;          // pair kernel: tiles taken whole; each later one in PARTS
    int parts, stages;
    uint32_t b_bytes;       // of a stage's tokens in one CTA
    int* err;
};

// ---- PTX --------------------------------------------------------------------

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The address of this CTA's shared ADDR in CTA RANK of the cluster.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
__device__ __forceinline__ int4 load_cluster(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ uint32_t load_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Signed 8-bit A and B (K-major), 32-bit integer D, M x N.
__host__ __device__ constexpr uint32_t instr_desc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Low word of the matrix descriptor of an operand at shared ADDR (under 256 KB);
// the high word is the same for all: K-major, SWIZZLE_128B, 8-row groups 1024
// bytes apart.
__device__ __forceinline__ uint32_t desc_low(uint32_t addr) { return (addr >> 4) | (1u << 16); }
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
#define CLQ_MMA_STAGE(CG)                                                                                            \
    "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t.reg .b32 x, y;\n\t"                                             \
    "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 q, %5, %5;\n\t"                                                            \
    "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"                                                             \
    "tcgen05.mma.cta_group::" CG ".kind::i8 [%0], da, db, %3, p;\n\t"                                                \
    "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 da, {x, %5};\n\tmov.b64 db, {y, %5};\n\t"                    \
    "tcgen05.mma.cta_group::" CG ".kind::i8 [%0], da, db, %3, q;\n\t"                                                \
    "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 da, {x, %5};\n\tmov.b64 db, {y, %5};\n\t"                    \
    "tcgen05.mma.cta_group::" CG ".kind::i8 [%0], da, db, %3, q;\n\t"                                                \
    "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 da, {x, %5};\n\tmov.b64 db, {y, %5};\n\t"                    \
    "tcgen05.mma.cta_group::" CG ".kind::i8 [%0], da, db, %3, q;\n\t}"
// The four MMAs (32 codes of K each) of one stage; A, B: low descriptor words.
// ACCUMULATE 0: the first of them overwrites the accumulator.
template <int CG>
__device__ __forceinline__ void mma_stage(uint32_t tmem, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    static_assert(kKB == 128, "four MMAs to a stage");
    if constexpr (CG == 1)
        asm volatile(CLQ_MMA_STAGE("1") ::"r"(tmem), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh) : "memory");
    else
        asm volatile(CLQ_MMA_STAGE("2") ::"r"(tmem), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh) : "memory");
}
#undef CLQ_MMA_STAGE
// Arrives on BAR once every MMA issued before has completed; CG 2: on the
// barriers at BAR's offset in both CTAs of the pair.
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"((uint16_t)3)
            : "memory");
}
// On BAR of this CTA alone.
__device__ __forceinline__ void mma_commit_here(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
    if constexpr (CG == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}
// 32 columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_load32(uint32_t addr, int (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void prefetch_map(const void* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// The loops that issue copies and MMAs run at the rate of one warp's
// instructions, so they work on 32-bit shared addresses throughout.
//
// A box of MAP at (X bytes, row Y) into this CTA's DST, counted on BAR; CG 2: BAR
// may lie in the pair's other CTA (a shared::cluster address).
template <int CG>
__device__ __forceinline__ void copy_box(uint32_t dst, const void* map, int x, int y, uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
            "[%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
}
__device__ __forceinline__ void arrive_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Whether the phase has completed: at once, or after the pause that try_wait may take.
__device__ __forceinline__ bool peek(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// One lane of a converged warp.  The copying and the issuing warp run their
// loops as whole warps and elect a lane around the asynchronous instructions
// alone: where a branch on the lane enclosed the loop, a tcgen05.commit after
// four MMAs cost about 800 cycles (0.30 us a stage whatever the tile; 256
// x 256 tiles took 0.41, and their MMAs alone need 0.28).
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
// Bounded wait of a whole warp that spins without sleeping (a stage is a few
// hundred cycles); every lane gets the same answer.  READY: what a peek at the
// barrier, made while other work was under way, found.
__device__ __forceinline__ bool wait_spin(uint32_t bar, uint32_t parity, int* err, bool ready = false) {
    if (__all_sync(0xffffffffu, ready)) return true;
    bool ok = test(bar, parity);
    if (!ok) {  // the pause of a poll has passed
        const uint32_t start = time_ns();
        while (!(ok = test(bar, parity)) && !*(volatile int*)err)
            if (time_ns() - start >= kWaitNs) atomicExch(err, CLQ_ERR_TIMEOUT);
    }
    return __all_sync(0xffffffffu, ok);
}
// A role's place in a ring of n stages: the stage and the parity of its round.
// Stepped rather than divided out of a count: the loops' rate is that of one
// warp's instructions (a division a stage cost 0.1 us of 0.28).
struct Ring {
    int n;
    int s = 0;
    uint32_t round = 0;
    __device__ __forceinline__ explicit Ring(int stages) : n(stages) {}
    __device__ __forceinline__ void next() {
        if (++s == n) {
            s = 0;
            round++;
        }
    }
    __device__ __forceinline__ uint32_t parity() const { return round & 1u; }
    __device__ __forceinline__ Ring after() const {
        Ring r = *this;
        r.next();
        return r;
    }
};
__device__ __forceinline__ uint8_t* align1024(uint8_t* p) {
    return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~(uintptr_t)1023);
}

// Outputs of weight row N (one per lane) for CNT <= 32 tokens from T0 on, from
// their sums; X: the scale of token T0 + lane.  Each loop is one straight run of
// independent instructions, and the pointers step by a row: with a test for the
// residual inside a single loop, or the product j * ldo for an address, 256
// columns took 9.0 us instead of 2.9.
template <typename OT, bool RES>
__device__ __forceinline__ void emit_columns(const Int8Product& p, const int (&v)[32], int64_t n, float wsn, int64_t t0,
                                             int cnt, float x) {
    if (n >= p.n) cnt = 0;
    float o[32];
    if constexpr (RES) {  // the residual's loads in flight before any is used
        const float* res = p.res + t0 * p.ldr + n;
#pragma unroll
        for (int j = 0; j < 32; j++, res += p.ldr) o[j] = j < cnt ? *res : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 32; j++) {
        const float y = int8_scaled(v[j], wsn, __shfl_sync(0xffffffffu, x, j));
        if constexpr (RES) o[j] = __fadd_rn(y, o[j]);
        else o[j] = y;
    }
    OT* out = static_cast<OT*>(p.out) + t0 * p.ldo + n;
#pragma unroll
    for (int j = 0; j < 32; j++, out += p.ldo)
        if (j < cnt) *out = int8_round<OT>(o[j]);
    __syncwarp();  // the next tensor-memory load wants the whole warp
}
template <typename OT>
__device__ __forceinline__ void emit32(const Int8Product& p, const int (&v)[32], int64_t n, float wsn, int64_t t0, int cnt,
                                       float x) {
    __syncwarp();
    if (p.res) emit_columns<OT, true>(p, v, n, wsn, t0, cnt, x);
    else emit_columns<OT, false>(p, v, n, wsn, t0, cnt, x);
}

// Four neighbouring outputs O of one token: one store where OUT allows it.
template <typename OT>
__device__ __forceinline__ void store4(OT* out, const float (&o)[4], int cnt) {
    if (cnt >= 4 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(OT)) == 0) {
        OT h[4];
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = int8_round<OT>(o[i]);
        if constexpr (sizeof(OT) == 4) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(h);
        else *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(h);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < cnt) out[i] = int8_round<OT>(o[i]);
    }
}

// Tokens T0, T0 + 4, .. (B of them) of rows N..N + 3, CNT of which exist: the
// SPLITS parts' sums at AT (this CTA's address of token T0's, a token 4 * kRows * 4
// bytes after the last) added up and written.  Two parts' loads are in flight
// together.
template <typename OT, int B, bool RES>
__device__ __forceinline__ void join_parts(const Int8Product& P, uint32_t at, int splits, int64_t t0, int64_t n, int cnt,
                                           const float (&wsn)[4], const float* xs) {
    float4 r[B] = {};
    if constexpr (RES) {
        const float* res = P.res + t0 * P.ldr + n;
#pragma unroll
        for (int b = 0; b < B; b++, res += 4 * P.ldr) {
            if (cnt > 0) r[b].x = res[0];
            if (cnt > 1) r[b].y = res[1];
            if (cnt > 2) r[b].z = res[2];
            if (cnt > 3) r[b].w = res[3];
        }
    }
    int4 a[B] = {};
    for (int q = 0; q < splits; q += 2) {
        const int once = q + 1 < splits ? -1 : 0;  // an odd last part is read twice and counted once
        const uint32_t one = map_rank(at, (uint32_t)q), two = map_rank(at, (uint32_t)(q - once));
        int4 v[B], v2[B];
#pragma unroll
        for (int b = 0; b < B; b++) {
            v[b] = load_cluster(one + b * 4 * kRows * 4);
            v2[b] = load_cluster(two + b * 4 * kRows * 4);
        }
#pragma unroll
        for (int b = 0; b < B; b++) {
            a[b].x += v[b].x + (v2[b].x & once);
            a[b].y += v[b].y + (v2[b].y & once);
            a[b].z += v[b].z + (v2[b].z & once);
            a[b].w += v[b].w + (v2[b].w & once);
        }
    }
    OT* out = static_cast<OT*>(P.out) + t0 * P.ldo + n;
#pragma unroll
    for (int b = 0; b < B; b++, out += 4 * P.ldo) {
        const float x = xs[4 * b];
        float o[4] = {int8_scaled(a[b].x, wsn[0], x), int8_scaled(a[b].y, wsn[1], x), int8_scaled(a[b].z, wsn[2], x),
                      int8_scaled(a[b].w, wsn[3], x)};
        if constexpr (RES) {
            o[0] = __fadd_rn(o[0], r[b].x);
            o[1] = __fadd_rn(o[1], r[b].y);
            o[2] = __fadd_rn(o[2], r[b].z);
            o[3] = __fadd_rn(o[3], r[b].w);
        }
        store4<OT>(out, o, cnt);
    }
}

// ---- tile kernel --------------------------------------------------------------

// Stages of a CTA that has an SM to itself (for 32 tokens fewer than fit: eight cover
// memory's latency), or shares it with one other.
constexpr int tile_stages(int tn, int per_sm) {
    return per_sm == 2 ? (tn == 64 ? 4 : 5) : tn == 256 ? 4 : tn == 128 ? 7 : tn == 64 ? 9 : 8;
}
constexpr size_t tile_smem(int tn, int stages) {
    return 1024 + (size_t)stages * (kABytes + (size_t)tn * kKB) + (2 * stages + 3) * 8 + (size_t)tn * 4;
}
constexpr bool tile_fits(int tn, int per_sm) {  // with the 1 KB that the system takes of each CTA's share
    return tile_smem(tn, tile_stages(tn, per_sm)) <= (kSmemPerSm + 1024) / per_sm - 1024 &&
           (size_t)tn * kRows * 4 <= (size_t)tile_stages(tn, per_sm) * (kABytes + (size_t)tn * kKB);  // the sums, over them
}
static_assert(tile_fits(256, 1) && tile_fits(128, 1) && tile_fits(64, 1) && tile_fits(32, 1) && tile_fits(64, 2) &&
              tile_fits(32, 2), "shared memory");

// CTA (blockIdx.x = row tile x SPLITS + part, blockIdx.y = token tile); the
// SPLITS parts of a tile form a cluster.  Each part leaves its sums in its own
// shared memory, over the stages it has done with, as [token][row], and part r
// finishes the tokens [r TN / SPLITS, (r + 1) TN / SPLITS) from all of them.  A part whose
// sums are not whole says so beside them, and none of the tile is written.
template <typename OT, int TN>
__global__ void __launch_bounds__(kThreads) int8_tile_kernel(const __grid_constant__ GemmI8 G, int splits) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const int NS = G.stages;
    constexpr uint32_t kBBytes = TN * kKB;
    uint8_t* A = align1024(smem_raw);
    uint8_t* B = A + (size_t)NS * kABytes;
    int* sums = reinterpret_cast<int*>(A);
    uint64_t* full = reinterpret_cast<uint64_t*>(B + (size_t)NS * kBBytes);
    uint64_t* empty = full + NS;
    uint64_t* done = empty + NS;  // the sums are whole
    uint64_t* last = done + 1;    // or, after a wait that gave up, the MMAs issued have ended
    uint32_t* slot = reinterpret_cast<uint32_t*>(last + 1);
    uint32_t* gave_up = slot + 1;
    float* xs = reinterpret_cast<float*>(slot + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = (int)(blockIdx.x % splits);
    const int64_t n0 = (int64_t)(blockIdx.x / splits) * kRows, t0 = (int64_t)blockIdx.y * TN;
    const int kb0 = (int)(G.kbt * part / splits), nk = (int)(G.kbt * (part + 1) / splits) - kb0;
    const Int8Product& P = G.p;

    if (warp == 5) {
        if (lane < 2 * NS + 2) mbar_init(full + lane, 1);  // full, empty, done, last
        mbar_init_fence();
    } else if (warp == 4) {
        if (lane < 2) prefetch_map(lane ? &G.xmap : &G.wmap);
        if (lane == 2) *gave_up = 0;
    } else if (warp == 0) {
        tmem_alloc<1>(slot, TN);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    grid_dependency_wait();
    allow_dependents();

    bool ok = false;
    const uint32_t fulls = smem_u32(full), empties = smem_u32(empty);
    if (warp == 4) {
        const uint32_t a0 = smem_u32(A), b0 = smem_u32(B);
        Ring r(NS);
        int it = 0;
        bool ready = false;
        for (; it < nk; it++, r.next()) {
            if (r.round && !wait_spin(empties + 8 * r.s, r.parity() ^ 1u, G.err, ready)) break;
            const Ring next = r.after();
            ready = next.round && peek(empties + 8 * next.s, next.parity() ^ 1u);
            if (elect_one()) {
                arrive_tx(fulls + 8 * r.s, kABytes + kBBytes);
                copy_box<1>(a0 + r.s * kABytes, &G.wmap, (kb0 + it) * kKB, (int)n0, fulls + 8 * r.s);
                copy_box<1>(b0 + r.s * kBBytes, &G.xmap, (kb0 + it) * kKB, (int)t0, fulls + 8 * r.s);
            }
            __syncwarp();
        }
        // what is in flight lands before the CTA exits
        for (int i = 0; i < NS; i++, r.next())
            if (r.round) mbar_drain(&full[r.s], r.parity() ^ 1u);
    } else if (warp == 5) {
        const uint32_t a0 = desc_low(smem_u32(A)), b0 = desc_low(smem_u32(B));
        constexpr uint32_t idesc = instr_desc_i8(kRows, TN);
        Ring r(NS);
        bool whole = true, ready = false;
        for (int it = 0; it < nk; it++, r.next()) {
            if (!(whole = wait_spin(fulls + 8 * r.s, r.parity(), G.err, ready))) break;
            const Ring next = r.after();
            ready = peek(fulls + 8 * next.s, next.parity());
            tc_fence_after();
            if (elect_one()) {
                mma_stage<1>(tmem, a0 + r.s * (kABytes >> 4), b0 + r.s * (kBBytes >> 4), idesc, it > 0);
                mma_commit<1>(empties + 8 * r.s);
            }
            __syncwarp();
        }
        uint64_t* ended = whole ? done : last;
        if (elect_one()) mma_commit<1>(smem_u32(ended));
        __syncwarp();
        mbar_drain(ended, 0);
    } else {
        for (int i = threadIdx.x; i < TN; i += 128) xs[i] = t0 + i < P.m ? P.xs[t0 + i] : 0.f;
        named_sync(1, 128);
        ok = __all_sync(0xffffffffu, mbar_wait(done, 0, G.err));
        tc_fence_after();
    }
    __syncwarp();

    const uint32_t lanes = tmem + ((uint32_t)(32 * warp) << 16);
    const int cols = P.m - t0 < TN ? (int)(P.m - t0) : TN;  // tokens of the tile
    if (splits == 1) {
        if (ok) {
            const int64_t n = n0 + 32 * warp + lane;
            const float wsn = n < P.n ? P.ws[n] : 0.f;
            for (int c = 0; c < cols; c += 32) {
                int v[32];
                tmem_load32(lanes + c, v);
                emit32<OT>(P, v, n, wsn, t0 + c, cols - c, xs[c + lane]);
            }
        }
    } else {
        const int64_t n = n0 + 4 * lane;  // four rows a lane, a token a warp
        float wsn[4] = {};
        if (ok) {
#pragma unroll
            for (int i = 0; i < 4; i++) wsn[i] = n + i < P.n ? P.ws[n + i] : 0.f;
            for (int c = 0; c < cols; c += 32) {
                int v[32];
                tmem_load32(lanes + c, v);
#pragma unroll
                for (int j = 0; j < 32; j++) sums[(c + j) * kRows + 32 * warp + lane] = v[j];
            }
        }
        if (warp < 4 && !ok && lane == 0) *gave_up = 1;
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp < 4) ok = !__any_sync(0xffffffffu, lane < splits && load_cluster_u32(map_rank(smem_u32(gave_up), (uint32_t)lane)));
        if (ok) {
            const int c0 = TN * part / splits, c1 = min(cols, TN * (part + 1) / splits);
            const uint32_t base = smem_u32(sums) + 16 * lane;
            const int cnt = P.n - n < 4 ? (int)(P.n - n) : 4;
            for (int c = c0 + warp; c < c1;) {  // eight tokens a warp at a time, then two
                const uint32_t at = base + (uint32_t)c * kRows * 4;
                if (c + 4 * 7 < c1) {
                    P.res ? join_parts<OT, 8, true>(P, at, splits, t0 + c, n, cnt, wsn, xs + c)
                          : join_parts<OT, 8, false>(P, at, splits, t0 + c, n, cnt, wsn, xs + c);
                    c += 4 * 8;
                } else if (c + 4 < c1) {
                    P.res ? join_parts<OT, 2, true>(P, at, splits, t0 + c, n, cnt, wsn, xs + c)
                          : join_parts<OT, 2, false>(P, at, splits, t0 + c, n, cnt, wsn, xs + c);
                    c += 4 * 2;
                } else {
                    P.res ? join_parts<OT, 1, true>(P, at, splits, t0 + c, n, cnt, wsn, xs + c)
                          : join_parts<OT, 1, false>(P, at, splits, t0 + c, n, cnt, wsn, xs + c);
                    c += 4;
                }
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();  // the other parts have read this CTA's sums
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_free<1>(tmem, TN);
    }
}

// ---- pair kernel --------------------------------------------------------------

constexpr int kPairTokens = 256, kGroup = 8;
constexpr uint32_t kPairB = kPairTokens / 2 * kKB;  // each CTA stages half of the tokens
constexpr uint32_t kPairRing = 6 * (kABytes + kPairB);  // six stages, or up to ten of fewer tokens
constexpr int kPairMaxStages = 10;
constexpr size_t kPairSmem = 1024 + kPairRing + (2 * kPairMaxStages + 5) * 8 + 16;
static_assert(kPairSmem <= kSmemPerSm, "shared memory of one SM");

// What a pair of SMs does at one time: rows [256 RT, ..) for TOKENS tokens from T0 on.
// The tiles of 256 rows x 256 tokens come in groups of kGroup row tiles, token
// tiles outermost within a group, so that those in flight at one time share both
// operands in L2.  The first G.whole of them, a multiple of the pairs, are taken
// whole; the rest would leave pairs idle for a whole round, so each is taken in
// G.parts ranges of its tokens.
struct PairUnit {
    int64_t rt, t0;
    int tokens;
};
__device__ __forceinline__ PairUnit pair_unit(const GemmI8& G, int64_t unit) {
    const int64_t late = unit - G.whole;
    const int64_t tile = late < 0 ? unit : G.whole + late / G.parts;
    const int64_t per = kGroup * G.token_tiles, g = tile / per, i = tile - g * per;
    const int64_t left = G.row_tiles - g * kGroup, width = left < kGroup ? left : kGroup;
    const int64_t tt = i / width;
    PairUnit u;
    u.rt = g * kGroup + (i - tt * width);
    u.tokens = late < 0 ? kPairTokens : kPairTokens / G.parts;
    u.t0 = tt * kPairTokens + (late < 0 ? 0 : late % G.parts * u.tokens);
    return u;
}

template <typename OT>
__global__ void __launch_bounds__(kThreads, 1) int8_pair_kernel(const __grid_constant__ GemmI8 G) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const int NS = G.stages;
    uint8_t* A = align1024(smem_raw);
    uint8_t* B = A + (size_t)NS * kABytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(A + kPairRing);            // used in the leader
    uint64_t* empty = full + kPairMaxStages;                                // in both
    uint64_t* acc_full = empty + kPairMaxStages;                            // [2], in both
    uint64_t* acc_empty = acc_full + 2;                                     // [2], in the leader
    uint64_t* last = acc_empty + 2;                                         // in the leader
    uint32_t* slot = reinterpret_cast<uint32_t*>(last + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const Int8Product& P = G.p;
    const int64_t tiles = G.whole + (G.row_tiles * G.token_tiles - G.whole) * G.parts;
    const int64_t first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const int nk = (int)G.kbt;

    if (warp == 5) {
        if (lane < 2 * kPairMaxStages + 5)  // acc_empty: both CTAs' epilogue warps
            mbar_init(full + lane, (lane & ~1) == 2 * kPairMaxStages + 2 ? 8 : 1);
        mbar_init_fence();
    } else if (warp == 4) {
        if (lane < 3) prefetch_map(lane == 0 ? &G.wmap : lane == 1 ? &G.xmap : &G.xmap_part);
    } else if (warp == 0) {
        tmem_alloc<2>(slot, 512);
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    tc_fence_after();
    const uint32_t tmem = *slot;
    grid_dependency_wait();
    allow_dependents();

    const uint32_t fulls = smem_u32(full), empties = smem_u32(empty);
    if (warp == 4) {
        const uint32_t a0 = smem_u32(A), b0 = smem_u32(B), fulls_leader = map_rank(fulls, 0);
        Ring r(NS);
        bool ok = true, ready = false;
        for (int64_t tile = first; tile < tiles && ok; tile += step) {
            const PairUnit u = pair_unit(G, tile);
            if (u.t0 >= P.m) break;  // a part past the last token, which is a CTA's last unit
            const int y_w = (int)(u.rt * 2 * kRows + rank * kRows), y_x = (int)(u.t0 + rank * (u.tokens / 2));
            const CUtensorMap* xmap = u.tokens == kPairTokens ? &G.xmap : &G.xmap_part;
            const uint32_t tx = 2u * (kABytes + (uint32_t)u.tokens / 2 * kKB);
            for (int kb = 0; kb < nk; kb++, r.next()) {
                if (r.round && !(ok = wait_spin(empties + 8 * r.s, r.parity() ^ 1u, G.err, ready))) break;
                const Ring next = r.after();
                ready = next.round && peek(empties + 8 * next.s, next.parity() ^ 1u);
                if (elect_one()) {
                    if (leader) arrive_tx(fulls + 8 * r.s, tx);
                    copy_box<2>(a0 + r.s * kABytes, &G.wmap, kb * kKB, y_w, fulls_leader + 8 * r.s);
                    copy_box<2>(b0 + r.s * G.b_bytes, xmap, kb * kKB, y_x, fulls_leader + 8 * r.s);
                }
                __syncwarp();
            }
        }
        // every stage has been read, and the leader's commits have arrived here, before the CTA exits
        for (int i = 0; i < NS && ok; i++, r.next())
            if (r.round) ok = wait_spin(empties + 8 * r.s, r.parity() ^ 1u, G.err);
        // after a wait that gave up, the copies in flight (their barrier may be the other CTA's) get
        // 100 us to land: a hundred times what one takes
        for (int i = 0; i < 100 && !ok; i++) __nanosleep(1000);
    } else if (warp == 5) {
        if (leader) {
            const uint32_t a0 = desc_low(smem_u32(A)), b0 = desc_low(smem_u32(B)), accs = smem_u32(acc_full);
            Ring r(NS);
            int64_t nt = 0;
            bool ok = true, ready = false;
            for (int64_t tile = first; tile < tiles && ok; tile += step, nt++) {
                const PairUnit u = pair_unit(G, tile);
                if (u.t0 >= P.m) break;
                const uint32_t idesc = instr_desc_i8(2 * kRows, u.tokens);
                const uint32_t buf = (uint32_t)(nt & 1), acc = tmem + buf * kPairTokens;
                if (nt >= 2 && !(ok = wait_spin(smem_u32(acc_empty) + 8 * buf, (uint32_t)((nt >> 1) - 1) & 1u, G.err))) break;
                tc_fence_after();
                for (int kb = 0; kb < nk; kb++, r.next()) {
                    if (!(ok = wait_spin(fulls + 8 * r.s, r.parity(), G.err, ready))) break;
                    const Ring next = r.after();
                    ready = peek(fulls + 8 * next.s, next.parity());
                    tc_fence_after();
                    if (elect_one()) {
                        mma_stage<2>(acc, a0 + r.s * (kABytes >> 4), b0 + r.s * (G.b_bytes >> 4), idesc, kb > 0);
                        mma_commit<2>(empties + 8 * r.s);
                    }
                    __syncwarp();
                }
                if (!ok) break;  // sums that are not whole are not handed on
                if (elect_one()) mma_commit<2>(accs + 8 * buf);
                __syncwarp();
            }
            // the MMAs issued last have read their operands before the CTA exits
            if (!ok) {
                if (elect_one()) mma_commit_here(smem_u32(last));
                __syncwarp();
                mbar_drain(last, 0);
            } else if (nt > 0) {
                mbar_drain(&acc_full[(nt - 1) & 1], (uint32_t)((nt - 1) >> 1) & 1u);
            }
            // where the other CTA may have stopped waiting, the commits' arrivals there get 10 us to land
            for (int i = 0; i < 10 && *(volatile int*)G.err; i++) __nanosleep(1000);
        }
    } else {
        int64_t nt = 0;
        for (int64_t tile = first; tile < tiles; tile += step, nt++) {
            const PairUnit u = pair_unit(G, tile);
            if (u.t0 >= P.m) break;
            const int buf = (int)(nt & 1);
            const int64_t n = u.rt * 2 * kRows + rank * kRows + 32 * warp + lane, t0 = u.t0;
            const float wsn = n < P.n ? P.ws[n] : 0.f;
            const int cols = P.m - t0 < u.tokens ? (int)(P.m - t0) : u.tokens;
            float x = lane < cols ? P.xs[t0 + lane] : 0.f;  // the scales of the 32 tokens to come
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (uint32_t)(nt >> 1) & 1u, G.err))) break;
            tc_fence_after();
            const uint32_t lanes = tmem + ((uint32_t)(32 * warp) << 16) + (uint32_t)(buf * kPairTokens);
            for (int c = 0; c < cols; c += 32) {
                const float next = c + 32 + lane < cols ? P.xs[t0 + c + 32 + lane] : 0.f;
                int v[32];
                tmem_load32(lanes + c, v);
                emit32<OT>(P, v, n, wsn, t0 + c, cols - c, x);
                x = next;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_cluster(map_rank(smem_u32(&acc_empty[buf]), 0));
        }
    }
    __syncwarp();
    tc_fence_before();
    cluster_arrive();
    cluster_wait();
    if (warp == 0) {
        tc_fence_after();
        tmem_free<2>(tmem, 512);
    }
}

// ---- host -----------------------------------------------------------------------

bool make_maps(GemmI8* g, int w_box, int x_box) {
    const Int8Product& p = g->p;
    return encode_swizzled_rows(&g->wmap, p.w, p.n, p.k, p.ldw, w_box) &&
           encode_swizzled_rows(&g->xmap, p.x, p.m, p.k, p.ldx, x_box);
}

template <typename OT, int TN>
cudaError_t launch_tile(GemmI8& g, int splits, int per_sm, cudaStream_t s) {
    const int64_t rt = (g.p.n + kRows - 1) / kRows, tt = (g.p.m + TN - 1) / TN;
    if (rt * splits > INT32_MAX || tt > 65535 || !make_maps(&g, kRows, TN)) return cudaErrorNotSupported;
    g.stages = tile_stages(TN, per_sm);
    const size_t smem = tile_smem(TN, g.stages);
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = allow_smem(int8_tile_kernel<OT, TN>, tile_smem(TN, tile_stages(TN, 1)), allowed);
    if (e != cudaSuccess) return e;
    return launch_cluster(int8_tile_kernel<OT, TN>, dim3((unsigned)(rt * splits), (unsigned)tt), kThreads, smem, splits, s, g,
                          splits);
}

// Into how many parts (1, 2, 4 or 8) each of LATE tiles goes so that PAIRS take them in one round.
int parts_of(int64_t late, int64_t pairs) {
    int parts = 1;
    while (parts < 8 && late * parts * 2 <= pairs) parts *= 2;
    return parts;
}

template <typename OT>
cudaError_t launch_pair(GemmI8& g, cudaStream_t s) {
    g.row_tiles = (g.p.n + 2 * kRows - 1) / (2 * kRows);
    g.token_tiles = (g.p.m + kPairTokens - 1) / kPairTokens;
    const int64_t tiles = g.row_tiles * g.token_tiles, pairs = sm_count() / 2;
    g.whole = tiles / pairs * pairs;
    g.parts = parts_of(tiles - g.whole, pairs);
    if (!make_maps(&g, kRows, kPairTokens / 2) ||
        !encode_swizzled_rows(&g.xmap_part, g.p.x, g.p.m, g.p.k, g.p.ldx, kPairTokens / 2 / g.parts))
        return cudaErrorNotSupported;
    // where every unit is a part, the ring holds more stages of fewer tokens
    g.b_bytes = kPairB / (g.whole ? 1u : (uint32_t)g.parts);
    g.stages = std::min<int>(kPairMaxStages, (int)(kPairRing / (kABytes + g.b_bytes)));
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = allow_smem(int8_pair_kernel<OT>, kPairSmem, allowed);
    if (e != cudaSuccess) return e;
    const int64_t units = g.whole + (tiles - g.whole) * g.parts;
    return launch_cluster(int8_pair_kernel<OT>, dim3((unsigned)(2 * std::min(units, pairs))), kThreads, kPairSmem, 2, s, g);
}

// Clusters of SPLITS tile CTAs that run at one time, counting one CTA to an SM (a
// cluster stays within a GPC: 148 SMs hold 74 pairs but 45 threes and 33 fours).
constexpr int kMaxSplits = 8;
int resident_clusters(int splits) {
    static std::atomic<int> known[kMaxSplits + 1];
    if (splits == 1) return sm_count();
    if (const int n = known[splits].load()) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(splits * sm_count()));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = tile_smem(256, tile_stages(256, 1));
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    static std::atomic<uint64_t> allowed{0};
    if (allow_smem(int8_tile_kernel<float, 256>, cfg.dynamicSmemBytes, allowed) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, int8_tile_kernel<float, 256>, &cfg) != cudaSuccess || n < 1) {
        (void)cudaGetLastError();
        return 1;  // not known: the split looks expensive and is not taken
    }
    known[splits].store(n);
    return n;
}

// The kernel for a request: the one of least time in microseconds by
//   max(rounds of resident tiles x columns of K x c, traffic) + rounds x e
// with c a 128-byte column's time and e a tile's start and end, fitted to every
// variant at 1024 to 14336 rows and K = 2051 to 14336.  For up to 128 tokens c is the
// issuing loop's: a column of operands in L2 takes 0.18 us for 32 or 64 tokens and 0.19
// for 128 with four CTAs at work, and 0.18, 0.19 and 0.21 with 144 (the same, so neither
// a copy's round trip, with seven or more stages in flight, nor L2, which then delivers
// 16 to 22 TB/s); the MMAs of 128 tokens alone take 0.14.  Those of 256 take 0.27, and
// their column 0.27 to 0.47 as more SMs work.  What it decides, at K = 4096 (us; the tile
// kernel as tokens / parts of K):
//   24 tokens, 4096 rows    32/4  7.5   32/1  8.7   pair 10.7
//   128 tokens, 4096 rows   64/2  9.0   64/1  9.4   pair 11.3
//   256 tokens, 6144 rows   128/1 11.8  pair 12.8   256/2 16.3
//   256 tokens, 14336 rows  pair 19.5   256/1 22.7  128/1 25.3
//   512 tokens, 4096 rows, K = 14336:  128/1 29.9  pair 30.3  256/2 31.2
struct Choice {
    int tn, splits, per_sm;  // tn 0: the pair kernel
};
Choice choose(const Int8Product& p, int64_t kbt) {
    static const struct {
        int tn;
        double c, e1, es, c2;  // es: with K split; c2: two to an SM
    } kTiles[] = {{32, 0.185, 1.15, 2.4, 0.45}, {64, 0.19, 1.5, 3.4, 0.55}, {128, 0.218, 2.3, 5.0, 0.}, {256, 0.364, 3.8, 7.9, 0.}};
    static const int kSplits[] = {1, 2, 3, 4, 6, 8};
    const auto rounds = [](int64_t tiles, int64_t at_once) { return (double)((tiles + at_once - 1) / at_once); };
    const double traffic = (double)(p.n + p.m) * (double)p.k / 6.2e6;
    const int64_t units = ((p.n + 2 * kRows - 1) / (2 * kRows)) * ((p.m + kPairTokens - 1) / kPairTokens);
    const int64_t pairs = sm_count() / 2;
    const int parts = parts_of(units % pairs, pairs);
    // the pair kernel's tiles overlap: only the last one's end, shorter in parts, is waited for
    Choice best = {0, 1, 1};
    double least = (double)kbt * (0.35 * (double)(units / pairs) + (units % pairs ? parts > 1 ? 0.225 : 0.322 : 0.));
    least = std::max(least, traffic) + (units % pairs == 0 || parts == 1 ? 5.0 : parts == 2 ? 3.85 : parts == 4 ? 2.5 : 2.3);
    for (const auto& t : kTiles) {
        const int64_t tiles = ((p.n + kRows - 1) / kRows) * ((p.m + t.tn - 1) / t.tn);
        if ((p.m + t.tn - 1) / t.tn > 65535) continue;
        for (const int splits : kSplits) {
            if (splits > 1 && 2 * splits > kbt) break;
            const double r = rounds(tiles, resident_clusters(splits));
            const double cost = std::max(r * (double)((kbt + splits - 1) / splits) * t.c, traffic) + r * (splits > 1 ? t.es : t.e1);
            if (cost <= least) {  // of equals, more parts: their copies are under way sooner
                least = cost;
                best = {t.tn, splits, 1};
            }
        }
        // more tiles than SMs: two to an SM, each at about half of its rate (32 tokens, 28672 rows
        // of 4096: 22.5 us, one to an SM 25.5; of 8192: 40.7 and 44.4)
        if (t.c2 > 0 && tiles > sm_count()) {
            const double r = rounds(tiles, 2 * sm_count());
            const double cost = std::max(r * (double)kbt * t.c2, traffic) + r * t.e1;
            if (cost < least) {
                least = cost;
                best = {t.tn, 1, 2};
            }
        }
    }
    return best;
}

template <typename OT>
cudaError_t launch_type(GemmI8& g, cudaStream_t s) {
    const Choice c = choose(g.p, g.kbt);
    switch (c.tn) {
    case 32: return launch_tile<OT, 32>(g, c.splits, c.per_sm, s);
    case 64: return launch_tile<OT, 64>(g, c.splits, c.per_sm, s);
    case 128: return launch_tile<OT, 128>(g, c.splits, c.per_sm, s);
    case 256: return launch_tile<OT, 256>(g, c.splits, c.per_sm, s);
    default: return launch_pair<OT>(g, s);
    }
}

}  // namespace

cudaError_t launch_int8_gemm(const Int8Product& p, cudaStream_t s) {
    if (!int8_aligned(p) || p.k < 1 || p.n > INT32_MAX - 512 || p.m > INT32_MAX - 512) return cudaErrorNotSupported;
    GemmI8 g = {};
    g.p = p;
    g.kbt = (p.k + kKB - 1) / kKB;
    g.err = device_status_word();
    if (!g.err) return cudaErrorNotSupported;
    switch (p.otype) {
    case CLQ_X_F32: return launch_type<float>(g, s);
    case CLQ_X_BF16: return launch_type<__nv_bfloat16>(g, s);
    case CLQ_X_F16: return launch_type<__half>(g, s);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace clq
