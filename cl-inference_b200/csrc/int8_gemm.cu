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
constexpr size_t kSmemMax = 227 * 1024;

struct GemmI8 {
    CUtensorMap wmap, xmap;
    Int8Product p;
    int64_t kbt;            // 128-wide columns of K
    int64_t row_tiles, token_tiles;
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
__device__ __forceinline__ void store_cluster(uint32_t addr, int v) {
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// K-major, SWIZZLE_128B, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
// Signed 8-bit A and B (K-major), 32-bit integer D, M x N.
__host__ __device__ constexpr uint32_t instr_desc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <int CG>
__device__ __forceinline__ void mma_i8(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}
// Arrives on BAR once every MMA issued before has completed; CG 2: on the
// barriers at BAR's offset in both CTAs of the pair.
template <int CG>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                     : "memory");
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)),
            "h"((uint16_t)3)
            : "memory");
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
// A box of MAP at (X bytes, row Y) into this CTA's DST, counted on BAR, a
// shared::cluster address that may lie in the pair's other CTA.
__device__ __forceinline__ void tensor_copy_pair(void* dst, const void* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// Bounded wait that spins without sleeping (a stage is a few hundred cycles).
__device__ __forceinline__ bool wait_spin(uint64_t* bar, uint32_t parity, int* err) {
    for (uint32_t i = 0; i < kWaitLimit; i++) {
        if (mbar_test(bar, parity)) return true;
        if ((i & 1023) == 1023 && *(volatile int*)err) return false;
    }
    atomicExch(err, CLQ_ERR_TIMEOUT);
    return false;
}
__device__ __forceinline__ uint8_t* align1024(uint8_t* p) {
    return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~(uintptr_t)1023);
}

// Outputs of weight row N (one per lane) for the 32 tokens T0.. from their sums.
template <typename OT>
__device__ __forceinline__ void emit32(const Int8Product& p, const int (&v)[32], int64_t n, float wsn, int64_t t0, int lane) {
    const float xs_lane = t0 + lane < p.m ? p.xs[t0 + lane] : 0.f;
    const bool in = n < p.n;
    const int cnt = p.m - t0 < 32 ? (int)(p.m - t0) : 32;
    OT* out = static_cast<OT*>(p.out) + t0 * p.ldo + n;
    const float* res = p.res ? p.res + t0 * p.ldr + n : nullptr;
    float r[32];
    if (res) {  // the residual's loads in flight before any is used
#pragma unroll
        for (int j = 0; j < 32; j++) r[j] = in && j < cnt ? res[j * p.ldr] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 32; j++) {
        float o = int8_scaled(v[j], wsn, __shfl_sync(0xffffffffu, xs_lane, j));
        if (res) o = __fadd_rn(o, r[j]);
        if (in && j < cnt) out[j * p.ldo] = int8_round<OT>(o);
    }
}

// ---- tile kernel --------------------------------------------------------------

constexpr int tile_stages(int tn) { return tn == 256 ? 4 : tn == 128 ? 5 : tn == 64 ? 8 : 9; }
size_t tile_smem(int tn, int splits) {
    return 1024 + (size_t)tile_stages(tn) * (kABytes + (size_t)tn * kKB) + (splits > 1 ? (size_t)tn * kRows * 4 : 0) +
           (2 * tile_stages(tn) + 1) * 8 + 16;
}

// CTA (blockIdx.x = row tile x SPLITS + part, blockIdx.y = token tile); the
// SPLITS parts of a tile form a cluster.  Part r of the cluster finishes the
// tokens [r TN / SPLITS, (r + 1) TN / SPLITS) of the tile.
template <typename OT, int TN>
__global__ void __launch_bounds__(kThreads) int8_tile_kernel(const __grid_constant__ GemmI8 G, int splits) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    constexpr int NS = tile_stages(TN);
    constexpr uint32_t kBBytes = TN * kKB;
    uint8_t* A = align1024(smem_raw);
    uint8_t* B = A + (size_t)NS * kABytes;
    int* sums = reinterpret_cast<int*>(B + (size_t)NS * kBBytes);  // [part][TN / splits][kRows]
    uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sums) + (splits > 1 ? TN * kRows * 4 : 0));
    uint64_t* empty = full + NS;
    uint64_t* done = empty + NS;
    uint32_t* slot = reinterpret_cast<uint32_t*>(done + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = (int)(blockIdx.x % splits);
    const int64_t n0 = (int64_t)(blockIdx.x / splits) * kRows, t0 = (int64_t)blockIdx.y * TN;
    const int kb0 = (int)(G.kbt * part / splits), nk = (int)(G.kbt * (part + 1) / splits) - kb0;
    const Int8Product& P = G.p;

    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        mbar_init_fence();
    }
    if (warp == 0) tmem_alloc<1>(slot, TN);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    if (splits > 1) cluster_arrive();  // the other parts may then write into this CTA's sums
    grid_dependency_wait();
    allow_dependents();

    bool ok = false;
    if (warp == 4) {
        if (lane == 0) {
            int it = 0;
            for (; it < nk; it++) {
                const int s = it % NS;
                if (it >= NS && !wait_spin(&empty[s], ((it / NS) - 1) & 1, G.err)) break;
                mbar_arrive_tx(&full[s], kABytes + kBBytes);
                tensor_copy_2d(A + (size_t)s * kABytes, &G.wmap, (kb0 + it) * kKB, (int)n0, &full[s]);
                tensor_copy_2d(B + (size_t)s * kBBytes, &G.xmap, (kb0 + it) * kKB, (int)t0, &full[s]);
            }
            // what is in flight lands before the CTA exits
            for (int i = it < NS ? 0 : it - NS; i < it; i++) mbar_drain(&full[i % NS], (i / NS) & 1);
        }
    } else if (warp == 5) {
        if (lane == 0) {
            constexpr uint32_t idesc = instr_desc_i8(kRows, TN);
            for (int it = 0; it < nk; it++) {
                const int s = it % NS;
                if (!wait_spin(&full[s], (it / NS) & 1, G.err)) break;
                tc_fence_after();
                const uint32_t a = smem_u32(A + (size_t)s * kABytes), b = smem_u32(B + (size_t)s * kBBytes);
#pragma unroll
                for (int j = 0; j < kKB / 32; j++)
                    mma_i8<1>(tmem, smem_desc(a + 32 * j), smem_desc(b + 32 * j), idesc, it > 0 || j > 0);
                mma_commit<1>(&empty[s]);
            }
            mma_commit<1>(done);
            mbar_drain(done, 0);
        }
    } else {
        ok = __all_sync(0xffffffffu, mbar_wait(done, 0, G.err));
        tc_fence_after();
    }
    __syncwarp();

    const int64_t n = n0 + 32 * warp + lane;
    const uint32_t lanes = tmem + ((uint32_t)(32 * warp) << 16);
    if (splits == 1) {
        if (ok) {
            const float wsn = n < P.n ? P.ws[n] : 0.f;
            for (int c = 0; c < TN && t0 + c < P.m; c += 32) {
                int v[32];
                tmem_load32(lanes + c, v);
                emit32<OT>(P, v, n, wsn, t0 + c, lane);
            }
        }
    } else {
        const int own = TN / splits;  // tokens that each part finishes
        cluster_wait();
        if (ok) {
            const uint32_t base = smem_u32(sums) + (uint32_t)((part * own) * kRows + 32 * warp + lane) * 4;
            for (int c = 0; c < TN && t0 + c < P.m; c += 32) {
                int v[32];
                tmem_load32(lanes + c, v);
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    const int col = c + j;
                    store_cluster(map_rank(base + (uint32_t)(col % own) * kRows * 4, (uint32_t)(col / own)), v[j]);
                }
            }
        }
        cluster_arrive();
        cluster_wait();
        if (ok) {
            const float wsn = n < P.n ? P.ws[n] : 0.f;
            for (int c = 0; c < own; c++) {
                const int64_t t = t0 + part * own + c;
                if (t >= P.m || n >= P.n) break;
                int sum = 0;
                for (int r = 0; r < splits; r++) sum += sums[(r * own + c) * kRows + 32 * warp + lane];
                float o = int8_scaled(sum, wsn, P.xs[t]);
                if (P.res) o = __fadd_rn(o, P.res[t * P.ldr + n]);
                static_cast<OT*>(P.out)[t * P.ldo + n] = int8_round<OT>(o);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_free<1>(tmem, TN);
    }
}

// ---- pair kernel --------------------------------------------------------------

constexpr int kPairTokens = 256, kPairStages = 6, kGroup = 8;
constexpr uint32_t kPairB = kPairTokens / 2 * kKB;  // each CTA stages half of the tokens
constexpr size_t kPairSmem = 1024 + (size_t)kPairStages * (kABytes + kPairB) + (2 * kPairStages + 4) * 8 + 16;
static_assert(kPairSmem <= kSmemMax, "shared memory of one SM");

// Tiles of 256 rows x 256 tokens in groups of kGroup row tiles, token tiles
// outermost within a group: the tiles in flight at one time share both operands in L2.
__device__ __forceinline__ void pair_tile(const GemmI8& G, int64_t tile, int64_t* rt, int64_t* tt) {
    const int64_t per = kGroup * G.token_tiles, g = tile / per, i = tile - g * per;
    const int64_t left = G.row_tiles - g * kGroup, width = left < kGroup ? left : kGroup;
    *tt = i / width;
    *rt = g * kGroup + (i - *tt * width);
}

template <typename OT>
__global__ void __launch_bounds__(kThreads, 1) int8_pair_kernel(const __grid_constant__ GemmI8 G) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    constexpr int NS = kPairStages;
    uint8_t* A = align1024(smem_raw);
    uint8_t* B = A + (size_t)NS * kABytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(B + (size_t)NS * kPairB);  // used in the leader
    uint64_t* empty = full + NS;                                            // in both
    uint64_t* acc_full = empty + NS;                                        // [2], in both
    uint64_t* acc_empty = acc_full + 2;                                     // [2], in the leader
    uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const Int8Product& P = G.p;
    const int64_t tiles = G.row_tiles * G.token_tiles, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const int nk = (int)G.kbt;

    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 8);  // the epilogue warps of both CTAs
        }
        mbar_init_fence();
    }
    if (warp == 0) tmem_alloc<2>(slot, 512);
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    tc_fence_after();
    const uint32_t tmem = *slot;
    grid_dependency_wait();
    allow_dependents();

    if (warp == 4) {
        if (lane == 0) {
            int64_t it = 0;
            bool ok = true;
            for (int64_t tile = first; tile < tiles && ok; tile += step) {
                int64_t rt, tt;
                pair_tile(G, tile, &rt, &tt);
                const int y_w = (int)(rt * 2 * kRows + rank * kRows), y_x = (int)(tt * kPairTokens + rank * (kPairTokens / 2));
                for (int kb = 0; kb < nk; kb++, it++) {
                    const int s = (int)(it % NS);
                    if (it >= NS && !(ok = wait_spin(&empty[s], (uint32_t)((it / NS) - 1) & 1u, G.err))) break;
                    if (leader) mbar_arrive_tx(&full[s], 2 * (kABytes + kPairB));
                    const uint32_t bar = map_rank(smem_u32(&full[s]), 0);
                    tensor_copy_pair(A + (size_t)s * kABytes, &G.wmap, kb * kKB, y_w, bar);
                    tensor_copy_pair(B + (size_t)s * kPairB, &G.xmap, kb * kKB, y_x, bar);
                }
            }
            // every stage has been read, and the leader's commits have arrived here, before the CTA exits
            for (int64_t i = it < NS ? 0 : it - NS; i < it && ok; i++)
                ok = wait_spin(&empty[i % NS], (uint32_t)(i / NS) & 1u, G.err);
            // after a wait that gave up, the copies in flight (their barrier may be the other CTA's) get
            // 100 us to land: a thousand times what one takes
            for (int i = 0; i < 100 && !ok; i++) __nanosleep(1000);
        }
    } else if (warp == 5) {
        if (leader && lane == 0) {
            constexpr uint32_t idesc = instr_desc_i8(2 * kRows, kPairTokens);
            int64_t it = 0, nt = 0;
            bool ok = true;
            for (int64_t tile = first; tile < tiles && ok; tile += step, nt++) {
                const int buf = (int)(nt & 1);
                if (nt >= 2 && !(ok = wait_spin(&acc_empty[buf], (uint32_t)((nt >> 1) - 1) & 1u, G.err))) break;
                tc_fence_after();
                for (int kb = 0; kb < nk; kb++, it++) {
                    const int s = (int)(it % NS);
                    if (!(ok = wait_spin(&full[s], (uint32_t)(it / NS) & 1u, G.err))) break;
                    tc_fence_after();
                    const uint32_t a = smem_u32(A + (size_t)s * kABytes), b = smem_u32(B + (size_t)s * kPairB);
#pragma unroll
                    for (int j = 0; j < kKB / 32; j++)
                        mma_i8<2>(tmem + (uint32_t)(buf * kPairTokens), smem_desc(a + 32 * j), smem_desc(b + 32 * j), idesc,
                                  kb > 0 || j > 0);
                    mma_commit<2>(&empty[s]);
                }
                mma_commit<2>(&acc_full[buf]);
            }
            // the MMAs issued last have read their operands before the CTA exits
            if (nt > 0) mbar_drain(&acc_full[(nt - 1) & 1], (uint32_t)((nt - 1) >> 1) & 1u);
        }
    } else {
        int64_t nt = 0;
        for (int64_t tile = first; tile < tiles; tile += step, nt++) {
            int64_t rt, tt;
            pair_tile(G, tile, &rt, &tt);
            const int buf = (int)(nt & 1);
            const int64_t n = rt * 2 * kRows + rank * kRows + 32 * warp + lane, t0 = tt * kPairTokens;
            const float wsn = n < P.n ? P.ws[n] : 0.f;
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (uint32_t)(nt >> 1) & 1u, G.err))) break;
            tc_fence_after();
            const uint32_t lanes = tmem + ((uint32_t)(32 * warp) << 16) + (uint32_t)(buf * kPairTokens);
            for (int c = 0; c < kPairTokens && t0 + c < P.m; c += 32) {
                int v[32];
                tmem_load32(lanes + c, v);
                emit32<OT>(P, v, n, wsn, t0 + c, lane);
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

template <typename Kern>
cudaError_t allow_smem(Kern kern, size_t smem) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
}

bool make_maps(GemmI8* g, int w_box, int x_box) {
    const Int8Product& p = g->p;
    return encode_swizzled_rows(&g->wmap, p.w, p.n, p.k, p.ldw, w_box) &&
           encode_swizzled_rows(&g->xmap, p.x, p.m, p.k, p.ldx, x_box);
}

template <typename OT, int TN>
cudaError_t launch_tile(GemmI8& g, int splits, cudaStream_t s) {
    const int64_t rt = (g.p.n + kRows - 1) / kRows, tt = (g.p.m + TN - 1) / TN;
    if (rt * splits > INT32_MAX || tt > 65535 || !make_maps(&g, kRows, TN)) return cudaErrorNotSupported;
    const size_t smem = tile_smem(TN, splits);
    const cudaError_t e = allow_smem(int8_tile_kernel<OT, TN>, smem);
    if (e != cudaSuccess) return e;
    return launch_cluster(int8_tile_kernel<OT, TN>, dim3((unsigned)(rt * splits), (unsigned)tt), kThreads, smem, splits, s, g,
                          splits);
}

template <typename OT>
cudaError_t launch_pair(GemmI8& g, cudaStream_t s) {
    g.row_tiles = (g.p.n + 2 * kRows - 1) / (2 * kRows);
    g.token_tiles = (g.p.m + kPairTokens - 1) / kPairTokens;
    if (!make_maps(&g, kRows, kPairTokens / 2)) return cudaErrorNotSupported;
    const cudaError_t e = allow_smem(int8_pair_kernel<OT>, kPairSmem);
    if (e != cudaSuccess) return e;
    const int64_t pairs = std::min<int64_t>(g.row_tiles * g.token_tiles, sm_count() / 2);
    return launch_cluster(int8_pair_kernel<OT>, dim3((unsigned)(2 * pairs)), kThreads, kPairSmem, 2, s, g);
}

template <typename OT>
cudaError_t launch_type(GemmI8& g, cudaStream_t s) {
    const Int8Product& p = g.p;
    if (p.m >= 512) return launch_pair<OT>(g, s);
    const int64_t rt = (p.n + kRows - 1) / kRows, sms = sm_count();
    const int tn = p.m <= 32 ? 32 : p.m <= 64 ? 64 : 128;
    const int64_t tiles = rt * ((p.m + tn - 1) / tn);
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= sms && splits * 2 * 4 <= g.kbt) splits *= 2;
    switch (tn) {
    case 32: return launch_tile<OT, 32>(g, splits, s);
    case 64: return launch_tile<OT, 64>(g, splits, s);
    default: return launch_tile<OT, 128>(g, splits, s);
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
