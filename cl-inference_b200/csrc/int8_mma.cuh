// int8_mma.cuh -- what the register-fed 8-bit products share: the integer MMA, and
// 16 codes of a row from any address.
#pragma once

#include <cstdint>

namespace clq {

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 codes from any address: the two 16-byte words around them, put together when
// they are used, so that loads stay in flight.  The words are read where both lie
// within the row, else its bytes alone.
struct Codes16 {
    uint4 a, b;
    uint32_t off;  // bytes of a before the first code

    // Codes [i, i + 16) of a row of K, zeros past its end.
    __device__ __forceinline__ void load(const int8_t* row, int64_t i, int64_t k) {
        if (i >= 15 && i + 32 <= k) {
            load_inside(row + i);
        } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 16; j++)
                if (i + j < k) w[j >> 2] |= (uint32_t)(uint8_t)row[i + j] << (8 * (j & 3));
            a = make_uint4(w[0], w[1], w[2], w[3]);
            b = make_uint4(0, 0, 0, 0);
            off = 0;
        }
    }
    // Codes [P, P + 16), with 15 more of the row before them and 16 after.
    __device__ __forceinline__ void load_inside(const int8_t* p) {
        off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
        const uint4* q = reinterpret_cast<const uint4*>(p - off);
        a = q[0];
        b = q[1];
    }
    __device__ __forceinline__ void zero() {
        a = b = make_uint4(0, 0, 0, 0);
        off = 0;
    }
    __device__ __forceinline__ uint4 codes() const {
        uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        if (off & 8) {
#pragma unroll
            for (int j = 0; j < 6; j++) w[j] = w[j + 2];
        }
        if (off & 4) {
#pragma unroll
            for (int j = 0; j < 5; j++) w[j] = w[j + 1];
        }
        const uint32_t bits = (off & 3) * 8;
        return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                          __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
    }
};

}  // namespace clq
