// The matrix instructions by storage type, and the direct HBM -> LDS load (gfx950, wave64).
//
// MFMA register conventions (32x32 family), lane l, l32 = l%32, lh = l/32:
//   fp32  v_mfma_f32_32x32x2_f32 :  a = A[i=l32][kk=lh]        b = B[kk=lh][j=l32]
//   16bit v_mfma_f32_32x32x16_*  :  a = A[i=l32][8*lh .. +7]   b = B[8*lh .. +7][j=l32]
//   accumulator register r holds D[i = 8*(r/4) + 4*lh + r%4][j = l32].
#pragma once
#include "common.hpp"

namespace wino {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Mma;
template <> struct Mma<float> {
    typedef floatx4 vec;
    static __device__ __forceinline__ void run(const vec& a, const vec& b, floatx16& acc) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
    }
};
template <> struct Mma<f16_t> {
    typedef halfx8 vec;
    static __device__ __forceinline__ void run(const vec& a, const vec& b, floatx16& acc) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
    }
};
template <> struct Mma<bf16_t> {
    typedef bf16x8 vec;
    static __device__ __forceinline__ void run(const vec& a, const vec& b, floatx16& acc) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
    }
};

// One direct-to-LDS load of 64 channel vectors (1 KB): lane l moves the 16 bytes at sbase + 16*l to
// lds_dst + 16*l.  sbase is wave-uniform (a scalar register pair, advanced with scalar adds): at
// 16-bit MFMA rates the address arithmetic of these loads, vector or scalar, costs as much as the
// multiplies of a stage, so the kernels keep one running address per load slot instead of
// recomputing row * pitch products.
// The instruction is written out rather than taken from the compiler's builtin: the compiler counts the builtin
// as an access of unknown kind, and while one is in flight (in these kernels: always) it can no longer tell in
// which order LDS reads return, so that every wait for an LDS read becomes a wait for ALL of them -- the read
// issued one instruction earlier included, which leaves a wave's matrix pipe idle for an LDS round trip at
// every step.  Written out, the load is invisible to that bookkeeping: every kernel that uses it waits for its
// rows itself (s_waitcnt vmcnt before the workgroup's barrier), which they did already.
// M0 is written here and not named as a clobber: it is a reserved register for this compiler (which refuses it on a
// clobber list as undefined behaviour), never holds a value across instructions, and is set by the compiler itself
// right before each of its own uses.
__device__ __forceinline__ void dma_row(uint64_t sbase, unsigned lane_off, void* lds_dst) {
    const unsigned dst = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) void*)lds_dst);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(lane_off), "s"(sbase) : "memory");
}

// a wave-uniform 64-bit value, for the compiler too (scalar registers): values that are uniform by construction
// (derived from the workgroup id and kernel arguments through a cursor the compiler keeps in memory) still have to
// reach the scalar operands of dma_row
__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return ((uint64_t)hi << 32) | lo;
}

}  // namespace wino
