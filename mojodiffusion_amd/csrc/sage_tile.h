// sage_tile.h — 16-bit tiles in LDS as the matrix instructions of the backward and of windowed attention take them: layout,
// copies from global memory, fragments along and across the rows.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sage {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __fp16 v2h __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

namespace {

// ---- LDS layouts -------------------------------------------------------------------------
// Tile [64 rows][D] bf16 in 16-byte chunks, CPR per row, the chunk position XORed with a function of the row.
// Two access patterns meet in it:  fragments along the channels (16 consecutive rows, one logical chunk:
// the 16 lanes must land in 16 different 16-byte bank groups), and transposed fragments (4 consecutive rows
// times 4 neighbouring chunks per 32 lanes, 8 bytes each: the 16 chunks must be different ones).  With the
// row's low two bits moved into the chunk's upper bits both are free of conflicts.
template <int CPR> __device__ __forceinline__ int nat_pos(int row, int c) {
    if constexpr (CPR >= 16) return c ^ (((row & 3) << 2) | ((row >> 2) & 3));
    else return c ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));       // (row & 1 is the half of the 64 banks)
}
template <int CPR> __device__ __forceinline__ int nat_off(int row, int c) { return (row * CPR + nat_pos<CPR>(row, c)) << 4; }

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// 16 (4) bytes per lane from global memory straight into LDS: lane l lands at base + 16*l (4*l).
__device__ __forceinline__ void dma16(const void* gbase_uniform, uint32_t goff, uint32_t lds_base_uniform) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds_base_uniform), "v"(goff), "s"(gbase_uniform)
                 : "memory");
}
__device__ __forceinline__ void dma4(const void* gbase_uniform, uint32_t goff, uint32_t lds_base_uniform) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 :
                 : "s"(lds_base_uniform), "v"(goff), "s"(gbase_uniform)
                 : "memory");
}
// Wait until at most N of this wave's copies are still in flight (they complete in order).
template <int N> __device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const v2f f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2bf));       // round to nearest even
}

// Transposed fragment of a tile: lane l gets channel (l & 31) of a 32-channel block, rows half * 4 + 0..3 in
// the first two registers and 8 + half * 4 + 0..3 in the others (half = l >> 5), counted from a 16-row block —
// the order in which an accumulator lane holds its rows, i.e. the A operand that goes with P and dS.
// ds_read_b64_tr_b16 works on 16 lanes: lane i names 8 bytes (row i / 4, channels (i % 4) * 4 .. + 3 of a
// 4 x 16 block) and receives channel i of the four rows.
typedef short v4s __attribute__((ext_vector_type(4)));
template <int CPR> __device__ __forceinline__ int tr_frag_off(int lane, int row0, int d) {
    const int row = row0 + (lane >> 5) * 4 + ((lane & 15) >> 2);
    const int ch = d * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    return nat_off<CPR>(row, ch >> 3) + (ch & 7) * 2;
}
__device__ __forceinline__ v4i tr_read(const uint8_t* lo, const uint8_t* hi) {
    using lds_v4s = __attribute__((address_space(3))) v4s;
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)lo));
    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)hi));
    return v4i{(int)a.x, (int)a.y, (int)b.x, (int)b.y};
}

}  // namespace

}  // namespace sage
