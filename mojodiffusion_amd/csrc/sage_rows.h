// sage_rows.h — rows of heads as the kernels that normalise and rotate them hold them: 16 channels to a lane, both partners of a pair in one
// lane in either pairing, in fp32.  Args: a kernel's arguments with cos, sin, table_type, table_rows, table_stride, halfsplit and gain_type.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sage_window.h"

namespace sage {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

// (the word by value: a bit cast of a vector's element reads the vector's first)
__device__ __forceinline__ float half_of(uint32_t w, int i) { return (float)__builtin_bit_cast(v2h, w)[i]; }

// 8 channels as they lie in memory
template <int T> struct Raw { u32x4 w[T == kF32 ? 2 : 1]; };

template <int T> __device__ __forceinline__ Raw<T> load8(const void* p, int64_t i) {
    Raw<T> r;
    const u32x4* s = reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(p) + i * (T == kF32 ? 4 : 2));
    r.w[0] = s[0];
    if constexpr (T == kF32) r.w[1] = s[1];
    return r;
}
template <int T> __device__ __forceinline__ float elem(const Raw<T>& r, int i) {
    if constexpr (T == kF32) return __uint_as_float(r.w[i >> 2][i & 3]);
    else if constexpr (T == kBF16) return __uint_as_float((i & 1) ? r.w[0][i >> 1] & 0xFFFF0000u : r.w[0][i >> 1] << 16);
    else return half_of(r.w[0][i >> 1], i & 1);
}
template <int T> __device__ __forceinline__ void store8(void* p, int64_t i, const float (&y)[8]) {
    u32x4* d = reinterpret_cast<u32x4*>(static_cast<uint8_t*>(p) + i * (T == kF32 ? 4 : 2));
    if constexpr (T == kF32) {
#pragma unroll
        for (int h = 0; h < 2; h++)
            d[h] = u32x4{__float_as_uint(y[h * 4]), __float_as_uint(y[h * 4 + 1]), __float_as_uint(y[h * 4 + 2]), __float_as_uint(y[h * 4 + 3])};
    } else {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const v2f f = {y[2 * e], y[2 * e + 1]};
            if constexpr (T == kBF16) w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2bf));
            else w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2h));
        }
        d[0] = w;
    }
}
// four neighbours of a gain or a table, whatever its type (uniform over the launch)
__device__ __forceinline__ void four(const void* p, int type, int64_t i, float* y) {
    if (type == kF32) {
        const v4f f = *reinterpret_cast<const v4f*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = f[e];
        return;
    }
    const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (type == kBF16) y[e] = __uint_as_float((e & 1) ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
        else y[e] = half_of(w[e >> 1], e & 1);
    }
}
template <class Args> __device__ __forceinline__ void load_gain(const Args& a, const void* gain, int c, float* y) {
    four(gain, a.gain_type, c, y);
    four(gain, a.gain_type, c + 4, y + 4);
}

// The lane's two runs of 8 channels: rotated ones half the rotated channels apart, the others likewise.
struct Lane { int c0, c1; bool on, rotated; };
template <int LPR> __device__ __forceinline__ Lane lane_channels(int D, int rot) {
    const int j = (int)threadIdx.x & (LPR - 1), nr = rot / 16;
    Lane l;
    l.on = j < D / 16;
    l.rotated = j < nr;
    l.c0 = l.rotated ? j * 8 : rot + (j - nr) * 8;
    l.c1 = l.c0 + (l.rotated ? rot / 2 : (D - rot) / 2);
    return l;
}

// cos and sin of the lane's 8 pairs.  Half-split: pair i is element i of both runs; interleaved: pairs 0..3 lie in the first
// run, 4..7 in the second.
struct Turn { float c[8], s[8]; };
template <class Args> __device__ __forceinline__ void load_turn_row(const Args& a, const Lane& l, int64_t row, Turn& t) {
    if (!l.rotated) return;
    const bool inside = row >= 0 && row < a.table_rows;
    const int64_t base = (inside ? row : 0) * a.table_stride;
    const int i0 = a.halfsplit ? l.c0 : l.c0 / 2, i1 = a.halfsplit ? l.c0 + 4 : l.c1 / 2;
    four(a.cos, a.table_type, base + i0, t.c);
    four(a.cos, a.table_type, base + i1, t.c + 4);
    four(a.sin, a.table_type, base + i0, t.s);
    four(a.sin, a.table_type, base + i1, t.s + 4);
    if (!inside) {                        // no such row: what depends on it must not look like a result
#pragma unroll
        for (int i = 0; i < 8; i++) t.c[i] = t.s[i] = __builtin_nanf("");
    }
}
// SIGN +1: z = R y, -1: y = R^T z
template <int SIGN> __device__ __forceinline__ void turn(const Turn& t, bool halfsplit, float (&y0)[8], float (&y1)[8]) {
    auto pair = [&](float& p, float& q, float c, float s) {
        s = SIGN * s;
        const float np = fmaf(p, c, -(q * s)), nq = fmaf(q, c, p * s);
        p = np;
        q = nq;
    };
    if (halfsplit) {
#pragma unroll
        for (int i = 0; i < 8; i++) pair(y0[i], y1[i], t.c[i], t.s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) pair(y0[2 * i], y0[2 * i + 1], t.c[i], t.s[i]);
#pragma unroll
        for (int i = 0; i < 4; i++) pair(y1[2 * i], y1[2 * i + 1], t.c[4 + i], t.s[4 + i]);
    }
}
// The sum over a group of 4, 8 or 16 lanes by moves between neighbours: the lane ^ 1, ^ 2, then the mirror image in 8 and in 16, whose four (eight) lanes hold one sum by then.
template <int CTRL> __device__ __forceinline__ float lane_moved(float x) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true)); }
template <int LPR> __device__ __forceinline__ float row_sum(float x) {
    static_assert(LPR == 4 || LPR == 8 || LPR == 16, "lanes of a row");
    x += lane_moved<0xB1>(x);
    x += lane_moved<0x4E>(x);
    if constexpr (LPR > 4) x += lane_moved<0x141>(x);
    if constexpr (LPR > 8) x += lane_moved<0x140>(x);
    return x;
}
template <int T> __device__ __forceinline__ float inv_root(float x) {
    if constexpr (T == kF32) return 1.0f / sqrtf(x);
    else return __builtin_amdgcn_rsqf(x);                 // (1 ulp of fp32, far below the rounding of the result)
}

}  // namespace

}  // namespace sage
