// sage_norm_rope.hip — RMSNorm of every query and key head and the position rotation, in one pass, and its gradient.
//
//     r = 1 / sqrt(mean_d x_d^2 + eps),  y_d = x_d r g_d,  z = R(pos) y      R: pairs (a, b) -> (a c - b s, b c + a s)
//     dy = R^T dz,  dg_d = sum over rows dy_d x_d r,
//     dx_d = r (u_d - x_d r m),  u = dy g,  m = mean_d u_d x_d r
// All sums and products in fp32, one rounding to the stored type at the end.
//
// Bound by memory: a row is read once and written once (backward: two reads, one write), about 25 operations per
// channel.  A group of LPR lanes owns a row, 16 channels to a lane: the 8 at j * 8 and the 8 at half the rotated
// channels behind them, so both partners of a pair sit in one lane in either pairing and the only exchange is the
// sum over the row.  The rows of a token's heads share one piece of the tables: a group takes HB heads of a token with
// cos, sin and the gain in registers, all its loads in flight at once.
// Measured: forward [2,4352,30 + 30,128] bf16 62 us, 4.3 TB/s; backward [1,16896,40 + 10,64] fp32 134 us, 4.9 TB/s of 4.8 that a large copy reaches.
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
__device__ __forceinline__ void load_gain(const NormRopeArgs& a, const void* gain, int c, float* y) {
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
__device__ __forceinline__ void load_turn(const NormRopeArgs& a, const Lane& l, int b, int s, Turn& t) {
    if (!l.rotated) return;
    int64_t row = s;
    if (a.positions != nullptr) {
        const int64_t at = b * a.pos_sb + s;
        row = a.pos64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
    }
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
template <int LPR> __device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int m = 1; m < LPR; m <<= 1) x += __shfl_xor(x, m);
    return x;
}
template <int T> __device__ __forceinline__ float inv_root(float x) {
    if constexpr (T == kF32) return 1.0f / sqrtf(x);
    else return __builtin_amdgcn_rsqf(x);                 // (1 ulp of fp32, far below the rounding of the result)
}

template <int T, int LPR, int HB>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a) {
    const bool is_k = (int)blockIdx.x >= a.wg_q;
    const NormRopeSide& x = is_k ? a.k : a.q;
    const int H = is_k ? a.Hk : a.Hq, nblk = (H + HB - 1) / HB;
    const int item = ((int)blockIdx.x - (is_k ? a.wg_q : 0)) * (256 / LPR) + (int)threadIdx.x / LPR;
    const int token = item / nblk, blk = item % nblk;
    const bool live = token < a.B * a.S;
    const int b = live ? token / a.S : 0, s = live ? token % a.S : 0;
    const Lane l = lane_channels<LPR>(a.D, a.rot);
    const bool on = live && l.on;

    // (heads blk, blk + nblk, ...: neighbouring groups take neighbouring heads)
    Raw<T> r0[HB], r1[HB];
    const int64_t base = b * x.sb + s * x.sn;
#pragma unroll
    for (int i = 0; i < HB; i++) {
        const int64_t row = base + min(blk + i * nblk, H - 1) * x.sh;
        if (on) {
            r0[i] = load8<T>(x.p, row + l.c0);
            r1[i] = load8<T>(x.p, row + l.c1);
        }
    }
    Turn t;
    float g0[8], g1[8];
    if (on) {
        load_turn(a, l, b, s, t);
        load_gain(a, x.gain, l.c0, g0);
        load_gain(a, x.gain, l.c1, g1);
    }
#pragma unroll
    for (int i = 0; i < HB; i++) {
        float y0[8], y1[8], sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            y0[e] = on ? elem<T>(r0[i], e) : 0.0f;
            y1[e] = on ? elem<T>(r1[i], e) : 0.0f;
            sum = fmaf(y0[e], y0[e], fmaf(y1[e], y1[e], sum));
        }
        const float r = inv_root<T>(row_sum<LPR>(sum) * a.inv_d + a.eps);
        const int h = blk + i * nblk;
        if (!on || h >= H) continue;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            y0[e] = y0[e] * r * g0[e];
            y1[e] = y1[e] * r * g1[e];
        }
        if (l.rotated) turn<1>(t, a.halfsplit, y0, y1);
        const int64_t row = b * x.osb + s * x.osn + h * x.osh;
        store8<T>(x.out, row + l.c0, y0);
        store8<T>(x.out, row + l.c1, y1);
    }
}

// The same walk with the gradient's two inputs.  A workgroup stays with one of Q and K and goes through its share of the
// tokens; the gain's gradient collects in registers, then over the workgroup's groups, and leaves as one row of D partial
// sums (launch 2 adds those up in fixed order: the same bits on every call).
template <int T, int LPR, int HB>
__global__ __launch_bounds__(256) void norm_rope_bwd_kernel(NormRopeArgs a) {
    __shared__ float red[4][LPR * 16];
    const bool is_k = (int)blockIdx.x >= a.wg_q;
    const NormRopeSide& x = is_k ? a.k : a.q;
    const int H = is_k ? a.Hk : a.Hq, nblk = (H + HB - 1) / HB;
    const int first = ((int)blockIdx.x - (is_k ? a.wg_q : 0)) * (256 / LPR) + (int)threadIdx.x / LPR;
    const int step = (is_k ? a.wg_k : a.wg_q) * (256 / LPR), items = a.B * a.S * nblk;
    const Lane l = lane_channels<LPR>(a.D, a.rot);

    float g0[8], g1[8], d0[8], d1[8];
#pragma unroll
    for (int e = 0; e < 8; e++) g0[e] = g1[e] = d0[e] = d1[e] = 0.0f;
    if (l.on) {
        load_gain(a, x.gain, l.c0, g0);
        load_gain(a, x.gain, l.c1, g1);
    }
    // (every group of a wave makes the same number of steps, so that the exchanges stay among live lanes)
    for (int it = first; it - (int)(threadIdx.x & 63) / LPR < items; it += step) {
        const bool on = it < items && l.on;
        const int token = on ? it / nblk : 0, blk = on ? it % nblk : 0;
        const int b = token / a.S, s = token % a.S;
        Raw<T> r0[HB], r1[HB], z0[HB], z1[HB];
#pragma unroll
        for (int i = 0; i < HB; i++) {
            const int h = min(blk + i * nblk, H - 1);
            const int64_t row = b * x.sb + s * x.sn + h * x.sh, drow = b * x.dsb + s * x.dsn + h * x.dsh;
            if (on) {
                r0[i] = load8<T>(x.p, row + l.c0), r1[i] = load8<T>(x.p, row + l.c1);
                z0[i] = load8<T>(x.d, drow + l.c0), z1[i] = load8<T>(x.d, drow + l.c1);
            }
        }
        Turn t;
        if (on) load_turn(a, l, b, s, t);
#pragma unroll
        for (int i = 0; i < HB; i++) {
            const int h = blk + i * nblk;
            const bool row_on = on && h < H;
            float x0[8], x1[8], y0[8], y1[8], sum = 0.0f, dot = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x0[e] = row_on ? elem<T>(r0[i], e) : 0.0f, x1[e] = row_on ? elem<T>(r1[i], e) : 0.0f;
                y0[e] = row_on ? elem<T>(z0[i], e) : 0.0f, y1[e] = row_on ? elem<T>(z1[i], e) : 0.0f;
                sum = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], sum));
            }
            const float r = inv_root<T>(row_sum<LPR>(sum) * a.inv_d + a.eps);
            if (row_on && l.rotated) turn<-1>(t, a.halfsplit, y0, y1);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x0[e] *= r, x1[e] *= r;
                if (row_on) d0[e] = fmaf(y0[e], x0[e], d0[e]), d1[e] = fmaf(y1[e], x1[e], d1[e]);
                y0[e] *= g0[e], y1[e] *= g1[e];
                dot = fmaf(y0[e], x0[e], fmaf(y1[e], x1[e], dot));
            }
            const float m = row_sum<LPR>(dot) * a.inv_d;
            if (!row_on) continue;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y0[e] = r * fmaf(-x0[e], m, y0[e]);
                y1[e] = r * fmaf(-x1[e], m, y1[e]);
            }
            const int64_t row = b * x.osb + s * x.osn + h * x.osh;
            store8<T>(x.out, row + l.c0, y0);
            store8<T>(x.out, row + l.c1, y1);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
#pragma unroll
        for (int m = LPR; m < 64; m <<= 1) d0[e] += __shfl_xor(d0[e], m), d1[e] += __shfl_xor(d1[e], m);
    }
    if ((threadIdx.x & 63) < LPR && l.on) {
#pragma unroll
        for (int e = 0; e < 8; e++) red[threadIdx.x >> 6][l.c0 + e] = d0[e], red[threadIdx.x >> 6][l.c1 + e] = d1[e];
    }
    __syncthreads();
    if ((int)threadIdx.x < a.D)
        a.partial[(int64_t)blockIdx.x * a.D + threadIdx.x] =
            (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// Launch 2: 16 channels to a workgroup, its 64 slices of the partial rows each in order, then the slices by a tree; in
// double, as there may be hundreds of them.
__global__ __launch_bounds__(1024) void norm_rope_gain_kernel(NormRopeArgs a) {
    __shared__ double red[64][16];
    const int per = (a.D + 15) / 16, is_k = (int)blockIdx.x / per, d = ((int)blockIdx.x % per) * 16 + (int)(threadIdx.x & 15);
    const int slice = (int)threadIdx.x >> 4, n = is_k ? a.wg_k : a.wg_q;
    const float* p = a.partial + (int64_t)(is_k ? a.wg_q : 0) * a.D + d;
    double sum = 0.0;
    for (int i = slice; i < n; i += 512) {
        float v[8];                      // (eight rows requested at a time: what this launch takes, 4 us, is latencies)
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = p[(int64_t)min(i + u * 64, n - 1) * a.D];
#pragma unroll
        for (int u = 0; u < 8; u++) sum += i + u * 64 < n ? (double)v[u] : 0.0;
    }
    red[slice][threadIdx.x & 15] = sum;
    __syncthreads();
    for (int m = 32; m > 0; m >>= 1) {
        if (slice < m) red[slice][threadIdx.x & 15] += red[slice + m][threadIdx.x & 15];
        __syncthreads();
    }
    if (slice == 0) (is_k ? a.d_gain_k : a.d_gain_q)[d] = (float)red[0][threadIdx.x & 15];
}

template <int T, int LPR, bool BWD> hipError_t launch(NormRopeArgs a, hipStream_t st) {
    constexpr int HB = BWD ? 2 : 4, GROUPS = 256 / LPR;
    const int64_t tokens = (int64_t)a.B * a.S;
    if constexpr (BWD) {
        norm_rope_bwd_split(a.B, a.S, a.Hq, a.Hk, a.D, &a.wg_q, &a.wg_k);
        hipLaunchKernelGGL((norm_rope_bwd_kernel<T, LPR, HB>), dim3(a.wg_q + a.wg_k), dim3(256), 0, st, a);
        hipLaunchKernelGGL(norm_rope_gain_kernel, dim3(2 * (a.D / 16)), dim3(1024), 0, st, a);
    } else {
        // Few rows: one to a group, the shortest chain; else HB share what they load of the tables.
        const bool few = tokens * (a.Hq + a.Hk) <= 256 * 16 * GROUPS;
        const int hb = few ? 1 : HB;
        a.wg_q = (int)((tokens * ((a.Hq + hb - 1) / hb) + GROUPS - 1) / GROUPS);
        a.wg_k = (int)((tokens * ((a.Hk + hb - 1) / hb) + GROUPS - 1) / GROUPS);
        if (few) hipLaunchKernelGGL((norm_rope_kernel<T, LPR, 1>), dim3(a.wg_q + a.wg_k), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((norm_rope_kernel<T, LPR, HB>), dim3(a.wg_q + a.wg_k), dim3(256), 0, st, a);
    }
    return hipGetLastError();
}
template <int T, bool BWD> hipError_t launch_d(const NormRopeArgs& a, hipStream_t st) {
    if (a.D <= 64) return launch<T, 4, BWD>(a, st);
    if (a.D <= 128) return launch<T, 8, BWD>(a, st);
    return launch<T, 16, BWD>(a, st);
}
template <bool BWD> hipError_t launch_t(const NormRopeArgs& a, hipStream_t st) {
    if (a.type == kBF16) return launch_d<kBF16, BWD>(a, st);
    if (a.type == kF16) return launch_d<kF16, BWD>(a, st);
    return launch_d<kF32, BWD>(a, st);
}

}  // namespace

// Workgroups of the backward's launch 1 for Q and for K: in proportion to their rows, no more than the chip holds at once
// (two to a compute unit, by their registers; 1024 on [1,4096,32 on 32,64] fp32: 143 us, 512: 134), no more than there are items.
void norm_rope_bwd_split(int B, int S, int Hq, int Hk, int D, int* wg_q, int* wg_k) {
    const int groups = 256 / (D <= 64 ? 4 : D <= 128 ? 8 : 16);
    const int64_t tokens = (int64_t)B * S;
    const int64_t nq = (tokens * ((Hq + 1) / 2) + groups - 1) / groups, nk = (tokens * ((Hk + 1) / 2) + groups - 1) / groups;
    constexpr int64_t kMost = 512;
    if (nq + nk <= kMost) {
        *wg_q = (int)nq, *wg_k = (int)nk;
        return;
    }
    const int64_t q = kMost * nq / (nq + nk);
    *wg_q = (int)(q < 1 ? 1 : q);
    *wg_k = (int)(kMost - q < 1 ? 1 : kMost - q);
}

hipError_t launch_norm_rope(const NormRopeArgs& a, hipStream_t st) { return launch_t<false>(a, st); }
hipError_t launch_norm_rope_bwd(const NormRopeArgs& a, hipStream_t st) { return launch_t<true>(a, st); }

}  // namespace sage
