// sage_kv_append.hip — new keys and values, normalised and rotated, into a paged cache of e4m3 codes, and the queries rotated beside them.
//
//     y = x g / sqrt(mean_d x_d^2 + eps),  z = R(pos) y       of every new row of K (and of Q, which leaves as rows); V as it is
//     e = the least with max |z| <= 448 * 2^e over a block's tokens so far,  code = e4m3(z 2^-e),  scale = 2^e
//
// Powers of two: e4m3's step is relative, so a finer scale would win nothing but the part of a binade that a largest value leaves unused, and codes
// that are there can be taken to a larger scale without a second rounding (but for what falls below e4m3's normal range).  So a block
// that fills token by token holds what it would hold had its tokens come at once, up to that.
//
// Bound by memory for prompts, by latency for single tokens.  A workgroup owns the new rows of one block and key head: a group of D / 16 lanes to a row, all rows
// in flight at once, one exchange for the two largest values, V turned through LDS.  Where a block's earlier codes stay, their 16-byte pieces that
// new rows share are read ahead and written back with them.  Queries are other workgroups of the same launch.
// Measured, bf16, 48 + 12 heads of 128: 31234 tokens of 6 prompts 224 us, 4.7 TB/s of 5.2 that a large copy reaches; one token of 32 sequences 6.7 us.
#include "sage_grid.h"
#include "sage_kv.h"
#include "sage_rows.h"

#include <algorithm>

namespace sage {

namespace {

// The least e with top <= 448 * 2^e = 1.75 * 2^(e + 8).
__device__ __forceinline__ int block_power(float top) {
    const uint32_t bits = __float_as_uint(top);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);        // (a subnormal top: far below the least)
    return max(e, kKvLeast);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int power_of(float scale) { return max(kKvLeast, min((int)(__float_as_uint(scale) >> 23 & 255) - 127, 120)); }
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
// x 2^-e; what is no finite number becomes NaN, the only such code.
__device__ __forceinline__ float scaled(float x, float mul) { return fabsf(x) < INFINITY ? x * mul : __builtin_nanf(""); }
// Codes of one scale as those of another, 2^-down of it.
__device__ __forceinline__ uint32_t rescale(uint32_t w, int down) {
    typedef float v2 __attribute__((ext_vector_type(2)));
    const v2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return four_codes(__builtin_amdgcn_ldexpf(lo[0], -down), __builtin_amdgcn_ldexpf(lo[1], -down), __builtin_amdgcn_ldexpf(hi[0], -down), __builtin_amdgcn_ldexpf(hi[1], -down));
}
// The larger of two sizes; what is no finite number does not count.
__device__ __forceinline__ float larger(float top, float x) { x = fabsf(x); return x < INFINITY ? fmaxf(top, x) : top; }

// First row and number of rows of sequence b.
struct Rows { int first, n; };
__device__ __forceinline__ Rows sequence_rows(const KvAppendArgs& a, int b) {
    if (a.cu == nullptr) return Rows{b * a.S, a.S};
    const int lo = b == 0 ? 0 : max(0, min(a.cu[b], a.rows)), hi = max(lo, min(a.cu[b + 1], a.rows));
    return Rows{lo, hi - lo};
}
__device__ __forceinline__ int64_t row_at(const KvAppendArgs& a, const Rows& r, int64_t sb, int64_t sn, int b, int i) {
    return a.cu == nullptr ? b * sb + i * sn : (int64_t)(r.first + i) * sn;
}
// Position of a sequence's first new token.  (A length below zero counts as zero, one beyond any table, 2^30, as that: positions of blocks stay within 32 bits.)
__device__ __forceinline__ int first_new(const KvAppendArgs& a, int b, int n) { return max(0, min(a.pool.lens[b], 1 << 30)) - n; }

// Workgroup slots of sequences that lie one behind the other: sequence b's begin at cu[b] / 32 + 2 b, which leaves n / 32 + 2 at the least, and n rows
// touch no more blocks than that.
__device__ __forceinline__ int first_slot(const KvAppendArgs& a, int b) { return max(0, min(a.cu[b], a.rows)) / kKvBlock + 2 * b; }
template <class F> __device__ __forceinline__ int last_not_above(int n, int x, F first) {        // the last b < n with first(b) <= x, first(0) <= x
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first(mid) <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// 16 channels of a row: 8 at l.c0, 8 at l.c1.
template <int T, int LPR> __device__ __forceinline__ void norm_row(const KvAppendArgs& a, const Lane& l, const void* gain, float (&y0)[8], float (&y1)[8]) {
    if (gain == nullptr) return;
    float sum = 0.0f, g0[8], g1[8];
#pragma unroll
    for (int e = 0; e < 8; e++) sum = fmaf(y0[e], y0[e], fmaf(y1[e], y1[e], sum));
    load_gain(a, gain, l.c0, g0);
    load_gain(a, gain, l.c1, g1);
    const float r = inv_root<T>(row_sum<LPR>(sum) * a.inv_d + a.eps);
#pragma unroll
    for (int e = 0; e < 8; e++) y0[e] = y0[e] * r * g0[e], y1[e] = y1[e] * r * g1[e];
}

template <int T, int D>
__device__ __forceinline__ void append_block(const KvAppendArgs& a, uint8_t* turned, float (&tops)[2 * D / 64][2], int slot, int h) {
    constexpr int LPR = D / 16, PITCH = kKvBlock + 4, NW = 2 * D / 64;
    const KvPool& c = a.pool;
    int b, i;
    if (a.cu == nullptr) {
        const int per = (a.S + 30) / kKvBlock + 1;
        b = slot / per;
        i = slot - b * per;
    } else {
        b = last_not_above(a.B, slot, [&](int s) { return s == 0 ? 0 : first_slot(a, s); });
        i = slot - (b == 0 ? 0 : first_slot(a, b));
    }
    const Rows rows = sequence_rows(a, b);
    const int start = first_new(a, b, rows.n), room = c.width << (5 + c.sub);
    const int block = max(start, 0) / kKvBlock + i, p0 = block * kKvBlock;
    if (p0 >= room) return;
    const int lo = max(max(start, 0), p0) - p0, hi = min(min(start + rows.n, room) - p0, kKvBlock);
    if (hi <= lo) return;
    const int page = c.table[b * c.table_stride + (block >> c.sub)];
    if (page < 0 || page >= c.pages) return;             // (no such page: its tokens go nowhere)
    const int64_t unit = (((int64_t)page << c.sub) + (block & ((1 << c.sub) - 1))) * c.Hk + h;
    uint8_t *ck = c.k + unit * kKvBlock * D, *cv = c.v + unit * kKvBlock * D;

    const int tid = threadIdx.x, r = tid / LPR, j = tid % LPR;
    const Lane l = lane_channels<LPR>(D, a.rot);
    const bool on = r >= lo && r < hi;
    // (a row that is not new takes the first new one's place in the loads)
    const int tok = p0 + (on ? r : lo) - start;
    const int64_t krow = row_at(a, rows, a.k.sb, a.k.sn, b, tok) + h * a.k.sh, vrow = row_at(a, rows, a.v.sb, a.v.sn, b, tok) + h * a.v.sh;
    const Raw<T> rk[2] = {load8<T>(a.k.p, krow + l.c0), load8<T>(a.k.p, krow + l.c1)};
    const Raw<T> rv[2] = {load8<T>(a.v.p, vrow + j * 16), load8<T>(a.v.p, vrow + j * 16 + 8)};
    // what is there: the scales, this thread's piece of V (16 tokens of a channel)
    float was_k = 0.0f, was_v = 0.0f;
    const bool whole = lo == 0 && hi == kKvBlock;
    const int ch = tid >> 1, half = (tid & 1) * 16;
    u32x4* const piece = reinterpret_cast<u32x4*>(cv + ch * kKvBlock + half);
    u32x4 had = {0u, 0u, 0u, 0u};
    if (lo > 0) was_k = c.ks[unit], was_v = c.vs[unit];
    if (!whole) had = *piece;

    float y0[8], y1[8], top[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 8; e++) y0[e] = elem<T>(rk[0], e), y1[e] = elem<T>(rk[1], e);
    norm_row<T, LPR>(a, l, a.k_gain, y0, y1);
    if (l.rotated) {
        Turn t;
        load_turn_row(a, l, p0 + (on ? r : lo), t);
        turn<1>(t, a.halfsplit, y0, y1);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        top[0] = larger(larger(top[0], y0[e]), y1[e]);
        top[1] = larger(larger(top[1], elem<T>(rv[0], e)), elem<T>(rv[1], e));
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top[0] = fmaxf(top[0], __shfl_xor(top[0], m)), top[1] = fmaxf(top[1], __shfl_xor(top[1], m));
    if ((tid & 63) == 0) tops[tid >> 6][0] = top[0], tops[tid >> 6][1] = top[1];
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) top[0] = fmaxf(top[0], tops[w][0]), top[1] = fmaxf(top[1], tops[w][1]);
    int ek = block_power(top[0]), ev = block_power(top[1]), up_k = 0, up_v = 0;
    if (lo > 0) {
        const int ok = power_of(was_k), ov = power_of(was_v);
        ek = max(ek, ok), ev = max(ev, ov);
        up_k = ek - ok, up_v = ev - ov;
    }
    const float mk = power_of_two(-ek), mv = power_of_two(-ev);
    if (on) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            w[e] = four_codes(scaled(y0[e * 4], mk), scaled(y0[e * 4 + 1], mk), scaled(y0[e * 4 + 2], mk), scaled(y0[e * 4 + 3], mk));
            w[2 + e] = four_codes(scaled(y1[e * 4], mk), scaled(y1[e * 4 + 1], mk), scaled(y1[e * 4 + 2], mk), scaled(y1[e * 4 + 3], mk));
        }
        *reinterpret_cast<u32x2*>(ck + r * D + l.c0) = u32x2{w[0], w[1]};
        *reinterpret_cast<u32x2*>(ck + r * D + l.c1) = u32x2{w[2], w[3]};
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const Raw<T>& v = rv[n >> 1];
            const int e0 = (n & 1) * 4;
            const uint32_t x = four_codes(scaled(elem<T>(v, e0), mv), scaled(elem<T>(v, e0 + 1), mv), scaled(elem<T>(v, e0 + 2), mv), scaled(elem<T>(v, e0 + 3), mv));
#pragma unroll
            for (int e = 0; e < 4; e++) turned[(j * 16 + n * 4 + e) * PITCH + r] = (uint8_t)(x >> (e * 8));
        }
    } else if (r < lo && up_k > 0) {
        u32x4* at = reinterpret_cast<u32x4*>(ck + r * D + j * 16);
        u32x4 w = *at;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = rescale(w[e], up_k);
        *at = w;
    }
    __syncthreads();
    // V: 16 tokens of a channel to a thread
    if (half < hi && (half + 16 > lo || up_v > 0)) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            uint32_t x = *reinterpret_cast<const uint32_t*>(turned + ch * PITCH + half + e * 4);
            if (!whole) {
                const uint32_t old = up_v > 0 ? rescale(had[e], up_v) : had[e];
                uint32_t out = 0;
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const int t = half + e * 4 + n;
                    out |= (t < lo ? old : t < hi ? x : had[e]) & (0xFFu << (n * 8));
                }
                x = out;
            }
            w[e] = x;
        }
        *piece = w;
    }
    if (tid == 0) c.ks[unit] = power_of_two(ek), c.vs[unit] = power_of_two(ev);
}

// HB heads of a token to a group of lanes, as in sage_norm_rope.hip.  (Two: four take registers from the other workgroups too; [3 x 1153 tokens, 18 + 6 heads x 256] 22.0
// and 20.7 us, one head 21.9; [31234 tokens, 48 + 12 x 128] 224, 224 and 272.)
template <int T, int D, int HB> __device__ __forceinline__ void rotate_queries(const KvAppendArgs& a, int wg) {
    constexpr int LPR = D / 16, GROUPS = 2 * D / LPR;
    const int nblk = (a.Hq + HB - 1) / HB, item = wg * GROUPS + (int)threadIdx.x / LPR, token = item / nblk, blk = item % nblk;
    if (token >= a.rows) return;
    int b;
    if (a.cu == nullptr) b = token / a.S;
    else b = last_not_above(a.B, token, [&](int s) { return a.cu[s]; });
    const Rows rows = sequence_rows(a, b);
    const int i = token - rows.first;
    const bool real = i >= 0 && i < rows.n;              // (else a row behind the last sequence: zeros)
    const Lane l = lane_channels<LPR>(D, a.rot);
    const int64_t base = row_at(a, rows, a.q.sb, a.q.sn, b, i), to = row_at(a, rows, a.qo_sb, a.qo_sn, b, i);
    Raw<T> r0[HB], r1[HB];
#pragma unroll
    for (int n = 0; n < HB; n++) {
        const int64_t row = base + min(blk + n * nblk, a.Hq - 1) * a.q.sh;
        r0[n] = load8<T>(a.q.p, row + l.c0), r1[n] = load8<T>(a.q.p, row + l.c1);
    }
    Turn t;
    load_turn_row(a, l, first_new(a, b, rows.n) + i, t);
#pragma unroll
    for (int n = 0; n < HB; n++) {
        float y0[8], y1[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y0[e] = elem<T>(r0[n], e), y1[e] = elem<T>(r1[n], e);
        norm_row<T, LPR>(a, l, a.q_gain, y0, y1);
        const int h = blk + n * nblk;
        if (h >= a.Hq) continue;
        if (l.rotated) turn<1>(t, a.halfsplit, y0, y1);
        if (!real)
#pragma unroll
            for (int e = 0; e < 8; e++) y0[e] = y1[e] = 0.0f;
        store8<T>(a.qo, to + h * a.qo_sh + l.c0, y0);
        store8<T>(a.qo, to + h * a.qo_sh + l.c1, y1);
    }
}

constexpr int kHeads = 2;
template <int T, int D> __global__ __launch_bounds__(2 * D) void kv_append_kernel(KvAppendArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t turned[D * (kKvBlock + 4)];
    __shared__ float tops[2 * D / 64][2];
    const int id = (int)blockIdx.x;
    if (id < a.kv_wgs) {
        const int item = xcd_item(id, a.kv_wgs);         // (the heads of a block, which share rows of the tables, go to one XCD)
        append_block<T, D>(a, turned, tops, item / a.pool.Hk, item % a.pool.Hk);
    }
    else rotate_queries<T, D, kHeads>(a, id - a.kv_wgs);
}

int64_t append_wgs(const KvAppendArgs& a) {
    const int64_t slots = a.cu ? (int64_t)a.rows / kKvBlock + 2 * (int64_t)a.B : (int64_t)a.B * ((a.S + 30) / kKvBlock + 1);
    return slots * a.pool.Hk;
}
int64_t query_wgs(const KvAppendArgs& a) { return a.q.p ? ((int64_t)a.rows * ((a.Hq + kHeads - 1) / kHeads) + 31) / 32 : 0; }

template <int T> hipError_t launch_t(const KvAppendArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(a.kv_wgs + query_wgs(a)));
    if (a.D == 64) hipLaunchKernelGGL((kv_append_kernel<T, 64>), grid, dim3(128), 0, st, a);
    else if (a.D == 128) hipLaunchKernelGGL((kv_append_kernel<T, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv_append_kernel<T, 256>), grid, dim3(512), 0, st, a);
    return hipGetLastError();
}

}  // namespace

// (rotate_queries numbers its groups of heads of a token, 32 to a workgroup, in 32 bits.)
bool kv_append_grid_ok(const KvAppendArgs& a) { return append_wgs(a) + query_wgs(a) <= 0x7FFFFFFF / 2 && query_wgs(a) <= 0x7FFFFFFF / 32; }

hipError_t launch_kv_append(const KvAppendArgs& args, hipStream_t st) {
    KvAppendArgs a = args;
    a.kv_wgs = (int)append_wgs(a);
    return a.type == kBF16 ? launch_t<kBF16>(a, st) : launch_t<kF16>(a, st);
}

}  // namespace sage
