// sage_window_bwd.hip — gradient of attention over a sliding window, bf16 or fp16, head dims 64 and 128.
//
//     P_ij = exp(scale q_i . k_j - L_i) for the keys j that query i sees, else 0
//     Delta_i = dO_i . O_i,  dS_ij = P_ij (dO_i . v_j - Delta_i)
//     dQ_i = scale sum_j dS_ij k_j,  dK_j = scale sum_i dS_ij q_i,  dV_j = sum_i P_ij dO_i
// where the sums over i of a shared key head run over the queries of all its heads.  No atomics: the same bits on every call.
//
// Launch 1: Delta_i (from O with what rounding left of it, where the caller kept that) and L_i log2(e).  Launch 2: one grid of two kinds of workgroups, as the full backward's (sage_bwd.hip, whose
// reasons for tiles, rings and the order of the work hold here): owners of rows, that walk the key tiles their window reaches -> dQ; and owners of
// 128 keys, that walk the (head, query tile) pairs that reach them -> dK, dV.  Blocks with sinks are reached by every later query; their
// pairs are dealt to as many workgroups as keep the longest of them near the others, which leave fp32 parts for launch 3
// to add up in order.  The same where there are too few key blocks to fill the chip.
#include "sage_grid.h"
#include "sage_window_common.h"

#include <algorithm>
#include <type_traits>

namespace sage {

namespace {

typedef __fp16 v2fp __attribute__((ext_vector_type(2)));

template <int D> constexpr int kWaves = D > 64 ? 8 : 4;
constexpr int kKeysWg = 128;
template <int D> constexpr int kRowsWg = kWaves<D> * 32;

template <int T> __device__ __forceinline__ float widen(uint32_t w, int i) {
    if constexpr (T == kBF16) return __uint_as_float(i ? w & 0xFFFF0000u : w << 16);
    else return (float)__builtin_bit_cast(v2hf, w)[i];
}

template <int T, int D>
__global__ __launch_bounds__(256) void window_bwd_prep_kernel(WindowBwdArgs a) {
    constexpr int CPR = D / 8, RPP = 256 / CPR;      // threads per row, rows per workgroup
    const int H = a.w.Hk * a.w.g;
    const int64_t row = (int64_t)blockIdx.x * RPP + threadIdx.x / CPR;                // over [B, H, sq_pad]
    if (row >= (int64_t)a.w.B * H * a.sq_pad) return;
    const int i = (int)(row % a.sq_pad), bh = (int)(row / a.sq_pad), b = bh / H, h = bh % H, col = (int)(threadIdx.x % CPR) * 8;
    const bool real = i < a.w.Sq;
    float sum = 0.0f;
    if (real) {
        const int64_t at = b * a.w.o_sb + h * a.w.o_sh + i * a.w.o_sn + col;
        const u32x4 o = *reinterpret_cast<const u32x4*>(a.w.o + at);
        const u32x4 rest = a.w.rest ? *reinterpret_cast<const u32x4*>(a.w.rest + at) : u32x4{0u, 0u, 0u, 0u};
        const u32x4 g = *reinterpret_cast<const u32x4*>(a.dout + b * a.do_sb + h * a.do_sh + i * a.do_sn + col);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t ow = o[e >> 1], rw = rest[e >> 1], gw = g[e >> 1];
            sum = fmaf(widen<T>(ow, e & 1) + widen<T>(rw, e & 1), widen<T>(gw, e & 1), sum);
        }
    }
#pragma unroll
    for (int m = 1; m < CPR; m <<= 1) sum += __shfl_xor(sum, m);
    if (col == 0) {
        const float l = real ? a.w.stats[(int64_t)bh * a.w.Sq + i] : -INFINITY;
        a.ndelta[row] = real ? -sum : 0.0f;
        a.lse2[row] = l == -INFINITY ? INFINITY : l * kLog2e;           // (nothing seen: every probability vanishes)
    }
}

// What the two passes see of a tile of y rows.
template <int D> struct PassLds {
    static constexpr int TILE = 64 * D * 2, SLOT = 2 * TILE, SLOTS = 3;
    static constexpr int ROWS = 2048;                // [slot][lse | -Delta][64], of query tiles
};

// ---- dQ: owners of 32 rows per wave, key tiles ---------------------------------------------------------------
template <int D> struct DqLds {
    static constexpr int SLOT = PassLds<D>::SLOT, OWN = kWaves<D> * 2 * 64 * D;
    static constexpr int CENTRE = 3 * SLOT, GROUPS = kWaves<D> * 64 / D;         // sums of a tile's keys, [group of rows][D] floats
    static constexpr int BYTES = CENTRE + GROUPS * D * 4 > SLOT + OWN ? CENTRE + GROUPS * D * 4 : SLOT + OWN;
};

template <int T, int D>
__device__ __forceinline__ void dq_body(const WindowBwdArgs& a, uint8_t* smem, int bh, int row0) {
    using L = PassLds<D>;
    using DL = DqLds<D>;
    constexpr int NW = kWaves<D>, CPR = D / 8, RPW = TilePieces<D, 64, NW>::N, KS = D / 16, DB = D / 32;
    const WindowArgs& w = a.w;
    const int rows = w.Sq * w.g, H = w.Hk * w.g;
    const int b = bh / w.Hk, kvh = bh % w.Hk;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int x0 = row0 + wave * 32, x = min(x0 + l32, rows - 1), i = x / w.g, hg = x - i * w.g;
    const int len = sequence_len(w, b), p0 = first_position(w, b, len);
    const int i_lo = row0 / w.g;
    const Span span = key_span<64>(w, p0 + i_lo, p0 + (min(row0 + NW * 32, rows) - 1) / w.g, len);
    const int wp_lo = p0 + min(x0, rows - 1) / w.g, wp_hi = p0 + min(x0 + 31, rows - 1) / w.g;
    const RowMask mask = {p0 + i - w.left, min(p0 + i + w.right, len - 1), w.sinks};

    const TilePieces<D, 64, NW> pieces(wave, lane);
    const uint32_t lds = lds_addr(smem);
    const uint16_t* kh = w.k + b * w.k_sb + kvh * w.k_sh;
    const uint16_t* vh = w.v + b * w.v_sb + kvh * w.v_sh;
    const uint32_t ks_b = (uint32_t)w.k_sn * 2u, vs_b = (uint32_t)w.v_sn * 2u;
    auto copy_tile = [&](int t, int slot) {
        const int j0 = span.tile(t) * 64;
        const uint16_t *kb = kh + (int64_t)j0 * w.k_sn, *vb = vh + (int64_t)j0 * w.v_sn;
#pragma unroll
        for (int n = 0; n < RPW; n++) {
            const uint32_t row = (uint32_t)(copied_key<64>(span, j0, j0 + pieces.row(n)) - j0);
            const uint32_t dst = lds + slot * L::SLOT + (n * NW + wave) * 1024;
            dma16(kb, row * ks_b + pieces.col(n, lane), __builtin_amdgcn_readfirstlane(dst));
            dma16(vb, row * vs_b + pieces.col(n, lane), __builtin_amdgcn_readfirstlane(dst + L::TILE));
        }
    };
    const Fragments<D> fr(lane);
    v4i b1[KS], b2[KS];
    const uint32_t own = L::SLOT + wave * 2 * 64 * D;
    query_rows_in<D>(w, w.q + b * w.q_sb + (int64_t)kvh * w.g * w.q_sh + (int64_t)i_lo * w.q_sn, w.q_sn, w.q_sh, i_lo, x0, lds + own, lane);
    query_rows_in<D>(w, a.dout + b * a.do_sb + (int64_t)kvh * w.g * a.do_sh + (int64_t)i_lo * a.do_sn, a.do_sn, a.do_sh, i_lo, x0, lds + own + 64 * D, lane);
    if (span.n > 0) copy_tile(0, 0);
    const int64_t at = ((int64_t)b * H + kvh * w.g + hg) * a.sq_pad + i;
    float lse = a.lse2[at], ndelta = a.ndelta[at];
    dma_wait<0>();
#pragma unroll
    for (int s = 0; s < KS; s++) b1[s] = fr.along(smem + own, s), b2[s] = fr.along(smem + own + 64 * D, s);
#pragma unroll
    for (int s = 0; s < KS; s++) asm volatile("" : "+v"(b1[s]), "+v"(b2[s]));
    asm volatile("" : "+v"(lse), "+v"(ndelta));
    __syncthreads();
    if (span.n > 1) copy_tile(1, 1);

    v16f acc[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[d][e] = 0.0f;
    const float c = w.scale * kLog2e;

    // A block of 32 keys: scores S = K Q^T and G = V dO^T, then dS, then dQ^T += K^T dS.
    auto scores_step = [&](const Fragments<D>& fr, const uint8_t* kt, v16f& s, v16f& g, int blk, int ks) {
        s = product<T>(fr.along(kt + blk * 64 * D, ks), b1[ks], s);
        g = product<T>(fr.along(kt + L::TILE + blk * 64 * D, ks), b2[ks], g);
    };
    auto pair = [&](const v16f& s, const v16f& g, int e, bool in0, bool in1) {
        const float y0 = __builtin_amdgcn_exp2f(in0 ? fmaf(s[e], c, -lse) : -INFINITY) * (g[e] + ndelta);
        const float y1 = __builtin_amdgcn_exp2f(in1 ? fmaf(s[e + 1], c, -lse) : -INFINITY) * (g[e + 1] + ndelta);
        return pack2<T>(y0, y1);
    };
    // Rows of dS sum to zero, but for the roundings of dS and of what Delta is made of; whatever their sum is, dS K multiplies it by the
    // keys' common offset.  So the rounded values are summed, and the sum times a vector c close to the mean key is
    // subtracted at the end: dQ = scale dS (K - c).
    float ds_sum = 0.0f;
    auto add_up = [&](uint32_t w) {
        if constexpr (T == kBF16) ds_sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, w), __builtin_bit_cast(v2bf, 0x3F803F80u), ds_sum, false);
        else ds_sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2fp, w), __builtin_bit_cast(v2fp, 0x3C003C00u), ds_sum, false);
    };
    auto acc_step = [&](const Fragments<D>& fr, const uint8_t* kt, const uint32_t (&ds)[8], int blk, int m) {
        const int j2 = m / DB, d = m % DB;
        const v4i sb = {(int)ds[j2 * 4], (int)ds[j2 * 4 + 1], (int)ds[j2 * 4 + 2], (int)ds[j2 * 4 + 3]};
        acc[d] = product<T>(fr.across(kt + (blk * 2 + j2) * 32 * D, d), sb, acc[d]);
    };
    // A whole tile, its two blocks overlapped: scores(0) | scores(1) + dS(0) | products(0) + dS(1) | products(1).
    auto whole = [&](const uint8_t* kt) {
        const Fragments<D> f = fr.fresh();
        v16f s[2], g[2];
        uint32_t ds[2][8];
#pragma unroll
        for (int blk = 0; blk < 2; blk++)
#pragma unroll
            for (int e = 0; e < 16; e++) s[blk][e] = g[blk][e] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) scores_step(f, kt, s[0], g[0], 0, ks);
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            scores_step(f, kt, s[1], g[1], 1, ks);
#pragma unroll
            for (int n = ks * (8 / KS); n < (ks + 1) * (8 / KS); n++) add_up(ds[0][n] = pair(s[0], g[0], n * 2, true, true));
        }
#pragma unroll
        for (int m = 0; m < 2 * DB; m++) {
            acc_step(f, kt, ds[0], 0, m);
#pragma unroll
            for (int n = m * (8 / (2 * DB)); n < (m + 1) * (8 / (2 * DB)); n++) add_up(ds[1][n] = pair(s[1], g[1], n * 2, true, true));
        }
#pragma unroll
        for (int m = 0; m < 2 * DB; m++) acc_step(f, kt, ds[1], 1, m);
    };
    // A tile on the window's edge, block by block (the registers that the mask takes).
    auto edge = [&](const uint8_t* kt, int j0) {
#pragma unroll 1
        for (int blk = 0; blk < 2; blk++) {
            const Fragments<D> f = fr.fresh();
            const RowMask rel = mask.from(j0 + blk * 32 + half * 4);
            v16f s, g;
            uint32_t ds[8];
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = g[e] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) scores_step(f, kt, s, g, blk, ks);
#pragma unroll
            for (int n = 0; n < 8; n++) {
                const int e = n * 2, key = (e >> 2) * 8 + (e & 3);
                add_up(ds[n] = pair(s, g, e, rel.sees(key), rel.sees(key + 1)));
            }
#pragma unroll
            for (int m = 0; m < 2 * DB; m++) acc_step(f, kt, ds, blk, m);
        }
    };

    int slot = 0;
    for (int t = 0; t < span.n; t++) {
        if (t + 1 < span.n) dma_wait<2 * RPW>();
        else dma_wait<0>();
        __syncthreads();
        if (t + 2 < span.n) copy_tile(t + 2, slot == 0 ? 2 : slot - 1);
        const int j0 = span.tile(t) * 64;
        const Seen what = x0 < rows ? seen<64>(w, wp_lo, wp_hi, len, j0) : Seen::kNone;
        const uint8_t* kt = smem + slot * L::SLOT;
        if (what == Seen::kAll) whole(kt);
        else if (what == Seen::kSome) edge(kt, j0);
        if (t == (span.n - 1) / 2) {           // c: the mean of those keys of the tile in the middle that some row here sees
            int me = tid;
            asm volatile("" : "+v"(me));
            const int ch = me % D, first = me / D * (64 / DL::GROUPS);
            float sum = 0.0f;
#pragma unroll 1
            for (int r = first; r < first + 64 / DL::GROUPS; r++) {
                const float k = widen<T>(*reinterpret_cast<const uint16_t*>(kt + nat_off<CPR>(r, ch >> 3) + (ch & 7) * 2), 0);
                sum += copied_key<64>(span, j0, j0 + r) == j0 + r ? k : 0.0f;
            }
            const int j1 = min(j0 + 63, span.hi), sinks = max(0, min(j1 + 1, span.s_end) - j0), others = max(0, j1 + 1 - max(max(j0, span.lo), span.s_end));
            reinterpret_cast<float*>(smem + DL::CENTRE)[me] = sum / (float)(sinks + others);
        }
        slot = slot == 2 ? 0 : slot + 1;
    }
    __syncthreads();
    uint8_t* os = smem + wave * 64 * D;
    if (span.n > 0) {
        const float rs = sum_halves(ds_sum);
        const float* centre = reinterpret_cast<const float*>(smem + DL::CENTRE);
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                v4f c4 = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int n = 0; n < DL::GROUPS; n++) c4 += *reinterpret_cast<const v4f*>(centre + n * D + d * 32 + g * 8 + half * 4);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[d][g * 4 + e] = fmaf(-rs, c4[e], acc[d][g * 4 + e]);
            }
    }
#pragma unroll
    for (int d = 0; d < DB; d++) row_put<T, D>(os, acc[d], d, w.scale, lane);
    if (x0 < rows) query_rows_out<D>(w, os, a.dq + b * a.dq_sb + (int64_t)kvh * w.g * a.dq_sh, a.dq_sn, a.dq_sh, x0, lane);
}

// ---- dK, dV: owners of keys, (head, query tile) pairs -----------------------------------------------------------
// The query tiles that reach keys k0 .. of a block: indices t0 .. t0 + nt - 1 of every head of the group.
struct QuerySpan { int t0, nt; };
__device__ __forceinline__ QuerySpan query_span(const WindowArgs& w, int k0, int p0, int len) {
    const int k1 = min(k0 + kKeysWg, len) - 1;
    const int64_t lo = (int64_t)k0 - w.right - p0;
    const int64_t hi = k0 < w.sinks ? (int64_t)w.Sq - 1 : (int64_t)k1 + w.left - p0;
    const int i0 = (int)(lo < 0 ? 0 : lo > w.Sq ? w.Sq : lo), i1 = (int)(hi < -1 ? -1 : hi > w.Sq - 1 ? w.Sq - 1 : hi);
    if (k1 < k0 || i1 < i0) return QuerySpan{0, 0};
    return QuerySpan{i0 >> 6, (i1 >> 6) - (i0 >> 6) + 1};
}
// Which of the queries at positions pa .. pb a wave's keys x0 .. x1 are seen by.
__device__ __forceinline__ Seen seen_by(const WindowArgs& w, int x0, int len, int pa, int pb) {
    const int x1 = x0 + 31;
    if (x0 >= len || x0 > pb + w.right || (x1 < pa - w.left && x0 >= w.sinks)) return Seen::kNone;
    return x1 < len && x1 <= pa + w.right && (x0 >= pb - w.left || x1 < w.sinks) ? Seen::kAll : Seen::kSome;
}
// Which rows of a workgroup's share: the walk over heads and tiles, one pair after the other.
struct Walk {
    int t0, nt, hg, qt;
    __device__ Walk(const QuerySpan& q, int first) : t0(q.t0), nt(q.nt), hg(0), qt(0) {
        if (nt > 0) hg = first / nt, qt = first - hg * nt;
    }
    __device__ void next() {
        if (++qt == nt) qt = 0, hg++;
    }
    __device__ int tile() const { return t0 + qt; }
};
// Positions of queries p that see the lane's key: lo <= p <= hi.  (Up to the last query: the padding of its tile stands at further ones.)
struct KeyMask {
    int lo, hi;
    __device__ bool sees(int n) const { return n >= lo && n <= hi; }
};
__device__ __forceinline__ KeyMask key_mask(const WindowArgs& w, int j, int len, int p0) {
    return j < len ? KeyMask{j - w.right, min(p0 + w.Sq - 1, j < w.sinks ? kWindowFar : j + w.left)} : KeyMask{kWindowFar, -kWindowFar};
}

// What a workgroup of this kind does: block of keys, chunk of its pairs, and where its result goes.
struct KeyWork { int k0, first, count; int64_t part; };          // part: index of its fp32 part, -1: straight to dK and dV
__device__ __forceinline__ KeyWork key_work(const WindowBwdArgs& a, int bh, int r, int total_blocks) {
    const int sink_wgs = a.sink_blocks * a.sink_chunks;
    int block, chunk;
    KeyWork k;
    k.part = -1;
    if (r < sink_wgs) {
        block = r / a.sink_chunks, chunk = r % a.sink_chunks;
        if (a.sink_chunks > 1) k.part = (int64_t)bh * ((a.sink_chunks > 1 ? sink_wgs : 0) + (a.chunks > 1 ? (total_blocks - a.sink_blocks) * a.chunks : 0)) + r;
    } else {
        r -= sink_wgs;
        block = a.sink_blocks + r / a.chunks, chunk = r % a.chunks;
        if (a.chunks > 1) {
            const int mine = a.sink_chunks > 1 ? sink_wgs : 0;
            k.part = (int64_t)bh * (mine + (total_blocks - a.sink_blocks) * a.chunks) + mine + r;
        }
    }
    k.k0 = block * kKeysWg;
    k.first = chunk * a.chunk_tiles;
    k.count = a.chunk_tiles;
    return k;
}

// 32 keys' gradients of a wave: fp32 registers -> the part's rows, or packed through LDS -> the caller's rows.
template <int T, int D>
__device__ __forceinline__ void key_rows_out(const WindowBwdArgs& a, const v16f (&acc)[D / 32], float mul, uint8_t* os, int64_t part, int which, uint16_t* out, int64_t sn,
                                             int x0, int k0, int lane) {
    constexpr int CPR = D / 8, RPI = 64 / CPR, DB = D / 32;
    asm volatile("" : "+v"(lane));
    if (part >= 0) {
        float* p = a.part + ((part * 2 + which) * kKeysWg + (x0 - k0) + (lane & 31)) * D + (lane >> 5) * 4;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<v4f*>(p + d * 32 + g * 8) = v4f{acc[d][g * 4] * mul, acc[d][g * 4 + 1] * mul, acc[d][g * 4 + 2] * mul, acc[d][g * 4 + 3] * mul};
        return;
    }
#pragma unroll
    for (int d = 0; d < DB; d++) row_put<T, D>(os, acc[d], d, mul, lane);
#pragma unroll
    for (int n = 0; n < 32 / RPI; n++) {
        const int r = n * RPI + lane / CPR;
        const u32x4 v = *reinterpret_cast<const u32x4*>(os + nat_off<CPR>(r, lane % CPR));
        if (x0 + r < a.w.Skv) *reinterpret_cast<u32x4*>(out + (int64_t)(x0 + r) * sn + (lane % CPR) * 8) = v;
    }
}
template <int D>
__device__ __forceinline__ void key_rows_in(const uint16_t* head, int64_t sn, int k0, int x0, int last, uint32_t dst, int lane) {
    constexpr int CPR = D / 8, RPI = 64 / CPR;
    const uint16_t* base = head + (int64_t)k0 * sn;          // (k0 <= last, or nothing of it is used)
#pragma unroll
    for (int n = 0; n < 32 / RPI; n++) {
        const int r = n * RPI + lane / CPR;
        dma16(base, (uint32_t)(max(min(x0 + r, last), k0) - k0) * (uint32_t)(sn * 2) + nat_pos<CPR>(r, lane % CPR) * 16, __builtin_amdgcn_readfirstlane(dst + n * 1024));
    }
}

// A query tile's copies: 64 rows of Q and of dO of one head, and their statistics.
template <int T, int D, int NW> struct QueryTiles {
    using L = PassLds<D>;
    static constexpr int RPW = TilePieces<D, 64, NW>::N;
    const WindowBwdArgs& a;
    int b, kvh, wave, lane;
    TilePieces<D, 64, NW> pieces;
    uint32_t rows_at, ring_at;
    __device__ QueryTiles(const WindowBwdArgs& a_, int b_, int kvh_, int wave_, int lane_, uint32_t rows_at_, uint32_t ring_at_)
        : a(a_), b(b_), kvh(kvh_), wave(wave_), lane(lane_), pieces(wave_, lane_), rows_at(rows_at_), ring_at(ring_at_) {}
    __device__ void copy(int hg, int qt, int slot) const {
        const WindowArgs& w = a.w;
        const int h = kvh * w.g + hg, i0 = qt * 64;
        const uint16_t* qb = w.q + b * w.q_sb + h * w.q_sh + (int64_t)i0 * w.q_sn;
        const uint16_t* gb = a.dout + b * a.do_sb + h * a.do_sh + (int64_t)i0 * a.do_sn;
        const int64_t row = ((int64_t)b * w.Hk * w.g + h) * a.sq_pad + i0;
        // (first, so that a wait for the copies below covers them)
        if (wave == 0) dma4(a.lse2 + row, lane * 4, __builtin_amdgcn_readfirstlane(rows_at + (slot * 2 + 0) * 256));
        if (wave == 1) dma4(a.ndelta + row, lane * 4, __builtin_amdgcn_readfirstlane(rows_at + (slot * 2 + 1) * 256));
#pragma unroll
        for (int n = 0; n < RPW; n++) {
            const uint32_t r = (uint32_t)min(pieces.row(n), w.Sq - 1 - i0);
            const uint32_t dst = ring_at + slot * L::SLOT + (n * NW + wave) * 1024;
            dma16(qb, r * (uint32_t)(w.q_sn * 2) + pieces.col(n, lane), __builtin_amdgcn_readfirstlane(dst));
            dma16(gb, r * (uint32_t)(a.do_sn * 2) + pieces.col(n, lane), __builtin_amdgcn_readfirstlane(dst + L::TILE));
        }
    }
};

// Head dim 64: a wave carries both products of its 32 keys.
template <int D> struct KeyLds {
    using L = PassLds<D>;
    static constexpr int OWN = kWaves<D> * 2 * 64 * D;
    static constexpr int BYTES = L::ROWS + (3 * L::SLOT > L::SLOT + OWN ? 3 * L::SLOT : L::SLOT + OWN);
};

template <int T, int D>
__device__ __forceinline__ void dkdv_body(const WindowBwdArgs& a, uint8_t* smem, int bh, const KeyWork& work) {
    using L = PassLds<D>;
    constexpr int NW = kWaves<D>, KS = D / 16, DB = D / 32, RPW = QueryTiles<T, D, NW>::RPW;
    static_assert(NW * 32 == kKeysWg, "a wave owns 32 keys");
    const WindowArgs& w = a.w;
    const int b = bh / w.Hk, kvh = bh % w.Hk;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int x0 = work.k0 + wave * 32, j = x0 + l32;
    const int len = sequence_len(w, b), p0 = first_position(w, b, len);
    const QuerySpan qs = query_span(w, work.k0, p0, len);
    const int n_tiles = max(0, min(qs.nt * w.g - work.first, work.count));
    const KeyMask mask = key_mask(w, j, len, p0);
    const uint32_t lds = lds_addr(smem);
    const QueryTiles<T, D, NW> tiles(a, b, kvh, wave, lane, lds, lds + L::ROWS);
    Walk ahead(qs, work.first), here = ahead;

    const Fragments<D> kept(lane);
    v4i b1[KS], b2[KS];
    const uint32_t own = L::ROWS + L::SLOT + wave * 2 * 64 * D;
    key_rows_in<D>(w.k + b * w.k_sb + kvh * w.k_sh, w.k_sn, min(work.k0, max(len - 1, 0)), x0, max(len - 1, 0), lds + own, lane);
    key_rows_in<D>(w.v + b * w.v_sb + kvh * w.v_sh, w.v_sn, min(work.k0, max(len - 1, 0)), x0, max(len - 1, 0), lds + own + 64 * D, lane);
    if (n_tiles > 0) tiles.copy(ahead.hg, ahead.tile(), 0), ahead.next();
    dma_wait<0>();
#pragma unroll
    for (int s = 0; s < KS; s++) b1[s] = kept.along(smem + own, s), b2[s] = kept.along(smem + own + 64 * D, s);
#pragma unroll
    for (int s = 0; s < KS; s++) asm volatile("" : "+v"(b1[s]), "+v"(b2[s]));
    __syncthreads();
    if (n_tiles > 1) tiles.copy(ahead.hg, ahead.tile(), 1), ahead.next();

    v16f dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) dk[d][e] = dv[d][e] = 0.0f;
    const float c = w.scale * kLog2e;

    auto tile = [&](auto masked_tag, int pa, int slot) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        const KeyMask rel = {mask.lo - pa - half * 4, mask.hi - pa - half * 4};
        const Fragments<D> fr = kept.fresh();
        const uint8_t* qt = smem + L::ROWS + slot * L::SLOT;
        const uint8_t* gt = qt + L::TILE;
        const uint8_t* rows = smem + slot * 512;
        v16f s[2], g[2];
        uint32_t pp[2][8], ds[2][8];
#pragma unroll
        for (int blk = 0; blk < 2; blk++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const v4f nd = *reinterpret_cast<const v4f*>(rows + 256 + (blk * 32 + q * 8 + half * 4) * 4);
#pragma unroll
                for (int e = 0; e < 4; e++) s[blk][q * 4 + e] = 0.0f, g[blk][q * 4 + e] = nd[e];
            }
        auto scores_step = [&](int blk, int ks) {
            s[blk] = product<T>(fr.along(qt + blk * 64 * D, ks), b1[ks], s[blk]);
            g[blk] = product<T>(fr.along(gt + blk * 64 * D, ks), b2[ks], g[blk]);
        };
        v4f lse;
        auto pair = [&](int blk, int e0) {
            if ((e0 & 3) == 0) lse = *reinterpret_cast<const v4f*>(rows + (blk * 32 + (e0 >> 2) * 8 + half * 4) * 4);
            float y[2], z[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int n = e0 + e;
                y[e] = __builtin_amdgcn_exp2f(fmaf(s[blk][n], c, -lse[n & 3]));
                z[e] = y[e] * g[blk][n];
                if constexpr (MASKED) {
                    const bool in = rel.sees(blk * 32 + (n >> 2) * 8 + (n & 3));
                    y[e] = in ? y[e] : 0.0f;
                    z[e] = in ? z[e] : 0.0f;             // (a key that nothing sees may hold anything)
                }
            }
            pp[blk][e0 >> 1] = pack2<T>(y[0], y[1]);
            ds[blk][e0 >> 1] = pack2<T>(z[0], z[1]);
        };
        auto acc_step = [&](int blk, int m) {
            const int which = m / (2 * DB), j2 = (m / DB) & 1, d = m % DB;
            const int at = (blk * 2 + j2) * 32 * D;
            const uint32_t(&r)[8] = which == 0 ? ds[blk] : pp[blk];
            const v4i sb = {(int)r[j2 * 4], (int)r[j2 * 4 + 1], (int)r[j2 * 4 + 2], (int)r[j2 * 4 + 3]};
            if (which == 0) dk[d] = product<T>(fr.across(qt + at, d), sb, dk[d]);
            else dv[d] = product<T>(fr.across(gt + at, d), sb, dv[d]);
        };
#pragma unroll
        for (int ks = 0; ks < KS; ks++) scores_step(0, ks);
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            scores_step(1, ks);
#pragma unroll
            for (int n = 0; n < 8 / KS; n++) pair(0, (ks * (8 / KS) + n) * 2);
        }
#pragma unroll
        for (int m = 0; m < 4 * DB; m++) {
            acc_step(0, m);
#pragma unroll
            for (int n = 0; n < 8 / (4 * DB); n++) pair(1, (m * (8 / (4 * DB)) + n) * 2);
        }
#pragma unroll
        for (int m = 0; m < 4 * DB; m++) acc_step(1, m);
    };

    int slot = 0;
    for (int t = 0; t < n_tiles; t++) {
        if (t + 1 < n_tiles) dma_wait<2 * RPW>();
        else dma_wait<0>();
        __syncthreads();
        if (t + 2 < n_tiles) tiles.copy(ahead.hg, ahead.tile(), slot == 0 ? 2 : slot - 1), ahead.next();
        const int pa = p0 + here.tile() * 64;
        here.next();
        const Seen what = seen_by(w, x0, len, pa, min(pa + 63, p0 + w.Sq - 1));
        if (what == Seen::kAll) tile(std::false_type{}, pa, slot);
        else if (what == Seen::kSome) tile(std::true_type{}, pa, slot);
        slot = slot == 2 ? 0 : slot + 1;
    }
    __syncthreads();
    uint8_t* os = smem + L::ROWS + wave * 64 * D;
    key_rows_out<T, D>(a, dk, w.scale, os, work.part, 0, a.dk + b * a.dk_sb + kvh * a.dk_sh, a.dk_sn, x0, work.k0, lane);
    key_rows_out<T, D>(a, dv, 1.0f, os, work.part, 1, a.dv + b * a.dv_sb + kvh * a.dv_sh, a.dv_sn, x0, work.k0, lane);
}

// Head dim 128: a pair of waves shares 32 keys, the P wave with K rows and dV, the S wave, one tile behind, with V rows and dK; P crosses
// over through LDS with some bits more than dS is rounded to: as fp16 pairs where that is bf16 (see sage_bwd.hip), as the upper three bytes of fp32
// where it is fp16 (with fp16 there dK's relative error was 3.5e-4, with these 2.9e-4).
template <int T, int D> struct PairLds {
    using L = PassLds<D>;
    static constexpr int WORDS = T == kBF16 ? 2 : 3;          // 16-byte words for the 16 values of a block
    static constexpr int HAND = 4 * 2 * WORDS * 64 * 16;      // [pair][32-row block][word][lane]
    static constexpr int RING = L::ROWS + 2 * HAND, BYTES = RING + 3 * L::SLOT;
    static_assert(BYTES <= 160 * 1024, "LDS of a compute unit");
    static_assert(8 * 64 * D <= 2 * L::SLOT, "the owner rows must fit behind the first slot");
};

// Four floats <-> the upper three bytes of each (15 bits behind the leading one).
__device__ __forceinline__ void pack24(const float (&y)[4], uint32_t* w) {
    const uint32_t a = __float_as_uint(y[0]), b = __float_as_uint(y[1]), c = __float_as_uint(y[2]), d = __float_as_uint(y[3]);
    w[0] = __builtin_amdgcn_perm(b, a, 0x05030201u);
    w[1] = __builtin_amdgcn_perm(c, b, 0x06050302u);
    w[2] = __builtin_amdgcn_perm(d, c, 0x07060503u);
}
__device__ __forceinline__ float unpack24(const uint32_t* w, int i) {
    return __uint_as_float(i == 0 ? w[0] << 8 : i == 1 ? __builtin_amdgcn_perm(w[1], w[0], 0x0504030Cu) : i == 2 ? __builtin_amdgcn_perm(w[2], w[1], 0x0403020Cu)
                                                                                                            : w[2] & 0xFFFFFF00u);
}

template <int T, int D, int ROLE>
__device__ __forceinline__ void dkdv_role(const WindowBwdArgs& a, uint8_t* smem, int bh, const KeyWork& work, int wave, int lane) {
    using L = PassLds<D>;
    using PL = PairLds<T, D>;
    constexpr int KS = D / 16, DB = D / 32;
    const WindowArgs& w = a.w;
    const int b = bh / w.Hk, kvh = bh % w.Hk;
    const int pr = wave & 3, half = lane >> 5, l32 = lane & 31;
    const int x0 = work.k0 + pr * 32, j = x0 + l32;
    const int len = sequence_len(w, b), p0 = first_position(w, b, len);
    const QuerySpan qs = query_span(w, work.k0, p0, len);
    const int n_tiles = max(0, min(qs.nt * w.g - work.first, work.count));
    const KeyMask mask = key_mask(w, j, len, p0);
    const uint32_t lds = lds_addr(smem);
    const QueryTiles<T, D, 8> tiles(a, b, kvh, wave, lane, lds, lds + PL::RING);
    Walk ahead(qs, work.first), here = ahead;

    const Fragments<D> kept(lane);
    v4i bx[KS];
    const uint32_t own = PL::RING + L::SLOT + wave * 64 * D;
    key_rows_in<D>(ROLE == 0 ? w.k + b * w.k_sb + kvh * w.k_sh : w.v + b * w.v_sb + kvh * w.v_sh, ROLE == 0 ? w.k_sn : w.v_sn, min(work.k0, max(len - 1, 0)), x0,
                   max(len - 1, 0), lds + own, lane);
    if (n_tiles > 0) tiles.copy(ahead.hg, ahead.tile(), 0), ahead.next();
    dma_wait<0>();
#pragma unroll
    for (int s = 0; s < KS; s++) bx[s] = kept.along(smem + own, s);
#pragma unroll
    for (int s = 0; s < KS; s++) asm volatile("" : "+v"(bx[s]));

    v16f acc[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[d][e] = 0.0f;
    const float c = w.scale * kLog2e;
    u32x4* hand = reinterpret_cast<u32x4*>(smem + L::ROWS) + pr * 2 * PL::WORDS * 64 + lane;

    auto tile = [&](auto masked_tag, int pa, int mine, int turn, auto&& copy_next) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        const KeyMask rel = {mask.lo - pa - half * 4, mask.hi - pa - half * 4};
        const Fragments<D> fr = kept.fresh();
        const uint8_t* nt = smem + PL::RING + mine * L::SLOT + ROLE * L::TILE;
        const uint8_t* rt = smem + PL::RING + mine * L::SLOT + (1 - ROLE) * L::TILE;
        const uint8_t* rowv = smem + (mine * 2 + ROLE) * 256;
        uint32_t hp[2][4 * PL::WORDS];   // P on its way to the S wave
        if constexpr (ROLE == 1) {
#pragma unroll
            for (int blk = 0; blk < 2; blk++)
#pragma unroll
                for (int n = 0; n < PL::WORDS; n++) {
                    const u32x4 v = hand[turn * (PL::HAND / 16) + (blk * PL::WORDS + n) * 64];
#pragma unroll
                    for (int e = 0; e < 4; e++) hp[blk][n * 4 + e] = v[e];
                }
        }
        v16f s[2];
        uint32_t pk[2][8];
        float last[2];
        v4f rv;
#pragma unroll
        for (int blk = 0; blk < 2; blk++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                v4f nd = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (ROLE == 1) nd = *reinterpret_cast<const v4f*>(rowv + (blk * 32 + q * 8 + half * 4) * 4);
#pragma unroll
                for (int e = 0; e < 4; e++) s[blk][q * 4 + e] = nd[e];
            }
        auto scores_step = [&](int blk, int ks) { s[blk] = product<T>(fr.along(nt + blk * 64 * D, ks), bx[ks], s[blk]); };
        auto pair = [&](int blk, int e0) {
            if (ROLE == 0 && (e0 & 3) == 0) rv = *reinterpret_cast<const v4f*>(rowv + (blk * 32 + (e0 >> 2) * 8 + half * 4) * 4);
            float y[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int n = e0 + e;
                if constexpr (ROLE == 0) {
                    y[e] = __builtin_amdgcn_exp2f(fmaf(s[blk][n], c, -rv[n & 3]));
                } else {
                    if constexpr (T == kBF16) y[e] = fmaf((float)__builtin_bit_cast(v2fp, hp[blk][e0 >> 1])[e], s[blk][n], 0.0f);
                    else y[e] = unpack24(&hp[blk][(n >> 2) * 3], n & 3) * s[blk][n];
                }
                if (MASKED && !rel.sees(blk * 32 + (n >> 2) * 8 + (n & 3))) y[e] = 0.0f;       // (in both: a key that nothing sees may hold anything)
            }
            pk[blk][e0 >> 1] = pack2<T>(y[0], y[1]);
            if constexpr (ROLE == 0) {
                if constexpr (T == kBF16) hp[blk][e0 >> 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(y[0], y[1]));
                else if (e0 & 2) pack24({last[0], last[1], y[0], y[1]}, &hp[blk][(e0 >> 2) * 3]);
                last[0] = y[0], last[1] = y[1];
            }
        };
        auto hand_over = [&](int blk) {
            if constexpr (ROLE == 0) {
                const auto& r = hp[blk];
#pragma unroll
                for (int n = 0; n < PL::WORDS; n++)
                    hand[turn * (PL::HAND / 16) + (blk * PL::WORDS + n) * 64] = u32x4{r[n * 4], r[n * 4 + 1], r[n * 4 + 2], r[n * 4 + 3]};
            }
        };
        auto acc_step = [&](int blk, int m) {
            const int j2 = m / DB, d = m % DB;
            const v4i sb = {(int)pk[blk][j2 * 4], (int)pk[blk][j2 * 4 + 1], (int)pk[blk][j2 * 4 + 2], (int)pk[blk][j2 * 4 + 3]};
            acc[d] = product<T>(fr.across(rt + (blk * 2 + j2) * 32 * D, d), sb, acc[d]);
        };
#pragma unroll
        for (int ks = 0; ks < KS; ks++) scores_step(0, ks);
        copy_next();
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            scores_step(1, ks);
#pragma unroll
            for (int n = 0; n < 8 / KS; n++) pair(0, (ks * (8 / KS) + n) * 2);
        }
        hand_over(0);
#pragma unroll
        for (int m = 0; m < 2 * DB; m++) {
            acc_step(0, m);
#pragma unroll
            for (int n = 0; n < 8 / (2 * DB); n++) pair(1, (m * (8 / (2 * DB)) + n) * 2);
        }
        hand_over(1);
#pragma unroll
        for (int m = 0; m < 2 * DB; m++) acc_step(1, m);
    };

    // iteration `it`: the P wave works on tile it, the S wave on tile it - 1
    int slot = 0;                        // it % 3
    for (int it = 0; n_tiles > 0 && it <= n_tiles; it++) {
        dma_wait<0>();
        __syncthreads();                 // this iteration's tile and the previous one's P are visible; the slot of tile it - 2 is free
        const int next = slot == 2 ? 0 : slot + 1;
        const int mine = ROLE == 0 ? slot : slot == 0 ? 2 : slot - 1;
        slot = next;
        bool copied = it + 1 >= n_tiles;
        auto copy_next = [&] {
            if (!copied) tiles.copy(ahead.hg, ahead.tile(), next), ahead.next();
            copied = true;
        };
        if (ROLE == 0 ? it < n_tiles : it > 0) {
            const int pa = p0 + here.tile() * 64, turn = (ROLE == 0 ? it : it - 1) & 1;
            here.next();
            const Seen what = seen_by(w, x0, len, pa, min(pa + 63, p0 + w.Sq - 1));
            if (what == Seen::kAll) tile(std::false_type{}, pa, mine, turn, copy_next);
            else if (what == Seen::kSome) tile(std::true_type{}, pa, mine, turn, copy_next);
        }
        copy_next();
    }
    __syncthreads();                     // (every copy has landed, every tile has been read: the ring takes the output rows)
    uint8_t* os = smem + PL::RING + wave * 64 * D;
    if constexpr (ROLE == 0) key_rows_out<T, D>(a, acc, 1.0f, os, work.part, 1, a.dv + b * a.dv_sb + kvh * a.dv_sh, a.dv_sn, x0, work.k0, lane);
    else key_rows_out<T, D>(a, acc, w.scale, os, work.part, 0, a.dk + b * a.dk_sb + kvh * a.dk_sh, a.dk_sn, x0, work.k0, lane);
}

template <int T, int D>
__global__ __launch_bounds__(kWaves<D> * 64, 2) void window_bwd_kernel(WindowBwdArgs a) {
    constexpr bool PAIRED = D > 64;
    constexpr int KV = PAIRED ? PairLds<T, D>::BYTES : KeyLds<D>::BYTES;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[KV > DqLds<D>::BYTES ? KV : DqLds<D>::BYTES];
    const int heads = a.w.B * a.w.Hk, rows = a.w.Sq * a.w.g;
    const int tq = (rows + kRowsWg<D> - 1) / kRowsWg<D>, blocks = (a.w.Skv + kKeysWg - 1) / kKeysWg;
    const int id = (int)blockIdx.x, nq = heads * tq;
    if (id < nq) {
        const int item = xcd_item(id, nq);
        dq_body<T, D>(a, smem, item / tq, (tq - 1 - item % tq) * kRowsWg<D>);
        return;
    }
    const int tk = a.sink_blocks * a.sink_chunks + (blocks - a.sink_blocks) * a.chunks, item = xcd_item(id - nq, heads * tk);
    const KeyWork work = key_work(a, item / tk, item % tk, blocks);
    if constexpr (PAIRED) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        if (wave < 4) dkdv_role<T, D, 0>(a, smem, item / tk, work, wave, lane);
        else dkdv_role<T, D, 1>(a, smem, item / tk, work, wave, lane);
    } else {
        dkdv_body<T, D>(a, smem, item / tk, work);
    }
}

// Launch 3: dK and dV of the blocks that several workgroups share, their parts added in order.  8 channels to a thread.
template <int T, int D>
__global__ __launch_bounds__(256) void window_bwd_join_kernel(WindowBwdArgs a) {
    constexpr int CPR = D / 8;
    const int blocks = (a.w.Skv + kKeysWg - 1) / kKeysWg;
    const int sink_parts = a.sink_chunks > 1 ? a.sink_blocks : 0, rest_parts = a.chunks > 1 ? blocks - a.sink_blocks : 0;
    const int64_t per_head = (int64_t)(sink_parts + rest_parts) * 2 * kKeysWg * CPR;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= (int64_t)a.w.B * a.w.Hk * per_head) return;
    const int bh = (int)(at / per_head), col = (int)(at % CPR) * 8;
    int64_t r = at % per_head / CPR;
    const int key = (int)(r % kKeysWg), which = (int)(r / kKeysWg & 1), n = (int)(r / (2 * kKeysWg));
    const bool sink = n < sink_parts;
    const int block = sink ? n : a.sink_blocks + n - sink_parts, chunks = sink ? a.sink_chunks : a.chunks;
    const int64_t sink_wgs = (int64_t)sink_parts * a.sink_chunks, wgs = sink_wgs + (int64_t)rest_parts * a.chunks;
    const int64_t part = bh * wgs + (sink ? (int64_t)n * a.sink_chunks : sink_wgs + (int64_t)(n - sink_parts) * a.chunks);
    const float* p = a.part + ((part * 2 + which) * kKeysWg + key) * D + col;
    float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int c = 0; c < chunks; c++) {
        const v4f u = *reinterpret_cast<const v4f*>(p + (int64_t)c * 2 * kKeysWg * D), v = *reinterpret_cast<const v4f*>(p + (int64_t)c * 2 * kKeysWg * D + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] += u[e], y[4 + e] += v[e];
    }
    const int j = block * kKeysWg + key, b = bh / a.w.Hk, kvh = bh % a.w.Hk;
    if (j >= a.w.Skv) return;
    uint16_t* out = which ? a.dv + b * a.dv_sb + kvh * a.dv_sh + j * a.dv_sn : a.dk + b * a.dk_sb + kvh * a.dk_sh + j * a.dk_sn;
    *reinterpret_cast<u32x4*>(out + col) = u32x4{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7])};
}

template <int T, int D> hipError_t launch_td(const WindowBwdArgs& a, hipStream_t st) {
    const int64_t heads = (int64_t)a.w.B * a.w.Hk, rows = (int64_t)a.w.Sq * a.w.g, blocks = (a.w.Skv + kKeysWg - 1) / kKeysWg;
    const int64_t prep = (heads * a.w.g * a.sq_pad * (D / 8) + 255) / 256;
    const int64_t grid = heads * ((rows + kRowsWg<D> - 1) / kRowsWg<D> + a.sink_blocks * a.sink_chunks + (blocks - a.sink_blocks) * a.chunks);
    const int64_t shared = (a.sink_chunks > 1 ? a.sink_blocks : 0) + (a.chunks > 1 ? blocks - a.sink_blocks : 0);
    const int64_t join = (heads * shared * 2 * kKeysWg * (D / 8) + 255) / 256;
    if (prep > 0x7FFFFFFF || grid > 0x7FFFFFFF || join > 0x7FFFFFFF) return hipErrorInvalidValue;
    hipLaunchKernelGGL((window_bwd_prep_kernel<T, D>), dim3((unsigned)prep), dim3(256), 0, st, a);
    hipLaunchKernelGGL((window_bwd_kernel<T, D>), dim3((unsigned)grid), dim3(kWaves<D> * 64), 0, st, a);
    if (join > 0) hipLaunchKernelGGL((window_bwd_join_kernel<T, D>), dim3((unsigned)join), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

// A key block's pairs without sinks: as many as its window spans.  They are dealt to several workgroups where whole blocks would leave the chip
// partly empty (two to a compute unit are wanted), down to 8 pairs; a block with sinks to as many as give each about that share too.
void window_bwd_plan(WindowBwdArgs* a) {
    const WindowArgs& w = a->w;
    const int64_t all = (w.Sq + 63) / 64, blocks = (w.Skv + kKeysWg - 1) / kKeysWg, heads = (int64_t)w.B * w.Hk;
    const int64_t tiles = std::min<int64_t>(all, ((int64_t)w.left + w.right + kKeysWg + 62) / 64 + 1), pairs = tiles * w.g;
    const int64_t want = std::max<int64_t>(1, 512 / (blocks * heads)), most = std::max<int64_t>(1, pairs / 8);
    const int64_t chunks = std::min(want, most), per = (pairs + chunks - 1) / chunks;
    a->chunks = (int)((pairs + per - 1) / per);
    a->chunk_tiles = (int)per;
    a->sink_blocks = tiles < all ? (w.sinks + kKeysWg - 1) / kKeysWg : 0;
    a->sink_chunks = (int)((all * w.g + per - 1) / per);
}
int64_t window_bwd_parts(const WindowBwdArgs& a) {
    const int64_t blocks = (a.w.Skv + kKeysWg - 1) / kKeysWg;
    return (int64_t)a.w.B * a.w.Hk * ((a.sink_chunks > 1 ? a.sink_blocks * a.sink_chunks : 0) + (a.chunks > 1 ? (blocks - a.sink_blocks) * a.chunks : 0));
}

hipError_t launch_window_bwd(const WindowBwdArgs& a, hipStream_t st) {
    if (a.w.D == 64) return a.w.type == kBF16 ? launch_td<kBF16, 64>(a, st) : launch_td<kF16, 64>(a, st);
    return a.w.type == kBF16 ? launch_td<kBF16, 128>(a, st) : launch_td<kF16, 128>(a, st);
}

}  // namespace sage
