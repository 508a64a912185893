// sage_window_bwd.hip — gradient of attention over a sliding window, bf16 or fp16, head dims 64 and 128.
//
//     P_ij = exp(scale q_i . k_j - L_i) for the keys j that query i sees, else 0
//     Delta_i = dO_i . O_i,  dS_ij = P_ij (dO_i . v_j - Delta_i)
//     dQ_i = scale sum_j dS_ij k_j,  dK_j = scale sum_i dS_ij q_i,  dV_j = sum_i P_ij dO_i
// where the sums over i of a shared key head run over the queries of all its heads.  No atomics: the same bits on every call.
//
// Launch 1: Delta_i (from O with what rounding left of it, where the caller kept that) and L_i log2(e).  Launch 2: one grid of two kinds of workgroups, as the full backward's (sage_bwd.hip, whose
// reasons for tiles, rings and the order of the work hold here): owners of rows, that walk the key tiles their window reaches -> dQ; and owners of
// 64 keys, that walk the (head, query tile) pairs that reach them -> dK, dV.  Blocks with sinks are reached by every later query; their
// pairs are dealt to several workgroups (window_bwd_plan), which leave fp32 parts for launch 3
// to add up in order.  The same where there are too few key blocks to fill the chip.
//
// The same for whole sequences that lie one behind the other: bf16, [20576 rows in 8, 24 on 8 heads x 64] causal 745 to 780 us, Delta 30; [2652 rows in 3, 30 x 128] full 200, 12.
#include "sage_grid.h"
#include "sage_window_common.h"

#include <algorithm>
#include <type_traits>

namespace sage {

namespace {

typedef __fp16 v2fp __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4, kRowsWg = kWaves * 32;
constexpr int kKeysWg = kWindowBwdKeys;                          // (pairs of waves share 32 keys)

// Weights are carried times 2^14 (by their statistic, at no cost): as fp16, which is how dV takes them where that is the type, and how they are handed on
// where it is bf16 (PairLds), those down to 2^-28 keep all bits.  What is made of them is multiplied by kWeightInv at the end.
constexpr float kWeightBits = 14.0f, kWeightInv = 0x1p-14f;
// fp16: the power of two that dS = P (dP - Delta) is rounded with, from the sum of its row's |dO|, or the largest such sum of the rows that meet in a dK.
// |dS| <= sum |dO| max |v| / 2, so that it stays within fp16's range for |v| < 511, and the largest keep all bits for weights down to 2^-18 or so,
// whatever the size of dO.  (Without it the relative error of dQ and dK was 3 times that of one rounding at dO of 1e-3 and 4 times at 1e-4.)
__device__ __forceinline__ int ds_power(float sum) { return 8 - __builtin_amdgcn_frexp_expf(sum); }

template <int T> __device__ __forceinline__ float widen(uint32_t w, int i) {
    if constexpr (T == kBF16) return __uint_as_float(i ? w & 0xFFFF0000u : w << 16);
    else return (float)__builtin_bit_cast(v2hf, w)[i];
}

// Row i of head bh, CPR threads to it; `at`: its place in the workspace.
template <int T, int D> __device__ __forceinline__ void prep_row(const WindowBwdArgs& a, int bh, int i, int64_t at_row) {
    constexpr int CPR = D / 8;
    const int H = a.w.Hk * a.w.g, b = bh / H, h = bh % H, col = (int)(threadIdx.x % CPR) * 8;
    const int len = sequence_len(a.w, b);
    const bool real = seeing(a.w, first_position(a.w, b, len), len).has(i);           // (rows that see nothing are not read: they may hold anything)
    float sum = 0.0f, size = 0.0f;
    if (real) {
        const int64_t at = b * a.w.o_sb + h * a.w.o_sh + i * a.w.o_sn + col;
        const u32x4 o = *reinterpret_cast<const u32x4*>(a.w.o + at);
        const u32x4 rest = a.w.rest ? *reinterpret_cast<const u32x4*>(a.w.rest + at) : u32x4{0u, 0u, 0u, 0u};
        const u32x4 g = *reinterpret_cast<const u32x4*>(a.dout + b * a.do_sb + h * a.do_sh + i * a.do_sn + col);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t ow = o[e >> 1], rw = rest[e >> 1], gw = g[e >> 1];
            sum = fmaf(widen<T>(ow, e & 1) + widen<T>(rw, e & 1), widen<T>(gw, e & 1), sum);
            if constexpr (T == kF16) size += fabsf(widen<T>(gw, e & 1));
        }
    }
#pragma unroll
    for (int m = 1; m < CPR; m <<= 1) {
        sum += __shfl_xor(sum, m);
        if constexpr (T == kF16) size += __shfl_xor(size, m);
    }
    if (col == 0) {
        const float l = real ? a.w.stats[(int64_t)bh * a.w.stats_n + i] : -INFINITY;
        a.ndelta[at_row] = real ? -sum : 0.0f;
        if constexpr (T == kF16) a.dsize[at_row] = size;
        a.lse2[at_row] = l == -INFINITY ? INFINITY : fmaf(l, kLog2e, -kWeightBits);           // (nothing seen: every probability vanishes)
    }
}

template <int T, int D>
__global__ __launch_bounds__(256) void window_bwd_prep_kernel(WindowBwdArgs a) {
    constexpr int CPR = D / 8, RPP = 256 / CPR;      // threads per row, rows per workgroup
    const int64_t row = (int64_t)blockIdx.x * RPP + threadIdx.x / CPR;                // over [B, H, sq_pad]
    if (row >= (int64_t)a.w.B * a.w.Hk * a.w.g * a.sq_pad) return;
    prep_row<T, D>(a, (int)(row / a.sq_pad), (int)(row % a.sq_pad), row);
}

// Both passes walk tiles of 32 rows, one after the other, and scores of pairs that do not see each other start, and stay, at -inf.  What hides the
// latencies of a tile (scores, exponentials, products, each waiting for the one before) is other workgroups' waves on the same SIMD: four of them at
// 64 channels, two at 128, where a wave's operands and sums alone are 128 and more registers.  (64 channels, [2,8192,24 on 8] window 1024 + 4, forward
// and backward, us: two waves with the next tile's scores taken beside this one's exponentials 732; three 645; four, with the pairs below, 635.)
// (Pairs for dQ as well, 64 rows to a workgroup, three waves to a SIMD at 128 channels: 114 -> 114 us at [2,1248,30,128] +-256, 452 -> 466 here; not kept.)
// Half of a SIMD's issue slots there are vector instructions, a third matrix instructions; slots that are known at compile time save a tenth of the former.

// ---- dQ: owners of rows, key tiles ------------------------------------------------------------------------------
// Two slots of K and V.  The owners' rows lie over the second at the start, and on their way out over the front.
template <int D> struct DqLds {
    static constexpr int TILE = 32 * D * 2, OWN = kWaves * 2 * 64 * D;
    static constexpr int CENTRE = 4 * TILE, GROUPS = kWaves * 64 / D;       // sums of a tile's keys, [group of rows][D] floats
    static constexpr int BYTES = OWN + 2 * TILE;
    static __device__ int keys(int t) { return t & 1 ? 0 : OWN; }
    static __device__ int values(int t) { return keys(t) + TILE; }
    static_assert(CENTRE + GROUPS * D * 4 <= OWN && kWaves * 64 * D <= CENTRE, "the centre lies behind the second slot and behind the rows on their way out");
};

// share, shares: which of the workgroups that the key tiles of these rows are dealt to; with several of them `part` takes the rows in fp32.
template <int T, int D>
__device__ __forceinline__ void dq_body(const WindowBwdArgs& a, uint8_t* smem, int bh, int row0, int share = 0, int shares = 1, float* part = nullptr) {
    using L = DqLds<D>;
    constexpr int NW = kWaves, CPR = D / 8, KS = D / 16, DB = D / 32;
    constexpr bool EARLY = D > 64;
    const WindowArgs& w = a.w;
    const int rows = w.Sq * w.g, H = w.Hk * w.g;
    const int b = bh / w.Hk, kvh = bh % w.Hk;
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int x0 = row0 + wave * 32, x = min(x0 + l32, rows - 1), i = x / w.g, hg = x - i * w.g;
    const int len = sequence_len(w, b), p0 = first_position(w, b, len);
    const int i_lo = row0 / w.g;
    const Span span = key_span<32>(w, p0 + i_lo, p0 + (min(row0 + NW * 32, rows) - 1) / w.g, len);
    const int wp_lo = p0 + min(x0, rows - 1) / w.g, wp_hi = p0 + min(x0 + 31, rows - 1) / w.g;
    const RowMask mask = {p0 + i - w.left, min(p0 + i + w.right, len - 1), w.sinks};

    const uint32_t lds = lds_addr(smem);
    const KeyTiles<D, NW> tiles(span, lds, wave, lane);
    const Range all = tiles.within(wp_hi - w.left, x0 < rows ? min(wp_lo + w.right, len - 1) : -1);
    const int each = (span.n + shares - 1) / shares, t_begin = min(share * each, span.n), t_end = min(t_begin + each, span.n);
    auto k = tiles.rows(w.k + b * w.k_sb + kvh * w.k_sh, w.k_sn, t_begin), v = tiles.rows(w.v + b * w.v_sb + kvh * w.v_sh, w.v_sn, t_begin);
    const Fragments<D> fr(lane);
    v4i b1[KS], b2[KS];
    const uint32_t own = wave * 2 * 64 * D;
    query_rows_in<D>(w, w.q + b * w.q_sb + (int64_t)kvh * w.g * w.q_sh + (int64_t)i_lo * w.q_sn, w.q_sn, w.q_sh, i_lo, x0, lds + own, lane);
    query_rows_in<D>(w, a.dout + b * a.do_sb + (int64_t)kvh * w.g * a.do_sh + (int64_t)i_lo * a.do_sn, a.do_sn, a.do_sh, i_lo, x0, lds + own + 64 * D, lane);
    if (t_end > t_begin) tiles.copy(k, t_begin, L::keys(0)), tiles.copy(v, t_begin, L::values(0));
    const int64_t at = ((int64_t)b * H + kvh * w.g + hg) * a.sq_pad + i;
    float lse = a.lse2[at], ndelta = a.ndelta[at], mul = w.scale * kWeightInv;
    if constexpr (T == kF16) mul = a.dsize[at];
    dma_wait<0>();
#pragma unroll
    for (int s = 0; s < KS; s++) b1[s] = fr.along(smem + own, s), b2[s] = fr.along(smem + own + 64 * D, s);
#pragma unroll
    for (int s = 0; s < KS; s++) asm volatile("" : "+v"(b1[s]), "+v"(b2[s]));
    if constexpr (T == kF16) {           // (a power of the row's own, for the weights' one)
        const int power = ds_power(mul);
        lse += kWeightBits - (float)power;
        mul = w.scale * __builtin_amdgcn_ldexpf(1.0f, -power);
        asm volatile("" : "+v"(mul));
    }
    asm volatile("" : "+v"(lse), "+v"(ndelta));

    v16f acc[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[d][e] = 0.0f;
    const float c = w.scale * kLog2e;
    // Rows of dS sum to zero, but for the roundings of dS and of what Delta is made of; whatever their sum is, dS K multiplies it by the
    // keys' common offset.  So the rounded values are summed, and the sum times a vector c close to the mean key is
    // subtracted at the end: dQ = scale dS (K - c).
    float ds_sum = 0.0f;

    // c: the mean of a tile's keys that some row here sees, of the first or of one from the window's middle, whichever has more of them.  (Of the
    // middle of all tiles, which may hold a single key: dQ's relative error 8% higher, [2,12456,2 on 1,128] window 36 + 77.)
    auto keys_of = [&](int t) {
        const int j0 = span.tile(t) * 32, j1 = min(j0 + 31, span.hi);
        return max(0, min(j1 + 1, span.s_end) - j0) + max(0, j1 + 1 - max(max(j0, span.lo), span.s_end));
    };
    int centre = 0;
    for (int n = 0; n < 2; n++) {
        const int t = span.first + (span.n - span.first - n) / 2;
        if (t >= 0 && t < span.n && keys_of(t) > keys_of(centre)) centre = t;
    }
    auto take_centre = [&](int t, int slot) {
        const int me = wave * 64 + lane_here(), ch = me % D, first = me / D * (32 / L::GROUPS), j0 = span.tile(t) * 32;
        const uint8_t* kt = smem + L::keys(slot);
        float sum = 0.0f;
#pragma unroll 1
        for (int r = first; r < first + 32 / L::GROUPS; r++) {
            const float key = widen<T>(*reinterpret_cast<const uint16_t*>(kt + nat_off<CPR>(r, ch >> 3) + (ch & 7) * 2), 0);
            sum += copied_key<32>(span, j0, j0 + r) == j0 + r ? key : 0.0f;
        }
        reinterpret_cast<float*>(smem + L::CENTRE)[me] = sum / (float)keys_of(t);
    };
    // Several workgroups: a row's dS sum to zero over all of them, so all take the same c; its tile is fetched ahead of the walk.
    if (shares > 1 && t_end > t_begin) {
        __syncthreads();                 // (every wave has its rows)
        auto kc = tiles.rows(w.k + b * w.k_sb + kvh * w.k_sh, w.k_sn, centre);
        tiles.copy(kc, centre, L::keys(1));
        dma_wait<0>();
        __syncthreads();
        take_centre(centre, 1);
    }
    auto tile = [&](int t, int slot) {
        dma_wait<0>();
        __syncthreads();                 // tile t is visible; every wave is done with tile t - 1
        if (t + 1 < t_end) tiles.copy(k, t + 1, L::keys(slot + 1)), tiles.copy(v, t + 1, L::values(slot + 1));
        const uint32_t keys = lds + L::keys(slot), values = lds + L::values(slot);
        const int j0 = span.tile(t) * 32;
        const Seen what = all.has(t) ? Seen::kAll : x0 < rows ? seen<32>(w, wp_lo, wp_hi, len, j0) : Seen::kNone;
        if (what != Seen::kNone) {
            const Fragments<D>& f = fr;
            // (128 channels leave room to request all fragments ahead of the first product, and those of the last product ahead of the exponentials)
            v4i kf[EARLY ? KS : 1], vf[EARLY ? KS : 1];
            auto key = [&](int ks) { return EARLY ? kf[EARLY ? ks : 0] : lds_read(keys + (f.nat ^ (ks << 5))); };
            auto value = [&](int ks) { return EARLY ? vf[EARLY ? ks : 0] : lds_read(values + (f.nat ^ (ks << 5))); };
            if constexpr (EARLY) {
#pragma unroll
                for (int ks = 0; ks < KS; ks++) kf[ks] = lds_read(keys + (f.nat ^ (ks << 5))), vf[ks] = lds_read(values + (f.nat ^ (ks << 5)));
                __builtin_amdgcn_sched_barrier(0);
            }
            v16f s, g;
            if (what == Seen::kAll) {
                s = product<T>(key(0), b1[0], v16f{});
            } else {
                const RowMask rel = mask.from(j0 + (lane_here() >> 5) * 4);
#pragma unroll
                for (int e = 0; e < 16; e++) s[e] = rel.sees((e >> 2) * 8 + (e & 3)) ? 0.0f : -INFINITY;
                s = product<T>(key(0), b1[0], s);
            }
            g = product<T>(value(0), b2[0], v16f{});
#pragma unroll
            for (int ks = 1; ks < KS; ks++) {
                s = product<T>(key(ks), b1[ks], s);
                g = product<T>(value(ks), b2[ks], g);
            }
            v4i rf[EARLY ? 2 * DB : 1];
            auto row = [&](int m) { return lds_read_across(keys + (f.tr[0] ^ (m % DB << 6)) + m / DB * 32 * D, keys + (f.tr[1] ^ (m % DB << 6)) + m / DB * 32 * D); };
            if constexpr (EARLY) {
#pragma unroll
                for (int m = 0; m < 2 * DB; m++) rf[m] = row(m);
                __builtin_amdgcn_sched_barrier(0);
            }
            uint32_t ds[8];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const float y0 = __builtin_amdgcn_exp2f(fmaf(s[e], c, -lse)) * (g[e] + ndelta), y1 = __builtin_amdgcn_exp2f(fmaf(s[e + 1], c, -lse)) * (g[e + 1] + ndelta);
                const uint32_t y = ds[e >> 1] = pack2<T>(y0, y1);
                if constexpr (T == kBF16) ds_sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, y), __builtin_bit_cast(v2bf, 0x3F803F80u), ds_sum, false);
                else ds_sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2fp, y), __builtin_bit_cast(v2fp, 0x3C003C00u), ds_sum, false);
            }
#pragma unroll
            for (int m = 0; m < 2 * DB; m++) {
                const int j2 = m / DB, d = m % DB;
                acc[d] = product<T>(EARLY ? rf[EARLY ? m : 0] : row(m), v4i{(int)ds[j2 * 4], (int)ds[j2 * 4 + 1], (int)ds[j2 * 4 + 2], (int)ds[j2 * 4 + 3]}, acc[d]);
            }
        }
        if (shares == 1 && t == centre) take_centre(t, slot);
    };
    if constexpr (D > 64) {
        for (int t = t_begin; t < t_end; t++) tile(t, (t - t_begin) & 1);
    } else {                             // (slots known ahead: addresses stay in registers, the slots in the reads' offsets)
        for (int t = t_begin; t < t_end; t += 2) {
            tile(t, 0);
            if (t + 1 < t_end) tile(t + 1, 1);
        }
    }
    __syncthreads();
    uint8_t* os = smem + wave * 64 * D;
    const int end_lane = lane_here(), end_half = end_lane >> 5;
    if (t_end > t_begin) {
        const float rs = sum_halves(ds_sum);
        const float* centre = reinterpret_cast<const float*>(smem + L::CENTRE);
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                v4f c4 = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int n = 0; n < L::GROUPS; n++) c4 += *reinterpret_cast<const v4f*>(centre + n * D + d * 32 + q * 8 + end_half * 4);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[d][q * 4 + e] = fmaf(-rs, c4[e], acc[d][q * 4 + e]);
            }
    }
    // Rows that see nothing: zeros, also where they or their upstream gradients are no numbers.
    const bool blind = !mask.sees_any();
    if (__any(blind)) {
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[d][e] = blind ? 0.0f : acc[d][e];
    }
    if (shares > 1) {
        float* p = part + (wave * 32 + (end_lane & 31)) * D + end_half * 4;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) *reinterpret_cast<v4f*>(p + d * 32 + g * 8) = v4f{acc[d][g * 4] * mul, acc[d][g * 4 + 1] * mul, acc[d][g * 4 + 2] * mul, acc[d][g * 4 + 3] * mul};
        return;
    }
#pragma unroll
    for (int d = 0; d < DB; d++) row_put<T, D>(os, acc[d], d, mul, end_lane);
    if (x0 < rows) query_rows_out<D>(w, os, a.dq + b * a.dq_sb + (int64_t)kvh * w.g * a.dq_sh, a.dq_sn, a.dq_sh, x0, end_lane);
}

// ---- dK, dV: owners of keys, (head, query tile) pairs --------------------------------------------------------------
// The tiles of 32 queries that reach `keys` keys from k0 on: indices t0 .. t0 + nt - 1 of every head of the group.
struct QuerySpan { int t0, nt; };
__device__ __forceinline__ QuerySpan query_span(const WindowArgs& w, int k0, int keys, int p0, int len) {
    const int k1 = min(k0 + keys, len) - 1;
    const int64_t lo = (int64_t)k0 - w.right - p0;
    const int64_t hi = k0 < w.sinks ? (int64_t)w.Sq - 1 : (int64_t)k1 + w.left - p0;
    const int i0 = (int)(lo < 0 ? 0 : lo > w.Sq ? w.Sq : lo), i1 = (int)(hi < -1 ? -1 : hi > w.Sq - 1 ? w.Sq - 1 : hi);
    if (k1 < k0 || i1 < i0) return QuerySpan{0, 0};
    return QuerySpan{i0 >> 5, (i1 >> 5) - (i0 >> 5) + 1};
}
// Which of the queries at positions pa .. pb a wave's keys x0 .. x0 + 31 are seen by.
__device__ __forceinline__ Seen seen_by(const WindowArgs& w, int x0, int len, int pa, int pb) {
    const int x1 = x0 + 31;
    if (x0 >= len || x0 > pb + w.right || (x1 < pa - w.left && x0 >= w.sinks)) return Seen::kNone;
    return x1 < len && x1 <= pa + w.right && (x0 >= pb - w.left || x1 < w.sinks) ? Seen::kAll : Seen::kSome;
}
// The tiles of 32 queries, by the first one's position, that all see all of a wave's keys, as far as one comparison can tell: what every tile of a walk would ask, answered once.
__device__ __forceinline__ Range all_seeing(const WindowArgs& w, int x0, int len) {
    const int x1 = x0 + 31, lo = x1 - w.right, hi = x1 < w.sinks ? kWindowFar : x0 + w.left - 31;
    return Range{lo, x1 < len && hi >= lo ? (unsigned)(hi - lo) + 1u : 0u};
}
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
template <int D> __device__ __forceinline__ KeyWork key_work(const WindowBwdArgs& a, int bh, int r, int total_blocks) {
    const int sink_wgs = a.sink_blocks * a.sink_chunks;
    int block, chunk;
    KeyWork k;
    k.part = -1;
    if (r < sink_wgs) {
        block = r / a.sink_chunks, chunk = r % a.sink_chunks;
        k.count = a.sink_tiles;
        if (a.sink_chunks > 1) k.part = (int64_t)bh * (sink_wgs + (a.chunks > 1 ? (total_blocks - a.sink_blocks) * a.chunks : 0)) + r;
    } else {
        r -= sink_wgs;
        block = a.sink_blocks + r / a.chunks, chunk = r % a.chunks;
        k.count = a.chunk_tiles;
        if (a.chunks > 1) {
            const int mine = a.sink_chunks > 1 ? sink_wgs : 0;
            k.part = (int64_t)bh * (mine + (total_blocks - a.sink_blocks) * a.chunks) + mine + r;
        }
    }
    k.k0 = block * kKeysWg;
    k.first = chunk * k.count;
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
// A wave's 32 keys from x0 on of the block at k0 -> LDS.  Keys that no query sees are not read: another row of the block stands in, whose gradient
// is dropped by probabilities of zero.  (`span`: of all queries.  A block that nothing sees reads some row and uses none.)
template <int D>
__device__ __forceinline__ void key_rows_in(const Span& span, const uint16_t* head, int64_t sn, int k0, int x0, uint32_t dst, int lane) {
    constexpr int CPR = D / 8, RPI = 64 / CPR;
    const int base = max(min(k0, span.hi), 0);
    const uint16_t* at = head + (int64_t)base * sn;
#pragma unroll
    for (int n = 0; n < 32 / RPI; n++) {
        const int r = n * RPI + lane / CPR;
        const int j = min(max(copied_key<kKeysWg>(span, k0, x0 + r), base), base + kKeysWg - 1);
        dma16(at, (uint32_t)(max(min(j, span.hi), base) - base) * (uint32_t)(sn * 2) + nat_pos<CPR>(r, lane % CPR) * 16, __builtin_amdgcn_readfirstlane(dst + n * 1024));
    }
}

// Q or dO on its way into LDS: tiles of 32 queries of one head after the other, then the next head's.
template <int D> struct QueryRows {
    using Pieces = TilePieces<D, 32, kWaves>;
    const uint16_t* at;                  // of the tile to be copied next
    int64_t tile, turn;                  // from a tile to the next, from a head's last to the next head's first
    uint32_t sn, off[Pieces::N];
    int qt, nt, t0;
    Seeing rows;                         // (others are not read: one of these stands in, with a statistic that makes its weights vanish)
    Range whole;                         // the tiles, from t0 on, that hold only such
    __device__ QueryRows(const Pieces& p, const uint16_t* head, int64_t sh, int64_t sn_, const QuerySpan& q, const Seeing& rows_, int first, int lane) {
        const int hg = q.nt > 0 ? first / q.nt : 0;
        nt = q.nt;
        t0 = q.t0;
        rows = rows_;
        whole = Range{(rows.lo + 31) / 32 - t0, (unsigned)max((rows.hi + 1) / 32 - (rows.lo + 31) / 32, 0)};
        qt = first - hg * nt;
        at = head + hg * sh + (int64_t)(t0 + qt) * 32 * sn_;
        tile = 32 * sn_;
        turn = sh - (nt - 1) * tile;
        sn = (uint32_t)sn_ * 2u;
#pragma unroll
        for (int n = 0; n < Pieces::N; n++) off[n] = p.row(n) * sn + p.col(n, lane);
    }
    __device__ void copy(const Pieces& p, uint32_t to, int wave, int lane) {
        auto place = [&](int n) { return __builtin_amdgcn_readfirstlane(to + (n * kWaves + wave) * 1024); };
        if (Pieces::N > 1 && whole.has(qt)) {
#pragma unroll
            for (int n = 0; n < Pieces::N; n++) dma16(at, off[n], place(n));
        } else {
#pragma unroll
            for (int n = 0; n < Pieces::N; n++) {
                uint32_t o = off[n];
                if (!whole.has(qt)) {    // (every tile that is copied holds one of them)
                    const int i0 = (t0 + qt) * 32;
                    o = (uint32_t)min(max(p.row(n), rows.lo - i0), rows.hi - i0) * sn + p.col(n, lane);
                }
                dma16(at, o, place(n));
            }
        }
        const bool last = qt == nt - 1;
        at += last ? turn : tile;
        qt = last ? 0 : qt + 1;
    }
};
// The statistics of the same tiles: 32 log-sum-exps and 32 -Delta, side by side.
struct QueryStats {
    const float* at;
    int64_t turn;
    uint32_t off;
    int qt, nt;
    __device__ QueryStats(const WindowBwdArgs& a, int64_t head, const QuerySpan& q, int first, int lane) {
        const int hg = q.nt > 0 ? first / q.nt : 0;
        nt = q.nt;
        qt = first - hg * nt;
        at = a.lse2 + (head + hg) * a.sq_pad + (q.t0 + qt) * 32;
        turn = a.sq_pad - (nt - 1) * 32;
        off = (uint32_t)(lane & 31) * 4u + (lane < 32 ? 0u : (uint32_t)((a.ndelta - a.lse2) * 4));
    }
    __device__ void copy(uint32_t to) {
        dma4(at, off, __builtin_amdgcn_readfirstlane(to));
        const bool last = qt == nt - 1;
        at += last ? turn : 32;
        qt = last ? 0 : qt + 1;
    }
};
// The largest sum of |dO| of the rows of those tiles.
__device__ __forceinline__ float largest_size(const WindowBwdArgs& a, int64_t head, const QuerySpan& q, int first, int n, int lane) {
    float top = 0.0f;
    for (int hg = q.nt > 0 ? first / q.nt : 0, qt = first - hg * q.nt; n > 0; hg++, qt = 0) {
        const int here = min(n, q.nt - qt);
        const v4f* at = reinterpret_cast<const v4f*>(a.dsize + (head + hg) * a.sq_pad + (q.t0 + qt) * 32);
#pragma unroll 4
        for (int e = lane; e < here * 8; e += 64) top = fmaxf(top, fmaxf(fmaxf(at[e][0], at[e][1]), fmaxf(at[e][2], at[e][3])));
        n -= here;
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(top)));
}
// Positions of the tiles' first queries.
struct QueryWalk {
    int p, qt, nt, p_first;
    __device__ QueryWalk(const QuerySpan& q, int first, int p0) {
        nt = q.nt;
        qt = nt > 0 ? first % nt : 0;
        p_first = p0 + q.t0 * 32;
        p = p_first + qt * 32;
    }
    __device__ void next() {
        const bool last = qt == nt - 1;
        p = last ? p_first : p + 32;
        qt = last ? 0 : qt + 1;
    }
};

// Scores of a tile of queries with the lane's key, where they start.
__device__ __forceinline__ void start_scores(v16f& s, const KeyMask& mask, int pa, int half) {
    const KeyMask rel = {mask.lo - pa - half * 4, mask.hi - pa - half * 4};
#pragma unroll
    for (int e = 0; e < 16; e++) s[e] = rel.sees((e >> 2) * 8 + (e & 3)) ? 0.0f : -INFINITY;
}

// A pair of waves shares 32 keys, the P wave with K rows and dV, the S wave, one tile behind, with V rows and dK; P crosses
// over through LDS with some bits more than dS is rounded to: as fp16 pairs, times 2^14, where that is bf16 (11 bits for weights down to 2^-28, fewer
// below, none below 2^-39), as the upper three bytes of fp32
// where it is fp16 (with fp16 there dK's relative error was 3.5e-4, with these 2.9e-4).  Three slots of Q, dO and their statistics: the tile on its way
// in, the P wave's and the S wave's.
template <int T, int D> struct PairLds {
    static constexpr int TILE = 32 * D * 2, WORDS = T == kBF16 ? 2 : 3;      // 16-byte words for the 16 values of a lane
    static constexpr int HAND = 2 * WORDS * 64 * 16;                          // [pair][word][lane]
    static constexpr int ROWS = 768, RING = ROWS + 2 * HAND, BYTES = RING + 6 * TILE;
    static __device__ int q(int slot) { return RING + (slot == 0 ? 4 : slot * 2 - 2) * TILE; }
    static __device__ int d(int slot) { return q(slot) + TILE; }
    static_assert(kWaves * 64 * D == 4 * TILE, "the owners' rows lie over all slots but the first, and over the front on their way out");
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
    using L = PairLds<T, D>;
    constexpr int KS = D / 16, DB = D / 32;
    static_assert(kWaves * 16 == kKeysWg, "a pair of waves owns 32 keys");
    const WindowArgs& w = a.w;
    const int b = bh / w.Hk, kvh = bh % w.Hk;
    const int pr = wave & 1, half = lane >> 5, l32 = lane & 31;
    const int x0 = work.k0 + pr * 32, j = x0 + l32;
    const int len = sequence_len(w, b), p0 = first_position(w, b, len), p_last = p0 + w.Sq - 1;
    const QuerySpan qs = query_span(w, work.k0, kKeysWg, p0, len);
    const int n_tiles = max(0, min(qs.nt * w.g - work.first, work.count));
    const Seeing real = seeing(w, p0, len);
    const KeyMask mask = key_mask(w, j, len, p0);
    const Range all = all_seeing(w, x0, len);
    const uint32_t lds = lds_addr(smem);
    const typename QueryRows<D>::Pieces pieces(wave, lane);
    QueryRows<D> q(pieces, w.q + b * w.q_sb + (int64_t)kvh * w.g * w.q_sh, w.q_sh, w.q_sn, qs, real, work.first, lane);
    QueryRows<D> d(pieces, a.dout + b * a.do_sb + (int64_t)kvh * w.g * a.do_sh, a.do_sh, a.do_sn, qs, real, work.first, lane);
    QueryStats st(a, (int64_t)b * w.Hk * w.g + kvh * w.g, qs, work.first, lane);
    QueryWalk walk(qs, work.first, p0);

    const Fragments<D> fr(lane);
    v4i bx[KS];
    const uint32_t own = L::RING + wave * 64 * D;
    const Span keys_seen = key_span<32>(w, p0, p_last, len);
    key_rows_in<D>(keys_seen, ROLE == 0 ? w.k + b * w.k_sb + kvh * w.k_sh : w.v + b * w.v_sb + kvh * w.v_sh, ROLE == 0 ? w.k_sn : w.v_sn, work.k0, x0, lds + own, lane);
    auto copy = [&](int slot) {
        if (wave == 0) st.copy(lds + slot * 256);
        q.copy(pieces, lds + L::q(slot), wave, lane);
        d.copy(pieces, lds + L::d(slot), wave, lane);
    };
    if (n_tiles > 0) copy(0);
    float ds_mul = 1.0f, out_mul = ROLE == 0 ? kWeightInv : w.scale * kWeightInv;
    if constexpr (T == kF16 && ROLE == 1) {
        const int power = ds_power(largest_size(a, (int64_t)b * w.Hk * w.g + kvh * w.g, qs, work.first, n_tiles, lane));
        ds_mul = __builtin_amdgcn_ldexpf(kWeightInv, power);
        out_mul = w.scale * __builtin_amdgcn_ldexpf(1.0f, -power);
    }
    dma_wait<0>();
#pragma unroll
    for (int s = 0; s < KS; s++) bx[s] = fr.along(smem + own, s);
#pragma unroll
    for (int s = 0; s < KS; s++) asm volatile("" : "+v"(bx[s]));

    v16f acc[DB];
#pragma unroll
    for (int n = 0; n < DB; n++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[n][e] = 0.0f;
    const float c = w.scale * kLog2e;
    u32x4* hand = reinterpret_cast<u32x4*>(smem + L::ROWS) + pr * L::WORDS * 64 + lane;

    // One tile of this wave's: scores (P wave: Q K^T, S wave: dO V^T - Delta), then the product with the rows (dO, Q) of the same tile.
    auto step = [&](Seen what, int pa, int slot, int parity) {
        const Fragments<D>& f = fr;
        const uint32_t score = lds + (ROLE == 0 ? L::q(slot) : L::d(slot)), rows = lds + (ROLE == 0 ? L::d(slot) : L::q(slot));
        const uint8_t* stats = smem + slot * 256 + ROLE * 128 + half * 16;
        // (128 channels leave room to request all fragments ahead of the first product: two waves to a SIMD do not cover the reads' latencies.  [2652 rows in 3, 30 x 128] a step
        // 279 -> 260 us with what dq_body does likewise; at 64 channels, where that takes a wave of four, no gain)
        constexpr bool EARLY = D > 64;
        v4i sf[EARLY ? KS : 1], rf[EARLY ? 2 * DB : 1];
        auto scores = [&](int ks) { return EARLY ? sf[EARLY ? ks : 0] : lds_read(score + (f.nat ^ (ks << 5))); };
        auto row = [&](int m) {
            const uint32_t lo = (f.tr[0] ^ (m % DB << 6)) + m / DB * 32 * D, hi = (f.tr[1] ^ (m % DB << 6)) + m / DB * 32 * D;
            return lds_read_across(rows + lo, rows + hi);
        };
        if constexpr (EARLY) {
#pragma unroll
            for (int ks = 0; ks < KS; ks++) sf[ks] = lds_read(score + (f.nat ^ (ks << 5)));
#pragma unroll
            for (int m = 0; m < 2 * DB; m++) rf[m] = row(m);
            __builtin_amdgcn_sched_barrier(0);
        }
        v16f s;
        if constexpr (ROLE == 0) {
            if (what != Seen::kAll) start_scores(s, mask, pa, half);
            s = what == Seen::kAll ? product<T>(scores(0), bx[0], v16f{}) : product<T>(scores(0), bx[0], s);
        } else {
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const v4f nd = *reinterpret_cast<const v4f*>(stats + n * 32);
#pragma unroll
                for (int e = 0; e < 4; e++) s[n * 4 + e] = nd[e];
            }
            s = product<T>(scores(0), bx[0], s);
        }
#pragma unroll
        for (int ks = 1; ks < KS; ks++) s = product<T>(scores(ks), bx[ks], s);
        uint32_t pk[8], hp[4 * L::WORDS];
        u32x4* mine = hand + parity * (L::HAND / 16);
        if constexpr (ROLE == 0) {
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const v4f lse = *reinterpret_cast<const v4f*>(stats + n * 32);
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = __builtin_amdgcn_exp2f(fmaf(s[n * 4 + e], c, -lse[e]));
                pk[n * 2] = pack2<T>(y[0], y[1]);
                pk[n * 2 + 1] = pack2<T>(y[2], y[3]);
                if constexpr (T == kBF16) {
                    hp[n * 2] = pack2<kF16>(y[0], y[1]);
                    hp[n * 2 + 1] = pack2<kF16>(y[2], y[3]);
                } else {
                    pack24(y, &hp[n * 3]);
                }
            }
#pragma unroll
            for (int n = 0; n < L::WORDS; n++) mine[n * 64] = u32x4{hp[n * 4], hp[n * 4 + 1], hp[n * 4 + 2], hp[n * 4 + 3]};
        } else {
#pragma unroll
            for (int n = 0; n < L::WORDS; n++) {
                const u32x4 v = mine[n * 64];
#pragma unroll
                for (int e = 0; e < 4; e++) hp[n * 4 + e] = v[e];
            }
#pragma unroll
            for (int n = 0; n < 16; n += 2) {
                float y[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    // (as a multiply-add: one instruction with the fp16 operand's conversion in it)
                    if constexpr (T == kBF16) y[e] = fmaf((float)__builtin_bit_cast(v2fp, hp[n >> 1])[e], s[n + e], 0.0f);
                    else y[e] = unpack24(&hp[(n >> 2) * 3], (n & 3) + e) * s[n + e] * ds_mul;
                }
                pk[n >> 1] = pack2<T>(y[0], y[1]);
            }
        }
#pragma unroll
        for (int m = 0; m < 2 * DB; m++) {
            const int j2 = m / DB, d = m % DB;
            acc[d] = product<T>(EARLY ? rf[EARLY ? m : 0] : row(m), v4i{(int)pk[j2 * 4], (int)pk[j2 * 4 + 1], (int)pk[j2 * 4 + 2], (int)pk[j2 * 4 + 3]}, acc[d]);
        }
    };
    auto tile = [&](int t, int slot) {   // slot: t % 3
        dma_wait<0>();
        __syncthreads();                 // tile t and P of t - 1 are visible; every wave is done with tile t - 2
        if (t + 1 < n_tiles) copy(slot == 2 ? 0 : slot + 1);
        if (ROLE == 0 ? t >= n_tiles : t == 0) return;
        const int pa = walk.p;
        const Seen what = all.has(pa) ? Seen::kAll : seen_by(w, x0, len, pa, min(pa + 31, p_last));
        walk.next();
        if (what != Seen::kNone) step(what, pa, ROLE == 0 ? slot : slot == 0 ? 2 : slot - 1, (t - ROLE) & 1);
    };
    if (n_tiles > 0) {
        if constexpr (D > 64) {
            for (int t = 0, slot = 0; t <= n_tiles; t++, slot = slot == 2 ? 0 : slot + 1) tile(t, slot);
        } else {                         // (slots known ahead, as above)
            for (int t = 0; t <= n_tiles; t += 3) {
                tile(t, 0);
                if (t + 1 <= n_tiles) tile(t + 1, 1);
                if (t + 2 <= n_tiles) tile(t + 2, 2);
            }
        }
    }
    __syncthreads();                     // (every copy has landed, every tile has been read: the ring takes the output rows)
    uint8_t* os = smem + L::RING + wave * 64 * D;
    if constexpr (ROLE == 0) key_rows_out<T, D>(a, acc, out_mul, os, work.part, 1, a.dv + b * a.dv_sb + kvh * a.dv_sh, a.dv_sn, x0, work.k0, lane);
    else key_rows_out<T, D>(a, acc, out_mul, os, work.part, 0, a.dk + b * a.dk_sb + kvh * a.dk_sh, a.dk_sn, x0, work.k0, lane);
}

template <int T, int D>
__global__ __launch_bounds__(kWaves * 64, D > 64 ? 2 : 4) void window_bwd_kernel(WindowBwdArgs a) {
    constexpr int KV = PairLds<T, D>::BYTES;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[KV > DqLds<D>::BYTES ? KV : DqLds<D>::BYTES];
    const int heads = a.w.B * a.w.Hk, rows = a.w.Sq * a.w.g;
    const int tq = (rows + kRowsWg - 1) / kRowsWg, blocks = (a.w.Skv + kKeysWg - 1) / kKeysWg;
    const int id = (int)blockIdx.x, nq = heads * tq;
    if (id < nq) {
        const int item = xcd_item(id, nq);
        dq_body<T, D>(a, smem, item / tq, (tq - 1 - item % tq) * kRowsWg);
        return;
    }
    const int tk = a.sink_blocks * a.sink_chunks + (blocks - a.sink_blocks) * a.chunks, item = xcd_item(id - nq, heads * tk);
    const KeyWork work = key_work<D>(a, item / tk, item % tk, blocks);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (wave < 2) dkdv_role<T, D, 0>(a, smem, item / tk, work, wave, lane);
    else dkdv_role<T, D, 1>(a, smem, item / tk, work, wave, lane);
}

// Launch 3: dK and dV of the blocks that several workgroups share, their parts added in order.  8 channels to a thread, which
// requests eight parts at a time (one after the other, each is a trip to memory).
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
    for (int c0 = 0; c0 < chunks; c0 += 8) {
        v4f u[8], v[8];
#pragma unroll
        for (int n = 0; n < 8; n++) {
            const float* at_c = p + (int64_t)min(c0 + n, chunks - 1) * 2 * kKeysWg * D;
            u[n] = *reinterpret_cast<const v4f*>(at_c);
            v[n] = *reinterpret_cast<const v4f*>(at_c + 4);
        }
#pragma unroll
        for (int n = 0; n < 8; n++) {
            if (c0 + n >= chunks) break;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] += u[n][e], y[4 + e] += v[n][e];
        }
    }
    const int j = block * kKeysWg + key, b = bh / a.w.Hk, kvh = bh % a.w.Hk;
    if (j >= a.w.Skv) return;
    uint16_t* out = which ? a.dv + b * a.dv_sb + kvh * a.dv_sh + j * a.dv_sn : a.dk + b * a.dk_sb + kvh * a.dk_sh + j * a.dk_sn;
    *reinterpret_cast<u32x4*>(out + col) = u32x4{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7])};
}

// ---- sequences one behind the other ----------------------------------------------------------------------
__device__ __forceinline__ WindowBwdArgs view(const PackedBwdArgs& all, const Sequence& s, int nq, int nk, int b) {
    WindowBwdArgs a = all.w;
    a.w = view(all.w.w, s, nq, nk);
    a.dout += s.q0 * a.do_sn;
    a.dq += s.q0 * a.dq_sn;
    a.dk += s.k0 * a.dk_sn;
    a.dv += s.k0 * a.dv_sn;
    const int row = (s.q0 / 32 + b) * 32;
    a.lse2 += row;
    a.ndelta += row;
    a.dsize += row;
    return a;
}
// (A workgroup's rows are of one tile of 32, so that head and sequence are found once for all of them.)
template <int T, int D> __global__ __launch_bounds__(256) void packed_bwd_prep_kernel(PackedBwdArgs a) {
    constexpr int CPR = D / 8, RPP = 256 / CPR;
    static_assert(32 % RPP == 0, "part of a tile");
    const uint32_t row0 = blockIdx.x * (uint32_t)RPP, tiles_head = (uint32_t)a.w.sq_pad / 32u, tile = row0 / 32u;
    const int h = (int)(tile / tiles_head), t = (int)(tile - (uint32_t)h * tiles_head);          // over [H, sq_pad]
    const Slots tiles = {a.p.cu_q, a.p.rows_q, 1, 32};
    const int b = tiles.owner(t, a.p.B), i = (t - tiles.first(b)) * 32 + (int)(row0 % 32u) + (int)threadIdx.x / CPR;
    const Sequence s = sequence(a.p, b);
    prep_row<T, D>(view(a, s, s.nq, b < a.p.B ? s.nk : 0, b), h, i, (int64_t)h * a.w.sq_pad + i);
}
// SPLIT: the rows' key tiles are dealt to several workgroups.
template <int T, int D, bool SPLIT>
__global__ __launch_bounds__(kWaves * 64, D > 64 ? 2 : 4) void packed_bwd_kernel(PackedBwdArgs a, int q_slots, int k_slots) {
    constexpr int KV = PairLds<T, D>::BYTES;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[KV > DqLds<D>::BYTES ? KV : DqLds<D>::BYTES];
    const int shares = SPLIT ? a.q_chunks : 1, nq = (int)spread_grid(a.w.w.Hk, q_slots * shares), id = (int)blockIdx.x;
    if (id < nq) {
        const HeadSlot at = spread_item(id, a.w.w.Hk, q_slots * shares);
        if (at.slot >= q_slots * shares) return;
        const int slot = SPLIT ? at.slot / shares : at.slot;
        const Found f = find_slot<false>(a.p, a.w.w.g, kRowsWg, slot);
        if (f.index >= f.n) return;
        const Sequence& s = f.s;
        const WindowBwdArgs v = view(a, s, s.nq, f.b < a.p.B ? s.nk : 0, f.b);
        const int row0 = (f.n - 1 - f.index) * kRowsWg;                // (the last rows first: they see most keys)
        if constexpr (SPLIT) dq_body<T, D>(v, smem, at.head, row0, at.slot - slot * shares, shares, a.q_part + ((int64_t)at.head * q_slots * shares + at.slot) * kRowsWg * D);
        else dq_body<T, D>(v, smem, at.head, row0);
        return;
    }
    const HeadSlot at = spread_item(id - nq, a.w.w.Hk, k_slots * a.chunks);
    if (at.slot >= k_slots * a.chunks) return;
    const int slot = at.slot / a.chunks, chunk = at.slot - slot * a.chunks;
    const Found f = find_slot<true>(a.p, 1, kKeysWg, slot);
    if (f.index >= f.n) return;
    const Sequence& s = f.s;
    const int k0 = f.index * kKeysWg;                    // (the first keys first: most queries see them)
    const WindowBwdArgs v = view(a, s, f.b < a.p.B ? s.nq : 0, s.nk, f.b);
    const QuerySpan qs = query_span(v.w, k0, kKeysWg, v.w.start, s.nk);
    KeyWork work;
    work.k0 = k0;
    work.count = (qs.nt * v.w.g + a.chunks - 1) / a.chunks;
    work.first = chunk * work.count;
    work.part = a.chunks > 1 ? ((int64_t)at.head * k_slots + slot) * a.chunks + chunk : -1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (wave < 2) dkdv_role<T, D, 0>(v, smem, at.head, work, wave, lane);
    else dkdv_role<T, D, 1>(v, smem, at.head, work, wave, lane);
}
// Eight channels of parts that lie `pitch` apart, added up in order, as above.
template <int T> __device__ __forceinline__ void join_parts(const float* p, int n, int64_t pitch, uint16_t* out) {
    float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int c0 = 0; c0 < n; c0 += 8) {
        v4f u[8], v[8];
#pragma unroll
        for (int m = 0; m < 8; m++) {
            const float* at_c = p + min(c0 + m, n - 1) * pitch;
            u[m] = *reinterpret_cast<const v4f*>(at_c);
            v[m] = *reinterpret_cast<const v4f*>(at_c + 4);
        }
#pragma unroll
        for (int m = 0; m < 8; m++) {
            if (c0 + m >= n) break;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] += u[m][e], y[4 + e] += v[m][e];
        }
    }
    *reinterpret_cast<u32x4*>(out) = u32x4{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7])};
}
// (A workgroup's threads are of one slot: 256 divides a slot's pieces.)
template <int T, int D> __global__ __launch_bounds__(256) void packed_bwd_join_kernel(PackedBwdArgs a, int q_slots, int k_slots) {
    constexpr int CPR = D / 8;
    const int Hk = a.w.w.Hk, g = a.w.w.g;
    const int64_t k_pieces = a.chunks > 1 ? (int64_t)Hk * k_slots * 2 * kKeysWg * CPR : 0;
    int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at < k_pieces) {
        const int col = (int)(at % CPR) * 8, key = (int)(at / CPR % kKeysWg), which = (int)(at / (CPR * kKeysWg) & 1);
        const int item = (int)(at / (2 * CPR * kKeysWg)), kvh = item / k_slots, slot = item - kvh * k_slots;
        const Found f = find_slot<true>(a.p, 1, kKeysWg, slot);
        const int j = f.index * kKeysWg + key;
        if (j >= f.s.nk) return;
        const int64_t row = f.s.k0 + j;
        join_parts<T>(a.w.part + (((int64_t)item * a.chunks * 2 + which) * kKeysWg + key) * D + col, a.chunks, 2 * kKeysWg * D,
                      (which ? a.w.dv + kvh * a.w.dv_sh + row * a.w.dv_sn : a.w.dk + kvh * a.w.dk_sh + row * a.w.dk_sn) + col);
        return;
    }
    at -= k_pieces;
    if (a.q_chunks == 1 || at >= (int64_t)Hk * q_slots * kRowsWg * CPR) return;
    const int col = (int)(at % CPR) * 8, r = (int)(at / CPR % kRowsWg), item = (int)(at / (CPR * kRowsWg)), kvh = item / q_slots, slot = item - kvh * q_slots;
    const Found f = find_slot<false>(a.p, g, kRowsWg, slot);
    const int x = (f.n - 1 - f.index) * kRowsWg + r;
    if (f.index >= f.n || x >= f.s.nq * g) return;
    const int i = x / g;
    join_parts<T>(a.q_part + ((int64_t)item * a.q_chunks * kRowsWg + r) * D + col, a.q_chunks, kRowsWg * D,
                  a.w.dq + (f.s.q0 + i) * a.w.dq_sn + (kvh * g + x - i * g) * a.w.dq_sh + col);
}
struct PackedGrid { int64_t q_slots, k_slots, prep, grid, join; };
PackedGrid packed_grid(const PackedBwdArgs& a) {
    const int64_t Hk = a.w.w.Hk, D = a.w.w.D;
    PackedGrid g;
    g.q_slots = slots_total(a.p.rows_q, a.w.w.g, kRowsWg, a.p.B);
    g.k_slots = slots_total(a.p.rows_k, 1, kKeysWg, a.p.B);
    g.prep = Hk * a.w.w.g * packed_stats_rows(a.p) * (D / 8) / 256;
    g.grid = spread_grid(Hk, g.q_slots * a.q_chunks) + spread_grid(Hk, g.k_slots * a.chunks);
    g.join = ((a.chunks > 1 ? Hk * g.k_slots * 2 * kKeysWg : 0) + (a.q_chunks > 1 ? Hk * g.q_slots * kRowsWg : 0)) * (D / 8) / 256;
    return g;
}
template <int T, int D> hipError_t launch_packed_td(const PackedBwdArgs& a, hipStream_t st) {
    const PackedGrid g = packed_grid(a);
    hipLaunchKernelGGL((packed_bwd_prep_kernel<T, D>), dim3((unsigned)g.prep), dim3(256), 0, st, a);
    if (a.q_chunks > 1) hipLaunchKernelGGL((packed_bwd_kernel<T, D, true>), dim3((unsigned)g.grid), dim3(kWaves * 64), 0, st, a, (int)g.q_slots, (int)g.k_slots);
    else hipLaunchKernelGGL((packed_bwd_kernel<T, D, false>), dim3((unsigned)g.grid), dim3(kWaves * 64), 0, st, a, (int)g.q_slots, (int)g.k_slots);
    if (g.join > 0) hipLaunchKernelGGL((packed_bwd_join_kernel<T, D>), dim3((unsigned)g.join), dim3(256), 0, st, a, (int)g.q_slots, (int)g.k_slots);
    return hipGetLastError();
}

template <int T, int D> hipError_t launch_td(const WindowBwdArgs& a, hipStream_t st) {
    const int64_t heads = (int64_t)a.w.B * a.w.Hk, rows = (int64_t)a.w.Sq * a.w.g, blocks = (a.w.Skv + kKeysWg - 1) / kKeysWg;
    const int64_t prep = (heads * a.w.g * a.sq_pad * (D / 8) + 255) / 256;
    const int64_t grid = heads * ((rows + kRowsWg - 1) / kRowsWg + (int64_t)a.sink_blocks * a.sink_chunks + (blocks - a.sink_blocks) * a.chunks);
    const int64_t shared = (a.sink_chunks > 1 ? a.sink_blocks : 0) + (a.chunks > 1 ? blocks - a.sink_blocks : 0);
    const int64_t join = (heads * shared * 2 * kKeysWg * (D / 8) + 255) / 256;
    if (prep > 0x7FFFFFFF || grid > 0x7FFFFFFF || join > 0x7FFFFFFF) return hipErrorInvalidValue;
    hipLaunchKernelGGL((window_bwd_prep_kernel<T, D>), dim3((unsigned)prep), dim3(256), 0, st, a);
    hipLaunchKernelGGL((window_bwd_kernel<T, D>), dim3((unsigned)grid), dim3(kWaves * 64), 0, st, a);
    if (join > 0) hipLaunchKernelGGL((window_bwd_join_kernel<T, D>), dim3((unsigned)join), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

// A key block's pairs without sinks: as many as its window spans.  They are dealt to several workgroups where whole blocks would leave the chip
// partly empty (four to a compute unit are wanted), down to 16 pairs.  A block with sinks is reached by every later query: its pairs go to as many workgroups as
// give each a window block's share, but to no more than two to a compute unit over all heads and blocks (the parts, 64 KiB each at 128 channels, stay within 32 MiB),
// and no more than twice the root of the pairs, since the join's time grows with the parts as the walks shrink.  (Gradients, us, with a window block's share whatever
// the length, one to a unit, two: [1,16896,8,128] window 16 + 4 187, 140, 140; [1,16896,30,128] 16 + 77 762, 617, 557; [1,65536,4 on 2,128] 63 + 4
// 381, 291, 287; [1,16896,2,128] 256 + 256 87, 100, 89.)
void window_bwd_plan(WindowBwdArgs* a) {
    constexpr int64_t kUnits = 256;
    const WindowArgs& w = a->w;
    const int64_t keys = kWindowBwdKeys;
    const int64_t all = (w.Sq + 31) / 32, blocks = (w.Skv + keys - 1) / keys, heads = (int64_t)w.B * w.Hk;
    const int64_t tiles = std::min<int64_t>(all, ((int64_t)w.left + w.right + keys + 30) / 32 + 1), pairs = tiles * w.g;
    const int64_t want = std::max<int64_t>(1, 4 * kUnits / (blocks * heads)), most = std::max<int64_t>(1, pairs / 16);
    const int64_t chunks = std::min(want, most), per = (pairs + chunks - 1) / chunks;
    a->chunks = (int)((pairs + per - 1) / per);
    a->chunk_tiles = (int)per;
    a->sink_blocks = tiles < all ? (int)((w.sinks + keys - 1) / keys) : 0;
    const int64_t sink_pairs = all * w.g, room = std::max<int64_t>(1, 2 * kUnits / std::max<int64_t>(1, a->sink_blocks * heads));
    int64_t n = std::min((sink_pairs + per - 1) / per, room);
    while (n * n > 4 * sink_pairs) n--;
    const int64_t sink_per = (sink_pairs + n - 1) / n;
    a->sink_tiles = (int)sink_per;
    a->sink_chunks = (int)((sink_pairs + sink_per - 1) / sink_per);
}
int64_t window_bwd_parts(const WindowBwdArgs& a) {
    const int64_t keys = kWindowBwdKeys, blocks = (a.w.Skv + keys - 1) / keys;
    return (int64_t)a.w.B * a.w.Hk * ((a.sink_chunks > 1 ? (int64_t)a.sink_blocks * a.sink_chunks : 0) + (a.chunks > 1 ? (blocks - a.sink_blocks) * a.chunks : 0));
}

hipError_t launch_window_bwd(const WindowBwdArgs& a, hipStream_t st) {
    if (a.w.D == 64) return a.w.type == kBF16 ? launch_td<kBF16, 64>(a, st) : launch_td<kF16, 64>(a, st);
    return a.w.type == kBF16 ? launch_td<kBF16, 128>(a, st) : launch_td<kF16, 128>(a, st);
}

int packed_stats_rows(const PackedArgs& a) { return (int)slots_total(a.rows_q, 1, 32, a.B) * 32; }
// Few key blocks: their pairs dealt to several workgroups until there are four to a compute unit, down to 8 pairs of the average and to no more than the root of
// the pairs, since the join's time grows with the parts.  (A step of [5 x 75 rows, 16 on 2 x 64] down to 16 pairs 40 us, 8: 31; of [1000 rows, 8 on 1 x 64] with
// 16 workgroups to a block 53, with 32 60.)
void packed_bwd_plan(PackedBwdArgs* a) {
    const int64_t blocks = (a->p.rows_k + kWindowBwdKeys - 1) / kWindowBwdKeys, heads = a->w.w.Hk;
    const int64_t pairs = (a->p.rows_q / std::max(a->p.B, 1) + 31) / 32 * a->w.w.g;
    int64_t n = std::max<int64_t>(1, std::min(1024 / (blocks * heads), pairs / 8));
    while (n > 1 && n * n > pairs) n--;
    a->chunks = (int)n;
    // Rows whose walk over the keys would take longer than the chip's average (four or two workgroups to a compute unit): their key tiles dealt out likewise, to no more
    // than half the places, since two rounds gain nothing ([1292 rows, 30 x 64] in two parts 88 -> 103 us), and to eight workgroups at the most.  A step with up to 1 / 4 / 8 / 16 of them, us:
    // [8000 rows, 1 x 64] 242 / 122 / 114 / 114, [4000, 1 x 64] 131 / 72 / 64 / 65, full [4096, 2 x 64] 136 / 92 / 95 / 94, [4000, 4 on 1 x 128] 192 / 149 / 149 / 149, [2048, 8 x 128] 120 / 105 / 105 / 105.
    // (All of it by averages over B, which counts empty sequences: [8000 rows, 1 x 64] with 63 of them behind it is dealt to one workgroup, 239 us.)
    const int64_t tiles = (a->p.rows_k / std::max(a->p.B, 1) + 31) / 32, row_blocks = (a->p.rows_q * a->w.w.g + kRowsWg - 1) / kRowsWg * heads, places = a->w.w.D == 64 ? 1024 : 512;
    const int64_t load = (row_blocks * tiles + blocks * heads * pairs) / (a->w.w.right < kWindowFar ? 2 : 1) / places;
    a->q_chunks = (int)std::max<int64_t>(1, std::min({tiles / std::max<int64_t>(load, 8), tiles / 8, places / 2 / row_blocks, (int64_t)8}));
}
int64_t packed_bwd_q_part_rows(const PackedBwdArgs& a) { return a.q_chunks > 1 ? a.w.w.Hk * slots_total(a.p.rows_q, a.w.w.g, kRowsWg, a.p.B) * a.q_chunks * kRowsWg : 0; }
int64_t packed_bwd_parts(const PackedBwdArgs& a) { return a.chunks > 1 ? (int64_t)a.w.w.Hk * slots_total(a.p.rows_k, 1, kWindowBwdKeys, a.p.B) * a.chunks : 0; }
bool packed_bwd_grid_ok(const PackedBwdArgs& a) {
    const PackedGrid g = packed_grid(a);
    return g.prep <= 0x7FFFFFFF && g.grid <= 0x7FFFFFFF && g.join <= 0x7FFFFFFF;
}
hipError_t launch_packed_bwd(const PackedBwdArgs& a, hipStream_t st) {
    if (a.w.w.D == 64) return a.w.w.type == kBF16 ? launch_packed_td<kBF16, 64>(a, st) : launch_packed_td<kF16, 64>(a, st);
    return a.w.w.type == kBF16 ? launch_packed_td<kBF16, 128>(a, st) : launch_packed_td<kF16, 128>(a, st);
}

}  // namespace sage
