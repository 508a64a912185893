// sage_window_common.h — what the forward and the backward kernels of windowed attention share: operands, positions, the key tiles that a
// block of rows sees.
#pragma once

#include "sage_tile.h"
#include "sage_window.h"

namespace sage {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2hf __attribute__((ext_vector_type(2)));

template <int T> __device__ __forceinline__ v16f product(v4i a, v4i b, v16f c) {
    if constexpr (T == kBF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
template <int T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (T == kBF16) return pack_bf16(a, b);
    const v2f f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2hf));
}
// fragments by their LDS address
__device__ __forceinline__ v4i lds_read(uint32_t at) { return *(const __attribute__((address_space(3))) v4i*)(uintptr_t)at; }
__device__ __forceinline__ v4i lds_read_across(uint32_t lo, uint32_t hi) {
    using lds_v4s = __attribute__((address_space(3))) v4s;
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(uintptr_t)lo));
    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(uintptr_t)hi));
    return v4i{(int)a.x, (int)a.y, (int)b.x, (int)b.y};
}
// the other half-wave's value of the same column
__device__ __forceinline__ float max_halves(float x) {
    const v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float sum_halves(float x) {
    const v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r.x) + __uint_as_float(r.y);
}

__device__ __forceinline__ int sequence_len(const WindowArgs& a, int b) { return a.lens ? max(0, min(a.lens[b], a.Skv)) : a.Skv; }
__device__ __forceinline__ int first_position(const WindowArgs& a, int b, int len) {
    if (a.at_end) return len - a.Sq;
    return a.starts ? max(-kWindowStart, min(a.starts[b], kWindowStart)) : a.start;
}

// The queries of a sequence that see a key: lo <= i <= hi.
struct Seeing {
    int lo, hi;
    __device__ bool has(int i) const { return i >= lo && i <= hi; }
};
__device__ __forceinline__ Seeing seeing(const WindowArgs& a, int p0, int len) {
    return Seeing{max(0, -a.right - p0), len == 0 ? -1 : a.sinks > 0 ? a.Sq - 1 : min(a.Sq - 1, len - 1 + a.left - p0)};
}

// The key tiles (KT keys each) that rows at positions p_lo .. p_hi see: `first` tiles with the sinks, then those from `next` on, n in all.
// Keys [0, s_end) and [lo, hi] are the ones that some row sees.
struct Span {
    int lo, hi, s_end, first, next, n;
    __device__ int tile(int t) const { return t < first ? t : next + t - first; }
};
template <int KT> __device__ __forceinline__ Span key_span(const WindowArgs& a, int p_lo, int p_hi, int len) {
    Span s;
    s.hi = min(p_hi + a.right, len - 1);
    s.lo = max(p_lo - a.left, 0);
    s.s_end = max(min(a.sinks, s.hi + 1), 0);
    s.first = (s.s_end + KT - 1) / KT;
    s.next = max(s.lo / KT, s.first);
    s.n = s.first + (s.hi >= s.lo ? max(s.hi / KT + 1 - s.next, 0) : 0);
    return s;
}
// The key whose row is copied for row j of the tile that starts at j0: j itself where some row of the workgroup sees it, else a neighbour that one sees.
template <int KT> __device__ __forceinline__ int copied_key(const Span& s, int j0, int j) {
    const int gap = s.lo <= min(j0 + KT - 1, s.hi) ? s.lo : s.s_end - 1;
    j = min(j, s.hi);                    // (first: a window that begins behind the last key leaves that key in the gap)
    return j >= s.s_end && j < s.lo ? gap : j;
}

// The keys a row sees: lo .. hi, and those below `sinks` up to hi.  (Relative to a key, so that a tile's comparisons are with constants.)
struct RowMask {
    int lo, hi, sinks;
    __device__ RowMask from(int j) const { return RowMask{lo - j, hi - j, sinks - j}; }
    __device__ bool sees(int j) const { return j <= hi && (j >= lo || j < sinks); }
    __device__ bool sees_any() const { return hi >= 0 && (hi >= lo || sinks > 0); }
};

// The lane's number, formed where it is used: not kept in a register through a loop for what follows it.
__device__ __forceinline__ int lane_here() {
    uint32_t all = 0xFFFFFFFFu;
    asm volatile("" : "+s"(all));
    return (int)__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0u));
}

// A wave's view of a tile: nothing of it, all of it, or some.
enum class Seen { kNone, kAll, kSome };
template <int KT> __device__ __forceinline__ Seen seen(const WindowArgs& a, int p_lo, int p_hi, int len, int j0) {
    const int j1 = j0 + KT - 1;
    if (j0 > min(p_hi + a.right, len - 1) || (j1 < p_lo - a.left && j0 >= a.sinks)) return Seen::kNone;
    return j1 <= min(p_lo + a.right, len - 1) && (j0 >= p_hi - a.left || j1 < a.sinks) ? Seen::kAll : Seen::kSome;
}

// Where a lane's fragments lie in a tile: along the channels by k-step s, across them by 32-channel block d (rows 0-7 and 8-15; 16-row
// blocks are + 32 * D bytes).  The layout XORs chunk numbers, so the offsets of all steps follow from one by an XOR with
// a constant, which the address's addition takes along; kept apart they are 16 registers.  (From 128 channels on: 256 bytes further.)
template <int D> struct Fragments {
    int nat, tr[2];
    __device__ explicit Fragments(int lane) {
        constexpr int CPR = D / 8;
        nat = nat_off<CPR>(lane & 31, lane >> 5);
        tr[0] = tr_frag_off<CPR>(lane, 0, 0);
        tr[1] = tr_frag_off<CPR>(lane, 8, 0);
    }
    // a copy whose offsets are formed where they are used, not ahead of a loop
    __device__ Fragments fresh() const {
        Fragments f = *this;
        asm volatile("" : "+v"(f.nat), "+v"(f.tr[0]), "+v"(f.tr[1]));
        return f;
    }
    __device__ v4i along(const uint8_t* tile, int s) const { return *reinterpret_cast<const v4i*>(tile + (nat ^ ((s & 7) << 5)) + (s >> 3) * 256); }
};

// The pieces of a [KT][D] tile that a lane of NW waves copies: piece n is 16 bytes of row(n).  Rows a multiple of 16 apart are laid out alike,
// so where the waves' passes are that far apart one column serves them all.
template <int D, int KT, int NW> struct TilePieces {
    static constexpr int CPR = D / 8, N = KT * D * 2 / 1024 / NW, PASS = NW * 64 / CPR;
    static_assert(KT * D * 2 / 1024 % NW == 0, "tile copies must divide over the waves");
    int row0, col0;
    __device__ TilePieces(int wave, int lane) {
        row0 = (wave * 64 + lane) / CPR;
        col0 = nat_pos<CPR>(row0, lane % CPR) * 16;
    }
    __device__ int row(int n) const { return row0 + n * PASS; }
    __device__ uint32_t col(int n, int lane) const { return (uint32_t)(PASS % 16 == 0 ? col0 : nat_pos<CPR>(row(n), lane % CPR) * 16); }
};

// Tiles of 32 keys of one head on their way into LDS: K and V each walk the tiles of a span, copied by NW waves.
struct Range {
    int first;
    unsigned n;
    __device__ bool has(int t) const { return (unsigned)(t - first) < n; }
};
template <int D, int NW> struct KeyTiles {
    static constexpr int KT = 32;
    using Pieces = TilePieces<D, KT, NW>;
    Span span;
    Pieces pieces;
    uint32_t lds;
    int wave, lane;
    Range whole;                         // which tiles of the window are copied as they are
    __device__ KeyTiles(const Span& s, uint32_t lds_, int wave_, int lane_) : span(s), pieces(wave_, lane_), lds(lds_), wave(wave_), lane(lane_) { whole = within(s.lo, s.hi); }
    // The tiles of the window whose keys all lie in lo .. hi: what every tile of a walk would ask, answered once.
    __device__ Range within(int lo, int hi) const {
        const int t0 = max((max(lo, 0) + KT - 1) / KT, span.next), t1 = hi + 1 < KT ? span.next : (hi + 1) / KT;
        return Range{t0 - span.next + span.first, (unsigned)max(t1 - t0, 0)};
    }
    struct Rows {                        // K or V: the tile to be copied next, and the lane's pieces where it is copied whole
        const uint16_t* at;
        int64_t tile;
        uint32_t sn, off[Pieces::N];
    };
    __device__ Rows rows(const uint16_t* head, int64_t sn, int t = 0) const {      // (from tile t on)
        Rows r;
        r.at = head + (int64_t)span.tile(t) * KT * sn;
        r.tile = KT * sn;
        r.sn = (uint32_t)sn * 2u;
#pragma unroll
        for (int i = 0; i < Pieces::N; i++) r.off[i] = pieces.row(i) * r.sn + pieces.col(i, lane);
        return r;
    }
    __device__ void copy(Rows& r, int t, int to) const {
        auto place = [&](int i) { return __builtin_amdgcn_readfirstlane(lds + to + (i * NW + wave) * 1024); };
        if (Pieces::N > 1 && whole.has(t)) {
#pragma unroll
            for (int i = 0; i < Pieces::N; i++) dma16(r.at, r.off[i], place(i));
        } else {
#pragma unroll
            for (int i = 0; i < Pieces::N; i++) {
                uint32_t off = r.off[i];
                if (!whole.has(t)) {
                    const int j0 = span.tile(t) * KT;
                    off = (uint32_t)(copied_key<KT>(span, j0, j0 + pieces.row(i)) - j0) * r.sn + pieces.col(i, lane);
                }
                dma16(r.at, off, place(i));
            }
        }
        r.at += (t + 1 == span.first ? span.next - t : 1) * r.tile;        // (from the tiles with sinks to the window's)
    }
};

// 32 rows x0 .. of (query, head) pairs -> LDS at dst; rows past the last repeat it.  `base` is query i_base's row of the group's first head.
template <int D>
__device__ __forceinline__ void query_rows_in(const WindowArgs& a, const uint16_t* base, int64_t sn, int64_t sh, int i_base, int x0, uint32_t dst, int lane) {
    constexpr int CPR = D / 8, RPI = 64 / CPR;
    const int last = a.Sq * a.g - 1;
#pragma unroll
    for (int n = 0; n < 32 / RPI; n++) {
        const int r = n * RPI + lane / CPR, x = min(x0 + r, last), i = x / a.g;
        const uint32_t off = ((uint32_t)(i - i_base) * (uint32_t)sn + (uint32_t)(x - i * a.g) * (uint32_t)sh) * 2u;
        dma16(base, off + nat_pos<CPR>(r, lane % CPR) * 16, __builtin_amdgcn_readfirstlane(dst + n * 1024));
    }
}
// ... and 32 finished rows from LDS (packed, laid out as a tile) to those below the last of `out`, the group's first head of the sequence
template <int D>
__device__ __forceinline__ void query_rows_out(const WindowArgs& a, const uint8_t* os, uint16_t* out, int64_t sn, int64_t sh, int x0, int lane) {
    constexpr int CPR = D / 8, RPI = 64 / CPR;
    const int rows = a.Sq * a.g;
    asm volatile("" : "+v"(lane));       // (the rows' numbers are formed again, not kept since they were read)
#pragma unroll
    for (int n = 0; n < 32 / RPI; n++) {
        const int r = n * RPI + lane / CPR, x = x0 + r, i = x / a.g;
        const u32x4 w = *reinterpret_cast<const u32x4*>(os + nat_off<CPR>(r, lane % CPR));
        if (x < rows) *reinterpret_cast<u32x4*>(out + i * sn + (int64_t)(x - i * a.g) * sh + (lane % CPR) * 8) = w;
    }
}
// what rounding to the type leaves of x
template <int T> __device__ __forceinline__ float rounded_off(float x) {
    if constexpr (T == kBF16) return x - (float)(__bf16)x;
    else return x - (float)(_Float16)x;
}
// Channels d * 32 + g * 8 + half * 4 .. + 3 of the lane's row, an accumulator's registers times `mul` -> LDS.
// REST: what rounding leaves of them.
template <int T, int D, bool REST = false> __device__ __forceinline__ void row_put(uint8_t* os, const v16f& acc, int d, float mul, int lane) {
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int g = 0; g < 4; g++) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            y[e] = acc[g * 4 + e] * mul;
            if constexpr (REST) y[e] = rounded_off<T>(y[e]);
        }
        *reinterpret_cast<u32x2*>(os + nat_off<D / 8>(lane & 31, d * 4 + g) + (lane >> 5) * 8) = u32x2{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3])};
    }
}

// ---- sequences one behind the other ----------------------------------------------------------------------
// Sequence b's rows, b = B: those behind the last sequence (queries without keys, keys without queries).
struct Sequence { int q0, nq, k0, nk; };
__device__ __forceinline__ int sequence_start(const int32_t* cu, int b, int rows) { return b == 0 ? 0 : max(0, min(cu[b], rows)); }
__device__ __forceinline__ Sequence sequence(const PackedArgs& a, int b) {
    Sequence s;
    s.q0 = sequence_start(a.cu_q, b, a.rows_q);
    s.k0 = sequence_start(a.cu_k, b, a.rows_k);
    s.nq = b < a.B ? max(0, min(a.cu_q[b + 1], a.rows_q) - s.q0) : a.rows_q - s.q0;
    s.nk = b < a.B ? max(0, min(a.cu_k[b + 1], a.rows_k) - s.k0) : a.rows_k - s.k0;
    return s;
}
// Its rows as a batch of one; where sides are asked for behind the last sequence, the other one is empty.
__device__ __forceinline__ WindowArgs view(const WindowArgs& all, const Sequence& s, int nq, int nk) {
    WindowArgs w = all;
    w.B = 1;
    w.q += s.q0 * w.q_sn;
    w.k += s.k0 * w.k_sn;
    w.v += s.k0 * w.v_sn;
    w.o += s.q0 * w.o_sn;
    if (w.rest != nullptr) w.rest += s.q0 * w.o_sn;
    if (w.stats != nullptr) w.stats += s.q0;
    w.Sq = nq;
    w.Skv = nk;
    w.lens = w.starts = nullptr;
    w.at_end = 0;
    w.start = nk - nq;
    return w;
}
// Slots of `rows` rows for a sequence's n: from cu[b] * per / rows + b on, which leaves n * per / rows + 1 at the least, so that a slot names its sequence without a
// sum over those before it.  With slots for the rows behind the last there are total(..).
struct Slots {
    const int32_t* cu;
    int rows_all, per, rows;
    __device__ int first(int b) const { return (int)((uint32_t)sequence_start(cu, b, rows_all) * (uint32_t)per / (uint32_t)rows) + b; }
    __device__ int owner(int slot, int B) const {
        int lo = 0, hi = B + 1;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first(mid) <= slot) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};
__host__ __device__ inline int64_t slots_total(int64_t rows_all, int64_t per, int64_t rows, int64_t B) { return rows_all * per / rows + B + 1; }

// The sequence that a slot names and which of its blocks of rows (KEYS: of keys), the heaviest first: sequences in the order of how much a block of theirs
// has to walk (up to 64 of them, a lane each; more are taken as they come, their slots as above).  The blocks of a sequence: `n`; an index of n or beyond: no work.
struct Found { int b, index, n; Sequence s; };
template <bool KEYS> __device__ __forceinline__ Found find_slot(const PackedArgs& a, int per, int rows, int slot) {
    if (a.B > 64) {
        const Slots slots = {KEYS ? a.cu_k : a.cu_q, KEYS ? a.rows_k : a.rows_q, per, rows};
        const int b = slots.owner(slot, a.B);
        const Sequence s = sequence(a, b);
        return Found{b, slot - slots.first(b), (int)(((uint32_t)(KEYS ? s.nk : s.nq) * (uint32_t)per + (uint32_t)rows - 1) / (uint32_t)rows), s};
    }
    const int lane = (int)threadIdx.x & 63;
    int count = 0, order = -1, start = 0, total = 0;
    Sequence s = {0, 0, 0, 0};
    if (lane < a.B) {
        s = sequence(a, lane);
        count = (int)(((uint32_t)(KEYS ? s.nk : s.nq) * (uint32_t)per + (uint32_t)rows - 1) / (uint32_t)rows);
        order = min(KEYS ? s.nq : s.nk, (1 << 25) - 1) << 6 | (63 - lane);
    }
    for (int j0 = 0; j0 < a.B; j0 += 4)
#pragma unroll
        for (int j = j0; j < j0 + 4; j++) {              // (lanes from B on: no blocks)
            const int order_j = __builtin_amdgcn_readlane(order, j), count_j = __builtin_amdgcn_readlane(count, j);
            start += order_j > order ? count_j : 0;
            total += count_j;
        }
    const unsigned long long here = __ballot(lane < a.B && slot >= start && slot < start + count);
    if (here == 0) {                     // (rows behind the last sequence, or nothing)
        s = sequence(a, a.B);
        return Found{a.B, slot - total, (int)(((uint32_t)(KEYS ? s.nk : s.nq) * (uint32_t)per + (uint32_t)rows - 1) / (uint32_t)rows), s};
    }
    const int b = (int)__builtin_ctzll(here);
    return Found{b, slot - __builtin_amdgcn_readlane(start, b), __builtin_amdgcn_readlane(count, b),
                 Sequence{__builtin_amdgcn_readlane(s.q0, b), __builtin_amdgcn_readlane(s.nq, b), __builtin_amdgcn_readlane(s.k0, b), __builtin_amdgcn_readlane(s.nk, b)}};
}

}  // namespace

}  // namespace sage
