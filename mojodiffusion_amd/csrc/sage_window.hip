// sage_window.hip — attention over a sliding window with a few first tokens that stay visible, bf16 or fp16.
//
//     S_ij = scale q_i . k_j  for the keys j that query i sees,  O_i = sum_j exp(S_ij - L_i) v_j,  L_i = log sum_j exp(S_ij)
//
// One pass over the visible key tiles with the running reference and sum of the softmax.  A wave owns 32 rows ("x": pairs of
// a query and a head of the group that shares keys) as the columns of its matrix products: a 32 x 32 block of scores
// S^T = K Q^T lands with the row as the lane's column, which is the operand layout of O^T += V^T P^T, so the
// probabilities go from registers into the next product; V^T comes from the row-major tile by the transposing LDS read.
// Scores, reference, sum and O are fp32; P is rounded to the inputs' type as a matrix operand (an error of at most
// half a step of each weight, unbiased over the keys), the sum is taken over the unrounded values.
//
// Which keys a workgroup walks follows from its rows' positions: the tiles of the first `sinks` keys, then those from the first
// row's left edge to the last row's right edge.  Tiles that every row of a wave sees whole take no mask; a wave leaves out tiles that
// none of its rows sees.  Rows of a tile that no row of the workgroup sees are not read at all (another key's row stands
// in), so whatever lies there, or behind a sequence's end, cannot reach a result.
#include "sage_grid.h"
#include "sage_window_common.h"

#include <algorithm>
#include <type_traits>

namespace sage {

namespace {

// What a lane keeps of its row, and the tile's part in it.
template <int D> struct RowState {
    v16f acc[D / 32];                // O^T: channels d * 32 + (i >> 2) * 8 + half * 4 + (i & 3)
    float ref, sum;                  // reference in log2 units, and this lane's part of the sum of exp2(S - ref)
    __device__ void clear() {
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[d][i] = 0.0f;
        ref = -INFINITY;
        sum = 0.0f;
    }
    // A new reference (log2 units), where `top` lies above the old one.
    __device__ void raise(float top) {
        const float r = fmaxf(ref, top), f = r == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - r);
        ref = r;
        sum *= f;
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[d][i] *= f;
    }
};
// FINE: the weights enter as two operands, what rounding leaves of them in a second product: for workgroups of
// at most kFineKeys keys, whose rows average over too few keys for the roundings of their weights to fade (relative error of dQ, whose row sums are
// taken from O, on a padded batch with sinks: 0.0027 without, 0.0024 with it; the products are a small part of what such a workgroup does).  By the keys of a workgroup, not of
// a row: rows of short windows in longer spans gain nothing from it (window 16 + 1 on [1,1024,heads,64], dQ: 0.00236 without it, one head to a group, 0.00234 with it, four).
constexpr int kFineKeys = 128;
template <int T, int D, bool FINE>
__device__ __forceinline__ void attend_tile(RowState<D>& st, const v4i (&q)[D / 16], uint32_t kt, uint32_t vt, const Fragments<D>& kept,
                                            Seen what, int j0, const RowMask& m, float c) {
    constexpr int KS = D / 16, DB = D / 32;
    const Fragments<D> f = D > 64 || FINE ? kept.fresh() : kept;         // (at 64 channels there is room for the addresses)
    auto key = [&](int ks) { return lds_read(kt + (f.nat ^ ((ks & 7) << 5)) + (ks >> 3) * 256); };
    v16f s = product<T>(key(0), q[0], v16f{});
#pragma unroll
    for (int ks = 1; ks < KS; ks++) s = product<T>(key(ks), q[ks], s);
    if (what != Seen::kAll) {
        const RowMask rel = m.from(j0 + (lane_here() >> 5) * 4);
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = rel.sees((i >> 2) * 8 + (i & 3)) ? s[i] : -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; i++) top = fmaxf(top, s[i]);
    top = max_halves(top) * c;
    // A new reference only where the old one lies more than 8 below: the weights stay under 2^8, and the sums have
    // room for that; O is multiplied on few tiles instead of on most.
    if (__any(top > st.ref + 8.0f)) st.raise(top);
    const float ref = st.ref == -INFINITY ? 0.0f : st.ref;       // (no key so far: every weight is exp2(-inf))
    uint32_t p[8], fine[FINE ? 8 : 1];
    float part[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[i], c, -ref)), y = __builtin_amdgcn_exp2f(fmaf(s[i + 1], c, -ref));
        part[0] += x;
        part[1] += y;
        p[i >> 1] = pack2<T>(x, y);
        if constexpr (FINE) fine[i >> 1] = pack2<T>(rounded_off<T>(x), rounded_off<T>(y));
    }
    st.sum += part[0] + part[1];
#pragma unroll
    for (int j2 = 0; j2 < 2; j2++)
#pragma unroll
        for (int d = 0; d < DB; d++) {
            const uint32_t at = vt + j2 * 32 * D + (d >> 2) * 256;
            const v4i vf = lds_read_across(at + (f.tr[0] ^ ((d & 3) << 6)), at + (f.tr[1] ^ ((d & 3) << 6)));
            st.acc[d] = product<T>(vf, v4i{(int)p[j2 * 4], (int)p[j2 * 4 + 1], (int)p[j2 * 4 + 2], (int)p[j2 * 4 + 3]}, st.acc[d]);
            if constexpr (FINE)
                st.acc[d] = product<T>(vf, v4i{(int)fine[j2 * 4], (int)fine[j2 * 4 + 1], (int)fine[j2 * 4 + 2], (int)fine[j2 * 4 + 3]}, st.acc[d]);
        }
}

// What a row's weighted sum is multiplied by.  A sum of zero is that of a row that sees no key, which gives zeros, or one whose scores are
// all -inf, which gives what exp(-inf + inf) is; the mask tells them apart.  (A NaN among the scores is in the sum.)
__device__ __forceinline__ float weight_of(const WindowArgs& a, float sum, int b, int i) {
    if (sum != 0.0f) return 1.0f / sum;
    const int len = sequence_len(a, b);
    return seeing(a, first_position(a, b, len), len).has(i) ? __builtin_nanf("") : 0.0f;
}

// The wave's finished rows: registers -> LDS (64 * D bytes at os) -> O, and the statistics.
template <int T, int D>
__device__ __forceinline__ void finish_rows(const WindowArgs& a, const RowState<D>& st, uint8_t* os, int b, int kvh, int x0, int lane) {
    const int rows = a.Sq * a.g, x = x0 + (lane & 31);
    const float sum = sum_halves(st.sum);
    const float inv = weight_of(a, sum, b, min(x, rows - 1) / a.g);
#pragma unroll
    for (int d = 0; d < D / 32; d++) row_put<T, D>(os, st.acc[d], d, inv, lane);
    if (a.stats != nullptr && lane < 32 && x < rows) {
        const int i = x / a.g;
        a.stats[((int64_t)b * a.Hk * a.g + kvh * a.g + (x - i * a.g)) * a.Sq + i] = sum == 0.0f ? -INFINITY : (st.ref + __builtin_amdgcn_logf(sum)) * kLn2;
    }
    const int64_t at = b * a.o_sb + (int64_t)kvh * a.g * a.o_sh;
    query_rows_out<D>(a, os, a.o + at, a.o_sn, a.o_sh, x0, lane);
    if (a.rest == nullptr) return;
#pragma unroll
    for (int d = 0; d < D / 32; d++) row_put<T, D, true>(os, st.acc[d], d, inv, lane);
    query_rows_out<D>(a, os, a.rest + at, a.o_sn, a.o_sh, x0, lane);
}

// Tiles of 32 keys, two slots.  The waves' own rows lie over all of them but K's first at the start, and over the front again at the end.
template <int D> struct WindowLds {
    static constexpr int NW = 4, KT = 32, TILE = KT * D * 2, OWN = NW * 64 * D;
    static constexpr int K0 = 3 * TILE > OWN ? 3 * TILE : OWN, BYTES = K0 + TILE;
    static __device__ int keys(int t) { return t & 1 ? 2 * TILE : K0; }
    static __device__ int values(int t) { return (t & 1) * TILE; }
};

// Workgroups of four waves, 128 rows.  A wave's step from scores to exponentials to products is one chain; what fills the gaps is the waves of other
// workgroups on the same SIMD, which meet no common barrier with it: five at 64 channels, three at 128, two at 256 (by registers: O, Q and one
// tile's scores are 64, 112, 208 of them).  The next tile's scores taken beside this one's weights, with a wave less, was slower: [1,16896,48 on 12,128]
// window 4096 + 4 1615 us, this form 1553; a training step of [2,1248,30,128] +-256 180, 175.  Two waves of this form at 128 channels: 1950.
template <int T, int D>
__global__ __launch_bounds__(256, D == 64 ? 5 : D == 128 ? 3 : 2) void window_kernel(WindowArgs a) {
    using L = WindowLds<D>;
    constexpr int NW = L::NW, KT = L::KT, KS = D / 16;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[L::BYTES];
    const int rows = a.Sq * a.g, blocks = (rows + NW * 32 - 1) / (NW * 32);
    const int item = xcd_item((int)blockIdx.x, a.B * a.Hk * blocks);
    const int bh = item / blocks, row0 = (blocks - 1 - item % blocks) * NW * 32;       // (the last rows first: without a left edge they see most keys)
    const int b = bh / a.Hk, kvh = bh % a.Hk;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int x0 = row0 + wave * 32;

    const int len = sequence_len(a, b), p0 = first_position(a, b, len);
    const int i_lo = row0 / a.g;
    const Span span = key_span<KT>(a, p0 + i_lo, p0 + (min(row0 + NW * 32, rows) - 1) / a.g, len);
    const int wp_lo = p0 + min(x0, rows - 1) / a.g, wp_hi = p0 + min(x0 + 31, rows - 1) / a.g;      // this wave's positions
    const int p = p0 + min(x0 + (lane & 31), rows - 1) / a.g;
    const RowMask mask = {p - a.left, min(p + a.right, len - 1), a.sinks};

    const uint32_t lds = lds_addr(smem);
    const KeyTiles<D, NW> tiles(span, lds, wave, lane);
    const Range all = tiles.within(wp_hi - a.left, x0 < rows ? min(wp_lo + a.right, len - 1) : -1);       // which this wave sees all of
    auto k = tiles.rows(a.k + b * a.k_sb + kvh * a.k_sh, a.k_sn), v = tiles.rows(a.v + b * a.v_sb + kvh * a.v_sh, a.v_sn);

    v4i q[KS];
    const Fragments<D> fr(lane);
    query_rows_in<D>(a, a.q + b * a.q_sb + (int64_t)kvh * a.g * a.q_sh + (int64_t)i_lo * a.q_sn, a.q_sn, a.q_sh, i_lo, x0, lds + wave * 64 * D, lane);
    if (span.n > 0) tiles.copy(k, 0, L::keys(0));
    dma_wait<0>();
#pragma unroll
    for (int s = 0; s < KS; s++) q[s] = fr.along(smem + wave * 64 * D, s);
#pragma unroll
    for (int s = 0; s < KS; s++) asm volatile("" : "+v"(q[s]));
    __syncthreads();                     // the rows' LDS becomes the rings' slots
    if (span.n > 0) tiles.copy(v, 0, L::values(0));

    RowState<D> st;
    st.clear();
    const float c = a.scale * kLog2e;
    auto walk = [&](auto fine) {
        auto tile = [&](int t, int slot) {
            dma_wait<0>();
            __syncthreads();             // tile t is visible; every wave is done with tile t - 1
            if (t + 1 < span.n) tiles.copy(k, t + 1, L::keys(slot + 1)), tiles.copy(v, t + 1, L::values(slot + 1));
            const int j0 = span.tile(t) * KT;
            const Seen what = all.has(t) ? Seen::kAll : x0 < rows ? seen<KT>(a, wp_lo, wp_hi, len, j0) : Seen::kNone;
            if (what != Seen::kNone) attend_tile<T, D, decltype(fine)::value>(st, q, lds + L::keys(slot), lds + L::values(slot), fr, what, j0, mask, c);
        };
        if constexpr (D == 64 && !decltype(fine)::value) {     // (slots known ahead: 147 -> 138 us at [2,8192,24 on 8] window 1024 + 4)
            for (int t = 0; t < span.n; t += 2) {
                tile(t, 0);
                if (t + 1 < span.n) tile(t + 1, 1);
            }
        } else {
            for (int t = 0; t < span.n; t++) tile(t, t & 1);
        }
    };
    if (D <= 128 && span.n * KT <= kFineKeys) walk(std::bool_constant<D <= 128>{});
    else walk(std::false_type{});
    __syncthreads();                     // (no copy is in flight: the last step's wait was for all of them)
    if (x0 < rows) finish_rows<T, D>(a, st, smem + wave * 64 * D, b, kvh, x0, lane);
}

// N neighbouring channels of a finished row, and what rounding left of them.
template <int T, int N> __device__ __forceinline__ void store_row(const WindowArgs& a, int64_t at, const float (&y)[N]) {
    auto put = [&](uint16_t* p, const float* x) {
        if constexpr (N == 1) p[0] = (uint16_t)pack2<T>(x[0], 0.0f);
        else if constexpr (N == 8) *reinterpret_cast<u32x4*>(p) = u32x4{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])};
        else
#pragma unroll
            for (int e = 0; e < N; e += 2) *reinterpret_cast<uint32_t*>(p + e) = pack2<T>(x[e], x[e + 1]);
    };
    put(a.o + at, y);
    if (a.rest == nullptr) return;
    float r[N];
#pragma unroll
    for (int e = 0; e < N; e++) r[e] = rounded_off<T>(y[e]);
    put(a.rest + at, r);
}

// ---- few rows: the keys split over waves and workgroups ---------------------------------------------------
// A workgroup owns 32 rows; its waves take tiles of 32 keys in turn, each with two slots of its own to copy into, so no wave waits for
// another before the end, where the waves' partial rows meet in LDS.  With several workgroups to a block of rows the partial rows go to
// memory in fp32 and window_join_kernel adds them up, in order.  Bound by the bytes of K and V.
template <int D> struct SplitLds {
    static constexpr int NW = 4, KT = 32, TILE = KT * D * 2, SLOT = 2 * TILE, SLOTS = D > 128 ? 1 : 2;
    static constexpr int RING = SLOTS * SLOT;                              // per wave
    static constexpr int MEET = NW * 32 * (D + 4) * 4;                     // per wave 32 rows of D floats (+ 4: banks)
    static constexpr int BYTES = NW * RING > MEET ? NW * RING : MEET;
    static_assert(64 * D <= RING, "a wave's rows pass through its ring");
};

template <int T, int D>
__global__ __launch_bounds__(256) void window_split_kernel(WindowArgs a) {
    using L = SplitLds<D>;
    constexpr int NW = L::NW, KT = L::KT, CPR = D / 8, RUNS = L::TILE / 1024, KS = D / 16, DB = D / 32;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[L::BYTES];
    __shared__ float meet_ml[NW][32][2];
    const int rows = a.Sq * a.g, blocks = (rows + 31) / 32;
    const int split = (int)blockIdx.x % a.splits, item = (int)blockIdx.x / a.splits;
    const int bh = item / blocks, x0 = item % blocks * 32;
    const int b = bh / a.Hk, kvh = bh % a.Hk;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    const int len = sequence_len(a, b), p0 = first_position(a, b, len);
    const int i_lo = x0 / a.g;
    const int p_lo = p0 + i_lo, p_hi = p0 + (min(x0 + 32, rows) - 1) / a.g;
    const Span span = key_span<KT>(a, p_lo, p_hi, len);
    const int p = p0 + min(x0 + l32, rows - 1) / a.g;
    const RowMask mask = {p - a.left, min(p + a.right, len - 1), a.sinks};
    const int share = span.n / a.splits, over = span.n - share * a.splits, t0 = share * split + min(split, over), t1 = t0 + share + (split < over ? 1 : 0);

    const uint32_t ring = lds_addr(smem) + wave * L::RING;
    const uint8_t* own = smem + wave * L::RING;
    const uint16_t* kh = a.k + b * a.k_sb + kvh * a.k_sh;
    const uint16_t* vh = a.v + b * a.v_sb + kvh * a.v_sh;
    const uint32_t ks_b = (uint32_t)a.k_sn * 2u, vs_b = (uint32_t)a.v_sn * 2u;
    auto copy_tile = [&](int t, int slot) {
        const int j0 = span.tile(t) * KT;
        const uint16_t *kb = kh + (int64_t)j0 * a.k_sn, *vb = vh + (int64_t)j0 * a.v_sn;
#pragma unroll
        for (int i = 0; i < RUNS; i++) {
            const int P = i * 64 + lane, r = P / CPR, col = nat_pos<CPR>(r, P % CPR) * 16;
            const uint32_t row = (uint32_t)(copied_key<KT>(span, j0, j0 + r) - j0);
            const uint32_t dst = ring + slot * L::SLOT + i * 1024;
            dma16(kb, row * ks_b + col, __builtin_amdgcn_readfirstlane(dst));
            dma16(vb, row * vs_b + col, __builtin_amdgcn_readfirstlane(dst + L::TILE));
        }
    };

    v4i q[KS];
    const Fragments<D> fr(lane);
    query_rows_in<D>(a, a.q + b * a.q_sb + (int64_t)kvh * a.g * a.q_sh + (int64_t)i_lo * a.q_sn, a.q_sn, a.q_sh, i_lo, x0, ring, lane);
    // (the first tile travels beside the rows where there is a slot for it)
    int t = t0 + wave, slot = L::SLOTS - 1;
    if (L::SLOTS == 2 && t < t1) {
        copy_tile(t, 1);
        dma_wait<2 * RUNS>();
    } else {
        dma_wait<0>();
    }
#pragma unroll
    for (int s = 0; s < KS; s++) q[s] = fr.along(own, s);
#pragma unroll
    for (int s = 0; s < KS; s++) asm volatile("" : "+v"(q[s]));

    RowState<D> st;
    st.clear();
    const float c = a.scale * kLog2e;
    // (a slot is filled again only when the reads of what it held have come back)
    auto reads_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
    reads_done();
    if (L::SLOTS == 1 && t < t1) copy_tile(t, 0);
    for (; t < t1; t += NW) {
        if (L::SLOTS == 2 && t + NW < t1) {
            reads_done();
            copy_tile(t + NW, slot ^ 1);
            dma_wait<2 * RUNS>();
        } else {
            dma_wait<0>();
        }
        const int j0 = span.tile(t) * KT;
        const uint32_t kt = ring + slot * L::SLOT;
        const Seen what = seen<KT>(a, p_lo, p_hi, len, j0);
        if (D <= 128 && span.n * KT <= kFineKeys) attend_tile<T, D, D <= 128>(st, q, kt, kt + L::TILE, fr, what, j0, mask, c);
        else attend_tile<T, D, false>(st, q, kt, kt + L::TILE, fr, what, j0, mask, c);
        if (L::SLOTS == 2) slot ^= 1;
        else if (t + NW < t1) {
            reads_done();
            copy_tile(t + NW, 0);
        }
    }

    // The waves' parts meet: every part is taken to the largest reference of its row.
    __syncthreads();
    const float wsum = sum_halves(st.sum);
    if (half == 0) meet_ml[wave][l32][0] = st.ref, meet_ml[wave][l32][1] = wsum;
    float* parts = reinterpret_cast<float*>(smem);
    constexpr int PR = D + 4;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *reinterpret_cast<v4f*>(parts + (wave * 32 + l32) * PR + d * 32 + g * 8 + half * 4) =
                v4f{st.acc[d][g * 4], st.acc[d][g * 4 + 1], st.acc[d][g * 4 + 2], st.acc[d][g * 4 + 3]};
    __syncthreads();
    // 8 lanes to a row, D / 8 channels each
    const int r = tid >> 3, x = x0 + r;
    float ref = -INFINITY, sum = 0.0f, f[NW];
#pragma unroll
    for (int w = 0; w < NW; w++) ref = fmaxf(ref, meet_ml[w][r][0]);
#pragma unroll
    for (int w = 0; w < NW; w++) {
        f[w] = ref == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(meet_ml[w][r][0] - ref);
        sum = fmaf(meet_ml[w][r][1], f[w], sum);
    }
    if (x >= rows) return;
    const int i = x / a.g, hg = x - i * a.g;
    const bool last = a.splits == 1;
    const float inv = last ? weight_of(a, sum, b, i) : 1.0f;
    float* po = a.part + ((int64_t)item * a.splits + split) * 32 * D + r * D;
    const int64_t at = b * a.o_sb + ((int64_t)kvh * a.g + hg) * a.o_sh + i * a.o_sn;
#pragma unroll
    for (int n = 0; n < D / 64; n++) {
        const int col = (n * 8 + (tid & 7)) * 8;
        float y[8];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            v4f sumv = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const v4f v = *reinterpret_cast<const v4f*>(parts + (w * 32 + r) * PR + col + h * 4);
#pragma unroll
                for (int e = 0; e < 4; e++) sumv[e] = fmaf(v[e], f[w], sumv[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) y[h * 4 + e] = sumv[e] * inv;
        }
        if (last) {
            store_row<T, 8>(a, at + col, y);
        } else {
            *reinterpret_cast<v4f*>(po + col) = v4f{y[0], y[1], y[2], y[3]};
            *reinterpret_cast<v4f*>(po + col + 4) = v4f{y[4], y[5], y[6], y[7]};
        }
    }
    if ((tid & 7) == 0) {
        if (!last) {
            float* ml = a.part_ml + (((int64_t)item * a.splits + split) * 32 + r) * 2;
            ml[0] = ref, ml[1] = sum;
        } else if (a.stats != nullptr) {
            a.stats[((int64_t)b * a.Hk * a.g + kvh * a.g + hg) * a.Sq + i] = sum == 0.0f ? -INFINITY : (ref + __builtin_amdgcn_logf(sum)) * kLn2;
        }
    }
}

// 64 lanes of D / 64 channels each to a row; WAVES of them share a row's parts and meet in LDS: four where there are more than eight parts, one else.
// What this launch takes is latencies (4 us of the 10 of one token against 1024 keys of 12 heads), so a wave requests eight parts (four, where
// no more are left) at a time, their statistics with them, and adds them up as the tiles are, by a running maximum.
constexpr int kJoinParts = 8;
template <int T, int D, int WAVES>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a) {
    constexpr int N = D / 64;
    typedef float vnf __attribute__((ext_vector_type(N)));
    const int rows = a.Sq * a.g, blocks = (rows + 31) / 32;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const uint32_t at = WAVES > 1 ? blockIdx.x : blockIdx.x * 4u + (uint32_t)wave;
    if (at >= (uint32_t)(a.B * a.Hk * rows)) return;
    const int lane = threadIdx.x & 63, bh = (int)(at / (uint32_t)rows), x = (int)at - bh * rows, b = bh / a.Hk, kvh = bh % a.Hk;
    const int64_t item = (int64_t)bh * blocks + x / 32;
    const float* ml = a.part_ml + (item * a.splits * 32 + x % 32) * 2;
    const float* part = a.part + (item * a.splits * 32 + x % 32) * D + lane * N;
    float ref = -INFINITY, sum = 0.0f, y[N];
#pragma unroll
    for (int e = 0; e < N; e++) y[e] = 0.0f;
    auto take = [&](auto count, int s0) {
        constexpr int AT_ONCE = decltype(count)::value;
        vnf v[AT_ONCE];
        float m[AT_ONCE], l[AT_ONCE], top = ref;
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const int64_t s = min(s0 + u, a.splits - 1);
            m[u] = ml[s * 64];
            l[u] = ml[s * 64 + 1];
            v[u] = *reinterpret_cast<const vnf*>(part + s * 32 * D);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) top = fmaxf(top, m[u]);
        // (no reference yet: parts that saw nothing, whose sums are zero, and parts whose scores were NaN, whose sums are: they pass as they are)
        const float f0 = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - top);
        ref = top;
        sum *= f0;
#pragma unroll
        for (int e = 0; e < N; e++) y[e] *= f0;
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            if (s0 + u >= a.splits) return;
            const float f = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[u] - ref);
            sum = fmaf(l[u], f, sum);
#pragma unroll
            for (int e = 0; e < N; e++) y[e] = fmaf(v[u][e], f, y[e]);
        }
    };
    for (int s0 = WAVES > 1 ? wave * kJoinParts : 0; s0 < a.splits; s0 += WAVES * kJoinParts) {
        if (a.splits - s0 > kJoinParts / 2) take(std::integral_constant<int, kJoinParts>{}, s0);
        else take(std::integral_constant<int, kJoinParts / 2>{}, s0);
    }
    if constexpr (WAVES > 1) {
        __shared__ float meet[WAVES][N + 2][64];
        meet[wave][N][lane] = ref, meet[wave][N + 1][lane] = sum;
#pragma unroll
        for (int e = 0; e < N; e++) meet[wave][e][lane] = y[e];
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int n = 1; n < WAVES; n++) ref = fmaxf(ref, meet[n][N][lane]);
        const float top = ref;
        sum = 0.0f;
#pragma unroll
        for (int e = 0; e < N; e++) y[e] = 0.0f;
#pragma unroll
        for (int n = 0; n < WAVES; n++) {
            const float f = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(meet[n][N][lane] - top);
            sum = fmaf(meet[n][N + 1][lane], f, sum);
#pragma unroll
            for (int e = 0; e < N; e++) y[e] = fmaf(meet[n][e][lane], f, y[e]);
        }
    }
    const int i = x / a.g, hg = x - i * a.g;
    const float inv = weight_of(a, sum, b, i);
#pragma unroll
    for (int e = 0; e < N; e++) y[e] *= inv;
    store_row<T, N>(a, b * a.o_sb + ((int64_t)kvh * a.g + hg) * a.o_sh + i * a.o_sn + lane * N, y);
    if (a.stats != nullptr && lane == 0)
        a.stats[((int64_t)b * a.Hk * a.g + kvh * a.g + hg) * a.Sq + i] = sum == 0.0f ? -INFINITY : (ref + __builtin_amdgcn_logf(sum)) * kLn2;
}

int64_t row_blocks(const WindowArgs& a, int rows) { return (int64_t)a.B * a.Hk * (((int64_t)a.Sq * a.g + rows - 1) / rows); }

template <int T, int D> hipError_t launch_td(const WindowArgs& a, const WindowPlan& p, hipStream_t st) {
    if (!p.splits) hipLaunchKernelGGL((window_kernel<T, D>), dim3((unsigned)row_blocks(a, 128)), dim3(256), 0, st, a);
    else {
        hipLaunchKernelGGL((window_split_kernel<T, D>), dim3((unsigned)(row_blocks(a, 32) * a.splits)), dim3(256), 0, st, a);
        const int64_t rows = (int64_t)a.B * a.Hk * a.Sq * a.g;
        if (a.splits > kJoinParts) hipLaunchKernelGGL((window_join_kernel<T, D, 4>), dim3((unsigned)rows), dim3(256), 0, st, a);
        else if (a.splits > 1) hipLaunchKernelGGL((window_join_kernel<T, D, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
    }
    return hipGetLastError();
}
template <int T> hipError_t launch_t(const WindowArgs& a, const WindowPlan& p, hipStream_t st) {
    if (a.D == 64) return launch_td<T, 64>(a, p, st);
    if (a.D == 128) return launch_td<T, 128>(a, p, st);
    return launch_td<T, 256>(a, p, st);
}

}  // namespace

// Blocks of 128 rows for half the chip: tiles shared by four waves.  (96 such blocks at 128 channels: 30 us, split 27; 192: 30, split 40.)  One token a
// sequence gains nothing from the sharing: there it takes as many blocks as compute units (128 blocks of 8192 keys: 197 us, split 104), and at 128
// channels, from 1024 keys on, the keys are split where that leaves the last round of workgroups full or nearly, since four waves with two tiles each on
// their way keep more bytes in flight (256 blocks of 8192 keys: 218 us, split 180; of 1024: 31, split 24; 384 of up to 8192: 291, in two parts 278; but 264
// of 1024: 32, in four parts 40; at 64 channels 512 of 2048 39, split 45, at 256 512 of 1024 96, split 105).
// Split: until the chip is full once, a workgroup's LDS leaving room for two on a compute unit at 64 channels, for one above.
// Down to 128 keys (one tile to a wave), counted as a row sees them on the average; and to the root of their number, since the join's time
// grows with the parts (one head against 65536 keys, us: 512 parts 37, 90 parts 16; 2048 keys: 9).
WindowPlan window_plan(const WindowArgs& a) {
    constexpr int64_t kUnits = 256;
    int64_t keys = a.right >= kWindowFar || a.left >= kWindowFar ? a.Skv
                                                                 : std::min<int64_t>(a.Skv, (int64_t)a.left + a.right + 32 / a.g + 1 + a.sinks);
    if (a.right < kWindowFar) keys -= std::min<int64_t>(a.Sq, keys) / 2;
    const int64_t room = a.D > 64 ? kUnits : 2 * kUnits, blocks = row_blocks(a, 32);
    int64_t splits = room / blocks;
    if (a.Sq * (int64_t)a.g > 32) {
        if (row_blocks(a, 128) >= kUnits / 2) return WindowPlan{0};
    } else if (blocks >= kUnits) {
        if (a.D != 128 || keys < 1024) return WindowPlan{0};
        auto full = [&](int64_t n) { const int64_t last = blocks * n % room; return last == 0 || last >= room * 3 / 4; };
        for (splits = 1; !full(splits); splits++)
            if (splits == 3) return WindowPlan{0};
    }
    splits = std::max<int64_t>(1, std::min(splits, keys / 128));
    while (splits * splits > std::max<int64_t>(1, keys / 8)) splits--;
    return WindowPlan{(int)splits};
}
bool window_grid_ok(const WindowArgs& a, const WindowPlan& p) {
    return row_blocks(a, 32) * std::max(p.splits, 1) <= 0x7FFFFFFF && (int64_t)a.B * a.Hk * a.Sq * a.g <= 0x7FFFFFFF;
}
size_t window_part_bytes(const WindowArgs& a, const WindowPlan& p) {
    return p.splits <= 1 ? 0 : (size_t)row_blocks(a, 32) * p.splits * 32 * (a.D + 2) * sizeof(float);
}

hipError_t launch_window(const WindowArgs& a, const WindowPlan& p, hipStream_t st) {
    return a.type == kBF16 ? launch_t<kBF16>(a, p, st) : launch_t<kF16>(a, p, st);
}

}  // namespace sage
