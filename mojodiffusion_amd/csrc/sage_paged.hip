// sage_paged.hip — attention of the last tokens of every sequence over its paged cache of e4m3 codes (sage_kv.h), bf16 or fp16.
//
//     S_ij = scale 2^ek(j) q_i . k_j  for the keys j up to query i's own position,  O_i = sum_j exp(S_ij - L_i) 2^ev(j) v_j,  L_i = log sum_j exp(S_ij)
//
// Bound by the bytes of K and V.  Codes have four significant bits, so they are operands of the inputs' type without a rounding (K's as they are, its scale goes to the scores; V's see
// RowState): one instruction widens two of them, and Q and the weights keep their own type.  A wave takes a block of 32 keys at a time, straight from memory into the
// registers that the matrix products read (no LDS): scores S^T = K Q^T with 16 keys as the rows, then O^T += V^T P^T over all 32.  The lane that holds the scores of
// a query's keys 8 q .. 8 q + 7 (q = lane / 16) hands just those to the second product, because the first takes its keys in that order; V lies a
// channel after the other, so those eight keys of a channel are eight bytes.  The next block is on its way while one is computed.
//
// Blocks of all sequences and heads are one list, dealt to the workgroups in equal shares, so sequences of any lengths fill the chip; rows whose
// blocks fall to several workgroups are left as parts in fp32 that a second launch adds up, in order: the same bits on every call.
// Measured, bf16, 48 on 12 heads of 128: one token of 32 sequences of 2 to 16 thousand keys 171 us, 5.4 TB/s; of one with 8192 keys 13 us, in launches of 8.4 and 3.2.
#include "sage_grid.h"
#include "sage_kv.h"
#include "sage_tile.h"
#include "sage_window.h"

#include <algorithm>

namespace sage {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2hf __attribute__((ext_vector_type(2)));
constexpr int kWaves = 4;

template <int T> __device__ __forceinline__ v4f product(v4i a, v4i b, v4f c) {
    if constexpr (T == kBF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
template <int T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (T == kBF16) return pack_bf16(a, b);
    const v2f f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2hf));
}
// Eight codes times a power of two, in the inputs' type.
template <int T> __device__ __forceinline__ v4i widen(uint32_t lo, uint32_t hi, float scale) {
    if constexpr (T == kBF16)
        return v4i{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
                   __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
    else
        return v4i{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true)),
                   __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true))};
}
// The four lanes of a query, 16 apart.
__device__ __forceinline__ float max_quads(float x) {
    const v2u a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a.x), __uint_as_float(a.y));
    const v2u b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b.x), __uint_as_float(b.y));
}
__device__ __forceinline__ float sum_quads(float x) {
    const v2u a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a.x) + __uint_as_float(a.y);
    const v2u b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b.x) + __uint_as_float(b.y);
}

__device__ __forceinline__ int cached(const PagedArgs& a, int b) { return max(0, min(a.pool.lens[b], a.pool.width << (5 + a.pool.sub))); }
// Blocks of a sequence; one at the least, so that rows which see nothing have an owner too.
__device__ __forceinline__ int blocks_of(int len) { return max(1, (len + kKvBlock - 1) / kKvBlock); }

// Sums over a wave's lanes by moves between neighbours, rows and halves (lane shuffles go through LDS; six of them are a fifth of a microsecond, of
// which a call of one token has few).
template <int CTRL, int ROWS = 0xF> __device__ __forceinline__ int moved(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, true); }
template <class F> __device__ __forceinline__ int wave_all(int x, F f) {
    x = f(x, moved<0xB1>(x));            // lanes ^ 1, ^ 2, then the other half of 8, of 16
    x = f(x, moved<0x4E>(x));
    x = f(x, moved<0x141>(x));
    x = f(x, moved<0x140>(x));
    const v2u a = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false);
    x = f((int)a.x, (int)a.y);
    const v2u b = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
    return __builtin_amdgcn_readfirstlane(f((int)b.x, (int)b.y));
}
__device__ __forceinline__ int wave_sum(int x) { return wave_all(x, [](int p, int q) { return p + q; }); }
__device__ __forceinline__ int wave_max(int x) { return wave_all(x, [](int p, int q) { return max(p, q); }); }
// Sums of the lanes up to and with each.
__device__ __forceinline__ int wave_scan(int x) {
    x += moved<0x111>(x);                // from 1, 2, 4, 8 lanes before in the row of 16
    x += moved<0x112>(x);
    x += moved<0x114>(x);
    x += moved<0x118>(x);
    x += moved<0x142, 0xA>(x);           // the row before, the half before
    x += moved<0x143, 0xC>(x);
    return x;
}

// The list of blocks: sequence after sequence, in each head after head, row block after row block, block after block.
// The share of a workgroup: all of them evenly, eight at the least (two to a wave; 16 from 96 row blocks on, 32 from 192: fewer parts where the chip is full without them), and at the least half the root of the longest sequence's
// blocks, since the second launch's time grows with the parts as the shares shrink.  Where shares are small (up to 32) a workgroup that had the
// end of one row's blocks and the beginning of another's would go through the chain of latencies twice, and all would wait for it: there every row's blocks are
// divided into shares of their own, of 8, 16 or 32.
struct Deal {
    int total, per;
    int len;                             // of the lane's sequence, of the first 64
    int shift;                           // log2 of the rows' own shares, or 0
    // places of a row with n blocks in the list: blocks, or shares
    __device__ int places(int n) const { return (n + (1 << shift) - 1) >> shift; }
};
__device__ __forceinline__ Deal deal(const PagedArgs& a, int mult, int lane) {
    Deal d;
    d.len = lane < a.B ? cached(a, lane) : 0;
    int sum = lane < a.B ? blocks_of(d.len) : 0, most = sum;
    for (int b0 = 64; b0 < a.B; b0 += 64) {
        const int n = b0 + lane < a.B ? blocks_of(cached(a, b0 + lane)) : 0;
        sum += n;
        most = max(most, n);
    }
    d.total = wave_sum(sum) * mult;
    most = wave_max(most);
    d.per = max(max((d.total + a.wgs - 1) / a.wgs, a.least), (int)(0.5f * sqrtf((float)most)));
    d.shift = a.more == 0 || d.per > 32 ? 0 : d.per > 16 ? 5 : d.per > 8 ? 4 : 3;
    if (d.shift > 0) d.per = 1;          // (places of the list)
    return d;
}
// The sequence that place t of the list belongs to, its first place in the list, its own blocks and its length.  n 0: behind the list's end.
struct Place { int b, begin, n, len; };
__device__ __forceinline__ Place place(const PagedArgs& a, const Deal& d, int mult, int t, int lane) {
    int begin = 0;
    for (int b0 = 0;; b0 += 64) {
        const int len = b0 == 0 ? d.len : b0 + lane < a.B ? cached(a, b0 + lane) : 0, n = b0 + lane < a.B ? blocks_of(len) : 0;
        const int here = d.places(n) * mult, end = begin + wave_scan(here);
        const unsigned long long past = __ballot(end > t);
        if (past != 0) {
            const int l = (int)__builtin_ctzll(past);
            return Place{b0 + l, __builtin_amdgcn_readlane(end - here, l), __builtin_amdgcn_readlane(n, l), __builtin_amdgcn_readlane(len, l)};
        }
        begin = __builtin_amdgcn_readlane(end, 63);
        if (b0 + 64 >= a.B) return Place{0, t, 0, 0};
    }
}

// A block's codes as a wave holds them.
template <int D> struct Block {
    u32x4 k[2][D / 64];                  // [16 keys][64 channels: 16 to a lane]
    u32x2 v[D / 16];                     // [16 channels]: 8 keys of one
};
template <int D> __device__ __forceinline__ void load_block(Block<D>& t, const uint8_t* k, const uint8_t* v, uint32_t k_off, uint32_t v_off) {
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int s = 0; s < D / 64; s++) t.k[m][s] = *reinterpret_cast<const u32x4*>(k + k_off + m * 4 * D + s * 64);
#pragma unroll
    for (int d = 0; d < D / 16; d++) t.v[d] = *reinterpret_cast<const u32x2*>(v + v_off + d * 16 * kKvBlock);
}

// Rows of a part: COLS groups of 16 queries.
// bf16: V's codes enter times their scale, which keeps all their bits.  fp16 has no exponents for that (below 2^-15 of its largest number a code loses bits, and a cache that
// bf16 tensors filled may hold what fp16 cannot): there the codes enter as they are, the weights take the scale, and O is held at 2^power of the scores' reference, so that the largest
// weight that it has met, scale included, lies near 2^7: what rounding takes from a weight is 2^-32 of that one at the most.  (fp16's numbers below 2^-14 lose bits, and its largest
// leaves room for 7 beside the 8 that a reference may be behind.  A whole power, so that a row of one key is that key's value.)
constexpr float kLift = 7.0f;
template <int D, int COLS> struct RowState {
    v4f acc[COLS][D / 16];               // O^T: channels d * 16 + q * 4 + i
    float ref[COLS], sum[COLS];
    int power[COLS];
    __device__ void clear() {
#pragma unroll
        for (int n = 0; n < COLS; n++) {
#pragma unroll
            for (int d = 0; d < D / 16; d++) acc[n][d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            ref[n] = -INFINITY;
            sum[n] = 0.0f;
            power[n] = 0;
        }
    }
    __device__ void scale_rows(int n, float f) {
#pragma unroll
        for (int d = 0; d < D / 16; d++) acc[n][d] *= f;
    }
};

// What lies behind a sequence's last key may be any code.  live: how many of the lane's eight keys are the sequence's.
template <int D> __device__ __forceinline__ void drop_values(Block<D>& t, int live) {
    const uint32_t lo = live >= 4 ? 0xFFFFFFFFu : live <= 0 ? 0u : (1u << (live * 8)) - 1u, hi = live >= 8 ? 0xFFFFFFFFu : live <= 4 ? 0u : (1u << ((live - 4) * 8)) - 1u;
#pragma unroll
    for (int d = 0; d < D / 16; d++) t.v[d] &= u32x2{lo, hi};
}

// rel[n]: the position of column n's query, less that of the block's first key and the lane's first; masked: some query does not see all of the block.
template <int T, int D, int COLS>
__device__ __forceinline__ void attend(RowState<D, COLS>& st, const v4i (&q)[COLS][D / 32], const Block<D>& t, float c, float vs, const int (&rel)[COLS], bool masked) {
    v4f s[COLS][2];
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int k = 0; k < D / 64; k++) {
            const v4i lo = widen<T>(t.k[m][k][0], t.k[m][k][1], 1.0f), hi = widen<T>(t.k[m][k][2], t.k[m][k][3], 1.0f);
#pragma unroll
            for (int n = 0; n < COLS; n++) {
                s[n][m] = product<T>(lo, q[n][2 * k], k == 0 ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : s[n][m]);
                s[n][m] = product<T>(hi, q[n][2 * k + 1], s[n][m]);
            }
        }
    if (masked) {
#pragma unroll
        for (int n = 0; n < COLS; n++)
#pragma unroll
            for (int e = 0; e < 8; e++) s[n][e >> 2][e & 3] = e <= rel[n] ? s[n][e >> 2][e & 3] : -INFINITY;
    }
    v4i p[COLS];
#pragma unroll
    for (int n = 0; n < COLS; n++) {
        float top = s[n][0][0];
#pragma unroll
        for (int e = 1; e < 8; e++) top = fmaxf(top, s[n][e >> 2][e & 3]);
        top *= c;
        // (a new reference only where the old one lies more than 8 below: the weights stay under 2^8)
        [[maybe_unused]] int take = 0;   // power of two that the weights take
        if constexpr (T == kBF16) {
            if (__any(top > st.ref[n] + 8.0f)) {
                const float r = fmaxf(st.ref[n], max_quads(top)), f = r == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.ref[n] - r);
                st.ref[n] = r;
                st.sum[n] *= f;
                st.scale_rows(n, f);
            }
        } else {
            const int ve = (int)(__float_as_uint(vs) >> 23 & 255) - 127;
            if (__any(top > st.ref[n] + 8.0f || top + (float)(ve - st.power[n]) > st.ref[n] + (8.0f + kLift))) {
                const float most = max_quads(top), r = fmaxf(st.ref[n], most), up = r == -INFINITY ? 0.0f : r - st.ref[n], was = (float)st.power[n];
                const float power = r == -INFINITY ? was : fmaxf(rintf(was - up), ceilf(most - r + ((float)ve - kLift)));
                st.ref[n] = r;
                st.sum[n] *= __builtin_amdgcn_exp2f(-up);
                st.scale_rows(n, __builtin_amdgcn_exp2f(was - power - up));
                st.power[n] = (int)power;
            }
            take = ve - st.power[n];
        }
        const float ref = st.ref[n] == -INFINITY ? 0.0f : st.ref[n];
        float part = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float y = __builtin_amdgcn_exp2f(fmaf(s[n][e >> 2][e & 3], c, -ref)), z = __builtin_amdgcn_exp2f(fmaf(s[n][e >> 2][(e & 3) + 1], c, -ref));
            part += y + z;
            if constexpr (T == kBF16) p[n][e >> 1] = (int)pack2<T>(y, z);
            else p[n][e >> 1] = (int)pack2<T>(__builtin_amdgcn_ldexpf(y, take), __builtin_amdgcn_ldexpf(z, take));
        }
        st.sum[n] += part;
    }
#pragma unroll
    for (int d = 0; d < D / 16; d++) {
        const v4i v = widen<T>(t.v[d][0], t.v[d][1], T == kBF16 ? vs : 1.0f);
#pragma unroll
        for (int n = 0; n < COLS; n++) st.acc[n][d] = product<T>(v, p[n], st.acc[n][d]);
    }
}

// A finished row's weight; a sum of zero is that of a row that sees no key, which gives zeros, or one whose scores are all -inf.
__device__ __forceinline__ float weight_of(float sum, bool blind) { return blind ? 0.0f : sum != 0.0f ? 1.0f / sum : __builtin_nanf(""); }
template <int T> __device__ __forceinline__ void store4(uint16_t* p, v4f y) { *reinterpret_cast<u32x2*>(p) = u32x2{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3])}; }

template <int T, int D, int COLS> __global__ __launch_bounds__(256, D == 256 ? 1 : D == 128 ? 2 : 5 - COLS) void paged_kernel(PagedArgs a) {
    constexpr int ROWS = 16 * COLS, PR = D + 4;
    __shared__ __attribute__((aligned(16))) float meet[kWaves * ROWS * PR];
    __shared__ float meet_ml[kWaves][ROWS][2];
    const int tid = threadIdx.x, lane = tid & 63, quad = lane >> 4, l16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rows = a.Sq * a.g, rblocks = (rows + ROWS - 1) / ROWS, mult = a.pool.Hk * rblocks;
    const Deal deal_ = deal(a, mult, lane);
    const Share share = share_of((int)blockIdx.x, deal_.per, deal_.total);
    const int t_begin = share.begin, t_end = share.end;
    const uint32_t k_off = (uint32_t)(((l16 >> 2) * 8 + (l16 & 3)) * D + quad * 16), v_off = (uint32_t)(l16 * kKvBlock + quad * 8);
    const KvPool& c = a.pool;

    Place at = {0, 0, 0, 0};
    for (int t = t_begin; t < t_end;) {
        if (t >= at.begin + deal_.places(at.n) * mult) at = place(a, deal_, mult, t, lane);
        if (at.n == 0) return;
        const int places = deal_.places(at.n), unit = (t - at.begin) / places, step = t - at.begin - unit * places;
        const int first = step << deal_.shift, n = min(at.n - first, (t_end - t) << deal_.shift);
        const int b = at.b, h = unit / rblocks, x0 = (unit - h * rblocks) * ROWS;
        const int len = at.len, p0 = len - a.Sq;
        const int p_lo = p0 + x0 / a.g, p_hi = p0 + (min(x0 + ROWS, rows) - 1) / a.g;

        v4i q[COLS][D / 32];
        int pos[COLS];
#pragma unroll
        for (int m = 0; m < COLS; m++) {
            const int x = min(x0 + m * 16 + l16, rows - 1), i = x / a.g;
            pos[m] = p0 + i;
            const uint16_t* row = a.q + b * a.q_sb + ((int64_t)h * a.g + (x - i * a.g)) * a.q_sh + i * a.q_sn + quad * 16;
#pragma unroll
            for (int k = 0; k < D / 64; k++) {
                q[m][2 * k] = *reinterpret_cast<const v4i*>(row + k * 64);
                q[m][2 * k + 1] = *reinterpret_cast<const v4i*>(row + k * 64 + 8);
            }
        }
        RowState<D, COLS> st;
        st.clear();
        // This wave's blocks: every fourth.  A lane looks one of 64 up: its page, its scales.
        const int mine = (n - wave + kWaves - 1) / kWaves;
        for (int i0 = 0; i0 < mine; i0 += 64) {
            const int look = first + wave + (i0 + lane) * kWaves;
            int unit_at = 0;
            float ks = 0.0f, vs = 0.0f;
            if (i0 + lane < mine && look * kKvBlock <= min(p_hi, len - 1)) {
                const int page = c.table[b * c.table_stride + (look >> c.sub)];
                const bool there = page >= 0 && page < c.pages;
                unit_at = there ? (page << c.sub) + (look & ((1 << c.sub) - 1)) : 0;
                ks = there ? c.ks[(int64_t)unit_at * c.Hk + h] : __builtin_nanf("");             // (no such page: no result)
                vs = c.vs[(int64_t)unit_at * c.Hk + h];
            }
            const int count = min(mine - i0, 64);
            auto fetch = [&](Block<D>& t, int i) {
                const int64_t base = ((int64_t)__builtin_amdgcn_readlane(unit_at, i) * c.Hk + h) * (kKvBlock * D);
                load_block<D>(t, c.k + base, c.v + base, k_off, v_off);
            };
            auto use = [&](Block<D>& t, int i) {
                const int j0 = (first + wave + (i0 + i) * kWaves) * kKvBlock;
                if (j0 > min(p_hi, len - 1)) return;
                const float kc = a.scale * kLog2e * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), i));
                const float vc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), i));
                int rel[COLS];
#pragma unroll
                for (int m = 0; m < COLS; m++) rel[m] = pos[m] - j0 - quad * 8;
                if (j0 + kKvBlock > len) drop_values(t, len - j0 - quad * 8);
                attend<T, D, COLS>(st, q, t, kc, vc, rel, j0 + kKvBlock - 1 > p_lo);
            };
            Block<D> even, odd;
            fetch(even, 0);
            for (int i = 0; i < count; i += 2) {
                if (i + 1 < count) fetch(odd, i + 1);
                use(even, i);
                if (i + 1 >= count) break;
                if (i + 2 < count) fetch(even, i + 2);
                use(odd, i + 1);
            }
        }

        // The waves' parts meet: every part is taken to the largest reference of its row.
#pragma unroll
        for (int m = 0; m < COLS; m++) {
            const float sum = sum_quads(st.sum[m]);
            if (quad == 0) meet_ml[wave][m * 16 + l16][0] = st.ref[m], meet_ml[wave][m * 16 + l16][1] = sum;
            if constexpr (T == kF16) st.scale_rows(m, __builtin_amdgcn_ldexpf(1.0f, st.power[m]));
#pragma unroll
            for (int d = 0; d < D / 16; d++) *reinterpret_cast<v4f*>(meet + (wave * ROWS + m * 16 + l16) * PR + d * 16 + quad * 4) = st.acc[m][d];
        }
        __syncthreads();
        const bool whole = n == at.n;
        const int64_t part = ((int64_t)blockIdx.x * 2 + (t == t_begin ? 0 : 1)) * ROWS;
        // 16 (8) threads to a row, four channels at a time
        constexpr int TPR = 256 / ROWS;
        const int r = tid / TPR, x = x0 + r;
        if (x < rows) {
            float ref = -INFINITY, sum = 0.0f, f[kWaves];
#pragma unroll
            for (int w = 0; w < kWaves; w++) ref = fmaxf(ref, meet_ml[w][r][0]);
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                f[w] = ref == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(meet_ml[w][r][0] - ref);
                sum = fmaf(meet_ml[w][r][1], f[w], sum);
            }
            const int i = x / a.g, hg = x - i * a.g;
            const bool blind = p0 + i < 0;
            const float inv = whole ? weight_of(sum, blind) : 1.0f;
            uint16_t* o = a.o + b * a.o_sb + ((int64_t)h * a.g + hg) * a.o_sh + i * a.o_sn;
            for (int col = tid % TPR * 4; col < D; col += TPR * 4) {
                v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    const v4f v = *reinterpret_cast<const v4f*>(meet + (w * ROWS + r) * PR + col);
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] = fmaf(v[e], f[w], y[e]);
                }
                if (whole) store4<T>(o + col, blind ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : y * inv);
                else *reinterpret_cast<v4f*>(a.part + (part + r) * D + col) = y;
            }
            if (!whole && tid % TPR == 0) a.part_ml[(part + r) * 2] = ref, a.part_ml[(part + r) * 2 + 1] = sum;
        }
        __syncthreads();
        t += deal_.places(n);
    }
}

// Rows whose blocks fell to several workgroups: their parts added up, in order, eight at a time.  What it takes are latencies.  SHARED: a workgroup to a
// row, whose waves share the parts: where a row of the table's length has more than eight (paged_shared); else a wave to a row.
constexpr int kJoinParts = 8;
template <int T, int D, bool SHARED> __global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a, int part_rows, int all_rows) {
    constexpr int N = D / 64, WAVES = SHARED ? kWaves : 1;
    typedef float vnf __attribute__((ext_vector_type(N)));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int rows = a.Sq * a.g, rblocks = (rows + part_rows - 1) / part_rows, mult = a.pool.Hk * rblocks;
    const Deal d = deal(a, mult, lane);
    const int first = SHARED ? (int)blockIdx.x : (int)blockIdx.x * kWaves + wave, step = (int)gridDim.x * (SHARED ? 1 : kWaves), share = SHARED ? wave : 0;
    for (int item = first; item < all_rows; item += step) {
        const int bh = item / rows, x = item - bh * rows, b = bh / a.pool.Hk, h = bh - b * a.pool.Hk;
        // where this row's blocks begin in the list, and how many they are
        int before = lane < b ? d.places(blocks_of(d.len)) : 0;
        for (int b0 = 64; b0 < b; b0 += 64) before += b0 + lane < b ? d.places(blocks_of(cached(a, b0 + lane))) : 0;
        const int len = b < 64 ? __builtin_amdgcn_readlane(d.len, b) : cached(a, b), n = d.places(blocks_of(len));
        const int u0 = wave_sum(before) * mult + (h * rblocks + x / part_rows) * n;
        const int w0 = u0 / d.per, w1 = (u0 + n - 1) / d.per;
        if (w0 == w1) continue;                          // (one workgroup had them all)
        const bool aligned = u0 == w0 * d.per;
        float ref = -INFINITY, sum = 0.0f, y[N];
#pragma unroll
        for (int e = 0; e < N; e++) y[e] = 0.0f;
        for (int s0 = w0 + share * kJoinParts; s0 <= w1; s0 += WAVES * kJoinParts) {
            vnf v[kJoinParts];
            float m[kJoinParts], l[kJoinParts], top = ref;
#pragma unroll
            for (int u = 0; u < kJoinParts; u++) {
                const int w = min(s0 + u, w1);
                const int64_t row = ((int64_t)w * 2 + (w == w0 && !aligned ? 1 : 0)) * part_rows + x % part_rows;
                m[u] = a.part_ml[row * 2];
                l[u] = a.part_ml[row * 2 + 1];
                v[u] = *reinterpret_cast<const vnf*>(a.part + row * D + lane * N);
            }
#pragma unroll
            for (int u = 0; u < kJoinParts; u++) top = fmaxf(top, m[u]);
            // (no reference yet: parts that saw nothing, whose sums are zero, and parts whose scores were NaN, whose sums are: they pass as they are)
            const float f0 = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - top);
            ref = top;
            sum *= f0;
#pragma unroll
            for (int e = 0; e < N; e++) y[e] *= f0;
#pragma unroll
            for (int u = 0; u < kJoinParts; u++) {
                // (no branch: the loads of all eight are to be on their way at once)
                const bool real = s0 + u <= w1;
                const float f = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[u] - ref);
                sum = real ? fmaf(l[u], f, sum) : sum;
#pragma unroll
                for (int e = 0; e < N; e++) y[e] = real ? fmaf(v[u][e], f, y[e]) : y[e];
            }
        }
        if constexpr (SHARED) {
            __shared__ float meet[kWaves][N + 2][64];
            __syncthreads();             // (the row before has been read)
            meet[wave][N][lane] = ref, meet[wave][N + 1][lane] = sum;
#pragma unroll
            for (int e = 0; e < N; e++) meet[wave][e][lane] = y[e];
            __syncthreads();
            if (wave > 0) continue;
#pragma unroll
            for (int m = 1; m < kWaves; m++) ref = fmaxf(ref, meet[m][N][lane]);
            sum = 0.0f;
#pragma unroll
            for (int e = 0; e < N; e++) y[e] = 0.0f;
#pragma unroll
            for (int m = 0; m < kWaves; m++) {
                const float f = ref == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(meet[m][N][lane] - ref);
                sum = fmaf(meet[m][N + 1][lane], f, sum);
#pragma unroll
                for (int e = 0; e < N; e++) y[e] = fmaf(meet[m][e][lane], f, y[e]);
            }
        }
        const int i = x / a.g, hg = x - i * a.g;
        const bool blind = len - a.Sq + i < 0;
        const float inv = weight_of(sum, blind);
        uint16_t* o = a.o + b * a.o_sb + ((int64_t)h * a.g + hg) * a.o_sh + i * a.o_sn + lane * N;
#pragma unroll
        for (int e = 0; e < N; e++) y[e] = blind ? 0.0f : y[e] * inv;
        if constexpr (N == 1) o[0] = (uint16_t)pack2<T>(y[0], 0.0f);
        else
#pragma unroll
            for (int e = 0; e < N; e += 2) *reinterpret_cast<uint32_t*>(o + e) = pack2<T>(y[e], y[e + 1]);
    }
}

// (fewer than 128 row blocks then: else the shares are larger.)  [8 x 4 tokens, 4429 keys, 40 on 10 heads x 64] 16.4 us with a wave to a row, 15.7; [32 x 16384 keys,
// 48 on 12 x 128], up to five parts, 173 and 174.
bool paged_shared(const PagedArgs& a) {
    const int64_t most = (int64_t)a.pool.width << a.pool.sub, per = std::max<int64_t>(8, (paged_tiles(a) + a.wgs - 1) / a.wgs);
    return most > kJoinParts * per;
}
// No row of the table's length has more blocks than a share of its own: nothing to add up.  (Shares are the rows' own up to 32 blocks: see deal.)
bool paged_whole(const PagedArgs& a) {
    const int64_t most = std::max<int64_t>(1, (int64_t)a.pool.width << a.pool.sub);
    return a.more > 0 && most <= a.least && paged_tiles(a) <= 32 * (int64_t)a.wgs;
}
int64_t all_rows(const PagedArgs& a) { return (int64_t)a.B * a.pool.Hk * a.Sq * a.g; }

template <int T, int D> hipError_t launch_td(const PagedArgs& a, hipStream_t st) {
    if (paged_rows(a) == 16) hipLaunchKernelGGL((paged_kernel<T, D, 1>), dim3((unsigned)(a.wgs + a.more)), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_kernel<T, D, 2>), dim3((unsigned)(a.wgs + a.more)), dim3(256), 0, st, a);
    const int64_t rows = all_rows(a);
    if (paged_whole(a)) return hipGetLastError();
    if (paged_shared(a)) hipLaunchKernelGGL((paged_join_kernel<T, D, true>), dim3((unsigned)rows), dim3(256), 0, st, a, paged_rows(a), (int)rows);
    else hipLaunchKernelGGL((paged_join_kernel<T, D, false>), dim3((unsigned)std::min<int64_t>((rows + 3) / 4, 4096)), dim3(256), 0, st, a, paged_rows(a), (int)rows);
    return hipGetLastError();
}
template <int T> hipError_t launch_t(const PagedArgs& a, hipStream_t st) {
    if (a.D == 64) return launch_td<T, 64>(a, st);
    if (a.D == 128) return launch_td<T, 128>(a, st);
    return launch_td<T, 256>(a, st);
}

}  // namespace

int paged_rows(const PagedArgs& a) { return a.Sq * a.g <= 16 ? 16 : 32; }
int64_t paged_tiles(const PagedArgs& a) {
    const int64_t rblocks = ((int64_t)a.Sq * a.g + paged_rows(a) - 1) / paged_rows(a);
    return (int64_t)a.B * a.pool.Hk * rblocks * std::max<int64_t>(1, (int64_t)a.pool.width << a.pool.sub);
}
// Workgroups for even shares, and how many more shares there may be where every row has its own: one for each row block (of a sequence and key head), up to 2048 of them; more row blocks go by even
// shares, whose parts take no more workspace as those grow.  (Own / even shares, us, 64 channels, rows of 100, 300, 1000 keys: 2048 row blocks 12 / 23, 18 / 24, 46 / 47; 2064: 13 / 26, 20 / 25,
// 49 / 50; 4096: 25 / 29, 35 / 36, 120 / 102; 8192: 58 / 43, 79 / 74, 205 / 204.  So the border bounds the workspace, and short rows just past it pay for that.)
// Blocks of a share at the least, 8 / 16 / 32, us, 128 channels, rows of 500, 1000, 2000 keys:
//    48 row blocks 10.1 / 7.4 / 7.4, 10.6 / 11.6 /  9.9, 12.0 / 12.0 / 14.1;   88: 10.3 / 7.4 / 7.4, 12.4 / 11.9 / 10.1, 17.2 / 15.9 / 15.7;
//   108 row blocks 10.4 / 7.4 / 7.4, 12.6 / 12.1 / 10.5, 19.2 / 17.7 / 16.3;  180: 12.1 / 7.5 / 7.6, 17.7 / 16.4 / 11.6, 23.9 / 23.8 / 22.6;
//   204 row blocks 12.4 / 7.7 / 7.9, 19.4 / 16.5 / 12.4, 27.1 / 27.2 / 24.0;  6000 keys: the same within 3 %.
// Rows of one share gain the most, since nothing is added up; few rows of some thousand keys are those that a larger least costs.
// The host knows the table's width, not the lengths: the second launch is left out only where a row of the table holds no more than one share (paged_whole).  With a table for 16384 tokens
// 32 sequences of 500 keys, 48 on 12 heads x 128, take 15.4 us for 12.6, 20 of 300, 40 on 10 x 64, 9.0 for 5.3.
void paged_plan(PagedArgs* a) {
    a->wgs = (int)std::min<int64_t>(1024, std::max<int64_t>(1, (paged_tiles(*a) + 7) / 8));
    const int64_t units = (int64_t)a->B * a->pool.Hk * (((int64_t)a->Sq * a->g + paged_rows(*a) - 1) / paged_rows(*a));
    a->more = units <= 2048 ? (int)units : 0;
    a->least = units < 96 ? 8 : units < 192 ? 16 : 32;
}
size_t paged_part_bytes(const PagedArgs& a) { return (size_t)(a.wgs + a.more) * 2 * paged_rows(a) * (a.D + 2) * sizeof(float); }

hipError_t launch_paged(const PagedArgs& a, hipStream_t st) { return a.type == kBF16 ? launch_t<kBF16>(a, st) : launch_t<kF16>(a, st); }

}  // namespace sage
