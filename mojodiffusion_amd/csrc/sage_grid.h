// sage_grid.h — which block of its launch's work a workgroup takes.  Plain arithmetic without any include, so that a
// host compiler can be asked for the same mapping (tests/test_grid_mapping.py).
#pragma once

namespace sage {

// Workgroup `id` of n -> item: consecutive ids go to the 8 XCDs in turn, and each XCD takes a contiguous range of items,
// so that those of a head, which all walk the same rows, share one L2.
__host__ __device__ inline int xcd_item(int id, int n) {
    const int per = n >> 3, extra = n & 7, xcd = id & 7;
    return xcd * per + (xcd < extra ? xcd : extra) + (id >> 3);
}

// The backward's grid: `heads` heads, each with tq blocks of query rows (dQ) and tk blocks of keys (dK, dV), the first lq
// and lk of which hold rows that count.  Those come first, dQ in front of dK/dV, each kind in even ranges over the XCDs;
// blocks of padding, which only store zeros, come last.  In ranges over all blocks, padding included, an XCD that does not
// get whole heads has up to twice another's blocks that count.  Launch 1 + 2 at 128 channels, rows / rows that count, us, so
// -> now:  12 heads  2304/1612 94.5 -> 75.8   4608/2304 149.8 -> 136.1   4608/3225 263.7 -> 230.9   4608/3916 373.5 -> 346.5
//          30 heads  1248/624 45.2 -> 38.8    1248/873 65.6 -> 61.1      4608/3225 580.8 -> 565.8
// Whole heads per XCD are even as they are and keep their order: the padding last measured 5 % behind that to 5 % ahead
// there (16 heads 4608/2304 158.1 -> 166.3, 24 heads 1248/873 57.1 -> 59.0, 24 heads 4608/3225 455.8 -> 432.2).
struct BwdBlock { bool dkdv; int head, tile; };
__host__ __device__ inline BwdBlock bwd_block(int id, int heads, int tq, int lq, int tk, int lk) {
    if ((heads & 7) == 0) lq = tq, lk = tk;
    const int nq = heads * lq, nk = heads * lk;
    if (id < nq) {
        const int i = xcd_item(id, nq);
        return BwdBlock{false, i / lq, i % lq};
    }
    if (id < nq + nk) {
        const int i = xcd_item(id - nq, nk);
        return BwdBlock{true, i / lk, i % lk};
    }
    const int j = id - nq - nk, pq = heads * (tq - lq);
    return j < pq ? BwdBlock{false, j / (tq - lq), lq + j % (tq - lq)} : BwdBlock{true, (j - pq) / (tk - lk), lk + (j - pq) % (tk - lk)};
}

// The encoders' grid where rows are rotated by tables.  What reads the same table rows — the Q and K blocks of one run of
// rows of one head, in every batch that shares the tables — is a set; its `members` go to one XCD, one soon after the other,
// so that the rows come from its L2 after the first.  Sets run over the heads first and are taken 32 at a time, member by
// member: consecutive ids read neighbours in memory, as everywhere in the quantizers.
constexpr int kSetGroup = 32;                    // (a multiple of the XCDs)
struct SetMember { int set, member; };
__host__ __device__ inline SetMember set_member(int id, int members) {
    const int at = id % (kSetGroup * members);
    return SetMember{id / (kSetGroup * members) * kSetGroup + at % kSetGroup, at / kSetGroup};
}
__host__ __device__ inline long long set_grid(long long sets, int members) {
    return (sets + kSetGroup - 1) / kSetGroup * kSetGroup * members;
}

// `slots` pieces of work of each of `heads` heads, of falling size, in even shares for the XCDs: where the heads do not divide among the 8, those that are shared are dealt out
// slot by slot (every second, fourth or eighth to one XCD), not in halves of which the first is the heavier.  A slot beyond the last: no work.
__host__ __device__ inline int spread_ways(int heads) { return (heads & 7) == 0 ? 1 : (heads & 3) == 0 ? 2 : (heads & 1) == 0 ? 4 : 8; }
__host__ __device__ inline long long spread_grid(long long heads, long long slots) {
    const int m = spread_ways((int)(heads & 7));
    return heads * m * ((slots + m - 1) / m);
}
struct HeadSlot { int head, slot; };
__host__ __device__ inline HeadSlot spread_item(int id, int heads, int slots) {
    const int m = spread_ways(heads), per = (slots + m - 1) / m, item = xcd_item(id, heads * m * per), p = item % (m * per);
    return HeadSlot{item / (m * per), p % per * m + p / per};
}

// Packed attention's workgroups.  kFull: 128 rows, a wave to 32, their key tiles shared; kPaired: two waves to 32 rows, even key tiles and odd; kFew: 32 rows whose waves take key tiles in
// turn.  By the workgroups of 128 rows (the last of a sequence half full, on the average) that `rows` rows (queries times the heads that share a key head) of B sequences make on `heads` key heads, and the keys of a
// sequence on the average (an empty sequence counts as any other): workgroups of 32 rows while one round holds them all (two to a compute unit at 64 channels, one above; two rounds
// where causal rows leave the second one short), two waves to 32 rows while every compute unit has about one workgroup, with short walks some fewer (the XCDs' shares are not even).
// Past 256 workgroups the others begin where the first end: with causal rows those are short, at 64 channels two fit a compute unit; else pairs would go through a second, nearly empty round.
// Measured over sequences of one length, bf16, few / paired / full in us:
//   64 channels, full attention of 4096 keys, 96 wgs 38 / 45 / 57, 160: 63 / 45 / 59, 256: 74 / 48 / 59, 320: 95 / 74 / 77; of 640, 95: 11 / 12 / 13, 190: 17 / 13 / 14, 255: 24 / 18 / 18;
//   128 channels, full, 4096 keys, 64: 47 / 67 / 95, 96: 91 / 67 / 95, 256: 182 / 78 / 96, 320: 228 / 141 / 118; causal, 128: 53 / 67 / 96; 333 keys, 96: 17 / 13 / 14,
//   192: 24 / 13 / 15, 225: 33 / 26 / 18;
//   256 channels, full, 4096 keys, 96: 151 / 121 / 180, 256: 284 / 143 / 182; causal, 128: 82 / 121 / 180;
// around one round, one sequence, paired / full, 256, 264 and 272 wgs of 8 heads: 64 channels, full 46 / 59, 69 / 70, 72 / 74; 128 channels, full 75 / 93, 135 / 110, 140 / 116, causal
// 67 / 94, 67 / 94, 69 / 96 (280: 73 / 102); 256 channels, full 129 / 170, 228 / 184, 238 / 192, causal 109 / 170, 109 / 170, 113 / 175.  Two sequences, 8 heads x 128, full: 2 x 2048 (256
// wgs) 41 / 50, 2000 + 2100 (264) 73 / 58: rows that B sequences of whole blocks make are taken for such.  (Sequences of very different lengths were not measured beyond that.)
enum class PackedForm { kFull, kPaired, kFew };
__host__ __device__ inline PackedForm packed_form_of(int D, bool causal, int B, long long heads, long long rows, long long keys) {
    const long long full = rows * heads / 128, wgs = full + B * heads / 2, apart = rows % (128LL * B) == 0 ? 0 : (B - 1) * heads / 2;
    if (full <= (D == 64 || (causal && keys >= 1024) ? 128 : 64)) return PackedForm::kFew;
    if (D > 64 && !causal && (rows + 127) / 128 * heads + apart > 256) return PackedForm::kFull;
    return wgs <= (keys >= 1024 ? 272 : 212) ? PackedForm::kPaired : PackedForm::kFull;
}

// Share `id` of a list of `total` places in shares of `per`: begin .. end - 1.  Ids go beyond the last share (nothing is left for those), and their products with
// `per` beyond 32 bits.
struct Share { int begin, end; };
__host__ __device__ inline Share share_of(int id, int per, int total) {
    const long long at = (long long)id * per;
    const int begin = at < total ? (int)at : total;
    return Share{begin, total - begin < per ? total : begin + per};
}

}  // namespace sage
