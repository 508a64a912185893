// sage_kv.h — launchers of the paged cache of e4m3 codes: appending keys and values (sage_kv_append.hip), attention of the last tokens
// over it (sage_paged.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sage {

// A block is 32 tokens of a page; of one key head it is 32 * D codes of K, a token after the other, 32 * D of V, a channel after the other, and two scales.
constexpr int kKvBlock = 32;
// Scales are 2^e.  The least: what is no larger than 2^-110 (half of e4m3's least step, 2^-9, times it) becomes zero.
constexpr int kKvLeast = -100;
struct KvPool {
    uint8_t *k, *v;                              // [page, block of the page, Hk, 32, D], [.., D, 32]
    float *ks, *vs;                              // [page, block of the page, Hk]
    int64_t pages;
    int sub;                                     // log2 of the blocks to a page
    const int32_t* table;                        // [B, width] pages of the sequences, in order
    int64_t table_stride;
    int width;
    const int32_t* lens;                         // [B] tokens of the sequences in the cache, new ones among them
    int Hk;
};

struct KvSide {
    const void* p;                               // rows, 16-byte aligned; element strides
    int64_t sb, sh, sn;
};
struct KvAppendArgs {
    KvPool pool;
    KvSide k, v, q;                              // q.p null: no queries
    void* qo;
    int64_t qo_sb, qo_sh, qo_sn;
    const int32_t* cu;                           // [B + 1]: first rows of the sequences that lie one behind the other, or null: S rows each
    int B, S, rows;                              // rows: of all sequences
    int Hq, D, type;
    const void *q_gain, *k_gain;                 // [D], or null: no norm
    int gain_type;
    float eps, inv_d;
    const void *cos, *sin;                       // [table_rows, rot / 2]
    int table_type, rot, halfsplit;
    int64_t table_rows, table_stride;
    int kv_wgs;                                  // filled by the launcher
};
bool kv_append_grid_ok(const KvAppendArgs& a);
hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t st);

struct PagedArgs {
    KvPool pool;
    const uint16_t* q;
    uint16_t* o;
    int64_t q_sb, q_sh, q_sn, o_sb, o_sh, o_sn;
    int B, g, Sq, D, type;                       // g query heads share a key head
    float scale;
    int wgs, more, least;                        // workgroups that the blocks are dealt to, blocks of a share at the least (paged_plan)
    float *part, *part_ml;                       // [workgroup, 2, rows, D], [workgroup, 2, rows, 2]: parts of rows that several workgroups share
};
int paged_rows(const PagedArgs& a);              // rows of a part: 16 or 32
int64_t paged_tiles(const PagedArgs& a);         // blocks times row blocks times heads, of the longest sequences that the table holds
void paged_plan(PagedArgs* a);
size_t paged_part_bytes(const PagedArgs& a);
hipError_t launch_paged(const PagedArgs& a, hipStream_t st);

}  // namespace sage
