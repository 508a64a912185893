// sage_window.h — launchers of the operators around windowed attention: norm and rotation of queries and keys
// (sage_norm_rope.hip), attention over a sliding window with first tokens that stay visible (sage_window*.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sage {

// ---- norm and rotation of queries and keys ---------------------------------------------------------
// Element types, as MI355_SAGE_BF16 / _FP16 / _F32 of the C ABI.
constexpr int kBF16 = 0, kF16 = 1, kF32 = 2;
struct NormRopeSide {
    const void* p;                   // rows, 16-byte aligned
    void* out;                       // the rotated rows, or (backward) the gradient of p's
    const void* d;                   // backward: upstream gradient
    const void* gain;                // [D]
    int64_t sb, sh, sn, osb, osh, osn, dsb, dsh, dsn;      // strides in elements
};
struct NormRopeArgs {
    NormRopeSide q, k;
    int B, S, Hq, Hk, D, type, gain_type, table_type;
    float eps, inv_d;
    const void *cos, *sin;           // [table_rows, rot / 2]
    int64_t table_rows, table_stride;
    int rot, halfsplit;              // rotated channels (0: none)
    const void* positions;           // [B, S], null: token s takes row s
    int64_t pos_sb;
    int pos64;
    float* partial;                  // backward: [wg_q + wg_k, D] partial sums of the gains' gradients
    float *d_gain_q, *d_gain_k;
    int wg_q, wg_k;                  // filled by the launcher
};
void norm_rope_bwd_split(int B, int S, int Hq, int Hk, int D, int* wg_q, int* wg_k);
hipError_t launch_norm_rope(const NormRopeArgs& a, hipStream_t st);
hipError_t launch_norm_rope_bwd(const NormRopeArgs& a, hipStream_t st);

// ---- attention over a sliding window ---------------------------------------------------------------
// A query at position p sees the keys j < len with j <= p + right and (j >= p - left or j < sinks).  Query i of sequence b stands
// at (at_end ? len - Sq : starts ? starts[b] : start) + i.  g query heads share a key head; the rows of a workgroup are
// (query, head of the group) pairs, heads first, so that they share one window.
constexpr int kWindowFar = (1 << 30) - 1;        // left, right: no bound
constexpr int kWindowStart = 1 << 29;            // positions are kept within this, so that sums with the above fit 32 bits
struct WindowArgs {
    const uint16_t *q, *k, *v;
    uint16_t *o, *rest;                          // rest: what rounding left of O, in O's type and strides, or null
    int64_t q_sb, q_sh, q_sn, k_sb, k_sh, k_sn, v_sb, v_sh, v_sn, o_sb, o_sh, o_sn;      // strides in elements
    int B, Hk, g, Sq, Skv, D, type;              // type: kBF16 or kF16
    int left, right, sinks;
    const int32_t *lens, *starts;                // [B] on the device, or null
    int start, at_end;
    float scale;                                 // > 0
    float* stats;                                // [B, Hk * g, Sq] natural log-sum-exp, or null
    // keys split over workgroups: unnormalised partial rows, their references and sums
    int splits;
    float *part, *part_ml;                       // [row block, split, 32, D], [row block, split, 32, 2]
};
struct WindowPlan {
    int splits;                                  // 0: tiles shared by the waves of a workgroup; else the keys split, so many workgroups to a block of 32 rows
};
WindowPlan window_plan(const WindowArgs& a);
bool window_grid_ok(const WindowArgs& a, const WindowPlan& p);
size_t window_part_bytes(const WindowArgs& a, const WindowPlan& p);
hipError_t launch_window(const WindowArgs& a, const WindowPlan& p, hipStream_t st);

// Its gradient.  w: the forward's arguments (o, stats as it wrote them).
struct WindowBwdArgs {
    WindowArgs w;
    const uint16_t* dout;
    uint16_t *dq, *dk, *dv;
    int64_t do_sb, do_sh, do_sn, dq_sb, dq_sh, dq_sn, dk_sb, dk_sh, dk_sn, dv_sb, dv_sh, dv_sn;
    // workspace
    float *lse2, *ndelta;                        // [B, Hk * g, sq_pad]: Stats * log2(e) less kWeightBits (+inf: no such row, or nothing seen), -rowsum(dO * O)
    float* dsize;                                // [B, Hk * g, sq_pad]: rowsum |dO| (fp16 only)
    int sq_pad;                                  // Sq rounded up to a multiple of 64
    // How a key block's (head, query tile) pairs are dealt: `sink_blocks` blocks of kWindowBwdKeys keys with sinks in them go to sink_chunks workgroups
    // each, of sink_tiles pairs, the others to chunks, of chunk_tiles pairs.
    int sink_blocks, sink_chunks, sink_tiles, chunks, chunk_tiles;
    float* part;                                 // [workgroup, 2, kWindowBwdKeys, D] fp32 parts of dK and dV of blocks with several workgroups
};
void window_bwd_plan(WindowBwdArgs* a);          // fills in the five above from a->w
constexpr int kWindowBwdKeys = 64;               // keys of a workgroup
int64_t window_bwd_parts(const WindowBwdArgs& a);        // workgroups that leave parts
hipError_t launch_window_bwd(const WindowBwdArgs& a, hipStream_t st);

}  // namespace sage
