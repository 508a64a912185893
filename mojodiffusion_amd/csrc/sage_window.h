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

}  // namespace sage
