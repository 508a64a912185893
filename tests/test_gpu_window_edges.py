"""Windowed attention where values, not sizes, are the hard part: queries that hold NaN or infinities, weights and upstream gradients far from
one, rows that see nothing, many sinks.  References and bounds: window_reference."""
import pytest
import torch

from mojodiffusion_amd import attention_window as W
from test_gpu_window import BF, FP, grads, tensors
from window_reference import backward, check_backward, forward

NAN, INF = float("nan"), float("inf")


# Tiles shared by four waves; keys of 32 rows in one workgroup, in 2 to 8, and in more, whose parts other lanes and waves join.
PLANS = [
    # B, Sq, Skv, Hq, Hk, D, type, left, sinks
    (8, 65, 200, 48, 16, 128, BF, 63, 4),
    (8, 100, 100, 16, 16, 256, FP, 16, 0),
    (4, 150, 150, 60, 12, 64, BF, -1, 0),
    (2, 1, 100, 4, 2, 64, FP, 40, 1),
    (1, 7, 200, 3, 1, 256, BF, -1, 0),
    (2, 1, 900, 8, 2, 128, BF, -1, 0),
    (1, 40, 1100, 2, 1, 64, FP, -1, 0),
    (1, 2, 700, 6, 3, 256, BF, 600, 4),
    (1, 1, 5000, 4, 1, 128, BF, -1, 0),
    (1, 2, 9000, 16, 1, 256, FP, 8191, 4),
    (1, 1, 6000, 8, 1, 64, BF, -1, 3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Sq,Skv,Hq,Hk,D,dtype,left,sinks", PLANS)
def test_a_query_that_is_not_finite(B, Sq, Skv, Hq, Hk, D, dtype, left, sinks):
    """Its row, and no other, is NaN, however the keys are shared out: by the formula all of its scores are NaN, or the largest is infinite, or
    all are -inf (and exp(-inf + inf) is no number); it is no row that sees nothing, which gives zeros."""
    q, k, v = (t.cuda() for t in tensors(B, Sq, Skv, Hq, Hk, D, dtype, 7))
    k[..., 0] = k[..., 0].abs() + 1
    lens = torch.full((B,), Skv - 3, dtype=torch.int32).cuda()
    calls = (lambda q: [W.sdpa_window_decode(q, k, v, lens, D ** -0.5, left, sinks)],
             lambda q: [(f := W.sdpa_window_train_fwd(q, k, v, D ** -0.5, left, 0, sinks, lens, Skv - 3 - Sq)).o, f.stats])
    b, i, h = B - 1, Sq // 2, Hq // 2
    for call in calls:
        want = call(q)
        for bad in (NAN, INF, -INF):
            q2 = q.clone()
            q2[b, i, h] = NAN if bad != bad else 0.0
            q2[b, i, h, 0] = bad
            got = call(q2)
            assert torch.isnan(got[0][b, i, h]).all(), bad
            if bad != bad and len(got) > 1:
                assert torch.isnan(got[1][b, h, i]).all()
            for x, y, at in zip(got, want, ((b, i, h), (b, h, i))):
                x = x.clone()
                x[at] = y[at]
                assert torch.equal(x, y), bad
            assert torch.isfinite(want[0]).all()
