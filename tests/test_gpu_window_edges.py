"""Windowed attention where values, not sizes, are the hard part: queries that hold NaN or infinities, weights and upstream gradients far from
one, rows that see nothing, many sinks.  References and bounds: window_reference."""
import pytest
import torch

from mojodiffusion_amd import attention_window as W
from mojodiffusion_amd.attention_sage import Error
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


def test_workspace_of_the_gradients():
    """Two fp32 statistics a query row (three at the most), and parts: those of the blocks with sinks no more than two for each of 256 compute units, those of the others
    no more than four.  (Sizes only: nothing runs.)"""
    from mojodiffusion_amd import _lib
    size = _lib.lib().mi355_sage_window_bwd_workspace_bytes
    for B, Hq, Hk, S, D, left, sinks in ((1, 8, 8, 16896, 128, 16, 4), (1, 30, 30, 16896, 128, 16, 77), (1, 40, 40, 16896, 128, 16, 1024), (1, 32, 32, 16384, 128, 128, 16384),
                                         (1, 8, 8, 131072, 128, 63, 4), (1, 8, 8, 131072, 128, 63, 77), (1, 8, 8, 16896, 128, 63, 16896), (2, 24, 8, 8192, 64, 1023, 4),
                                         (1, 1, 1, 1 << 22, 64, 0, 1 << 22), (1, 2, 1, 1 << 27, 64, 0, 1 << 27), (1, 64, 1, 1 << 20, 64, 1, 1 << 27), (1, 1, 1, 300, 64, 2, 300),
                                         (4, 4, 2, 1000, 128, 999, 3), (1, 1, 1, 131072, 64, 16, 1), (64, 32, 8, 4096, 128, 64, 64)):
        stats = 3 * 4 * B * Hq * (S + 63)
        got = size(B, Hq, Hk, S, S, D, left, 0, sinks)
        assert 0 < got <= stats + 4 * 256 + (512 + 1024) * 2 * 64 * D * 4, (S, left, sinks, got)
        plain = size(B, Hq, Hk, S, S, D, left, 0, 0)
        assert got <= plain + 256 + 512 * 2 * 64 * D * 4, (S, left, sinks, got)


# Many sinks on short windows: whole blocks of them, ends inside a block, all keys, and one block whose pairs many workgroups share.
SINKS = [
    # B, S, Hq, Hk, D, type, left, sinks, lens
    (1, 1500, 2, 2, 64, BF, 16, 1024, None),
    (1, 1500, 3, 1, 128, FP, 16, 1500, [1490]),
    (2, 900, 2, 1, 64, FP, 0, 130, [900, 100]),
    (1, 5000, 2, 2, 64, BF, 16, 4, None),
    (1, 3500, 1, 1, 128, BF, 8, 70, [3400]),
    (1, 700, 40, 20, 64, BF, 30, 700, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,Hq,Hk,D,dtype,left,sinks,lens", SINKS)
def test_gradients_with_many_sinks(B, S, Hq, Hk, D, dtype, left, sinks, lens):
    q, k, v = tensors(B, S, S, Hq, Hk, D, dtype, S)
    d = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).to(dtype)
    n = [S] * B if lens is None else lens
    want = backward(q, k, v, d, D ** -0.5, forward(q, k, v, D ** -0.5, left, 0, sinks, n, [0] * B), Hq // Hk)
    lens = None if lens is None else torch.tensor(lens, dtype=torch.int32).cuda()
    args = (q.cuda(), k.cuda(), v.cuda(), d.cuda(), D ** -0.5, left, 0, sinks)
    got = grads(*args, lens=lens)[1]
    check_backward(got, want)
    for x, y in zip(got, grads(*args, lens=lens)[1]):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("B,H", [(1, 2), (64, 8)])
def test_a_key_between_the_sinks_and_a_window_behind_the_last(B, H):
    """Queries so far behind a sequence's end that their window holds no key: they see the sinks alone, and the last key may hold anything."""
    q, k, v = (t.cuda() for t in tensors(B, 3, 64, H, H, 64, BF, 1))
    lens = torch.full((B,), 20, dtype=torch.int32).cuda()
    call = lambda k, v: W.sdpa_window(q, k, v, 0.125, 8, 0, 4, kv_lens=lens, q_start=30)
    want = call(k, v)
    for bad in (NAN, INF, -3e38):
        k2, v2 = k.clone(), v.clone()
        k2[:, 4:], v2[:, 4:] = bad, bad
        assert torch.equal(call(k2, v2), want), bad
    assert torch.isfinite(want).all()


# Queries before the first key (right edge), behind the last (left edge, no sinks), both; of one sequence and of some.
BLIND = [
    # B, Sq, Skv, Hq, Hk, D, type, left, right, lens, first
    (1, 70, 64, 2, 1, 64, BF, 8, 0, [20], 0),
    (2, 200, 200, 3, 3, 128, FP, 30, 2, [200, 77], -11),
    (1, 300, 130, 4, 2, 64, FP, 9, 0, [130], -40),
    (2, 45, 45, 2, 2, 128, BF, 3, 1, [0, 5], 0),
    (1, 500, 100, 5, 1, 128, BF, 50, 60, [90], -150),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Sq,Skv,Hq,Hk,D,dtype,left,right,lens,first", BLIND)
def test_gradients_past_queries_that_see_nothing(B, Sq, Skv, Hq, Hk, D, dtype, left, right, lens, first):
    """Whatever such rows and their upstream gradients hold: zeros for their dQ, the same bits for the rest."""
    q, k, v = (t.cuda() for t in tensors(B, Sq, Skv, Hq, Hk, D, dtype, 3))
    d = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    p = first + torch.arange(Sq)
    blind = torch.stack([(p + right < 0) | (p - left > x - 1) | (x == 0) for x in lens])
    assert blind.any() and not blind.all()
    run = lambda q, d: grads(q, k, v, d, D ** -0.5, left, right, 0, lens=n, first=first)[1]
    want = run(q, d)
    for bad in (NAN, INF, -6e4):
        q2, d2 = q.clone(), d.clone()
        q2[blind.cuda()], d2[blind.cuda()] = bad, bad
        got = run(q2, d2)
        for name, x, y in zip(("dQ", "dK", "dV"), got, want):
            assert torch.equal(x, y), (name, bad)
    assert (want[0].cpu()[blind] == 0).all() and all(torch.isfinite(x).all() for x in want)


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hq,Hk", [(64, 2, 2), (128, 4, 2)])
def test_gradients_of_keys_with_small_weights(D, Hq, Hk):
    """Half of the keys lie 12 lower than the others: weights about 2^-25.  The bounds are relative to every weight."""
    S = 300
    q, k, v = tensors(1, S, S, Hq, Hk, D, BF, 11)
    q, k = q * 0.25, k * 0.25
    q[..., 0], k[..., 0] = 4.0, 0.0
    k[:, S // 3:, :, 0] = -3.0
    q, k = q.to(BF), k.to(BF)
    d = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).to(BF)
    ref = forward(q, k, v, 1.0, -1, -1, 0, [S], [0])
    assert 2.0 ** -30 < float(ref[2].min()) < 2.0 ** -23
    want = list(backward(q, k, v, d, 1.0, ref, Hq // Hk))
    # (the bounds grant a weight that is handed on 2^-10 of it: half a step of fp16 and as much again.  Carried times 2^14, a weight below 2^-28 is below fp16's
    # normal range there: half a step is 2^-25 / 2^14 whatever the weight.  That much of |dP - Delta| |q| comes on top of dK's bound.)
    extra = torch.zeros_like(want[1][1])
    for h in range(Hq):
        dp = d[0, :, h].double() @ v[0, :, h // (Hq // Hk)].double().T
        away = (dp - (ref[2][0, h] * dp).sum(1, keepdim=True)).abs() * (ref[2][0, h] < 2.0 ** -28)
        extra[0, :, h // (Hq // Hk)] += 2.0 ** -39 * away.T @ q[0, :, h].double().abs()
    want[1] = (want[1][0], want[1][1] + extra)
    assert float(extra.max()) < 0.02 * float(want[1][0][:, S // 3:].abs().max())
    check_backward(grads(q.cuda(), k.cuda(), v.cuda(), d.cuda(), 1.0, -1, -1, 0)[1], want)


@pytest.mark.gpu
@pytest.mark.parametrize("power", [-16, -12, -6])
@pytest.mark.parametrize("S,Hq,Hk,D,left,sinks", [(1500, 2, 1, 64, -1, 0), (333, 3, 3, 128, 40, 3), (900, 1, 1, 128, -1, 0)])
def test_fp16_gradients_of_small_upstream_gradients(power, S, Hq, Hk, D, left, sinks):
    """Gradients are linear in the upstream gradient.  Of size 2^power, which fp16 holds exactly here, it gives those of size 1 times 2^power but for one rounding
    of either result: half a step, 2^-11 of the value, 2^-25 below fp16's normal range.

    And but for single dS that are rounded another way: a row's power is added to its statistic in fp32, a sum of less than 64 in size (off by 2^-19 at most, either
    time: weights by 2^-18 relatively), so a dS within 2^-18 of a tie may fall on its other side.  Ties are a step of 2^-11 to 2^-10 apart: that is 2^-6 of the
    dS at most, by a step, 2^-10 of each, of either sign.  Elementwise that is more than the bounds of results near zero (a restatement of dQ's roundings on the CPU, in which the
    statistics' sums are all that differs, has two rows of 1500 beyond them, by 1.69), so norms are compared: 2^-10 sqrt(2^-6) of the root sum
    of the squared terms comes on top."""
    q, k, v = (t.cuda() for t in tensors(1, S, S, Hq, Hk, D, FP, 5))
    d = (torch.randint(-64, 65, q.shape, generator=torch.Generator().manual_seed(4)) / 64.0).to(FP)
    small = (d.double() * 2.0 ** power).to(FP)
    assert torch.equal(small.double(), d.double() * 2.0 ** power)
    got, one = (grads(q, k, v, x.cuda(), D ** -0.5, left, 0, sinks)[1] for x in (small, d))
    w, g = forward(q, k, v, D ** -0.5, left, 0, sinks, [S], [0])[2], Hq // Hk
    terms = [torch.zeros(x.shape, dtype=torch.float64) for x in one]
    for h in range(Hq):
        qh, dh, kh, vh = (x[0, :, y].double().cpu() for x, y in ((q, h), (d, h), (k, h // g), (v, h // g)))
        dp = dh @ vh.T
        ds = w[0, h] * (dp - (w[0, h] * dp).sum(1, keepdim=True)) * D ** -0.5
        terms[0][0, :, h] = ds.square() @ kh.square()
        terms[1][0, :, h // g] += ds.T.square() @ qh.square()
        terms[2][0, :, h // g] += w[0, h].T.square() @ dh.square()
    for name, x, y, t in zip(("dQ", "dK", "dV"), got, one, terms):
        x, y = x.double(), y.double() * 2.0 ** power
        bound = 2.0 ** -10 * 1.001 * y.abs() + 2.0 ** -25 + 2.0 ** (power - 25)
        other = 2.0 ** (power - 13) * float(t.sum().sqrt())
        assert float((x - y).norm()) <= float(bound.norm()) + other, (name, float((x - y).norm()), float(bound.norm()), other)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_gradients_of_large_upstream_gradients(D):
    """dS beyond fp16's range where dQ, dK and dV are not: the bounds of an upstream gradient of size 1, times 2^13."""
    S, scale, size = 16, 2.0 ** -10, 2.0 ** 13
    q, k, v = tensors(1, S, S, 2, 2, D, FP, 5)
    v = v * 8.0
    d = (torch.randint(-64, 65, q.shape, generator=torch.Generator().manual_seed(4)) / 64.0).to(FP)
    ref = forward(q, k, v, scale, -1, 0, 0, [S], [0])
    want = [(x * size, y * size) for x, y in backward(q, k, v, d, scale, ref, 1)]
    ds = ref[2][0, 0] * (d[0, :, 0].double() @ v[0, :, 0].double().T)
    assert float(ds.abs().max()) * size > 65504 and all(float(x.abs().max()) < 6e4 for x, _ in want)
    check_backward(grads(q.cuda(), k.cuda(), v.cuda(), (d * size).cuda(), scale, -1, 0, 0)[1], want)


@pytest.mark.gpu
def test_lengths_and_positions_past_32_bits():
    q, k, v = (t.cuda() for t in tensors(2, 3, 90, 2, 2, 64, BF, 2))
    call = lambda lens: W.sdpa_window_decode(q, k, v, torch.tensor(lens).cuda(), 0.125, 30)
    assert torch.equal(call([2 ** 32 + 5, 90]), call([90, 90])) and torch.equal(call([-2 ** 32 + 60, 90]), call([0, 90]))
    call = lambda starts: W.sdpa_window(q, k, v, 0.125, 30, q_start=torch.tensor(starts).cuda())
    assert torch.equal(call([2 ** 32 + 40, -2 ** 33 + 40]), call([2 ** 29, -2 ** 29]))
    assert (call([2 ** 32 + 40, -2 ** 33 + 40]) == 0).all()


def test_positions_past_32_bits_are_refused():
    q, k = torch.zeros((2, 4, 4, 64), dtype=BF), torch.zeros((2, 6, 2, 64), dtype=BF)
    for start in (2 ** 29 + 1, -2 ** 29 - 1, 2 ** 32, 2 ** 32 + 5, -2 ** 64):
        for call in (W.sdpa_window, W.sdpa_window_train_fwd):
            with pytest.raises(Error, match="q_start"):
                call(q, k, k, 0.1, 3, q_start=start)
        with pytest.raises(Error, match="q_start"):
            W.sdpa_window_backward(W.SdpaWindowFwd(q, q, torch.zeros((2, 4, 4, 1)), q, k, k, 0.1, 3, 0, 0, None, start), q)
    for start in (2 ** 29, -2 ** 29):
        with pytest.raises(Error, match="must live on the GPU"):
            W.sdpa_window(q, k, k, 0.1, 3, q_start=start)
    assert W._int32(torch.tensor([2 ** 32 + 5, -2 ** 33, 7])).tolist() == [2 ** 31 - 1, -2 ** 31, 7]


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hq,Hk,dtype", [(64, 2, 1, FP), (128, 3, 3, BF)])
def test_gradients_past_queries_before_the_sinks(D, Hq, Hk, dtype):
    """With sinks every later query sees something: those before the first key alone do not, and an empty sequence's."""
    B, Sq, Skv, left, right, sinks, first = 2, 300, 130, 9, 1, 5, -40
    q, k, v = tensors(B, Sq, Skv, Hq, Hk, D, dtype, 3)
    d = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).to(dtype)
    lens = [120, 0]
    blind = torch.stack([(first + torch.arange(Sq) + right < 0) | (n == 0) for n in lens])
    want = backward(q, k, v, d, D ** -0.5, forward(q, k, v, D ** -0.5, left, right, sinks, lens, [first] * B), Hq // Hk)
    q[blind], d[blind] = NAN, INF
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    fwd, got = grads(q.cuda(), k.cuda(), v.cuda(), d.cuda(), D ** -0.5, left, right, sinks, lens=n, first=first)
    check_backward(got, want)
    assert (fwd.o.cpu()[blind] == 0).all() and (got[0].cpu()[blind] == 0).all()


@pytest.mark.gpu
def test_fp16_gradients_captured():
    """A graph whose upstream gradient changes its size between replays, with the program's own calls in between."""
    B, S, H, D = 2, 300, 2, 64
    q, k, v = (t.cuda() for t in tensors(B, S, S, H, H, D, FP, 8))
    first = torch.randn(q.shape, generator=torch.Generator().manual_seed(1)).cuda()
    d = first.half()
    step = lambda: grads(q, k, v, d, 0.125, 80, 0, 3)[1]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for power in (0, -14, 10, -8, 3):
        d.copy_(first * 2.0 ** power)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        want = step()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y) and torch.isfinite(x).all() and x.abs().max() > 0, power
